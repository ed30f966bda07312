"""Each kernel of the block-scaled FP8 products at sizes that reach it, which every
test checks before it runs, at random places and in the last rows and columns (GPU)."""
import numpy as np
import pytest

import block_ref as R
import mxfp4hip as M
from test_block_rules import tile_rows
from test_gpu_block import dequant, expert_case, expert_ref, quantize, run_experts, weights

pytestmark = pytest.mark.gpu
F, H, B = M.DT_F32, M.DT_F16, M.DT_BF16


def four_waves(row_tiles, n, swiglu):
    """Whether the weight streams of 16-row tiles have four waves, and not eight."""
    return row_tiles * -(-n // 32) * (2 if swiglu else 1) >= 256


def half_round(tiles):
    """Whether 256-row tiles have whole rounds and a last one for at most half of the CUs."""
    per = -(-tiles // 8)  # of an XCD and its 32 CUs
    return per > 32 and 1 <= per % 32 <= 16


def check_matmul(dev, m, n, k, dtypes, cores):
    rng = np.random.default_rng(m + n + k)
    x = (rng.normal(0, 1, (m, k)) * np.exp(rng.normal(0, 1, (m, 1)))).astype(np.float32)
    q, s = quantize(dev, x, F)
    rs = R.act_scales(x)
    wq, ws, wv = weights(dev, rng, 1, n, k)
    rows = np.unique(np.r_[rng.integers(0, m, 50), 0, m - 1])
    cols = np.unique(np.r_[rng.integers(0, n, 300), 0, max(0, n - 20):n])
    a = R.act_codes(x, rs) * np.repeat(rs.T, 128, 1)[:, :k].astype(np.float64)
    ref, err = R.product(a[rows], wv[0][cols], cores=cores)
    for ct in dtypes:
        c = dev.upload(np.full(m * n + 64, 9, R.np_type(ct)))
        dev.block_matmul(q, s, wq, ws, c, ct, m, n, k)
        got = dev.download(c, R.np_type(ct), m * n + 64)
        c.free()
        assert (got[m * n:] == 9).all()
        diff = np.abs(R.values_of(got[:m * n].reshape(m, n)[np.ix_(rows, cols)], ct) - ref)
        assert np.all(diff <= R.rounded(ref, err, ct)), (ct, diff.max())


@pytest.mark.parametrize("m,n,k", [(1700, 8323, 400), (2050, 2051, 272), (1600, 8200, 144), (1153, 4100, 1040)])
def test_f32_results_by_128_rows(dev, m, n, k):
    assert tile_rows(m, 1, n, k, F) == 128
    check_matmul(dev, m, n, k, [F], False)


@pytest.mark.parametrize("m,n,k", [(1, 8193, 1040), (16, 8193, 272), (1, 8225, 4112), (13, 8209, 4240)])
def test_streams_of_16_rows_with_four_waves(dev, m, n, k):
    assert tile_rows(m, 1, n, k, H) == 16 and four_waves(1, n, False)
    check_matmul(dev, m, n, k, [F, H, B], False)


@pytest.mark.parametrize("m,n,k", [(24, 14337, 272), (17, 6177, 1040), (32, 6161, 4112), (25, 6145, 4240)])
def test_streams_of_32_rows(dev, m, n, k):
    assert tile_rows(m, 1, n, k, H) == 32
    check_matmul(dev, m, n, k, [F, H, B], False)


@pytest.mark.parametrize("m,n,k", [(2300, 8441, 144), (2560, 7300, 400), (1800, 9999, 272)])
def test_256_rows_in_rounds_and_half_a_round(dev, m, n, k):
    assert tile_rows(m, 1, n, k, H) == 256 and half_round(-(-m // 256) * -(-n // 256))
    check_matmul(dev, m, n, k, [H, B], True)


@pytest.mark.parametrize("t,h,i,rows", [(1, 272, 4112, 16), (5, 4240, 4112, 16), (24, 272, 4128, 32), (30, 4112, 4144, 32)])
def test_format_mlp_streams(dev, t, h, i, rows):
    assert tile_rows(t, 1, i, h, H, True) == rows and (rows > 16 or four_waves(1, i, True))
    rng = np.random.default_rng(t)
    x = R.bits_of(rng.normal(0, 1, (t, h)), H)
    ws = [weights(dev, rng, 1, n, k, std=0.05) for n, k in ((i, h), (i, h), (h, i))]
    out = dev.alloc(t * h * 2)
    dev.fmt_mlp_forward(M.WFMT_FP8_BLOCK, t, h, i, dev.upload(x), M.Device.weights(*[w[:2] for w in ws]), out)
    y, err = R.mlp(dequant(x, H), *[w[2][0] for w in ws])
    got = R.values_of(dev.download(out, np.float16, (t, h)), H)
    assert np.all(np.abs(got - y) <= R.rounded(y, err, H))


def sampled_experts(dev, t, h, i, e, k, dtype, cores, drop=0.0, tokens=40):
    """Experts of all tokens, compared at some of them."""
    x, ids, w, ws, base = expert_case(dev, t, h, i, e, k, dtype, t + h, drop=drop)
    got = run_experts(dev, x, ids, w, ws, base, dtype)
    some = np.unique(np.r_[np.random.default_rng(t).integers(0, t, tokens), 0, t - 1])
    ref, err = expert_ref(x[some], ids[some], w[some], ws, base[some], dtype, cores=cores)
    assert np.all(np.abs(got[some] - ref) <= err)
    assert np.isfinite(got).all()
    for v in ws:
        v[0].free(), v[1].free()
    return ids


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("h,i,e,k", [(2064, 1040, 6, 4), (4240, 528, 8, 8)])
def test_one_token_with_four_waves(dev, dtype, h, i, e, k):
    assert four_waves(k, i, True) and four_waves(k, h, False)
    sampled_experts(dev, 1, h, i, e, k, dtype, False)


@pytest.mark.parametrize("h,i", [(8208, 144), (144, 8208)])
def test_one_token_past_the_direct_rows(dev, h, i):
    sampled_experts(dev, 1, h, i, 2, 2, H, False)


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("t,h,i,e,k,rows", [(20, 4240, 528, 8, 2, 16), (50, 4240, 528, 8, 2, 32)])
def test_expert_streams_of_long_rows(dev, dtype, t, h, i, e, k, rows):
    assert tile_rows(t * k, e, i, h, dtype, True) == rows
    assert rows == 32 or (four_waves(e + t * k // 16, i, True) and four_waves(e + t * k // 16, h, False))
    sampled_experts(dev, t, h, i, e, k, dtype, False)


@pytest.mark.parametrize("t,rows", [(10, 16), (24, 32)])
def test_expert_streams_of_long_middles(dev, t, rows):
    h, i, e, k = 2064, 4112, 4, 2
    assert tile_rows(t * k, e, i, h, H, True) == rows
    assert rows == 32 or four_waves(e + t * k // 16, h, False)
    sampled_experts(dev, t, h, i, e, k, H, False)


@pytest.mark.parametrize("dtype", [H, B])
def test_experts_of_256_rows_in_rounds_and_half_a_round(dev, dtype):
    t, h, i, e, k = 4000, 4112, 2064, 4, 1
    assert tile_rows(t * k, e, i, h, dtype, True) == 256
    ids = sampled_experts(dev, t, h, i, e, k, dtype, True, drop=0.02)
    row_tiles = sum(-(-int((ids == x).sum()) // 256) for x in range(e))
    assert half_round(row_tiles * -(-i // 128)) and half_round(row_tiles * -(-h // 256))


def test_experts_of_more_slots_than_a_workgroup_counts(dev):
    """More than 65536 slots: their order comes from a table of counts."""
    sampled_experts(dev, 33000, 128, 128, 5, 2, B, True, drop=0.05)


def test_experts_of_nothing_leave_the_output(dev):
    x, ids, w, ws, _ = expert_case(dev, 1, 128, 128, 2, 1, H, 0)
    out = dev.upload(np.full(128, 0x1234, np.uint16))
    dev.moe_block_forward(0, 128, 128, 2, 1, dev.upload(x), H, dev.upload(ids), dev.upload(w), M.Device.weights(*[v[:2] for v in ws]), out)
    assert (dev.download(out, np.uint16, 128) == 0x1234).all()

"""Routed block-FP8 experts: their rows up to the weighted sum (GPU)."""
import numpy as np
import pytest

import block_ref as R
import mxfp4hip as M
from test_gpu_block import dequant, expert_ref, weights

pytestmark = pytest.mark.gpu
H, B = M.DT_F16, M.DT_BF16


def forward(dev, x, dtype, ids, w, mats, inter, experts):
    t, h = x.shape
    out = dev.alloc(t * h * 2)
    dev.moe_block_forward(t, h, inter, experts, ids.shape[1], dev.upload(x), dtype, dev.upload(ids), dev.upload(w),
                          M.Device.weights(*mats), out)
    return R.values_of(dev.download(out, x.dtype, (t, h)), dtype)


@pytest.mark.parametrize("t", [1, 8, 30, 60, 300])
def test_rows_past_f16_in_a_sum_that_is_not(dev, t):
    """Rows up to 1e5 to 2e6, which f16 does not hold, weighted by 2^-6.  (Two experts:
    direct, 16- and 32-row streams, tiles of 64 and 256 rows.)"""
    h = i = 256
    rng = np.random.default_rng(t)
    x = R.bits_of(rng.normal(0, 1, (t, h)), H)
    ws = [weights(dev, rng, 2, n, k, std=s) for n, k, s in ((i, h, 0.3), (i, h, 0.3), (h, i, 75))]
    ids = (np.arange(t, dtype=np.int32) % 2).reshape(t, 1)
    got = forward(dev, x, H, ids, np.full((t, 1), 2.0 ** -6, np.float32), [v[:2] for v in ws], i, 2)
    most = 0.0
    for e in range(2):
        at = np.nonzero(ids[:, 0] == e)[0]
        if not at.size:
            continue
        y, err = R.mlp(dequant(x, H)[at], *[v[2][e] for v in ws], cores=True)
        most = max(most, np.abs(y).max())
        y, err = y * 2.0 ** -6, err * 2.0 ** -6 + 4 * R.EPS * np.abs(y) * 2.0 ** -6
        assert np.abs(y).max() < 60000
        assert np.all(np.abs(got[at] - y) <= R.rounded(y, err, H))
    assert most > 65536


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("t", [4, 14, 30, 60, 300])
def test_rows_that_nearly_cancel(dev, dtype, t):
    """Expert 1 is expert 0 with its down product 1 + 2^-6 times as large: their
    difference is 2^-6 of expert 0's row.  A row's one block of K makes both rows
    the same sum times scales that are rounded three times (scale, product of scales,
    row) and the weighted sum once: 8 roundings of 2^-24 of a row, 2^6 as much of the
    difference; each of the two results is rounded to the rows' type."""
    h, i = 256, 128
    rng = np.random.default_rng(t)
    x = R.bits_of(rng.normal(0, 1, (t, h)), dtype)
    mats = []
    for n, k in ((i, h), (i, h), (h, i)):
        q, s, _ = weights(dev, rng, 1, n, k, std=0.1)
        codes = dev.download(q, np.uint8, (n, k))
        scales = dev.download(s, np.float32, (R.blocks(n), R.blocks(k)))
        other = scales * np.float32(1 + 2.0 ** -6) if n == h else scales
        mats.append((dev.upload(np.stack([codes, codes])), dev.upload(np.stack([scales, other]))))
    ids = np.tile(np.array([1, 0], np.int32), (t, 1))
    diff = forward(dev, x, dtype, ids, np.tile(np.array([1, -1], np.float32), (t, 1)), mats, i, 2)
    one = forward(dev, x, dtype, ids, np.tile(np.array([0, 2.0 ** -6], np.float32), (t, 1)), mats, i, 2)
    assert np.abs(one).max() > 1e-3
    size = np.abs(one) * (1 + 2 * R.HALF_ULP[dtype])
    tol = 2 * (R.HALF_ULP[dtype] * size * 1.01 + R.TINY[dtype]) + 8 * 2.0 ** 6 * R.EPS / 2 * size
    assert np.all(np.abs(diff - one) <= tol)


def test_batches_in_parts(dev):
    """16400 tokens of 65536: the last 17 are a part of their own."""
    t, h, i, e, k = 16400, 65536, 32, 3, 2
    rng = np.random.default_rng(0)
    x, out = dev.alloc(t * h * 2), dev.alloc(t * h * 2)
    dev.fill_normal(x, H, t * h, seed=1)
    dev.memset(out, 0xff)
    ids = rng.integers(-1, e, (t, k)).astype(np.int32)
    w = rng.random((t, k)).astype(np.float32)
    ws = [weights(dev, rng, e, n, kk, std=0.05) for n, kk in ((i, h), (i, h), (h, i))]
    dev.moe_block_forward(t, h, i, e, k, x, H, dev.upload(ids), dev.upload(w), M.Device.weights(*[v[:2] for v in ws]), out)
    some = np.r_[0, 1, 5000, 16381:16386, t - 1]

    def rows(buf):
        return np.concatenate([dev.download(buf.offset(int(r) * h * 2), np.float16, (1, h)) for r in some])

    ref, err = expert_ref(rows(x), ids[some], w[some], ws, None, H, cores=True)
    got = rows(out).astype(np.float64)
    x.free(), out.free()
    assert np.all(np.abs(got - ref) <= err)

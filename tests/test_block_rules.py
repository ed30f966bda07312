"""Which kernels the block-scaled FP8 products run on, their step names, and the
oracle of their tests (host logic, no GPU)."""
import ctypes

import numpy as np
import pytest

import block_ref as R
import mxfp4hip as M


def tile_rows(rows, groups, n, k, dtype, swiglu=False):
    f = getattr(M.load(), "_ZN2mx15block_tile_rowsEliiiib")
    f.argtypes = [ctypes.c_long] + [ctypes.c_int] * 4 + [ctypes.c_bool]
    return f(rows, groups, n, k, dtype, swiglu)


def splits(m, n, k, rows):
    return getattr(M.load(), "_ZN2mx12block_splitsEiiii")(m, n, k, rows)


# sides measured, us: the row's tile height / another
@pytest.mark.parametrize("m,n,k,dtype,rows", [
    (1, 4096, 4096, M.DT_F16, 16), (16, 14336, 4096, M.DT_F32, 16),
    (24, 4096, 4096, M.DT_F16, 16),          # 9.8 / 11.7 with 32
    (24, 14336, 4096, M.DT_F16, 32),         # 18.6 / 25.3 with 16
    (100, 14336, 4096, M.DT_F16, 64), (300, 4096, 4096, M.DT_BF16, 64),
    (1000, 4096, 4096, M.DT_F16, 64),        # 30 / 38 with 256
    (1000, 4096, 4096, M.DT_F32, 64),        # 41.5 / 56 with 128
    (2000, 8192, 4096, M.DT_F32, 128),       # 112 / 137 with 64
    (4096, 14336, 4096, M.DT_BF16, 256),
])
def test_dense_tile_heights(m, n, k, dtype, rows):
    assert tile_rows(m, 1, n, k, dtype) == rows


@pytest.mark.parametrize("rows,groups,want", [(8, 8, 16), (44, 16, 16), (320, 32, 32), (512, 16, 64), (2048, 64, 64), (4096, 64, 256)])
def test_expert_tile_heights(rows, groups, want):
    assert tile_rows(rows, groups, 2048, 7168, M.DT_F16, True) == want


def test_parts_of_k():
    assert splits(46, 1221, 3968, 64) == 7       # 10 tiles, 31 blocks of K
    assert splits(257, 2080, 5536, 64) == 3      # 85 tiles
    assert splits(300, 4096, 4096, 64) == 1      # 160 tiles: the parts' sum costs more
    assert splits(40, 128, 128, 64) == 1         # one block of K
    assert splits(4096, 4096, 4096, 256) == 1 and splits(1, 4096, 4096, 16) == 1


def test_step_names():
    def names(t, h, i):
        cfg = M.MlpConfig(t, h, i)
        got = [M.load().mx_fmt_mlp_kernel_name(M.WFMT_FP8_BLOCK, ctypes.byref(cfg), s) for s in range(5)]
        return [g.decode() for g in got if g]

    assert names(1, 4096, 14336) == ["block_quantize_x", "block_gemm_gate_up_swiglu", "block_quantize_mid", "block_gemm_down"]
    assert names(512, 4096, 14336) == ["block_quantize_x", "block_gemm_gate_up_swiglu_quantize", "block_gemm_down"]


# ---- the oracle ------------------------------------------------------------------------
def test_e4m3_rounds_to_the_nearest_code():
    grid = R.e4m3_values(np.arange(256, dtype=np.uint8))
    grid = np.unique(grid[np.isfinite(grid)])
    assert grid.max() == 448 and (grid > 0).sum() == 126
    assert np.array_equal(R.e4m3(grid), grid)
    mid = (grid[1:] + grid[:-1]) / 2
    step = np.diff(grid)
    assert np.array_equal(R.e4m3(mid - step * 0.01), grid[:-1]) and np.array_equal(R.e4m3(mid + step * 0.01), grid[1:])
    codes = {v: c for c, v in enumerate(R.e4m3_values(np.arange(127, dtype=np.uint8)))}
    assert all(codes[abs(v)] % 2 == 0 for v in R.e4m3(mid))  # ties: the even code


def test_route_oracle():
    """Ties, the bias' part in the choice, and the groups."""
    logits = np.array([[1.0, 1.0, 0.0, 3.0]])
    s = 1 / (1 + np.exp(-logits[0]))
    ids, w, _ = R.route(logits, np.array([0.0, 0.0, 1.0, 0.0]), 2, True, 1, 1, 1, False, 1.0)
    assert ids[0].tolist() == [2, 3] and np.allclose(w[0], s[[2, 3]])  # chosen with the bias, weighted without
    assert R.route(logits, None, 3, True, 1, 1, 1, False, 1.0)[0][0].tolist() == [3, 0, 1]
    assert R.route(logits, None, 2, True, 2, 1, 1, False, 1.0)[0][0].tolist() == [3, 2]
    assert R.route(logits, None, 2, True, 2, 1, 2, False, 1.0)[0][0].tolist() == [0, 1]  # 0.731 + 0.731 > 0.953 + 0.5


def test_product_bounds_hold_for_f32_sums():
    rng = np.random.default_rng(0)
    a, w = rng.normal(0, 1, (5, 300)), rng.normal(0, 1, (7, 300))
    a, w = a.astype(np.float32).astype(np.float64), w.astype(np.float32).astype(np.float64)
    c, err = R.product(a, w)
    seq = np.zeros((5, 7), np.float32)
    for k in range(300):
        seq += (a[:, k, None] * w[:, k]).astype(np.float32)
    assert np.all(np.abs(seq - c) <= err) and np.all(R.product(a, w, cores=True)[1] > err)

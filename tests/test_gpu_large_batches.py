"""Batches whose tokens pass what one launch holds, up to the entry points' limits (GPU)."""
import ctypes

import numpy as np
import pytest

import mxfp4hip as M

pytestmark = pytest.mark.gpu
H = M.DT_F16
MANY = (1 << 24) + 3


def test_dispatch_and_combine(dev):
    rng = np.random.default_rng(0)
    ids = rng.integers(-1, 4, MANY).astype(np.int32)
    x = rng.integers(0, 0x7c00, MANY).astype(np.uint16)
    order = np.concatenate([np.nonzero(ids == e)[0] for e in range(4)])
    want = np.full(MANY, -1, np.int32)
    want[order] = np.arange(order.size)
    bufs = [dev.upload(ids), dev.alloc(16), dev.alloc(4 * MANY), dev.upload(x), dev.upload(np.zeros_like(x)), dev.upload(np.full(MANY, 2, np.float32)), dev.alloc(2 * MANY)]
    i, counts, rows, xb, xs, w, out = bufs
    dev.moe_dispatch(MANY, 1, 4, i, counts, rows, xb, H, 1, xs)
    assert np.array_equal(dev.download(counts, np.int32, 4), np.bincount(ids[ids >= 0], minlength=4))
    assert np.array_equal(dev.download(rows, np.int32, MANY), want)
    assert np.array_equal(dev.download(xs, np.uint16, MANY)[:order.size], x[order])
    dev.moe_combine(MANY, 1, 1, xs, H, rows, w, out, H, add=xb)
    v = x.view(np.float16).astype(np.float32)
    with np.errstate(over="ignore"):
        both = np.where(ids >= 0, v + 2 * v, v).astype(np.float16)
    assert np.array_equal(dev.download(out, np.uint16, MANY), both.view(np.uint16))
    for b in bufs:
        b.free()


def test_route(dev):
    t = (1 << 26) - 1
    logits = np.zeros(t, np.float16)
    logits[::7] = -np.inf
    bufs = [dev.upload(logits), dev.alloc(4 * t), dev.alloc(4 * t)]
    dev.moe_route(t, 1, 1, bufs[0], H, bufs[1], bufs[2], scale=3.0)
    gone = np.isneginf(logits)
    assert np.array_equal(dev.download(bufs[1], np.int32, t), np.where(gone, -1, 0))
    assert np.array_equal(dev.download(bufs[2], np.float32, t), np.where(gone, 0, 3).astype(np.float32))
    for b in bufs:
        b.free()


def test_rows_past_a_grid_are_refused(dev):
    L, c, p = M.load(), dev.ctx, dev.alloc(4096).p
    assert L.mx_block_quantize(c, p, M.DT_F32, 1 << 28, 16, p, p) == M.MX_EINVAL
    assert L.mx_block_matmul(c, p, p, p, p, p, H, 1 << 28, 16, 16) == M.MX_EINVAL
    assert L.mx_block_matmul(c, p, p, p, p, p, H, 1, 1 << 28, 16) == M.MX_EINVAL
    q = M.QMatrix(p.value, p.value)
    cfg, w = M.MlpConfig(1 << 28, 16, 16), M.MlpWeights(q, q, q)
    assert L.mx_fmt_mlp_forward(c, M.WFMT_FP8_BLOCK, ctypes.byref(cfg), p, ctypes.byref(w), p) == M.MX_EINVAL


def test_sizes_past_an_int_are_refused(dev):
    L, c, p = M.load(), dev.ctx, dev.alloc(4096).p
    for hidden in (1 << 28, 0x7fffffff):
        assert L.mx_moe_dispatch(c, 1, 1, 1, p, p, p, p, H, hidden, p) == M.MX_EINVAL
        assert L.mx_moe_combine(c, 1, 1, hidden, p, H, p, p, None, p, H) == M.MX_EINVAL
    assert L.mx_fmt_quantize(c, M.WFMT_FP8_BLOCK, p, 1 << 28, 16, p, p) == M.MX_EINVAL
    assert L.mx_fmt_quantize(c, M.WFMT_FP8_BLOCK, p, 0x7fffffff, 16, p, p) == M.MX_EINVAL
    assert L.mx_fmt_quantize(c, M.WFMT_FP8_BLOCK, p, 1, 65552, p, p) == M.MX_EINVAL


def test_one_long_row(dev):
    """The longest row of a token out and back."""
    hidden = (1 << 28) - 1
    x = dev.alloc(2 * hidden)
    xs, out = dev.alloc(2 * hidden), dev.alloc(2 * hidden)
    dev.fill_normal(x, H, hidden, seed=3)
    dev.memset(out, 0)
    ids, counts, rows, w = dev.upload(np.zeros(1, np.int32)), dev.alloc(4), dev.alloc(4), dev.upload(np.ones(1, np.float32))
    dev.moe_dispatch(1, 1, 1, ids, counts, rows, x, H, hidden, xs)
    dev.moe_combine(1, 1, hidden, xs, H, rows, w, out, H)
    got, want = dev.download(out, np.float16, hidden), dev.download(x, np.float16, hidden)
    for b in (x, xs, out):
        b.free()
    assert np.array_equal(got, want)

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

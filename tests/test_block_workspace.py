"""The workspace of the block-FP8 calls: the largest shape's holds every smaller one's,
so that calls after a captured one do not free what its graph points at."""
import ctypes

import numpy as np
import pytest

import block_ref as R
import mxfp4hip as M
from test_block_rules import splits, tile_rows

PARTS = ["xq", "xs", "rows", "src", "counts", "tiles", "n_tiles", "hist", "mid", "mq", "ms", "y", "total"]


class Layout(ctypes.Structure):
    _fields_ = [(n, ctypes.c_size_t) for n in PARTS]


def layout(t, h, i, e, k):
    f = M.load()._ZN2mx14experts_layoutEiiiii
    f.restype = Layout
    got = f(t, h, i, e, k)
    return {n: getattr(got, n) for n in PARTS}


def split_bytes(m, n, k):
    f = M.load()._ZN2mx17block_split_bytesEiii
    f.restype = ctypes.c_size_t
    return f(m, n, k)


SHAPES = [(7168, 2048, 64, 8), (256, 256, 8, 2), (4096, 1408, 32, 1), (1024, 512, 1, 1), (512, 256, 1, 64), (128, 384, 512, 8), (9216, 128, 4, 4)]


@pytest.mark.parametrize("h,i,e,k", SHAPES)
def test_experts_need_no_less_for_more_tokens(h, i, e, k):
    need = [layout(t, h, i, e, k)["total"] for t in list(range(1, 700)) + list(range(700, 20000, 97))]
    assert need == sorted(need)
    assert layout(100, h, i, e, k)["total"] <= layout(100, h + 16, i + 16, e + 1, k)["total"]


@pytest.mark.parametrize("h,i,e,k", SHAPES)
def test_experts_parts_hold_what_is_written(h, i, e, k):
    for t in list(range(1, 200)) + [255, 256, 1000, 4096, 8192, 8193]:
        n, l = t * k, layout(t, h, i, e, k)
        ends = [l[p] for p in PARTS[1:]]
        size = {p: end - l[p] for p, end in zip(PARTS, ends)}
        used = min(n, e)
        rows = tile_rows(n, used, i, h, M.DT_F16, True)
        want = {"xq": t * h, "xs": t * R.blocks(h) * 4, "rows": n * 4, "src": n * 4, "counts": e * 4, "tiles": (used + n // rows) * 16,
                "n_tiles": 4, "hist": -(-n // 4096) * e * 4 if n > 65536 else 0, "mid": n * i * 4 if rows <= 32 or t == 1 else 0,
                "mq": n * i, "ms": n * R.blocks(i) * 4, "y": n * h * 4}
        assert all(size[p] >= want[p] for p in want), (t, size, want)
        assert all(l[p] % 256 == 0 for p in PARTS)


@pytest.mark.parametrize("n,k", [(4096, 4096), (1221, 3968), (128, 1024), (1, 65536), (2080, 5536), (512, 2048), (640, 128)])
def test_products_need_no_less_for_more_rows(n, k):
    need = [split_bytes(m, n, k) for m in range(1, 3000)]
    assert need == sorted(need)
    for m in range(1, 3000):
        for dtype in (M.DT_F16, M.DT_F32):
            s = splits(m, n, k, tile_rows(m, 1, n, k, dtype))
            assert s == 1 or need[m - 1] >= s * m * n * 4, (m, s)


@pytest.mark.gpu
def test_smaller_calls_beside_a_captured_one():
    """The largest batch once, a smaller one captured, others of every kernel called
    in between: each replay gives what the call itself does."""
    h, i, e, k, n, kk = 256, 256, 8, 2, 512, 2048
    L, vp, byref = M.load(), ctypes.c_void_p, ctypes.byref
    with M.Device(0) as dev:
        rng = np.random.default_rng(0)
        bufs = {}

        def codes(count, rows, cols):
            q = rng.integers(0, 127, (count, rows, cols)).astype(np.uint8) | (rng.integers(0, 2, (count, rows, cols)) * 128).astype(np.uint8)
            s = rng.uniform(1e-3, 2e-3, (count, R.blocks(rows), R.blocks(cols))).astype(np.float32)
            return dev.upload(q), dev.upload(s)

        mats = codes(e, i, h), codes(e, i, h), codes(e, h, i)
        wt = M.Device.weights(*mats)
        a, b = codes(1, 1024, kk), codes(1, n, kk)
        sc = dev.upload(rng.uniform(1e-3, 2e-3, R.blocks(kk) * 1024).astype(np.float32))
        x = dev.upload(rng.normal(0, 1, (300, h)).astype(np.float16))
        ids = dev.upload(rng.integers(0, e, (300, k)).astype(np.int32))
        w = dev.upload(rng.random((300, k)).astype(np.float32))

        def step(t, m):
            if (t, m) not in bufs:
                bufs[t, m] = dev.alloc(t * h * 2), dev.alloc(m * n * 2)
            out, c = bufs[t, m]
            dev.moe_block_forward(t, h, i, e, k, x, M.DT_F16, ids, w, wt, out)
            dev.block_matmul(a[0], sc, b[0], b[1], c, M.DT_F16, m, n, kk)
            return out, c

        def results(t, m, of):
            return dev.download(of[0], np.uint16, t * h), dev.download(of[1], np.uint16, m * n)

        step(300, 1024)
        out = bufs[60, 64] = dev.alloc(60 * h * 2), dev.alloc(64 * n * 2)
        side, graph, replay = vp(), vp(), vp()
        assert L.hipStreamCreateWithFlags(byref(side), 1) == 0
        assert L.mx_set_stream(dev.ctx, side) == M.MX_OK
        try:
            assert L.hipStreamBeginCapture(side, 1) == 0
            step(60, 64)
            assert L.hipStreamEndCapture(side, byref(graph)) == 0
        finally:
            L.mx_set_stream(dev.ctx, None)
        assert L.hipGraphInstantiate(byref(replay), graph, None, None, vp(0)) == 0
        want = results(60, 64, step(60, 64))
        assert np.isfinite(want[0].view(np.float16)).all() and np.isfinite(want[1].view(np.float16)).all()
        for other in ((1, 1), (40, 40), (80, 100), (161, 200), (299, 700)):
            step(*other)
            for o in out:
                dev.memset(o, 0xff)
            dev.sync()
            assert L.hipGraphLaunch(replay, side) == 0 and L.hipStreamSynchronize(side) == 0
            got = results(60, 64, out)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])

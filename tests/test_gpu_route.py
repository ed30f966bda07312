"""Router, dispatch and combine against their definitions in 64 bits (GPU)."""
import ctypes

import numpy as np
import pytest

import block_ref as R
import mxfp4hip as M

pytestmark = pytest.mark.gpu
F, H, B = M.DT_F32, M.DT_F16, M.DT_BF16


def run_route(dev, logits, dtype, topk, bias=None, stride=0, **kw):
    t, e = logits.shape
    buf = np.full((t, stride or e), 7.0)
    buf[:, :e] = logits
    ids, w = dev.alloc(t * topk * 4), dev.alloc(t * topk * 4)
    dev.moe_route(t, e, topk, dev.upload(R.bits_of(buf, dtype)), dtype, ids, w,
                  bias=None if bias is None else dev.upload(bias.astype(np.float32)), stride=stride, **kw)
    return dev.download(ids, np.int32, (t, topk)), dev.download(w, np.float32, (t, topk))


def check_route(dev, logits, dtype, topk, bias=None, stride=0, sure_share=0.9, **kw):
    logits = R.values_of(R.bits_of(logits, dtype), dtype)
    ids, w = run_route(dev, logits, dtype, topk, bias, stride, **kw)
    rids, rw, sure = R.route(logits, bias, topk, kw.get("score", M.ROUTE_SOFTMAX) == M.ROUTE_SIGMOID, kw.get("groups", 1),
                             kw.get("topk_groups", 1), kw.get("group_top", 1), kw.get("renormalize", False), kw.get("scale", 1.0))
    assert sure.mean() >= sure_share
    assert np.array_equal(ids[sure], rids[sure])
    # f32 scores: the exponential within 2 ulp of its argument's 2^-24 (arguments past 104 give 0), a quotient, the sum, two products
    tol = (min(104, np.abs(logits[np.isfinite(logits)]).max(initial=0)) * 2 + 16) * R.EPS
    assert np.all(np.abs(w - rw)[sure] <= tol * np.abs(rw)[sure] + 1e-37)
    return ids, w


@pytest.mark.parametrize("score", [M.ROUTE_SOFTMAX, M.ROUTE_SIGMOID])
@pytest.mark.parametrize("dtype", [F, H, B])
@pytest.mark.parametrize("tokens,experts,topk", [(1, 1, 1), (1, 64, 8), (3, 8, 8), (5, 65, 3), (37, 128, 6), (9, 257, 64), (65, 512, 9)])
def test_route(dev, score, dtype, tokens, experts, topk):
    rng = np.random.default_rng(tokens * experts + topk)
    logits = rng.normal(0, 1.5, (tokens, experts))
    for bias in (None, rng.integers(-100, 101, experts) * 0.001):
        for renorm in (False, True):
            check_route(dev, logits, dtype, topk, bias, score=score, renormalize=renorm, scale=2.5, sure_share=0.0)


@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("tokens,experts,groups,kept,topk", [(33, 256, 8, 4, 8), (17, 64, 4, 1, 16), (7, 96, 32, 3, 5), (4, 64, 64, 64, 2),
                                                             (64, 60, 3, 2, 4), (3, 512, 2, 1, 32)])
def test_route_groups(dev, tokens, experts, groups, kept, topk, group_top):
    rng = np.random.default_rng(experts + groups)
    logits = rng.normal(0, 1.5, (tokens, experts))
    bias = rng.integers(-100, 101, experts) * 0.001
    for b, score in ((bias, M.ROUTE_SIGMOID), (None, M.ROUTE_SOFTMAX), (bias, M.ROUTE_SOFTMAX)):
        check_route(dev, logits, F, topk, b, score=score, groups=groups, topk_groups=kept, group_top=group_top, renormalize=True, sure_share=0.0)


@pytest.mark.parametrize("score", [M.ROUTE_SOFTMAX, M.ROUTE_SIGMOID])
@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 3)])
def test_route_ties_take_the_lowest_index(dev, score, groups, kept):
    rng = np.random.default_rng(5)
    logits = rng.integers(0, 3, (50, 128)).astype(np.float64)
    logits[0] = 0
    ids, _ = check_route(dev, logits, F, 16, score=score, groups=groups, topk_groups=kept, sure_share=1.0)
    assert ids[0].tolist() == list(range(16))


@pytest.mark.parametrize("score", [M.ROUTE_SOFTMAX, M.ROUTE_SIGMOID])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_masks(dev, score, groups):
    """Masked experts, rows left with few or none, infinities, the type's lowest value."""
    inf, low = np.inf, float(np.finfo(np.float32).min)
    logits = np.tile(np.linspace(-1, 1, 32), (8, 1))
    logits[1] = -inf
    logits[2] = np.nan
    logits[3] = -inf
    logits[3, [4, 30]] = [0.5, 0.25]
    logits[4, 3] = inf
    logits[5, 1:] = low
    logits[6, ::2] = np.nan
    logits[7] = low
    ids, w = check_route(dev, logits, F, 4, score=score, groups=groups, topk_groups=max(1, groups - 1), group_top=2, renormalize=True, sure_share=1.0)
    for r in (1, 2):
        assert (ids[r] == -1).all() and (w[r] == 0).all()
    assert ids[3].tolist() == [4, 30, -1, -1] and (w[3, 2:] == 0).all()
    assert np.isfinite(w).all()


def test_route_bias_can_mask(dev):
    logits = np.tile(np.linspace(1, -1, 16), (3, 1))
    bias = np.zeros(16)
    bias[[0, 2]] = -np.inf, np.nan
    ids, _ = run_route(dev, logits, F, 16, bias, score=M.ROUTE_SIGMOID)
    assert ids[0].tolist() == [1] + list(range(3, 16)) + [-1, -1]


@pytest.mark.parametrize("dtype", [F, H])
def test_route_stride(dev, dtype):
    logits = np.random.default_rng(1).normal(0, 1, (11, 24))
    a = run_route(dev, logits, dtype, 5)
    b = run_route(dev, logits, dtype, 5, stride=37)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


# ---- dispatch ----------------------------------------------------------------------
@pytest.mark.parametrize("tokens,topk,experts", [(1, 1, 1), (1, 8, 64), (2, 3, 5), (255, 8, 64), (256, 8, 64), (257, 8, 512), (1000, 5, 7),
                                                 (4096, 8, 256), (5001, 3, 33)])
@pytest.mark.parametrize("drop", [False, True])
def test_dispatch_order(dev, tokens, topk, experts, drop):
    rng = np.random.default_rng(tokens + topk)
    ids = (experts * rng.random((tokens, topk)) ** 2).astype(np.int32)  # uneven, with repeats in a token
    if drop:
        ids[rng.random(ids.shape) < 0.3] = -1
        ids[0, 0] = experts  # out of range too
    counts, rows = dev.alloc(experts * 4), dev.alloc(tokens * topk * 4)
    dev.moe_dispatch(tokens, topk, experts, dev.upload(ids), counts, rows)
    rc, rr, _ = R.dispatch(ids, experts)
    assert np.array_equal(dev.download(counts, np.int32, experts), rc)
    assert np.array_equal(dev.download(rows, np.int32, ids.shape), rr)


def test_dispatch_of_nothing(dev):
    counts = dev.upload(np.full(9, 5, np.int32))
    dev.moe_dispatch(0, 4, 9, dev.alloc(4), counts, dev.alloc(4))
    assert not dev.download(counts, np.int32, 9).any()
    ids = dev.upload(np.full((3, 2), -1, np.int32))
    rows = dev.alloc(24)
    dev.moe_dispatch(3, 2, 9, ids, counts, rows)
    assert not dev.download(counts, np.int32, 9).any()
    assert (dev.download(rows, np.int32, 6) == -1).all()


@pytest.mark.parametrize("dtype", [F, H, B])
@pytest.mark.parametrize("hidden", [1, 7, 16, 130, 4096])
def test_dispatch_rows(dev, dtype, hidden):
    rng = np.random.default_rng(hidden)
    tokens, topk, experts = 45, 3, 11
    ids = rng.integers(-1, experts, (tokens, topk)).astype(np.int32)
    x = R.bits_of(rng.normal(0, 1, (tokens, hidden)), dtype)
    counts, rows = dev.alloc(experts * 4), dev.alloc(tokens * topk * 4)
    mark = np.full((tokens * topk, hidden), 3, x.dtype)
    xs = dev.upload(mark)
    dev.moe_dispatch(tokens, topk, experts, dev.upload(ids), counts, rows, dev.upload(x), dtype, hidden, xs)
    _, _, slots = R.dispatch(ids, experts)
    got = dev.download(xs, x.dtype, mark.shape)
    assert np.array_equal(got[:slots.size], x[slots // topk])
    assert np.array_equal(got[slots.size:], mark[slots.size:])  # nothing past the last pair


# ---- combine -----------------------------------------------------------------------
@pytest.mark.parametrize("yt,ot", [(H, H), (B, B), (F, F), (F, H), (F, B), (H, F)])
@pytest.mark.parametrize("tokens,topk,hidden", [(1, 1, 8), (1, 8, 7168), (33, 3, 130), (7, 64, 1), (200, 8, 2056)])
@pytest.mark.parametrize("add", [False, True])
def test_combine(dev, yt, ot, tokens, topk, hidden, add):
    rng = np.random.default_rng(tokens + hidden)
    n = tokens * topk
    rows = rng.permutation(n).astype(np.int32).reshape(tokens, topk)
    rows[rng.random(rows.shape) < 0.2] = -1
    w = rng.normal(0, 1, (tokens, topk)).astype(np.float32)
    w[rows < 0] = np.nan  # not used
    y = R.bits_of(rng.normal(0, 1, (n, hidden)), yt)
    base = R.bits_of(rng.normal(0, 1, (tokens, hidden)), ot)
    out = dev.upload(base)
    dev.moe_combine(tokens, topk, hidden, dev.upload(y), yt, dev.upload(rows), dev.upload(w), out, ot, add=out if add else None)
    ref = R.values_of(base, ot) if add else np.zeros((tokens, hidden))
    size = np.abs(ref)
    yv = R.values_of(y, yt)
    for s in range(topk):
        term = np.where(rows[:, s, None] >= 0, np.nan_to_num(w[:, s, None].astype(np.float64)) * yv[rows[:, s]], 0)
        ref, size = ref + term, size + np.abs(term)
    err = R.rounded(ref, (topk + 1) * R.EPS * size, ot)
    assert np.all(np.abs(R.values_of(dev.download(out, base.dtype, base.shape), ot) - ref) <= err)


# ---- refusals ------------------------------------------------------------------------
def refused(rc):
    return rc == M.MX_EINVAL


def test_refusals(dev):
    L, c = M.load(), dev.ctx
    buf = dev.alloc(4096)
    p, odd = buf.p, buf.offset(2)

    def route(logits=p, dtype=F, stride=0, ids=p, w=p, **kw):
        cfg = M.RouteConfig(**{**dict(tokens=2, experts=8, topk=2, score=0, groups=1, topk_groups=1, group_top=1, renormalize=0, scale=1.0), **kw})
        return L.mx_moe_route(c, ctypes.byref(cfg), logits, dtype, stride, None, ids, w)

    bad = [dict(experts=0), dict(experts=513), dict(topk=0), dict(topk=9), dict(topk=65, experts=512), dict(score=2), dict(groups=3),
           dict(groups=65, experts=130), dict(groups=4, topk_groups=0), dict(groups=4, topk_groups=5), dict(groups=4, topk_groups=2, group_top=3),
           dict(groups=4, topk_groups=1, topk=3), dict(stride=7), dict(dtype=M.DT_I8), dict(logits=None), dict(ids=None), dict(w=None),
           dict(logits=odd), dict(ids=odd), dict(tokens=0x80000000)]
    for kw in bad:
        assert refused(route(**kw)), kw
        assert dev_error(dev)
    assert refused(L.mx_moe_route(c, None, p, F, 0, None, p, p))
    assert route(tokens=0, logits=None) == M.MX_OK

    def dispatch(tokens=2, topk=2, experts=8, ids=p, counts=p, rows=p, x=None, dtype=F, hidden=4, xs=None):
        return L.mx_moe_dispatch(c, tokens, topk, experts, ids, counts, rows, x, dtype, hidden, xs)

    for kw in [dict(tokens=-1), dict(topk=0), dict(topk=65), dict(tokens=1 << 26, topk=64), dict(experts=0), dict(experts=513), dict(ids=None),
               dict(counts=None), dict(rows=None), dict(ids=odd), dict(x=p), dict(xs=p), dict(x=p, xs=p, dtype=M.DT_U8),
               dict(x=p, xs=p, hidden=0), dict(x=odd, xs=p)]:
        assert refused(dispatch(**kw)), kw

    def combine(tokens=2, topk=2, hidden=8, y=p, yt=F, rows=p, w=p, add=None, out=p, ot=F):
        return L.mx_moe_combine(c, tokens, topk, hidden, y, yt, rows, w, add, out, ot)

    for kw in [dict(tokens=-1), dict(topk=0), dict(hidden=0), dict(y=None), dict(yt=M.DT_I32), dict(rows=None), dict(w=None), dict(out=None),
               dict(ot=M.DT_U8), dict(y=odd), dict(add=odd), dict(out=odd), dict(w=odd)]:
        assert refused(combine(**kw)), kw
    assert combine(tokens=0, y=None) == M.MX_OK


def dev_error(dev):
    return len(M.load().mx_last_error(dev.ctx)) > 0

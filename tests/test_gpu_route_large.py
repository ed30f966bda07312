"""Router rows whose choice is certain, or is checked by its keys; dispatch and combine
of the sizes that each of their kernels takes (GPU)."""
import numpy as np
import pytest

import block_ref as R
import mxfp4hip as M
from test_gpu_route import check_route, run_route

pytestmark = pytest.mark.gpu
F, H, B = M.DT_F32, M.DT_F16, M.DT_BF16


def spaced_logits(rng, tokens, experts, top):
    """Logits whose softmax decides by more than 1e-5: all ranks of up to 256 experts
    (uneven steps, 2e-5 at least), the first `top` of more."""
    rank = np.argsort(rng.random((tokens, experts)), 1)
    if experts <= 256:
        steps = np.cumsum(rng.uniform(1, 2, (tokens, experts)), 1)
        p = np.take_along_axis(steps, experts - 1 - rank, 1)
        p /= p.sum(1, keepdims=True)
    else:
        p = np.where(rank < top, 0.004 + (top - rank) * 5e-5, rng.uniform(0.0005, 0.002, rank.shape))
    v = np.log(p)
    return v - v.max(1, keepdims=True)


@pytest.mark.parametrize("tokens,experts,topk", [(5, 65, 3), (9, 257, 64), (65, 512, 9), (17, 512, 64), (33, 256, 16)])
def test_route_of_spaced_keys(dev, tokens, experts, topk):
    rng = np.random.default_rng(tokens + experts)
    logits = spaced_logits(rng, tokens, experts, topk + 2)
    bias = rng.permutation(experts) * 0.01
    for renorm in (False, True):
        check_route(dev, logits, F, topk, None, score=M.ROUTE_SOFTMAX, renormalize=renorm, scale=2.5, sure_share=1.0)
        for score in (M.ROUTE_SOFTMAX, M.ROUTE_SIGMOID):
            check_route(dev, logits * 0.01, F, topk, bias, score=score, renormalize=renorm)


@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("tokens,experts,groups,kept,topk", [(3, 512, 2, 1, 32), (4, 64, 64, 64, 2), (9, 96, 32, 3, 5), (33, 256, 8, 4, 8)])
def test_route_groups_of_spaced_keys(dev, tokens, experts, groups, kept, topk, group_top):
    rng = np.random.default_rng(experts + groups)
    logits = spaced_logits(rng, tokens, experts, 4 * topk)
    check_route(dev, logits, F, topk, None, score=M.ROUTE_SOFTMAX, groups=groups, topk_groups=kept, group_top=group_top, renormalize=True,
                sure_share=0.4)  # (two keys' sums are close more often)


@pytest.mark.parametrize("score", [M.ROUTE_SOFTMAX, M.ROUTE_SIGMOID])
@pytest.mark.parametrize("dtype", [F, H, B])
@pytest.mark.parametrize("tokens,experts,topk", [(9, 257, 64), (65, 512, 9), (21, 512, 64), (37, 128, 6)])
def test_route_of_any_keys(dev, score, dtype, tokens, experts, topk):
    """Whichever of two close keys comes first: distinct experts whose keys are, rank
    by rank, the best, and their weights."""
    rng = np.random.default_rng(tokens + experts)
    logits = R.values_of(R.bits_of(rng.normal(0, 1.5, (tokens, experts)), dtype), dtype)
    ids, w = run_route(dev, logits, dtype, topk, score=score, scale=2.5)
    if score == M.ROUTE_SIGMOID:
        p = 1 / (1 + np.exp(-logits))
    else:
        p = np.exp(logits - logits.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
    assert ids.min() >= 0 and ids.max() < experts
    assert all(len(set(row)) == topk for row in ids.tolist())
    mine = np.take_along_axis(p, ids, 1)
    # f32 scores: the exponential of an argument within 2^-24 of 20, a quotient, the sum, a product
    tol = (20 * 2 + 16) * R.EPS
    assert np.all(np.abs(mine - -np.sort(-p, 1)[:, :topk]) <= 2 * tol * mine)
    assert np.all(np.abs(w - 2.5 * mine) <= tol * 2.5 * mine)


# ---- dispatch ----------------------------------------------------------------------
def order(ids, experts):
    flat = ids.reshape(-1)
    slots = np.argsort(np.where((flat >= 0) & (flat < experts), flat, experts), kind="stable")
    counts = np.bincount(flat[(flat >= 0) & (flat < experts)], minlength=experts)
    slots = slots[:counts.sum()]
    rows = np.full(flat.size, -1, np.int32)
    rows[slots] = np.arange(slots.size)
    return counts, rows.reshape(ids.shape), slots


@pytest.mark.parametrize("dtype,tokens,topk,experts,hidden", [
    (H, 300, 8, 64, 2100), (F, 256, 4, 9, 1030), (B, 257, 8, 512, 2049),     # one workgroup a token, rows past 4096 bytes
    (H, 100, 8, 64, 5001),                                                   # rows split over workgroups
    (H, 1500, 5, 33, 1055), (B, 5000, 3, 7, 9), (F, 1025, 4, 16, 2051), (H, 520, 64, 128, 17),  # order, then rows
    (H, 65537, 1, 33, 3), (B, 12501, 8, 512, 11), (F, 33333, 3, 1, 5),       # by a table of counts
])
@pytest.mark.parametrize("drop", [False, True])
def test_dispatch_rows_of_larger_batches(dev, dtype, tokens, topk, experts, hidden, drop):
    rng = np.random.default_rng(tokens + hidden)
    ids = (experts * rng.random((tokens, topk)) ** 2).astype(np.int32)
    if drop:
        ids[rng.random(ids.shape) < 0.3] = -1
        ids[0, 0], ids[-1, -1] = experts, -5
    x = R.bits_of(rng.normal(0, 1, (tokens, hidden)), dtype)
    mark = np.full((tokens * topk, hidden), 3, x.dtype)
    bufs = [dev.upload(ids), dev.alloc(experts * 4), dev.alloc(ids.size * 4), dev.upload(x), dev.upload(mark)]
    i, counts, rows, xb, xs = bufs
    dev.moe_dispatch(tokens, topk, experts, i, counts, rows, xb, dtype, hidden, xs)
    rc, rr, slots = order(ids, experts)
    assert np.array_equal(dev.download(counts, np.int32, experts), rc)
    assert np.array_equal(dev.download(rows, np.int32, ids.shape), rr)
    got = dev.download(xs, x.dtype, mark.shape)
    for b in bufs:
        b.free()
    assert np.array_equal(got[:slots.size], x[slots // topk])
    assert np.array_equal(got[slots.size:], mark[slots.size:])


@pytest.mark.parametrize("n", [65536, 65537, 69632, 100001])
@pytest.mark.parametrize("experts", [1, 33, 512])
def test_dispatch_order_of_many_slots(dev, n, experts):
    rng = np.random.default_rng(n + experts)
    ids = rng.integers(-1, experts + 1, (n, 1)).astype(np.int32)
    counts, rows = dev.alloc(experts * 4), dev.alloc(n * 4)
    dev.moe_dispatch(n, 1, experts, dev.upload(ids), counts, rows)
    rc, rr, _ = order(ids, experts)
    assert np.array_equal(dev.download(counts, np.int32, experts), rc)
    assert np.array_equal(dev.download(rows, np.int32, ids.shape), rr)


@pytest.mark.parametrize("yt,ot", [(H, H), (B, B), (F, H), (F, B), (B, F), (F, F)])
@pytest.mark.parametrize("tokens,topk,hidden", [(33, 3, 9), (5, 8, 1055), (12, 2, 2049), (3, 1, 4103)])
@pytest.mark.parametrize("add", [False, True])
def test_combine_of_odd_rows(dev, yt, ot, tokens, topk, hidden, add):
    rng = np.random.default_rng(tokens + hidden)
    n = tokens * topk
    rows = rng.permutation(n).astype(np.int32).reshape(tokens, topk)
    rows[rng.random(rows.shape) < 0.2] = -1
    w = rng.normal(0, 1, (tokens, topk)).astype(np.float32)
    y, base = R.bits_of(rng.normal(0, 1, (n, hidden)), yt), R.bits_of(rng.normal(0, 1, (tokens, hidden)), ot)
    out = dev.upload(np.concatenate([base.reshape(-1), np.full(32, 5, base.dtype)]))
    dev.moe_combine(tokens, topk, hidden, dev.upload(y), yt, dev.upload(rows), dev.upload(w), out, ot, add=out if add else None)
    got = dev.download(out, base.dtype, base.size + 32)
    assert (got[base.size:] == 5).all()
    ref = R.values_of(base, ot) if add else np.zeros((tokens, hidden))
    size = np.abs(ref)
    yv = R.values_of(y, yt)
    for s in range(topk):
        term = np.where(rows[:, s, None] >= 0, w[:, s, None].astype(np.float64) * yv[rows[:, s]], 0)
        ref, size = ref + term, size + np.abs(term)
    err = R.rounded(ref, (topk + 1) * R.EPS * size, ot)
    assert np.all(np.abs(R.values_of(got[:base.size].reshape(base.shape), ot) - ref) <= err)

"""Block-scaled FP8 against its definition in 64 bits (GPU)."""
import ctypes

import numpy as np
import pytest

import block_ref as R
import mxfp4hip as M

pytestmark = pytest.mark.gpu
F, H, B = M.DT_F32, M.DT_F16, M.DT_BF16


def quantize(dev, x, dtype):
    rows, k = x.shape
    q, s = dev.alloc(rows * k), dev.alloc(R.blocks(k) * rows * 4)
    dev.block_quantize(dev.upload(x), dtype, rows, k, q, s)
    return q, s


def weights(dev, rng, count, n, k, std=0.02):
    """`count` matrices through the library's quantizer: (data, scales) buffers and values."""
    qs, ss, vs = [], [], []
    for _ in range(count):
        w = rng.normal(0, std, (n, k)).astype(np.float32)
        w *= np.exp(rng.normal(0, 1, (R.blocks(n), R.blocks(k)))).astype(np.float32).repeat(128, 0).repeat(128, 1)[:n, :k]  # blocks differ
        q, s = dev.alloc(n * k), dev.alloc(R.blocks(n) * R.blocks(k) * 4)
        dev.fmt_quantize(M.WFMT_FP8_BLOCK, dev.upload(w), n, k, q, s)
        qs.append(dev.download(q, np.uint8, (n, k)))
        ss.append(dev.download(s, np.float32, (R.blocks(n), R.blocks(k))))
        vs.append(R.e4m3_values(qs[-1]) * R.spread_w(ss[-1], n, k))
    return dev.upload(np.stack(qs)), dev.upload(np.stack(ss)), vs


# ---- quantizers ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F, H, B])
@pytest.mark.parametrize("rows,k", [(1, 16), (1, 128), (3, 144), (17, 1024), (33, 2080), (16, 112), (130, 256)])
def test_activation_codes_and_scales(dev, dtype, rows, k):
    rng = np.random.default_rng(rows * k)
    x = rng.normal(0, 1, (rows, k)) * np.exp(rng.normal(0, 2, (rows, 1)))
    x[0, :16] = 0
    if rows > 2:
        x[2] = 0
    b = R.bits_of(x, dtype)
    q, s = quantize(dev, b, dtype)
    v = R.values_of(b, dtype)
    rs = R.act_scales(v)
    assert np.array_equal(dev.download(s, np.float32, (R.blocks(k), rows)), rs)
    assert np.array_equal(R.e4m3_values(dev.download(q, np.uint8, (rows, k))), R.act_codes(v, rs))


def test_activation_extremes(dev):
    """The largest and the smallest f32, subnormals, and blocks with a NaN or an infinity."""
    x = np.zeros((6, 256), np.float32)
    top = np.finfo(np.float32).max
    x[0, :4] = top, -top, top / 3, 1
    x[1, :3] = 1e-45, -3e-45, 0
    x[2, :3] = 2.0 ** -126, 2.0 ** -130, -(2.0 ** -118)
    x[3, 5], x[3, 200] = np.nan, 2
    x[4, 5], x[4, 6], x[4, 200] = -np.inf, 1, 2
    x[5] = np.linspace(-448, 448, 256)
    q, s = quantize(dev, x, F)
    codes = R.e4m3_values(dev.download(q, np.uint8, x.shape))
    sc = dev.download(s, np.float32, (2, 6))
    got = codes * np.repeat(sc.T, 128, 1)
    fine = np.ones(x.shape, bool)
    fine[3:5, :128] = False
    rs = R.act_scales(x[:3])
    assert np.array_equal(sc[:, :3], rs)
    assert np.array_equal(codes[:3], R.act_codes(x[:3], rs))
    two = 448 * float(2 * R.PER_448)
    assert np.isfinite(got[fine]).all() and got[3, 200] == two and got[4, 200] == two
    with np.errstate(invalid="ignore"):
        assert np.isnan(got[3, :128]).all() and np.isnan(got[4, :128]).all()


@pytest.mark.parametrize("n,k", [(128, 128), (1, 16), (130, 144), (300, 512)])
def test_weight_codes_and_scales(dev, n, k):
    rng = np.random.default_rng(n)
    w = rng.normal(0, 0.02, (n, k)).astype(np.float32)
    w[-1, -1] = 3.0
    q, s = dev.alloc(n * k), dev.alloc(R.blocks(n) * R.blocks(k) * 4)
    dev.fmt_quantize(M.WFMT_FP8_BLOCK, dev.upload(w), n, k, q, s)
    p = np.zeros((R.blocks(n) * 128, R.blocks(k) * 128), np.float32)
    p[:n, :k] = np.abs(w)
    rs = p.reshape(R.blocks(n), 128, R.blocks(k), 128).max((1, 3)) * R.PER_448
    assert np.array_equal(dev.download(s, np.float32, rs.shape), rs)
    want = R.e4m3((w / np.repeat(np.repeat(rs, 128, 0)[:n], 128, 1)[:, :k]).astype(np.float64))
    assert np.array_equal(R.e4m3_values(dev.download(q, np.uint8, (n, k))), want)


# ---- product ------------------------------------------------------------------------------
SIZES = [(1, 1, 16), (1, 128, 128), (1, 4096, 7168), (2, 130, 144), (5, 100, 1040), (8, 256, 512), (15, 513, 272), (16, 512, 2048), (17, 96, 4096),
         (31, 1000, 640), (33, 64, 128), (48, 384, 4112), (63, 257, 528), (64, 2048, 1024), (65, 129, 1024), (100, 640, 400), (127, 300, 2080),
         (128, 1024, 1024), (129, 128, 256), (200, 512, 144), (255, 1025, 384), (256, 256, 1152), (257, 2080, 5536), (400, 777, 896), (513, 512, 1040),
         (1000, 1536, 640)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(dev, m, n, k):
    rng = np.random.default_rng(m + n + k)
    x = (rng.normal(0, 1, (m, k)) * np.exp(rng.normal(0, 1, (m, 1)))).astype(np.float32)
    q, s = quantize(dev, x, F)
    rs = R.act_scales(x)
    wq, ws, wv = weights(dev, rng, 1, n, k)
    ref, err = R.product(R.act_codes(x, rs) * np.repeat(rs.T, 128, 1)[:, :k].astype(np.float64), wv[0])
    for ct in (F, H, B):
        c = dev.upload(np.full(m * n + 64, 9, R.np_type(ct)))
        dev.block_matmul(q, s, wq, ws, c, ct, m, n, k)
        got = dev.download(c, R.np_type(ct), m * n + 64)
        assert (got[m * n:] == 9).all()
        diff = np.abs(R.values_of(got[:m * n].reshape(m, n), ct) - ref)
        assert np.all(diff <= R.rounded(ref, err, ct)), (ct, diff.max())


@pytest.mark.parametrize("m,n,k", [(700, 16384, 272), (385, 16400, 400), (2050, 4100, 656), (4096, 2048, 128), (257, 32768, 144)])
@pytest.mark.parametrize("ct", [H, B])
def test_matmul_on_the_fp8_cores(dev, ct, m, n, k):
    """Sizes of the 256-row tiles, at random places and in the last rows and columns."""
    rng = np.random.default_rng(m + n + k)
    x = (rng.normal(0, 1, (m, k)) * np.exp(rng.normal(0, 1, (m, 1)))).astype(np.float32)
    q, s = quantize(dev, x, F)
    rs = R.act_scales(x)
    wq, ws, wv = weights(dev, rng, 1, n, k)
    rows = np.unique(np.r_[rng.integers(0, m, 60), 0, m - 1])
    cols = np.unique(np.r_[rng.integers(0, n, 400), 0, n - 20:n])
    a = R.act_codes(x, rs) * np.repeat(rs.T, 128, 1)[:, :k].astype(np.float64)
    ref, err = R.product(a[rows], wv[0][cols], cores=True)
    c = dev.upload(np.full(m * n + 64, 9, R.np_type(ct)))
    dev.block_matmul(q, s, wq, ws, c, ct, m, n, k)
    got = dev.download(c, R.np_type(ct), m * n + 64)
    assert (got[m * n:] == 9).all()
    diff = np.abs(R.values_of(got[:m * n].reshape(m, n)[np.ix_(rows, cols)], ct) - ref)
    assert np.all(diff <= R.rounded(ref, err, ct)), diff.max()


@pytest.mark.parametrize("m", [1, 20, 200])
def test_matmul_repeats_bit_for_bit(dev, m):
    rng = np.random.default_rng(m)
    n, k = 640, 2064
    q, s = quantize(dev, rng.normal(0, 1, (m, k)).astype(np.float32), F)
    wq, ws, _ = weights(dev, rng, 1, n, k)
    got = []
    for _ in range(3):
        c = dev.alloc(m * n * 4)
        dev.block_matmul(q, s, wq, ws, c, F, m, n, k)
        got.append(dev.download(c, np.uint32, m * n))
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


@pytest.mark.parametrize("m", [3, 150])
def test_matmul_nan_stays_in_its_row(dev, m):
    """A row with a NaN activation is NaN throughout; the other rows are untouched."""
    rng = np.random.default_rng(m)
    n, k = 200, 400
    x = rng.normal(0, 1, (m, k)).astype(np.float32)
    clean = x.copy()
    x[1, 390] = np.nan
    clean[1, 390] = 0
    wq, ws, _ = weights(dev, rng, 1, n, k)
    out = []
    for v in (x, clean):
        q, s = quantize(dev, v, F)
        c = dev.alloc(m * n * 4)
        dev.block_matmul(q, s, wq, ws, c, F, m, n, k)
        out.append(dev.download(c, np.float32, (m, n)))
    assert np.isnan(out[0][1]).all() and np.isfinite(out[1]).all()
    keep = np.arange(m) != 1
    assert np.array_equal(out[0][keep], out[1][keep])


# ---- MLPs ------------------------------------------------------------------------------------
def dequant(x, dtype):
    v = R.values_of(x, dtype)
    s = R.act_scales(v)
    return R.act_codes(v, s) * np.repeat(s.T, 128, 1)[:, :v.shape[1]].astype(np.float64)


@pytest.mark.parametrize("t,h,i", [(1, 256, 512), (3, 144, 272), (16, 512, 256), (40, 1024, 400), (130, 640, 1024), (300, 400, 384)])
def test_format_mlp(dev, t, h, i):
    rng = np.random.default_rng(t)
    x = R.bits_of(rng.normal(0, 1, (t, h)), H)
    ws = [weights(dev, rng, 1, n, k, std=0.05) for n, k in ((i, h), (i, h), (h, i))]
    out = dev.alloc(t * h * 2)
    dev.fmt_mlp_forward(M.WFMT_FP8_BLOCK, t, h, i, dev.upload(x), M.Device.weights(*[w[:2] for w in ws]), out)
    y, err = R.mlp(dequant(x, H), *[w[2][0] for w in ws])
    got = R.values_of(dev.download(out, np.float16, (t, h)), H)
    assert np.all(np.abs(got - y) <= R.rounded(y, err, H))


def expert_case(dev, t, h, i, e, k, dtype, seed, drop=0.0, one=None):
    rng = np.random.default_rng(seed)
    x = R.bits_of(rng.normal(0, 1, (t, h)), dtype)
    ids = np.argsort(rng.normal(0, 1, (t, e)) + rng.normal(0, 0.7, e), 1)[:, :k].astype(np.int32)
    if one is not None:
        ids[:] = one
    ids[rng.random(ids.shape) < drop] = -1
    w = rng.random((t, k)).astype(np.float32)
    ws = [weights(dev, rng, e, n, kk, std=0.05) for n, kk in ((i, h), (i, h), (h, i))]
    return x, ids, w, ws, R.bits_of(rng.normal(0, 1, (t, h)), dtype)


def expert_ref(x, ids, w, ws, add, dtype, cores=False):
    """Sum and bound; a slot's row may be rounded once to the rows' type."""
    xv = dequant(x, dtype)
    ref = np.zeros(x.shape) if add is None else R.values_of(add, dtype)
    err = np.zeros(x.shape)
    size = np.abs(ref)
    for e in range(len(ws[0][2])):
        t, s = np.nonzero(ids == e)
        if t.size:
            y, ey = R.mlp(xv[t], *[v[2][e] for v in ws], cores=cores)
            ey = R.rounded(y, ey, dtype)
            wt = w[t, s].astype(np.float64)[:, None]
            np.add.at(ref, t, wt * y)
            np.add.at(size, t, np.abs(wt * y))
            np.add.at(err, t, np.abs(wt) * ey)
    return ref, R.rounded(ref, err + (ids.shape[1] + 2) * R.EPS * size, dtype)


def run_experts(dev, x, ids, w, ws, add, dtype):
    t, h = x.shape
    i = ws[0][2][0].shape[0]
    out = dev.upload(add) if add is not None else dev.alloc(t * h * 2)
    dev.moe_block_forward(t, h, i, len(ws[0][2]), ids.shape[1], dev.upload(x), dtype, dev.upload(ids), dev.upload(w),
                          M.Device.weights(*[v[:2] for v in ws]), out, add=out if add is not None else None)
    return R.values_of(dev.download(out, x.dtype, x.shape), dtype)


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("t,h,i,e,k", [(1, 256, 128, 8, 2), (1, 512, 272, 4, 4), (2, 144, 144, 3, 1), (7, 256, 384, 16, 4), (20, 400, 256, 2, 1),
                                       (64, 256, 256, 8, 3), (150, 384, 144, 4, 2), (300, 256, 256, 3, 2), (520, 128, 400, 2, 1)])
@pytest.mark.parametrize("add", [False, True])
def test_experts(dev, dtype, t, h, i, e, k, add):
    x, ids, w, ws, base = expert_case(dev, t, h, i, e, k, dtype, t + h)
    ref, err = expert_ref(x, ids, w, ws, base if add else None, dtype)
    got = run_experts(dev, x, ids, w, ws, base if add else None, dtype)
    assert np.all(np.abs(got - ref) <= err)


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("t,h,i,e,k", [(1100, 256, 2064, 4, 1), (1000, 400, 1040, 8, 2)])
def test_experts_on_the_fp8_cores(dev, dtype, t, h, i, e, k):
    x, ids, w, ws, base = expert_case(dev, t, h, i, e, k, dtype, t + h, drop=0.05)
    ref, err = expert_ref(x, ids, w, ws, base, dtype, cores=True)
    got = run_experts(dev, x, ids, w, ws, base, dtype)
    assert np.all(np.abs(got - ref) <= err)


def test_format_mlp_on_the_fp8_cores(dev):
    t, h, i = 600, 272, 8208
    rng = np.random.default_rng(t)
    x = R.bits_of(rng.normal(0, 1, (t, h)), H)
    ws = [weights(dev, rng, 1, n, k, std=0.05) for n, k in ((i, h), (i, h), (h, i))]
    out = dev.alloc(t * h * 2)
    dev.fmt_mlp_forward(M.WFMT_FP8_BLOCK, t, h, i, dev.upload(x), M.Device.weights(*[w[:2] for w in ws]), out)
    rows = np.unique(np.r_[rng.integers(0, t, 40), 0, t - 1])
    y, err = R.mlp(dequant(x, H)[rows], *[w[2][0] for w in ws], cores=True)
    got = R.values_of(dev.download(out, np.float16, (t, h)), H)[rows]
    assert np.all(np.abs(got - y) <= R.rounded(y, err, H))


@pytest.mark.parametrize("t", [1, 40, 300])
def test_experts_with_empty_slots_and_rows(dev, t):
    x, ids, w, ws, base = expert_case(dev, t, 256, 256, 6, 3, H, t, drop=0.5)
    ids[0] = -1
    w[ids < 0] = np.nan
    ref, err = expert_ref(x, ids, np.nan_to_num(w), ws, base, H)
    got = run_experts(dev, x, ids, w, ws, base, H)
    assert np.all(np.abs(got - ref) <= err)
    assert np.array_equal(got[0], R.values_of(base[0], H))


@pytest.mark.parametrize("t", [5, 200])
def test_experts_all_on_one(dev, t):
    x, ids, w, ws, _ = expert_case(dev, t, 256, 256, 5, 1, B, t, one=3)
    ref, err = expert_ref(x, ids, w, ws, None, B)
    assert np.all(np.abs(run_experts(dev, x, ids, w, ws, None, B) - ref) <= err)


def test_experts_of_nothing(dev):
    M.load().mx_moe_block_forward  # tokens = 0 touches no buffer
    x, ids, w, ws, _ = expert_case(dev, 1, 128, 128, 2, 1, H, 0)
    dev.moe_block_forward(0, 128, 128, 2, 1, dev.upload(x), H, dev.upload(ids), dev.upload(w), M.Device.weights(*[v[:2] for v in ws]), dev.alloc(16))
    dev.sync()


def test_route_to_experts_in_a_graph(dev):
    """Router, experts: captured once on a stream of the caller's, replayed with
    other logits and rows; every replay as the calls themselves give it."""
    t, h, i, e, k = 12, 256, 128, 16, 4
    rng = np.random.default_rng(3)
    _, _, _, ws, _ = expert_case(dev, t, h, i, e, k, H, 9)
    wt = M.Device.weights(*[v[:2] for v in ws])
    x, logits = dev.alloc(t * h * 2), dev.alloc(t * e * 4)
    ids, w, out = dev.alloc(t * k * 4), dev.alloc(t * k * 4), dev.alloc(t * h * 2)
    L = M.load()

    def step():
        dev.moe_route(t, e, k, logits, F, ids, w, renormalize=True)
        dev.moe_block_forward(t, h, i, e, k, x, H, ids, w, wt, out)

    def fill(seed):
        r = np.random.default_rng(seed)
        dev.upload(r.normal(0, 1, (t, h)).astype(np.float16), x)
        dev.upload(r.normal(0, 1, (t, e)).astype(np.float32), logits)

    fill(0)
    step()
    dev.sync()
    vp, byref = ctypes.c_void_p, ctypes.byref
    side, graph, replay = vp(), vp(), vp()
    assert L.hipStreamCreateWithFlags(byref(side), 1) == 0
    assert L.mx_set_stream(dev.ctx, side) == M.MX_OK
    try:
        assert L.hipStreamBeginCapture(side, 1) == 0
        step()
        assert L.hipStreamEndCapture(side, byref(graph)) == 0
    finally:
        L.mx_set_stream(dev.ctx, None)
    assert L.hipGraphInstantiate(byref(replay), graph, None, None, vp(0)) == 0
    for seed in range(1, 5):
        fill(seed)
        step()
        want = dev.download(out, np.uint16, (t, h))
        dev.memset(out, 0xff)
        dev.sync()
        assert L.hipGraphLaunch(replay, side) == 0 and L.hipStreamSynchronize(side) == 0
        assert np.array_equal(dev.download(out, np.uint16, (t, h)), want)


# ---- refusals ------------------------------------------------------------------------------------
def test_refusals(dev):
    L, c = M.load(), dev.ctx
    buf = dev.alloc(1 << 16)
    p, odd = buf.p, buf.offset(8)

    def quant(src=p, dtype=F, rows=2, k=32, q=p, s=p):
        return L.mx_block_quantize(c, src, dtype, rows, k, q, s)

    for kw in [dict(rows=-1), dict(k=0), dict(k=24), dict(dtype=M.DT_U8), dict(src=None), dict(q=None), dict(s=None), dict(src=odd), dict(q=odd),
               dict(s=buf.offset(2))]:
        assert quant(**kw) == M.MX_EINVAL, kw
    assert quant(rows=0, src=None) == M.MX_OK

    def mul(a=p, as_=p, b=p, bs=p, out=p, ct=F, m=2, n=4, k=32):
        return L.mx_block_matmul(c, a, as_, b, bs, out, ct, m, n, k)

    for kw in [dict(m=-1), dict(n=0), dict(k=0), dict(k=40), dict(ct=M.DT_I32), dict(a=None), dict(as_=None), dict(b=None), dict(bs=None),
               dict(out=None), dict(a=odd), dict(b=odd), dict(out=odd), dict(bs=buf.offset(1))]:
        assert mul(**kw) == M.MX_EINVAL, kw
    assert mul(m=0, a=None) == M.MX_OK

    q = M.QMatrix(buf.ptr, buf.ptr)

    def experts(t=2, h=32, i=32, e=2, k=1, x=p, dtype=H, ids=p, w=p, mats=(q, q, q), add=None, out=p):
        cfg, ws = M.MlpConfig(t, h, i), M.MlpWeights(*mats)
        return L.mx_moe_block_forward(c, ctypes.byref(cfg), e, k, x, dtype, ids, w, ctypes.byref(ws), add, out)

    none, shifted = M.QMatrix(None, buf.ptr), M.QMatrix(buf.ptr + 8, buf.ptr)
    for kw in [dict(h=0), dict(h=24), dict(i=40), dict(e=0), dict(e=513), dict(k=0), dict(k=65), dict(x=None), dict(x=odd), dict(dtype=F),
               dict(ids=None), dict(w=None), dict(out=None), dict(out=odd), dict(add=odd), dict(mats=(none, q, q)), dict(mats=(q, q, shifted)),
               dict(t=1 << 30, k=4)]:
        assert experts(**kw) == M.MX_EINVAL, kw
    assert L.mx_moe_block_forward(c, None, 2, 1, p, H, p, p, None, None, p) == M.MX_EINVAL
    cfg, ws = M.MlpConfig(2, 40, 32), M.MlpWeights(q, q, q)
    assert L.mx_fmt_mlp_forward(c, M.WFMT_FP8_BLOCK, ctypes.byref(cfg), p, ctypes.byref(ws), p) == M.MX_EINVAL
    assert L.mx_fmt_quantize(c, M.WFMT_FP8_BLOCK, p, 2, 24, p, p) == M.MX_EINVAL

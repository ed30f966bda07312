"""Measured cases of the routed-experts operators of libmxfp4hip on one MI355X.

  route     gate logits to expert ids and weights (mx_moe_route)
  dispatch  a batch's rows into expert order, with the counts (mx_moe_dispatch)
  combine   the experts' rows back into token order, weighted (mx_moe_combine)
  project   one linear layer with FP8 weights and a scale per 128 x 128 block:
            activations quantized per 1 x 128, then the product
            (mx_block_quantize, mx_block_matmul)
  experts   the MLP of each token's experts in that format, from token rows to
            token rows (mx_moe_block_forward)

`own` chooses between the library's calls and the plain form: elementary torch
operations in 32 bits.  exact() is written from the definitions in 64 bits.

Data: activations ~ N(0, 1), weights ~ N(0, 0.02) quantized here, logits ~
N(0, 1) with an offset per expert, so that experts are unevenly popular.
"""
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
FLT_MAX = 3.4028234663852886e38
BLOCK = 128

_M = None
_dev = None


def lib():
    """The library's binding, and the context that a program keeps for its life."""
    global _M, _dev
    if _M is None:
        sys.path.insert(0, os.path.join(ROOT, "mpp-4.1-fp4-fp8-block_amd"))
        import mxfp4hip
        _M, _dev = mxfp4hip, mxfp4hip.Device(0)
    return _M, _dev


# ---- the cases -------------------------------------------------------------------
def listed():
    return [
        # the gate of a decode step with one sequence
        {"name": "route_1", "kind": "route", "tokens": 1, "experts": 64, "topk": 8, "score": "softmax", "bias": False,
         "groups": 1, "topk_groups": 1, "group_top": 1, "renormalize": True, "logits": "f32"},
        # the gate of a prefill: sigmoid scores, a balance bias, the best 4 of 8 groups
        {"name": "route_8192", "kind": "route", "tokens": 8192, "experts": 256, "topk": 8, "score": "sigmoid",
         "bias": True, "groups": 8, "topk_groups": 4, "group_top": 2, "renormalize": True, "logits": "f32"},
        # a decode batch's rows to the experts, and a prefill's
        {"name": "dispatch_64", "kind": "dispatch", "tokens": 64, "experts": 64, "topk": 8, "hidden": 7168, "type": "f16"},
        {"name": "dispatch_4096", "kind": "dispatch", "tokens": 4096, "experts": 64, "topk": 8, "hidden": 7168, "type": "f16"},
        # and back
        {"name": "combine_64", "kind": "combine", "tokens": 64, "topk": 8, "hidden": 7168, "type": "f16", "add": False},
        {"name": "combine_4096", "kind": "combine", "tokens": 4096, "topk": 8, "hidden": 7168, "type": "bf16", "add": True},
        # a projection of one decoded token; of an odd batch at sizes off the block grid; of a prefill
        {"name": "project_1", "kind": "project", "m": 1, "n": 14336, "k": 4096, "a": "f16", "c": "f16"},
        {"name": "project_ragged_257", "kind": "project", "m": 257, "n": 2080, "k": 5536, "a": "f32", "c": "f32"},
        {"name": "project_4096", "kind": "project", "m": 4096, "n": 14336, "k": 4096, "a": "bf16", "c": "bf16"},
        # the experts of one decoded token, of a decode batch, of a prefill
        {"name": "experts_1", "kind": "experts", "tokens": 1, "experts": 64, "topk": 8, "hidden": 7168, "inter": 2048,
         "type": "f16", "add": False},
        {"name": "experts_256", "kind": "experts", "tokens": 256, "experts": 64, "topk": 8, "hidden": 7168, "inter": 2048,
         "type": "f16", "add": False},
        {"name": "experts_4096", "kind": "experts", "tokens": 4096, "experts": 64, "topk": 8, "hidden": 7168,
         "inter": 2048, "type": "bf16", "add": True},
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99))))


def _size(rng, lo, hi, step):
    return max(step, _log(rng, lo, hi) // step * step)


def draw(rng):
    kind = rng.choice(["route", "dispatch", "combine", "project", "project", "experts", "experts"])
    half = rng.choice(["f16", "bf16"])
    if kind == "route":
        groups = rng.choice([1, 1, 4, 8])
        kept = rng.randint(1, groups)
        experts = groups * rng.randint(-(-8 // groups), 384 // groups)
        return {"kind": kind, "tokens": _log(rng, 1, 16384), "experts": experts,
                "topk": rng.randint(1, min(16, experts // groups * kept)), "score": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.5, "groups": groups, "topk_groups": kept, "group_top": rng.choice([1, 2]),
                "renormalize": rng.random() < 0.7, "logits": rng.choice(["f32", "f32", "f16", "bf16"])}
    if kind == "dispatch":
        experts = rng.randint(8, 256)
        return {"kind": kind, "tokens": _log(rng, 1, 8192), "experts": experts, "topk": rng.randint(1, 8),
                "hidden": _size(rng, 512, 7168, rng.choice([1, 8, 64])), "type": half}
    if kind == "combine":
        return {"kind": kind, "tokens": _log(rng, 1, 8192), "topk": rng.randint(1, 8),
                "hidden": _size(rng, 512, 7168, rng.choice([1, 8, 64])), "type": half, "add": rng.random() < 0.5}
    if kind == "project":
        n = _size(rng, 512, 16384, 128) if rng.random() < 0.6 else _log(rng, 512, 16384)
        return {"kind": kind, "m": _log(rng, 1, 4096), "n": n, "k": _size(rng, 512, 8192, rng.choice([16, 128, 128])),
                "a": rng.choice([half, half, "f32"]), "c": rng.choice([half, half, "f32"])}
    experts = rng.choice([8, 16, 32, 64])
    step = rng.choice([16, 128, 128])
    return {"kind": kind, "tokens": _log(rng, 1, 4096), "experts": experts, "topk": rng.randint(1, 8),
            "hidden": _size(rng, 1024, 7168, step), "inter": _size(rng, 512, 2048, step), "type": half,
            "add": rng.random() < 0.5}


# ---- inputs ------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _logits(tokens, experts, g):
    return (torch.randn(tokens, experts, device="cuda", generator=g)
            + 0.6 * torch.randn(experts, device="cuda", generator=g))


def _blocks(n):
    return -(-n // BLOCK)


def _weights(count, n, k, g):
    """`count` random matrices [n][k]: E4M3 codes, and f32 scales [n / 128][k / 128] (amax / 448), rounded up."""
    q = torch.empty(count, n, k, dtype=torch.uint8, device="cuda")
    s = torch.empty(count, _blocks(n), _blocks(k), device="cuda")
    for e in range(count):
        w = torch.randn(n, k, device="cuda", generator=g) * 0.02
        p = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK))
        s[e] = p.reshape(_blocks(n), BLOCK, _blocks(k), BLOCK).abs().amax((1, 3)) / 448.0
        q[e] = (w / _spread(s[e], n, k)).to(torch.float8_e4m3fn).view(torch.uint8)
    return q, s


def _spread(s, n, k):
    """Block scales as one value per weight."""
    return s.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _inputs(case, seed):
    """The tensors of one call, from the seed alone."""
    g = _gen(seed)
    kind = case["kind"]
    if kind == "route":
        s = {"logits": _logits(case["tokens"], case["experts"], g).to(DTYPES[case["logits"]])}
        # a balance bias: moved in steps of 0.001 while a model trains
        s["bias"] = torch.randint(-100, 101, (case["experts"],), device="cuda", generator=g) * 0.001 if case["bias"] else None
        return s
    if kind == "project":
        a = torch.randn(case["m"], case["k"], device="cuda", generator=g).to(DTYPES[case["a"]])
        q, w = _weights(1, case["n"], case["k"], g)
        return {"a": a, "wq": q[0], "ws": w[0]}
    t, k, h, dt = case["tokens"], case["topk"], case["hidden"], DTYPES[case["type"]]
    if kind == "combine":
        s = {"y": torch.randn(t * k, h, device="cuda", generator=g).to(dt),
             "rows": torch.randperm(t * k, device="cuda", generator=g).int().reshape(t, k),
             "weights": torch.rand(t, k, device="cuda", generator=g)}
        s["weights"] /= s["weights"].sum(1, keepdim=True)
        s["add"] = torch.randn(t, h, device="cuda", generator=g).to(dt) if case["add"] else None
        return s
    top = _logits(t, case["experts"], g).topk(k, 1)
    s = {"x": torch.randn(t, h, device="cuda", generator=g).to(dt), "ids": top[1].int()}
    if kind == "experts":
        i, e = case["inter"], case["experts"]
        s["weights"] = torch.softmax(top[0], 1)
        s["w"] = [_weights(e, i, h, g), _weights(e, i, h, g), _weights(e, h, i, g)]
        s["add"] = torch.randn(t, h, device="cuda", generator=g).to(dt) if case["add"] else None
    return s


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    kind = case["kind"]

    def new(dt, *shape):
        return torch.empty(*shape, dtype=dt, device="cuda")

    if kind == "route":
        s["ids"] = new(torch.int32, case["tokens"], case["topk"])
        s["weights"] = new(torch.float32, case["tokens"], case["topk"])
    elif kind == "project":
        s["aq"] = new(torch.uint8, case["m"], case["k"])
        s["as"] = new(torch.float32, _blocks(case["k"]), case["m"])
        s["c"] = new(DTYPES[case["c"]], case["m"], case["n"])
    else:
        t, k, h, dt = case["tokens"], case["topk"], case["hidden"], DTYPES[case["type"]]
        if kind == "dispatch":
            s["counts"], s["rows"] = new(torch.int32, case["experts"]), new(torch.int32, t, k)
            s["xs"] = new(dt, t * k, h)
        else:
            s["out"] = new(dt, t, h)
    torch.cuda.synchronize()  # the library works on a stream of its own
    return s


# ---- one pass: the library -----------------------------------------------------------
def _handles(s):
    """Device buffers of a state's tensors, as a program makes them once."""
    if "bufs" not in s:
        M, dev = lib()

        def buf(t):
            return None if t is None else M.DevBuf(dev, t.data_ptr(), t.numel() * t.element_size())

        s["bufs"] = {n: buf(t) for n, t in s.items() if t is None or isinstance(t, torch.Tensor)}
        if "w" in s:
            s["bufs"]["w"] = M.Device.weights(*[(buf(q), buf(c)) for q, c in s["w"]])
    return s["bufs"]


def _run_own(s):
    M, dev = lib()
    case, b = s["case"], _handles(s)
    dt = {"f32": M.DT_F32, "f16": M.DT_F16, "bf16": M.DT_BF16}
    kind = case["kind"]
    if kind == "route":
        dev.moe_route(case["tokens"], case["experts"], case["topk"], b["logits"], dt[case["logits"]], b["ids"], b["weights"],
                      bias=b["bias"], score=M.ROUTE_SIGMOID if case["score"] == "sigmoid" else M.ROUTE_SOFTMAX,
                      groups=case["groups"], topk_groups=case["topk_groups"], group_top=case["group_top"],
                      renormalize=case["renormalize"], scale=2.5)
        return [s["ids"], s["weights"]]
    if kind == "project":
        dev.block_quantize(b["a"], dt[case["a"]], case["m"], case["k"], b["aq"], b["as"])
        dev.block_matmul(b["aq"], b["as"], b["wq"], b["ws"], b["c"], dt[case["c"]], case["m"], case["n"], case["k"])
        return s["c"]
    t, k, h = case["tokens"], case["topk"], case["hidden"]
    if kind == "dispatch":
        dev.moe_dispatch(t, k, case["experts"], b["ids"], b["counts"], b["rows"], b["x"], dt[case["type"]], h, b["xs"])
        return [s["counts"], s["rows"], s["xs"]]
    if kind == "combine":
        dev.moe_combine(t, k, h, b["y"], dt[case["type"]], b["rows"], b["weights"], b["out"], dt[case["type"]], add=b["add"])
        return s["out"]
    dev.moe_block_forward(t, h, case["inter"], case["experts"], k, b["x"], dt[case["type"]], b["ids"], b["weights"],
                          b["w"], b["out"], add=b["add"])
    return s["out"]


# ---- one pass: the plain form ------------------------------------------------------------
def _quantized(x):
    """Activations as their block-FP8 values, in f32: E4M3(x / s) s with s = amax / 448 over 128 values."""
    rows, k = x.shape
    p = torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).reshape(rows, _blocks(k), BLOCK)
    amax = p.abs().amax(2, keepdim=True)
    s = torch.where(amax > 0, (amax / 448.0).clamp(min=2.0 ** -126), torch.ones_like(amax))
    return ((p / s).to(torch.float8_e4m3fn).float() * s).reshape(rows, -1)[:, :k]


def _values(q, s):
    """Weights as f32 values."""
    return q.view(torch.float8_e4m3fn).float() * _spread(s, *q.shape[-2:])


def _route(s):
    case = s["case"]
    t, e, groups = case["tokens"], case["experts"], case["groups"]
    low = float("-inf")
    v = s["logits"].float()
    here = v > low  # neither masked nor NaN
    v = torch.where(here, v.clamp(max=FLT_MAX), 0.0)
    if case["score"] == "sigmoid":
        p = 1.0 / (1.0 + torch.exp(-v))
    else:
        top = torch.where(here, v, -FLT_MAX).amax(1, keepdim=True)
        p = torch.where(here, torch.exp(v - top), 0.0)
        # summed in 64 bits, so that the choice does not depend on the order of the sum
        p = p / p.double().sum(1, keepdim=True).float()
    p = torch.where(here, p, 0.0)
    key = p + s["bias"] if s["bias"] is not None else p
    key = torch.where(here & (key > low), key, low)
    if groups > 1:
        best = key.reshape(t, groups, e // groups).sort(dim=2, descending=True)[0]
        score = best[:, :, 0]
        if case["group_top"] == 2 and e // groups > 1:
            score = score + torch.where(best[:, :, 1] > low, best[:, :, 1], 0.0)
        rank = score.sort(dim=1, descending=True, stable=True)[1]
        keep = torch.zeros(t, groups, dtype=torch.bool, device=v.device).scatter_(1, rank[:, :case["topk_groups"]], True)
        key = torch.where(keep.repeat_interleave(e // groups, 1), key, low)
    best, ids = key.sort(dim=1, descending=True, stable=True)  # ties: the lowest index first
    best, ids = best[:, :case["topk"]], ids[:, :case["topk"]]
    w = torch.where(best > low, p.gather(1, ids), 0.0)
    if case["renormalize"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return [torch.where(best > low, ids, -1).int(), w * 2.5]


def _in_order(ids, experts):
    """(expert order of the flat slots, their experts in that order, rows of [t][slot])"""
    flat = ids.reshape(-1).long()
    sorted_ids, order = flat.sort(stable=True)
    rows = torch.empty_like(order)
    rows[order] = torch.arange(order.numel(), device=order.device)
    return order, sorted_ids, rows.reshape(ids.shape)


def _dispatch(s):
    case = s["case"]
    order, sorted_ids, rows = _in_order(s["ids"], case["experts"])
    counts = torch.zeros(case["experts"], dtype=torch.int32, device=order.device)
    counts.scatter_add_(0, sorted_ids, torch.ones_like(sorted_ids, dtype=torch.int32))
    return [counts, rows.int(), s["x"][order // case["topk"]]]


def _weighted(y, rows, weights, add, dt):
    out = (y[rows.reshape(-1).long()].float().reshape(*rows.shape, -1) * weights.unsqueeze(2)).sum(1)
    return (out + add.float() if add is not None else out).to(dt)


def _experts(s):
    """The slots sorted by expert, every used expert's rows padded to the largest count, batched f32 products."""
    case, x = s["case"], _quantized(s["x"])
    order, sorted_ids, rows = _in_order(s["ids"], case["experts"])
    used, which, counts = torch.unique_consecutive(sorted_ids, return_inverse=True, return_counts=True)
    at = torch.arange(order.numel(), device=x.device) - (counts.cumsum(0) - counts)[which]
    xs = torch.zeros(used.numel(), int(counts.max()), case["hidden"], device=x.device)
    xs[which, at] = x[order // case["topk"]]
    gate, up, down = [(q[used], c[used]) for q, c in s["w"]]
    g = torch.bmm(xs, _values(*gate).transpose(1, 2).contiguous())
    u = torch.bmm(xs, _values(*up).transpose(1, 2).contiguous())
    mid = g / (1.0 + torch.exp(-g)) * u
    mid = _quantized(mid.reshape(-1, case["inter"])).reshape(mid.shape)
    y = torch.bmm(mid, _values(*down).transpose(1, 2).contiguous())[which, at]
    return _weighted(y, rows, s["weights"], s["add"], s["x"].dtype)


def run(s):
    if own:
        return _run_own(s)
    kind = s["case"]["kind"]
    if kind == "route":
        return _route(s)
    if kind == "dispatch":
        return _dispatch(s)
    if kind == "combine":
        return _weighted(s["y"], s["rows"], s["weights"], s["add"], s["out"].dtype)
    if kind == "project":
        return (_quantized(s["a"]) @ _values(s["wq"], s["ws"]).T).to(s["c"].dtype)
    return _experts(s)


# ---- what a pass cannot do without --------------------------------------------------------
def _matrix_bytes(n, k):
    return n * k + 4 * _blocks(n) * _blocks(k)


def work(case):
    kind = case["kind"]
    if kind == "route":
        t, e, k = case["tokens"], case["experts"], case["topk"]
        return {"bytes": t * e * SIZE[case["logits"]] + (4 * e if case["bias"] else 0) + 8 * t * k, "flops": 4 * t * e}
    if kind == "project":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * SIZE[case["a"]] + _matrix_bytes(n, k) + m * n * SIZE[case["c"]], "flops": 2 * m * n * k}
    t, k, h, size = case["tokens"], case["topk"], case["hidden"], SIZE[case["type"]]
    add = t * h * size if case.get("add") else 0
    if kind == "dispatch":
        return {"bytes": 8 * t * k + 4 * case["experts"] + t * h * size + t * k * h * size, "flops": 0}
    if kind == "combine":
        return {"bytes": 8 * t * k + t * k * h * size + add + t * h * size, "flops": 2 * t * k * h}
    i, e = case["inter"], case["experts"]
    used = e * (1.0 - (1.0 - k / e) ** t)  # experts that evenly spread tokens reach
    weights = used * (2 * _matrix_bytes(i, h) + _matrix_bytes(h, i))
    return {"bytes": weights + 8 * t * k + 2 * t * h * size + add, "flops": 6 * t * k * h * i}


# ---- 64 bits ----------------------------------------------------------------------------
def _e4m3_f64(v):
    """The nearest E4M3 value, ties to even."""
    exp = torch.frexp(v)[1].clamp(min=-5) - 4  # of the last of three mantissa bits; subnormals below 2^-6
    return torch.ldexp(torch.ldexp(v, -exp).round(), exp).clamp(-448.0, 448.0)


def _act_f64(x):
    # the format's scale is an f32 and its codes are those of an f32 division:
    # f16 values meet their ties often
    x = x.float()
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for lo in range(0, x.shape[1], BLOCK):
        b = x[:, lo:lo + BLOCK]
        amax = b.abs().amax(1, keepdim=True)
        s = torch.where(amax > 0, torch.clamp(amax / 448.0, min=2.0 ** -126), 1.0)
        out[:, lo:lo + BLOCK] = _e4m3_f64((b / s).double()) * s.double()
    return out


def _weights_f64(q, s):
    n, k = q.shape
    at = torch.arange(n, device=q.device).unsqueeze(1) // BLOCK, torch.arange(k, device=q.device) // BLOCK
    code = torch.arange(256, device=q.device)
    e, m = (code >> 3) & 15, (code & 7).double()
    value = torch.where(e > 0, torch.ldexp(1.0 + m / 8.0, e - 7), torch.ldexp(m / 8.0, torch.full_like(e, -6)))
    value = torch.where(code > 127, -value, value)
    return value[q.long()] * s.double()[at]


def _exact_route(case, s):
    v = s["logits"].double()
    p = torch.sigmoid(v) if case["score"] == "sigmoid" else torch.softmax(v, 1)
    key = p if s["bias"] is None else p + s["bias"].double()
    t, e, groups = case["tokens"], case["experts"], case["groups"]
    if groups > 1:
        top = min(case["group_top"], e // groups)
        score = key.reshape(t, groups, -1).topk(top, 2)[0].sum(2)
        out = torch.ones(t, groups, dtype=torch.bool, device=v.device)
        out.scatter_(1, score.topk(case["topk_groups"], 1)[1], False)
        key = key.masked_fill(out.repeat_interleave(e // groups, 1), float("-inf"))
    w = p.gather(1, key.topk(case["topk"], 1)[1])
    return [None, (w / w.sum(1, keepdim=True) if case["renormalize"] else w) * 2.5]


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "route":
        return _exact_route(case, s)
    if kind == "project":
        return _act_f64(s["a"]) @ _weights_f64(s["wq"], s["ws"]).T
    if kind == "dispatch":
        return [None, None, s["x"].double()[torch.argsort(s["ids"].reshape(-1), stable=True) // case["topk"]]]
    if kind == "combine":
        t, k = s["rows"].shape
        out = s["add"].double() if case["add"] else torch.zeros(t, case["hidden"], dtype=torch.float64, device="cuda")
        for slot in range(k):
            out = out + s["y"][s["rows"][:, slot].long()].double() * s["weights"][:, slot:slot + 1].double()
        return out
    x = _act_f64(s["x"])
    out = s["add"].double() if case["add"] else torch.zeros_like(x)
    for e in range(case["experts"]):
        token, slot = (s["ids"] == e).nonzero(as_tuple=True)
        if token.numel():
            gate, up, down = [_weights_f64(q[e], c[e]) for q, c in s["w"]]
            g, u = x[token] @ gate.T, x[token] @ up.T
            y = _act_f64(g * torch.sigmoid(g) * u) @ down.T
            out.index_add_(0, token, y * s["weights"][token, slot].double().unsqueeze(1))
    return out

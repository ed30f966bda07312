"""A mixture-of-experts layer on libmxfp4hip: gate, router, experts, shared expert.

  python3 examples/moe_layer.py [--tokens 64] [--hidden 1024] [--inter 512] [--experts 32] [--topk 4]

The layer runs twice on the same tokens, and the results are compared:

  block FP8  gate product -> mx_moe_route -> mx_moe_block_forward, with the
             shared expert's rows (mx_fmt_mlp_forward) added; nothing but the
             launches happens on the host
  MXFP4      the same routes through mx_moe_dispatch, mx_moe_forward (which takes
             its counts on the host) and mx_moe_combine
"""
import argparse
import os
import sys
import time

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mpp-4.1-fp4-fp8-block_amd"))
import mxfp4hip as M  # noqa: E402


def blocks(n):
    return -(-n // 128)


def part(buf, i, nbytes):
    """The i-th run of nbytes of a buffer."""
    return M.DevBuf(buf.dev, buf.ptr + i * nbytes, nbytes)


class Layer:
    """Random weights in f32, quantized on the device to both formats."""

    def __init__(self, dev, hidden, inter, experts, topk, seed=0):
        self.dev, self.h, self.i, self.e, self.k = dev, hidden, inter, experts, topk
        rng = np.random.default_rng(seed)
        self.gate = dev.upload((rng.normal(0, 1, (experts, hidden)) / np.sqrt(hidden)).astype(np.float16))
        self.bias = dev.upload((rng.integers(-50, 51, experts) * 0.001).astype(np.float32))
        shapes = ((inter, hidden), (inter, hidden), (hidden, inter))
        fp8, mx = [], []
        for n, k in shapes:
            w = dev.upload(rng.normal(0, 1 / np.sqrt(k), (experts * n, k)).astype(np.float32))
            q, s = dev.alloc(experts * n * k), dev.alloc(experts * blocks(n) * blocks(k) * 4)
            for e in range(experts):  # a block's scale covers rows of one expert only
                dev.fmt_quantize(M.WFMT_FP8_BLOCK, part(w, e, n * k * 4), n, k, part(q, e, n * k),
                                 part(s, e, blocks(n) * blocks(k) * 4))
            fp8.append((q, s))
            p, e8 = dev.alloc(experts * n * k // 2), dev.alloc(experts * n * k // 32)
            dev.mxfp4_quantize(w, M.DT_F32, experts * n, k, p, e8)
            mx.append((p, e8))
            dev.sync()
            w.free()
        self.fp8, self.mx = M.Device.weights(*fp8), M.Device.weights(*mx)
        self.shared = self.fp8  # its pointers are at expert 0, which serves as the shared expert too

    def buffers(self, tokens):
        a = self.dev.alloc
        n = tokens * self.k
        return {"logits": a(tokens * self.e * 4), "ids": a(n * 4), "weights": a(n * 4), "shared": a(tokens * self.h * 2),
                "out": a(tokens * self.h * 2), "counts": a(self.e * 4), "rows": a(n * 4), "xs": a(n * self.h * 2),
                "ys": a(n * self.h * 2)}

    def route(self, x, tokens, b):
        d = self.dev
        d.gemm_f16(x, M.DT_F16, self.gate, b["logits"], tokens, self.e, self.h)
        d.moe_route(tokens, self.e, self.k, b["logits"], M.DT_F32, b["ids"], b["weights"], bias=self.bias,
                    score=M.ROUTE_SIGMOID, renormalize=True)
        d.fmt_mlp_forward(M.WFMT_FP8_BLOCK, tokens, self.h, self.i, x, self.shared, b["shared"])

    def block_fp8(self, x, tokens, b):
        self.route(x, tokens, b)
        self.dev.moe_block_forward(tokens, self.h, self.i, self.e, self.k, x, M.DT_F16, b["ids"], b["weights"], self.fp8,
                                   b["out"], add=b["shared"])
        return b["out"]

    def mxfp4(self, x, tokens, b):
        d = self.dev
        self.route(x, tokens, b)
        d.moe_dispatch(tokens, self.k, self.e, b["ids"], b["counts"], b["rows"], x, M.DT_F16, self.h, b["xs"])
        counts = d.download(b["counts"], np.int32, self.e)
        d.moe_forward(self.h, self.i, counts.tolist(), b["xs"], self.mx, b["ys"])
        d.moe_combine(tokens, self.k, self.h, b["ys"], M.DT_F16, b["rows"], b["weights"], b["out"], M.DT_F16, add=b["shared"])
        return b["out"]


def run(tokens=64, hidden=1024, inter=512, experts=32, topk=4, device=0, steps=20):
    """(cosine between the two formats' results, us a pass of each)"""
    with M.Device(device) as dev:
        layer = Layer(dev, hidden, inter, experts, topk)
        x = dev.upload(np.random.default_rng(1).normal(0, 1, (tokens, hidden)).astype(np.float16))
        b = layer.buffers(tokens)
        got, us = [], []
        for path in (layer.block_fp8, layer.mxfp4):
            got.append(dev.download(path(x, tokens, b), np.float16, (tokens, hidden)).astype(np.float64).ravel())
            start = time.perf_counter()
            for _ in range(steps):
                path(x, tokens, b)
            dev.sync()
            us.append((time.perf_counter() - start) / steps * 1e6)
        return float(got[0] @ got[1] / np.sqrt((got[0] @ got[0]) * (got[1] @ got[1]))), us


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("tokens", 64), ("hidden", 1024), ("inter", 512), ("experts", 32), ("topk", 4)):
        ap.add_argument("--" + name, type=int, default=value)
    cosine, us = run(**vars(ap.parse_args()))
    print(f"block FP8 {us[0]:.1f} us, MXFP4 {us[1]:.1f} us a layer; cosine of their results {cosine:.4f}")

"""Runs the 4-bit operators of one build of the library in a process of its own.

    python tests/fp4_cases.py {product|checked} OUT.npz   odd shapes through every path, outputs saved
    python tests/fp4_cases.py capture                     the process's first calls are captured in a graph
"""
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

import t0_web_b200._lib as L  # noqa: E402

if sys.argv[1] == "checked":
    L.LIB_PATH = os.path.join(os.path.dirname(L.LIB_PATH), "libt0b_checked.so")

import torch  # noqa: E402

from t0_web_b200 import fp4, t0_fast  # noqa: E402

DEV = "cuda:0"


def rnd(seed, *shape, dev=1.0):
    return torch.from_numpy((np.random.default_rng(seed).standard_normal(shape) * dev).astype(np.float32)).to(DEV)


def mat(eng, fmt, rows, k):
    m = fp4.Fp4Matrix.empty(fmt, rows, k, DEV, 2.0 ** -6 if fmt == "nv" else 1.0)
    m.codes.fill_(255)
    m.scales.fill_(255)
    return m


def save(path):
    eng = t0_fast.Engine(0)
    out = {}
    # one and a few tokens, one tile and several, one K slice and several, both kernels, unaligned rows
    for fmt in ("mx", "nv"):
        for m, f, k, pad in ((1, 130, 300, 0), (17, 257, 1001, 1), (70, 100, 70, 0), (130, 384, 2500, 3), (300, 1001, 96, 0),
                             (700, 2000, 520, 1)):
            x = rnd(m + k, m, k + pad)[:, :k]
            w0, w2 = (fp4.quantize(eng, rnd(i, r, c, dev=0.05), mat(eng, fmt, r, c)) for i, r, c in ((1, 2 * f, k), (2, k, f)))
            y = torch.full((m, k + pad), float("nan"), device=DEV)[:, :k]
            h = torch.full((m, 2 * f), float("nan"), dtype=torch.float16, device=DEV)
            z = torch.full((m, f), float("nan"), device=DEV)
            zq = mat(eng, fmt, m, f)
            fp4.mlp(eng, w0, w2, x, mat(eng, fmt, m, k), zq, y, rnd(3, 2 * f), rnd(4, k))
            fp4.linear(eng, w0, x, mat(eng, fmt, m, k), h)
            xq = fp4.quantize(eng, x, mat(eng, fmt, m, k))
            fp4.glu(eng, w0, xq, z)
            back = fp4.dequantize(eng, xq, torch.full((m, k), float("nan"), dtype=torch.bfloat16, device=DEV))
            fp4.sync(eng)
            for name, t in (("y", y), ("h", h), ("z", z), ("back", back)):
                out[f"{fmt}_{m}_{name}"] = t.float().cpu().numpy()
            for name, t in (("zc", zq.codes), ("zs", zq.scales), ("xc", xq.codes), ("xs", xq.scales)):
                out[f"{fmt}_{m}_{name}"] = t.cpu().numpy()
    np.savez(sys.argv[2], **out)


def capture():
    eng = t0_fast.Engine(0)
    cases = []
    for m in (3, 600):  # both product kernels
        f, k = 512, 256
        x, (w0, w2) = rnd(m, m, k), (mat(eng, "nv", r, c) for r, c in ((2 * f, k), (k, f)))
        cases.append([x, w0, w2, rnd(1, 2 * f, k, dev=0.1), rnd(2, k, f, dev=0.1), mat(eng, "nv", m, k), mat(eng, "nv", m, f),
                      torch.full((m, k), float("nan"), device=DEV), torch.full((m, k), float("nan"), device=DEV)])
    torch.cuda.synchronize()

    def run(i):
        for x, w0, w2, v0, v2, xq, zq, *y in cases:
            fp4.quantize(eng, v0, w0)
            fp4.quantize(eng, v2, w2)
            fp4.mlp(eng, w0, w2, x, xq, zq, y[i])

    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        run(0)
    g.replay()
    g.replay()
    torch.cuda.synchronize()
    run(1)
    fp4.sync(eng)
    for c in cases:
        assert torch.isfinite(c[7]).all() and torch.equal(c[7], c[8])


if __name__ == "__main__":
    capture() if sys.argv[1] == "capture" else save(sys.argv[2])

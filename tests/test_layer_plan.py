"""Which kernel computes a product of the MLP layer, and that the tests' shapes reach every one of them (no GPU)."""
import ctypes
import os
import random
import subprocess

import pytest

import test_layer as L
import test_layer_range as R
from conftest import PKG

SOURCE = """
#include "linear_plan.h"
// bn (0: the pair kernel), cluster size, whether a CTA adds partial sums
extern "C" void plan_of(int op, int type, int out_type, int rows, int cols, int depth, int* out) {
  mlpg::LinearArgs a = {};
  a.op = op, a.type = type, a.out_type = out_type;
  a.rows = rows, a.cols = cols, a.depth = depth, a.num_sms = 148;
  const mlpg::Plan p = mlpg::plan(a);
  const int blocks = (depth + mlpg::kKb - 1) / mlpg::kKb;
  out[0] = p.bn, out[1] = p.split, out[2] = (blocks + p.split - 1) / p.split > mlpg::segment_blocks(out_type);
}
"""
OPS = {"linear": 0, "dx": 1, "dw": 2}
TYPES = {"f16": 0, "bf16": 1, "f32": 2}


@pytest.fixture(scope="module")
def plan_of(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cc").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(PKG, "csrc"), "-I",
                    "/usr/local/cuda/include", str(d / "plan.cc"), "-o", str(d / "plan.so")], check=True)
    fn = ctypes.CDLL(str(d / "plan.so")).plan_of

    def plan(op, type, out, N, K, M):
        """The kernel of a product: its template arguments, and whether it adds partial sums."""
        rows, cols, depth = {"linear": (N, M, K), "dx": (N, K, M), "dw": (K, M, N)}[op]
        o = (ctypes.c_int * 3)()
        fn(OPS[op], TYPES[type], TYPES[out], rows, cols, depth, o)
        return (op, type, out, o[0], bool(o[2]))
    return plan


def covered():
    """(op, type, type of the result, N, K, M) of the tests that compare whole products with 64 bits."""
    for t in ("f16", "bf16"):
        for s in L.SIZES:
            yield ("linear", t, t) + s
        for s in L.GRAD_SIZES:
            yield ("dx", t, t) + s
            yield ("dw", t, t) + s
            yield ("dw", t, "f32") + s
    yield from R.KERNELS


def drawn(n):
    """Products over the whole range that fit a GPU: up to 2^16 rows and columns, contractions up to 2^21."""
    rng = random.Random(5)
    while n:
        op = rng.choice(list(OPS))
        t = rng.choice(["f16", "bf16"])
        sizes = [int(2 ** rng.uniform(0, 16)) for _ in range(3)]
        if rng.random() < 0.5:
            sizes[{"linear": 1, "dx": 2, "dw": 0}[op]] = int(2 ** rng.uniform(10, 21))
        N, K, M = sizes
        if max(N * K, K * M, N * M) > 2 ** 32:
            continue
        n -= 1
        yield (op, t, rng.choice([t, "f32"]) if op == "dw" else t) + (N, K, M)


def test_every_kernel_has_a_shape(plan_of):
    # a change of the time model may move a shape to another kernel: then R.KERNELS needs new ones
    have = {plan_of(*p) for p in covered()}
    missing = {}
    for p in drawn(60000):
        k = plan_of(*p)
        if k not in have:
            q = missing.setdefault(k, p)
            if p[3] * p[4] * p[5] < q[3] * q[4] * q[5]:
                missing[k] = p
    assert not missing, "\n".join(f"{k}: e.g. {p}" for k, p in sorted(missing.items()))


def test_partial_sums_fit(plan_of):
    # what a CTA of the split kernel takes fits its accumulators, at any length of the contraction
    import itertools
    for (op, t, out), depth in itertools.product((("linear", "f16", "f16"), ("linear", "bf16", "bf16"), ("dw", "bf16", "f32")),
                                                 (1, 4096, 32768, 32769, 1 << 18, (1 << 18) + 1, 1 << 21, 1 << 30)):
        for rows, cols in ((64, 128), (64, 40000), (500, 500), (4096, 64)):
            N, K, M = {"linear": (rows, depth, cols), "dw": (depth, rows, cols)}[op]
            _, _, _, bn, _ = plan_of(op, t, out, N, K, M)
            most = {"f16": 64, "bf16": 512, "f32": 8}[out] * 64 * 8 * (2 if bn == 256 else 256 // bn if bn else 0)
            assert bn == 0 or depth <= most, (op, out, depth, rows, cols, bn)

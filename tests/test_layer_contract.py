"""What the MLP layer's entry points refuse, and the bindings' checks (no GPU needed)."""
import pytest

from mlpgemm import lib as G
from test_layer import P, refused


def test_workspace_of_refused_arguments_is_0():
    # an operand off its element, rows closer together than their length: no size, as the header says
    ws = G.linear_workspace
    for op, ca, cb in ((G.OP_LINEAR, 64, 72), (G.OP_DX, 72, 72), (G.OP_DW, 64, 72)):    # the operands' row lengths
        good = (op, P + 2, P + 2, 4, 64, 72)
        assert ws(*good, ca, cb) > 0
        for lda, ldb in ((ca - 1, cb), (ca, cb - 1), (-3, cb), (ca, -3), (1, 0), (0, 1)):
            assert ws(*good, lda, ldb) == 0, (op, lda, ldb)
        assert ws(op, P + 1, P + 2, 4, 64, 72) == 0 and ws(op, P + 2, P + 3, 4, 64, 72) == 0
        assert ws(op, P + 2, P + 2, 4, 64, (1 << 30) + 1) == 0


# ---- torch tensors: what they are against what the call takes them for ------------------------------
# Tensors of the CPU belong to device -1, which no call gets past its arguments with.
N, K, M = 4, 64, 72
OPERANDS = {   # name -> rows, columns, its row length's name
    "linear": {"X": (N, K, "ldx"), "W": (K, M, "ldw"), "Y": (N, M, "ldy"), "residual": (N, M, "ldr"), "preact": (N, M, "ldz")},
    "linear_dx": {"dZ": (N, M, "lddz"), "W": (K, M, "ldw"), "dX": (N, K, "lddx"), "residual": (N, K, "ldr")},
    "linear_dw": {"X": (N, K, "ldx"), "dZ": (N, M, "lddz"), "dW": (K, M, "lddw"), "residual": (K, M, "ldr")},
    "act_grad": {"dY": (N, M, "lddy"), "Z": (N, M, "ldz"), "dZ": (N, M, "lddz")},
    "dropout": {"X": (N, M, "ldx"), "Y": (N, M, "ldy"), "residual": (N, M, "ldr")}}
EACH = [(op, name) for op in OPERANDS for name in OPERANDS[op]]


def call(op, device=-1, **change):
    import torch
    kw = dict(type=1, N=N, M=M)
    if op.startswith("linear"):
        kw.update(K=K)
    kw.update({n: torch.zeros(r, c, dtype=torch.bfloat16) for n, (r, c, _) in OPERANDS[op].items()})
    if op == "act_grad":
        kw.update(act=2, dbias=torch.zeros(M))
    if op == "dropout":
        kw.update(p=0.5, seed=0, offset=0)
    kw.update(change)
    getattr(G, op)(device, **kw)


def passes(op, **change):
    with pytest.raises(G.GemmError) as e:
        call(op, **change)
    assert e.value.code == G.GEMM_ERR_INIT, e.value


@pytest.mark.parametrize("op,name", EACH)
def test_tensors_have_to_be_what_they_are_taken_for(op, name):
    import torch
    rows, cols, ld = OPERANDS[op][name]
    bf16 = torch.bfloat16
    passes(op)
    passes(op, **{name: torch.zeros(rows * cols + 5, dtype=bf16)})                              # a flat buffer
    passes(op, **{name: torch.zeros(2, rows // 2, cols, dtype=bf16)})                           # batched, dense
    wide = torch.zeros(rows + 1, cols + 8, dtype=bf16)[:rows, :cols]
    passes(op, **{name: wide, ld: cols + 8})
    refused(lambda: call(op, device=0, **{n: P + 4096 * i for i, n in enumerate(OPERANDS[op]) if n != name}), name, "cpu")
    refused(lambda: call(op, **{name: torch.zeros(rows, cols, dtype=torch.float16)}), name, "elements of")
    refused(lambda: call(op, **{name: torch.zeros(cols, rows, dtype=bf16).t()}), name, "strides")
    refused(lambda: call(op, **{name: wide}), name, "strides")
    refused(lambda: call(op, **{name: wide, ld: cols + 16}), name, "strides")
    refused(lambda: call(op, **{name: torch.zeros(1, cols, dtype=bf16).expand(rows, cols)}), name, "strides")
    refused(lambda: call(op, **{name: torch.zeros(rows - 1, cols, dtype=bf16)}), name, "needed")
    refused(lambda: call(op, **{name: torch.zeros(rows, cols, dtype=bf16), ld: cols + 8}), name, "needed")
    refused(lambda: call(op, **{name: wide[1:], ld: cols + 8}), name, "needed")


def test_the_other_buffers():
    import torch
    refused(lambda: call("linear", bias=torch.zeros(M - 1, dtype=torch.bfloat16)), "bias", "needed")
    refused(lambda: call("linear", bias=torch.zeros(M)), "bias", "elements of")
    refused(lambda: call("act_grad", dbias=torch.zeros(M, dtype=torch.bfloat16)), "dbias", "elements of")
    refused(lambda: call("act_grad", dbias=torch.zeros(M - 1)), "dbias", "needed")
    refused(lambda: call("linear_dw", out_type=2), "dW", "elements of")
    passes("linear_dw", out_type=2, dW=torch.zeros(K, M), residual=torch.zeros(K, M))
    word = torch.zeros(1, dtype=torch.int64)
    passes("linear", offset_ptr=word, dropout_p=0.5)
    for op in ("linear", "act_grad", "dropout"):
        refused(lambda: call(op, device=0, offset_ptr=word, **{n: P + 4096 * i for i, n in enumerate(OPERANDS[op])},
                             **({"dbias": P} if op == "act_grad" else {})), "offset_ptr", "cpu")
    refused(lambda: call("linear", workspace=torch.zeros(16, dtype=torch.uint8), workspace_bytes=32), "workspace")


def test_sizes_that_ctypes_would_cut():
    for op in OPERANDS:
        for n in ("N", "M") + (("K",) if op.startswith("linear") else ()):
            for v in ((1 << 32) + 4, -(1 << 32) + 4, 1 << 31):
                with pytest.raises(G.GemmError) as e:
                    getattr(G, op)(0, **{**dict(type=0, N=N, M=M), **({"K": K} if op.startswith("linear") else {}),
                                         **({"p": 0.5, "seed": 0, "offset": 0} if op == "dropout" else {}),
                                         **({"dbias": P} if op == "act_grad" else {}),
                                         **{x: P + (i << 16) for i, x in enumerate(OPERANDS[op])}, n: v})
                assert e.value.code == G.GEMM_ERR_ARGS, e.value


def test_sizes_of_other_integer_types():
    import numpy as np
    i = np.int64
    passes("linear", N=i(N), K=i(K), M=i(M), type=i(1), ldx=i(K), act=i(2))
    passes("linear_dx", N=i(N), K=i(K), M=i(M))
    passes("linear_dw", N=i(N), out_type=i(1))
    passes("act_grad", N=i(N), act=i(1))
    passes("dropout", M=i(M), seed=5, offset=7)


# ---- results in an input's buffer --------------------------------------------------------------
def in_place(kw_of, *words):
    """kw_of(ld of the result, rows): refused where the input's rows are 80 apart and the result's are not."""
    refused(lambda: kw_of(96, 4), *words)
    refused(lambda: kw_of(0, 2), *words)
    for ld, rows in ((80, 4), (96, 1), (0, 1)):        # the same rows, or a single one
        with pytest.raises(G.GemmError) as e:
            kw_of(ld, rows)
        assert e.value.code == G.GEMM_ERR_INIT, e.value


def test_results_in_place_have_the_inputs_rows():
    Q, R = P + (1 << 16), P + (2 << 16)
    in_place(lambda ld, n: G.linear(-1, 0, P, Q, R, n, 64, 72, residual=R, ldr=80, ldy=ld), "Y", "residual")
    in_place(lambda ld, n: G.linear_dx(-1, 0, P, Q, R, n, 72, 64, residual=R, ldr=80, lddx=ld), "dX", "residual")
    in_place(lambda ld, k: G.linear_dw(-1, 0, P, Q, R, 64, 8 * (k > 1) or 1, 72, out_type=2, residual=R, ldr=80, lddw=ld,
                                       ldx=8), "dW", "residual")
    in_place(lambda ld, n: G.act_grad(-1, 0, P, Q, P, None, n, 72, act=2, lddy=80, lddz=ld), "dZ", "dY")
    in_place(lambda ld, n: G.act_grad(-1, 0, P, Q, Q, None, n, 72, act=2, ldz=80, lddz=ld), "dZ", "Z's buffer")
    in_place(lambda ld, n: G.dropout(-1, 0, P, P, n, 72, 0.5, 1, 2, ldx=80, ldy=ld), "Y", "X")
    in_place(lambda ld, n: G.dropout(-1, 0, P, Q, n, 72, 0.5, 1, 2, residual=Q, ldr=80, ldy=ld), "Y", "residual")
    refused(lambda: G.linear(-1, 0, P, Q, R, 4, 64, 72, bias=R), "bias", "same buffer")
    refused(lambda: G.linear(-1, 0, P, Q, R, 4, 64, 72, bias=R + 4096, preact=R + 4096), "preact", "same buffer")

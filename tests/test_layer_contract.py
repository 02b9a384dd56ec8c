"""What the MLP layer's entry points refuse, and the bindings' checks (no GPU needed)."""
import pytest

from mlpgemm import lib as G
from test_layer import P


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

"""Calls of the attention operators' C entry points at the ends of their ranges
that no kernel is needed for: batches of no rows, sizes and scalars that are
refused before any launch."""
import ctypes

import pytest

from flashlog_amd import _lib


def _logits_op(**kw):
    op = _lib.FlLogits(x=1, rows=4, cols=40, ldx=40, inner=1, repetition=1.0, temperature=1.0)
    for k, v in kw.items():
        setattr(op, k, v)
    return op


@pytest.mark.parametrize("table", [dict(allowed=1, allowed_rows=3, allowed_ld=2), dict(bias=1, bias_rows=3)])
def test_no_rows_need_no_group(table):
    """An empty group tensor has the address 0: with no rows it is not missing."""
    lib = _lib.lib()
    op = _logits_op(rows=0, group=None, **table)
    assert lib.fl_logits_constrain(None, op, None) == 0
    assert lib.fl_logits_softmax(None, op, None, None, 0) == 0
    assert lib.fl_logits_grad(None, op, None, None, None, None, None, 0) == 0
    op.rows = 1
    assert lib.fl_logits_constrain(None, op, ctypes.c_void_p(1)) == 1

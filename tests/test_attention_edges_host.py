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


def test_more_tiles_than_a_launch_holds():
    """A launch has fewer than 2^32 threads along a dimension; the products' tiles lie along one."""
    lib = _lib.lib()
    one, ws = ctypes.c_void_p(1), ctypes.c_void_p(4096)

    def refused(rc):
        assert rc == 1 and "shape" in lib.fl_last_error().decode()

    op = _lib.FlLinear(M=(1 << 31) - 1, N=64, K=1, groups=1, x=1, ldx=1, weight=1, ldw=1)
    refused(lib.fl_linear_forward(None, op, one, None, None, 0))
    # the activation's gradient of 2^34 values, the weight gradient of 2^31 x 256, the bias gradients of 2^24 groups
    op = _lib.FlLinear(M=1 << 20, N=1 << 14, K=0, groups=1, act=2)
    refused(lib.fl_linear_backward(None, op, one, one, None, None, None, 0, ws, 1 << 60))
    op = _lib.FlLinear(M=1, N=(1 << 31) - 1, K=256, groups=1, x=1, ldx=256, weight=1, ldw=256)
    refused(lib.fl_linear_backward(None, op, one, None, None, one, None, 0, ws, 1 << 60))
    op = _lib.FlLinear(M=1, N=1, K=0, groups=1 << 24, order=1, offsets=1, tiles=1)
    refused(lib.fl_linear_backward(None, op, one, None, None, None, one, 0, ws, 1 << 60))
    op = _lib.FlLinear(M=1 << 24, N=1 << 14, K=0, groups=1 << 19, act=2, dtype=1, order=1, offsets=1, tiles=1)
    refused(lib.fl_linear_backward(None, op, one, one, None, None, one, 0, ws, 1 << 60))


@pytest.mark.parametrize("name,bad,good", [("temperature", 1e39, 2.0 ** 126), ("temperature", 1e-39, 2.0 ** -126),
                                           ("repetition", 1e39, 2.0 ** 126), ("repetition", 1e-40, 2.0 ** -126),
                                           ("presence", 1e39, 3e38), ("frequency", -1e39, -3e38),
                                           ("frequency", float("nan"), 0.0)])
def test_scalars_that_float32_cannot_divide_by(name, bad, good):
    """Finite numbers of 64 bits that are infinite, or have an infinite reciprocal, in 32."""
    lib = _lib.lib()
    one = ctypes.c_void_p(1)
    op = _logits_op(**{name: bad})
    for rc in (lib.fl_logits_constrain(None, op, one), lib.fl_logits_softmax(None, op, one, None, 0),
               lib.fl_logits_grad(None, op, None, one, one, None, None, 0)):
        assert rc == 1 and "range" in lib.fl_last_error().decode()
    assert lib.fl_logits_constrain(None, _logits_op(rows=0, **{name: good}), one) == 0

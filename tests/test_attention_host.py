"""Refusals of the attention operators' entry points that need no GPU: CPU
tensors, and arguments of the C-ABI that are turned down before any launch."""
import ctypes

import pytest
import torch

from flashlog_amd import _lib
from flashlog_amd import attention as fa


def _error(rc):
    assert rc == 1
    return _lib.lib().fl_last_error().decode()


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 3), torch.zeros(4, 3)
    for call in (lambda: fa.linear(x, w), lambda: fa.group_rows(torch.zeros(2, dtype=torch.long), 1),
                 lambda: fa.constrain_logits(x), lambda: fa.hop_attention(x),
                 lambda: fa.pack_allowed(torch.ones(3, dtype=torch.bool)),
                 lambda: fa.history_from_pairs(torch.zeros(1, dtype=torch.long), torch.zeros(1, dtype=torch.long), 1)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        fa.linear([1.0], w)


def test_group_rows_arguments():
    lib = _lib.lib()
    one = ctypes.c_void_p(1)
    assert "range" in _error(lib.fl_group_rows(None, one, -1, 3, one, one, one, None, 0))
    assert "range" in _error(lib.fl_group_rows(None, one, 5, 0, one, one, one, None, 0))
    assert "range" in _error(lib.fl_group_rows(None, one, 5, 1 << 24, one, one, one, None, 0))
    assert "null" in _error(lib.fl_group_rows(None, None, 5, 3, one, one, one, None, 0))
    assert lib.fl_group_rows_bytes(16384, 4095) == 0 and lib.fl_group_rows_bytes(16385, 4095) > 0
    assert "workspace" in _error(lib.fl_group_rows(None, one, 20000, 3, one, one, one, one, 16))
    # enough tiles for any sizes of the groups
    for rows in (1, 31, 1000, 70000):
        for groups in (1, 2, 500, 5000):
            block = lib.fl_group_block(rows, groups)
            g = min(rows, groups + 1)  # worst: every group one row over whole tiles
            worst = g + (rows - g) // block
            assert lib.fl_group_tiles(rows, groups) >= worst
    assert lib.fl_group_tiles(0, 4) == 0


def _linear_op(**kw):
    op = _lib.FlLinear(M=4, N=3, K=5, groups=1, x=1, ldx=5, weight=1, ldw=5)
    for k, v in kw.items():
        setattr(op, k, v)
    return op


def test_linear_arguments():
    lib = _lib.lib()
    one = ctypes.c_void_p(1)
    fwd = lambda op, y=one: _error(lib.fl_linear_forward(None, op, y, None, None, 0))
    assert "type" in fwd(_linear_op(dtype=3))
    assert "activation" in fwd(_linear_op(act=6))
    assert "shape" in fwd(_linear_op(M=-1))
    assert "shape" in fwd(_linear_op(groups=0))
    assert "plan" in fwd(_linear_op(groups=2))
    assert "plan" in fwd(_linear_op(groups=2, offsets=1))
    assert "null" in fwd(_linear_op(x=None))
    assert "null" in fwd(_linear_op(), None)
    back = lambda op, gy, pre, dx, dw, db, ws, n: _error(lib.fl_linear_backward(None, op, gy, pre, dx, dw, db, 0, ws, n))
    assert "null" in back(_linear_op(), None, None, one, None, None, None, 0)
    assert "null" in back(_linear_op(act=2), one, None, one, None, None, one, 1 << 20)
    assert "null" in back(_linear_op(weight=None), one, None, one, None, None, None, 0)
    assert "null" in back(_linear_op(x=None), one, None, None, one, None, None, 0)
    assert "workspace" in back(_linear_op(), one, None, None, None, one, None, 0)
    assert "workspace" in back(_linear_op(act=2), one, one, one, None, None, None, 0)
    long = _linear_op(M=100_000)
    need = lib.fl_linear_backward_bytes(long, 0, 1, 0)
    assert need > 0 and "workspace" in back(long, one, None, None, one, None, one, need - 1)
    # nothing to do is no error
    assert lib.fl_linear_forward(None, _linear_op(M=0), None, None, None, 0) == 0


def _logits_op(**kw):
    op = _lib.FlLogits(x=1, rows=4, cols=40, ldx=40, inner=1, repetition=1.0, temperature=1.0)
    for k, v in kw.items():
        setattr(op, k, v)
    return op


def test_logits_arguments():
    lib = _lib.lib()
    one = ctypes.c_void_p(1)
    fwd = lambda op, y=one: _error(lib.fl_logits_constrain(None, op, y))
    assert "type" in fwd(_logits_op(dtype=7))
    assert "shape" in fwd(_logits_op(inner=3))
    assert "shape" in fwd(_logits_op(inner=0))
    assert "range" in fwd(_logits_op(temperature=0.0))
    assert "range" in fwd(_logits_op(temperature=float("nan")))
    assert "range" in fwd(_logits_op(repetition=-2.0))
    assert "allowed" in fwd(_logits_op(allowed=1, allowed_rows=1, allowed_ld=1))
    assert "allowed" in fwd(_logits_op(allowed=1, allowed_rows=2, allowed_ld=2))
    assert "bias" in fwd(_logits_op(bias=1, bias_rows=2))
    assert "history" in fwd(_logits_op(history=1, history_len=-1))
    assert "null" in fwd(_logits_op(x=None))
    assert "null" in fwd(_logits_op(), None)
    long = _logits_op(cols=20000, ldx=20000)
    need = lib.fl_logits_softmax_bytes(long)
    assert need > 0 and "workspace" in _error(lib.fl_logits_softmax(None, long, one, one, need - 1))
    back = lambda op, w, g, dx, db, ws, n: _error(lib.fl_logits_grad(None, op, w, g, dx, db, ws, n))
    assert "bias" in back(_logits_op(), None, one, one, one, None, 0)
    assert "null" in back(_logits_op(), None, None, one, None, None, 0)
    for op in (_logits_op(rows=100_000, bias=1, bias_rows=1), _logits_op(bias=1, bias_rows=2, group=1)):
        need = lib.fl_logits_grad_bytes(op, 0, 1, 1)
        assert need > 0 and "workspace" in back(op, None, one, one, one, one, need - 1)
        assert "aligned" in back(op, None, one, one, one, one, need)
    assert "shape" in _error(lib.fl_pack_bits(None, one, -1, 3, one))
    assert lib.fl_logits_constrain(None, _logits_op(rows=0), None) == 0

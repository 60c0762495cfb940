"""Refusals of layer_norm's and the losses' entry points that need no GPU: CPU
tensors, and arguments of the C-ABI that are turned down before any launch."""
import ctypes

import pytest
import torch

from flashlog_amd import _lib, attention, losses

ONE = ctypes.c_void_p(16)


def _error(rc):
    assert rc == 1
    return _lib.lib().fl_last_error().decode()


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 3), torch.zeros(4, 3)
    ids, teacher = torch.zeros(2, 1, dtype=torch.long), torch.zeros(2, 1)
    for call in (lambda: attention.layer_norm(x), lambda: losses.linear_cross_entropy(x, w, ids[:, 0]),
                 lambda: losses.linear_distillation(x, w, ids, teacher), lambda: losses.distillation(x, ids, teacher)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        losses.distillation([1.0], ids, teacher)


def test_norm_arguments():
    lib = _lib.lib()

    def op(**kw):
        p = _lib.FlNorm(x=16, M=4, N=3, ldx=3, eps=1e-5)
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    fwd = lambda p, y=ONE: _error(lib.fl_norm_forward(None, p, y, None))
    assert "type" in fwd(op(dtype=3)) and "type" in fwd(op(dtype=-1))
    assert "shape" in fwd(op(M=-1)) and "shape" in fwd(op(N=1 << 31))
    assert "null" in fwd(op(x=None)) and "null" in fwd(op(), None)
    assert lib.fl_norm_forward(None, op(M=0), None, None) == 0
    assert "null" in _error(lib.fl_norm_backward(None, op(), None, ONE, ONE, ONE, ONE, ONE, 1 << 20))
    assert "workspace" in _error(lib.fl_norm_backward(None, op(), ONE, ONE, ONE, ONE, ONE, ONE, 8))
    assert "shape" in _error(lib.fl_norm_backward(None, op(M=0), ONE, ONE, ONE, ONE, ONE, ONE, 1 << 20))
    for N in (1, 2048, 2049, 8192, 8193, 50000):
        assert lib.fl_norm_backward_bytes(op(N=N), 1) >= 8 * N and lib.fl_norm_backward_bytes(op(N=N), 0) == 0


def _lists(**kw):
    p = _lib.FlLists(rows=4, k=2, ids=16, teacher=16, temperature=1.0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


LISTS = [("shape", dict(k=4097)), ("shape", dict(k=-1)), ("shape", dict(rows=-1)), ("shape", dict(teacher=None)),
         ("null", dict(ids=None)), ("temperature", dict(temperature=0.0)),
         ("temperature", dict(temperature=float("nan"))), ("temperature", dict(temperature=float("inf"))),
         ("temperature", dict(temperature=-1.0)), ("temperature", dict(temperature=2.0 ** -61)),
         ("temperature", dict(temperature=2.0 ** 61))]


def test_scores_arguments():
    lib = _lib.lib()

    def op(lists=None, **kw):
        p = _lib.FlScores(lists=lists or _lists(), logits=16, cols=5, ld=5)
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    fwd = lambda p, loss=ONE, size=1 << 20: _error(lib.fl_scores_forward(None, p, loss, ONE, ONE, size))
    for word, kw in LISTS:
        assert word in fwd(op(_lists(**kw)))
    assert "type" in fwd(op(dtype=5)) and "shape" in fwd(op(cols=-1)) and "null" in fwd(op(logits=None))
    assert "null" in fwd(op(), None) and "workspace" in fwd(op(), ONE, 8)
    assert lib.fl_scores_forward(None, op(_lists(rows=0)), None, None, None, 0) == 0
    assert "null" in _error(lib.fl_scores_backward(None, op(), None, ONE, ONE))
    assert lib.fl_scores_forward_bytes(op(cols=4097)) == 4 * 3 * 8
    assert lib.fl_lists_state_bytes(_lists()) >= 4 * 8 + 4 * 2 * 8


def test_vocab_arguments():
    lib = _lib.lib()

    def op(lists=None, **kw):
        p = _lib.FlVocab(lists=lists or _lists(), M=4, V=6, K=3, x=16, ldx=3, weight=16, ldw=3, train=1)
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    fwd = lambda p, loss=ONE, size=1 << 20: _error(lib.fl_vocab_forward(None, p, loss, ONE, None, ONE, size))
    for word, kw in LISTS:
        if kw != dict(rows=-1):
            assert word in fwd(op(_lists(**kw)))
    assert "type" in fwd(op(dtype=3)) and "shape" in fwd(op(V=0)) and "shape" in fwd(op(K=-1))
    assert "shape" in fwd(op(M=3)) and "null" in fwd(op(x=None)) and "null" in fwd(op(weight=None))
    assert "null" in fwd(op(), None) and "workspace" in fwd(op(), ONE, 0)
    back = lambda p, ws=ONE, size=1 << 30, g=ONE: _error(
        lib.fl_vocab_backward(None, p, g, ONE, None, ONE, ONE, ONE, ws, size))
    assert "null" in back(op(), g=None) and "workspace" in back(op(), size=16)
    assert "16-byte" in back(op(), ctypes.c_void_p(24))
    assert "train" in back(op(train=0))
    assert lib.fl_vocab_backward(None, op(_lists(rows=0), M=0), None, None, None, None, None, None, None, 0) == 0
    large = op(_lists(rows=4096), M=4096, V=4096, K=64, ldx=64, ldw=64)
    assert lib.fl_vocab_layout_bytes(large) > 4 * 2 * 4096 * 64 and lib.fl_vocab_layout_bytes(op()) == 0
    assert "null" in fwd(large)


def test_many_bfloat16_inputs_in_training():
    lib = _lib.lib()
    op = lambda K, **kw: _lib.FlVocab(lists=_lists(), M=4, V=6, K=K, x=16, ldx=K, weight=16, ldw=K, dtype=1, **kw)
    fwd = lambda p: _error(lib.fl_vocab_forward(None, p, ONE, ONE, ONE, ONE, 0))
    assert "inputs" in fwd(op((1 << 23) + 1, train=1))
    assert "inputs" not in fwd(op(1 << 23, train=1)) and "inputs" not in fwd(op((1 << 23) + 1))
    assert lib.fl_vocab_layout_bytes(op(1 << 23, train=1)) > 2 * 10 << 23


def test_layouts_lie_on_16_bytes():
    lib = _lib.lib()
    op = _lib.FlVocab(lists=_lists(), M=4, V=6, K=64, x=16, ldx=64, weight=16, ldw=64, dtype=1, train=1)
    assert lib.fl_vocab_layout_bytes(op) > 0
    off = ctypes.c_void_p(24)
    assert "layout" in _error(lib.fl_vocab_forward(None, op, ONE, ONE, off, ONE, 1 << 20))
    assert "layout" in _error(lib.fl_vocab_backward(None, op, ONE, ONE, off, ONE, ONE, ONE, ONE, 1 << 30))

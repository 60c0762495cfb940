"""Losses that train relation logits and entity scores, on the gfx950 HIP
library, with their gradients.

  linear_cross_entropy  softmax cross entropy of hidden states over a
                        vocabulary of relations or entities with a row of
                        weights each (``attention.linear`` and a softmax's
                        loss in one), the logits not kept;
  linear_distillation   the same against a teacher's top answers;
  distillation          the same on score rows that exist: what a hop's states
                        add up to, or ``attention.constrain_logits`` rows, in
                        which masked columns are -inf.

(The reference trains on dense target rows, ``log_loss``, src/utils.py:28-34.)
All give one float32 loss a row, so that a mean, weights or a mask of the rows
are the caller's.  Operands, streams, graphs and derivatives are as in
``attention``: float32, bfloat16 or float16 tensors on the GPU, sums and
softmax statistics in float32, once and backward differentiable, on torch's
current stream, nothing kept between calls.
"""
import math

import torch
from torch import autograd
from torch.autograd.function import once_differentiable

from ._lib import FlLists, FlScores, FlVocab
from .attention import (_TYPES, _differentiated, _integers, _launch, _lib_handle, _need_gpu, _ptr, _rows_of,
                        _workspace)

__all__ = ["linear_cross_entropy", "linear_distillation", "distillation"]


class _Lists:
    """The checked ids and teacher logits of a call, laid out as [rows, k]."""

    __slots__ = ("rows", "k", "ids", "teacher", "temperature")

    def op(self):
        return FlLists(self.rows, self.k, self.ids.data_ptr(), _ptr(self.teacher), self.temperature, 0)


def _targets(what, lead, target):
    if target.shape != lead:
        raise ValueError("%s: target must be %s" % (what, list(lead)))
    out = _Lists()
    out.ids, out.teacher, out.temperature = _integers(what, "target", target), None, 1.0
    out.rows, out.k = target.numel(), 1
    return out


def _lists(what, lead, ids, teacher, temperature):
    if ids.dim() < 1 or ids.shape[:-1] != lead:
        raise ValueError("%s: ids must be [%s], one list a row" % (what, ", ".join([str(n) for n in lead] + ["k"])))
    if teacher.shape != ids.shape:
        raise ValueError("%s: teacher must be %s, as ids" % (what, list(ids.shape)))
    if teacher.dtype not in _TYPES:
        raise TypeError("%s: teacher must be float32, bfloat16 or float16" % what)
    if teacher.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s: the teacher has no gradient; detach it" % what)
    temperature = float(temperature)
    if not 2.0 ** -60 <= temperature <= 2.0 ** 60:
        raise ValueError("%s: temperature must be within 2^-60 and 2^60" % what)
    out = _Lists()
    out.ids, out.teacher, out.temperature = _integers(what, "ids", ids), teacher.float().contiguous(), temperature
    out.rows, out.k = math.prod(lead), ids.shape[-1]
    return out


# ---------------------------------------------------------------------------
# Rows that are a product


def _vocab_op(x, weight, bias, lists, train):
    return FlVocab(lists.op(), x.shape[0], weight.shape[0], weight.shape[1], x.data_ptr(), x.stride(0),
                   weight.data_ptr(), weight.stride(0), _ptr(bias), _TYPES[x.dtype],
                   int(bias is not None and bias.dtype is torch.float32), train, 0)


def _vocab_forward(what, x, weight, bias, lists, train):
    """(losses, x, weight and bias as the call took them, the state and the layout for the backward)."""
    dev, lib = x.device, _lib_handle()
    loss = x.new_empty(x.shape[:-1], dtype=torch.float32)
    x = _rows_of(x, x.shape[-1])
    if weight.shape[1] > 1 and weight.stride(1) != 1:
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    op = _vocab_op(x, weight, bias, lists, train)
    state = _workspace(lib.fl_lists_state_bytes(op.lists), dev)
    layout = _workspace(lib.fl_vocab_layout_bytes(op), dev)
    nbytes = lib.fl_vocab_forward_bytes(op)
    ws = _workspace(nbytes, dev)
    _launch(what, lib.fl_vocab_forward, dev, op, loss.data_ptr(), _ptr(state), _ptr(layout), _ptr(ws), nbytes)
    return loss, x, weight, bias, state, layout


class _VocabFunction(autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, lists, what):
        loss, x2, w2, b2, state, layout = _vocab_forward(what, x, weight, bias, lists, True)
        ctx.save_for_backward(x2, w2, b2, state, layout, lists.ids, lists.teacher)
        ctx.lists, ctx.what, ctx.shape = lists, what, x.shape
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, bias, state, layout = ctx.saved_tensors[:5]
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dev, lib, grad = x.device, _lib_handle(), grad.contiguous()
        make = x.new_empty if x.shape[0] else x.new_zeros  # the sums over no rows
        dx = x.new_empty(ctx.shape) if need_x else None
        dw = make(weight.shape) if need_w else None
        db = make(weight.shape[0], dtype=bias.dtype) if need_b else None
        if x.shape[0]:
            op = _vocab_op(x, weight, bias, ctx.lists, True)
            if lib.fl_vocab_layout_bytes(op) != (0 if layout is None else layout.numel()):
                # a hook on saved tensors has them on other strides than the forward had
                state, layout = _vocab_forward(ctx.what, x, weight, bias, ctx.lists, True)[4:]
            nbytes = lib.fl_vocab_backward_bytes(op, need_x, need_w, need_b)
            ws = _workspace(nbytes, dev)
            _launch(ctx.what, lib.fl_vocab_backward, dev, op, grad.data_ptr(), _ptr(state), _ptr(layout), _ptr(dx),
                    _ptr(dw), _ptr(db), _ptr(ws), nbytes)
        return dx, dw, db, None, None


def _vocab_operands(what, x, weight, bias):
    """Checks them; the shape of the rows."""
    if x.dtype not in _TYPES:
        raise TypeError("%s: x must be float32, bfloat16 or float16" % what)
    if weight.dtype is not x.dtype:
        raise TypeError("%s: x and weight must be of one type" % what)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError("%s: weight must be [vocabulary, inputs] and x [..., inputs]" % what)
    if weight.shape[0] < 1:
        raise ValueError("%s: an empty vocabulary" % what)
    if bias is not None:
        if bias.dtype is not x.dtype and bias.dtype is not torch.float32:
            raise TypeError("%s: bias must be of x's type or float32" % what)
        if bias.shape != weight.shape[:1]:
            raise ValueError("%s: bias must be [%d]" % (what, weight.shape[0]))
    return x.shape[:-1]


def _vocab_loss(what, x, weight, bias, lists):
    if _differentiated(x, weight, bias):
        return _VocabFunction.apply(x, weight, bias, lists, what)
    return _vocab_forward(what, x, weight, bias, lists, False)[0]


def linear_cross_entropy(x, weight, target, bias=None):
    """The cross entropy of every row of ``softmax(x @ weight.T + bias)``.

    x [..., inputs], weight [vocabulary, inputs], bias [vocabulary] (x's type
    or float32; -inf takes a column out), target [...] integers; float32
    [...].  A row whose target is outside [0, vocabulary) has loss 0 and gives
    no gradient; its x may be any finite values, but 0 times an infinity is NaN
    in weight's gradient.  A target that the bias takes out has loss inf, a row
    of which nothing is left 0 without a gradient.

    In training, bfloat16 has up to 2^23 inputs.

    No logits are kept: the backward computes them again, a piece of the
    vocabulary at a time.  Its workspace is up to 1 GB of their gradient (256
    columns where there are more rows than that holds), float32 sums of x's
    gradient (of its size where the vocabulary takes several pieces, else up to
    64 MB) and of weight's (up to 64 MB), and a copy of 16-bit x.  Held from the
    forward to the backward are copies of x and weight, where large products
    lay them out: float32 as three bfloat16 planes (1.5 times their size; all
    of their 24 bits, at float32's range), half whose rows are not whole steps
    of 64 inputs on 16 bytes, and bfloat16, always, as scaled half (a value is
    off by nothing, or by 2^-38 of the largest of its row of x or of weight).

    The logits' gradient is an operand of two products and a term of the
    bias's: float32's is held as such; of 16-bit operands the softmax's terms
    less what the row is held to are held as half (2^-11 of themselves or
    2^-39; of up to 64 rows of half with what rounding leaves), whatever the
    losses' gradients are, and in weight's gradient each row's input times its
    loss's (2^-38 of the largest of all rows).
    Softmax terms are off by 2^-23 of themselves times 1 + their logit's
    distance from the largest (at least 16 over large vocabularies), whatever
    all logits have in common; a bias whose quotient by the temperature
    overflows float32 counts as infinite."""
    _need_gpu("linear_cross_entropy", x, weight, target, bias)
    lead = _vocab_operands("linear_cross_entropy", x, weight, bias)
    return _vocab_loss("linear_cross_entropy", x, weight, bias, _targets("linear_cross_entropy", lead, target))


def linear_distillation(x, weight, ids, teacher, bias=None, temperature=1.0):
    """``distillation`` of the logits ``x @ weight.T + bias``, which are not
    kept: operands and gradients as in ``linear_cross_entropy``."""
    _need_gpu("linear_distillation", x, weight, ids, teacher, bias)
    lead = _vocab_operands("linear_distillation", x, weight, bias)
    return _vocab_loss("linear_distillation", x, weight, bias,
                       _lists("linear_distillation", lead, ids, teacher, temperature))


# ---------------------------------------------------------------------------
# Rows that are given


def _scores_op(logits, lists):
    return FlScores(lists.op(), logits.data_ptr(), logits.shape[1], logits.stride(0), _TYPES[logits.dtype], 0)


def _scores_forward(logits, lists):
    """(losses, the laid out logits, the state for the backward)."""
    dev, lib = logits.device, _lib_handle()
    loss = logits.new_empty(logits.shape[:-1], dtype=torch.float32)
    x = _rows_of(logits, logits.shape[-1])
    op = _scores_op(x, lists)
    state = _workspace(lib.fl_lists_state_bytes(op.lists), dev)
    nbytes = lib.fl_scores_forward_bytes(op)
    ws = _workspace(nbytes, dev)
    _launch("distillation", lib.fl_scores_forward, dev, op, loss.data_ptr(), _ptr(state), _ptr(ws), nbytes)
    return loss, x, state


class _ScoresFunction(autograd.Function):
    @staticmethod
    def forward(ctx, logits, lists):
        loss, x, state = _scores_forward(logits, lists)
        ctx.save_for_backward(x, state, lists.ids, lists.teacher)
        ctx.lists, ctx.shape = lists, logits.shape
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, state = ctx.saved_tensors[:2]
        dx = x.new_empty(ctx.shape)
        if dx.numel():
            _launch("distillation", _lib_handle().fl_scores_backward, x.device, _scores_op(x, ctx.lists),
                    grad.contiguous().data_ptr(), _ptr(state), dx.data_ptr())
        return dx, None


def distillation(logits, ids, teacher, temperature=1.0):
    """How far rows of logits or scores [..., n] are from a teacher's top
    answers: ids [..., k] (integers; k up to 4096) and the teacher's logits for
    them; float32 [...].

    With u = logits / temperature over all n columns and q the softmax of
    teacher / temperature over the row's listed ids::

        loss = temperature^2 * sum_j q_j (log q_j - u[ids_j] + log sum exp u)

    (the divergence of the row's softmax from q; the factor keeps gradients of
    one size).  Ids outside [0, n) pad a list; an id whose logit is -inf, as
    ``constrain_logits`` leaves masked columns, and one whose teacher logit is
    -inf are left out of it.  An id listed twice counts twice.  A row with
    nothing listed, or with nothing left (every logit -inf), has loss 0 and no
    gradient; a NaN or +inf among its logits makes both NaN.  Masked columns
    have a gradient of 0.  The teacher has none (one that requires it is
    refused)."""
    _need_gpu("distillation", logits, ids, teacher)
    if logits.dtype not in _TYPES:
        raise TypeError("distillation: logits must be float32, bfloat16 or float16")
    if logits.dim() < 1:
        raise ValueError("distillation: logits must be [..., columns]")
    lists = _lists("distillation", logits.shape[:-1], ids, teacher, temperature)
    if _differentiated(logits):
        return _ScoresFunction.apply(logits, lists)
    return _scores_forward(logits, lists)[0]

"""The operators between a rule generator's hidden states, the hops and the
answers, on the gfx950 HIP library.

A hop takes attention ``w [B, L, n]`` over the n = 2R+1 relation operators
(``flashlog_kernel.dense_csr_sum_cuda`` and the sparse classes), and the
evaluation takes score rows ``[Q, E]``.  The reference's model files make w
with torch (linear layers, then ``softmax(w_all[:, t] / tau_1)``,
src/model_DRUM_kernel.py:90-117); it has no constraints on either.  Here:

  linear           act(x W^T + b) + residual in one pass: generator layers and
                   the head that makes relation logits;
  relation_linear  the same with weights of its own for every head relation,
                   over rows in any order (``group_rows`` groups them);
  constrain_logits masks (which relations a rule body may use, which entities
                   an answer may be), priors, and penalties for ids that a row
                   has had already, on logits or score rows;
  hop_attention    the same, then the softmax over what is allowed: a hop's w,
                   fp32, exactly 0 where nothing is allowed (the hops skip
                   weights that are not positive).

Operands are float32, bfloat16 or float16 tensors on the GPU (CPU tensors
raise); sums, softmax statistics and gradients of tables are float32.  All
four are differentiable (once and backward: a second derivative and
forward-mode tangents raise), run on torch's current stream, allocate with
torch, and neither synchronise nor keep anything between calls, so they can be
captured into a graph.  A captured backward needs leaves whose gradient graph
was not begun outside the capture, as everywhere in torch.
"""
import math

import torch
from torch import autograd
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import FlLinear, FlLogits, check

__all__ = ["RowGroups", "group_rows", "linear", "relation_linear", "pack_allowed", "history_from_pairs",
           "constrain_logits", "hop_attention"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "silu": 3, "tanh": 4, "sigmoid": 5}
_raw_stream = torch._C._cuda_getCurrentRawStream  # the current stream's handle, without a Stream object
_LIB = None


def _lib_handle():
    global _LIB
    if _LIB is None:
        _LIB = _lib.lib()
    return _LIB


def _launch(what, fn, dev, *args):
    """Calls an entry point on the device's current stream, with the device current."""
    i = dev.index
    if i == torch.cuda.current_device():
        rc = fn(_raw_stream(i), *args)
    else:
        with torch.cuda.device(dev):
            rc = fn(_raw_stream(i), *args)
    if rc:
        check(rc, what)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _need_gpu(what, *tensors):
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not torch.is_tensor(t):
            raise TypeError("%s: expected tensors, got %s" % (what, type(t).__name__))
        if not t.is_cuda:
            raise RuntimeError("%s runs on the GPU only; got a CPU tensor" % what)
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError("%s: tensors on different devices" % what)
    return dev


def _differentiated(*operands):
    """Whether a call has to go through its autograd function: for the
    backward, or, inside a forward-mode level, to have it refuse tangents
    (dual tensors need not require gradients)."""
    if forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in operands)


def _integers(what, name, t):
    if t.dtype is torch.int64 and t.is_contiguous():
        return t
    if t.dtype not in (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8):
        raise TypeError("%s: %s must hold integers" % (what, name))
    return t.long().contiguous()


def _workspace(nbytes, dev):
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


# ---------------------------------------------------------------------------
# Rows by relation


class RowGroups:
    """Rows grouped by an index (``group_rows``): ``order`` int32 [rows], the
    rows of a group together and in their own order; ``offsets`` int32
    [groups + 1], where each group begins.  Rows whose id was outside
    [0, groups) come behind ``offsets[groups]``."""

    __slots__ = ("rows", "groups", "_plan", "_at")

    def __init__(self, rows, groups, plan):
        self.rows, self.groups, self._plan = rows, groups, plan  # order, offsets, the products' tiles
        base = plan.data_ptr()
        self._at = (base, base + 4 * rows, base + 4 * (rows + groups + 1))

    @property
    def order(self):
        return self._plan[:self.rows]

    @property
    def offsets(self):
        return self._plan[self.rows:self.rows + self.groups + 1]

    @property
    def tiles(self):
        return self._plan[self.rows + self.groups + 1:]


def group_rows(index, groups):
    """Groups rows by ``index`` (integers of any shape, a row each), each in
    [0, groups); rows with another id belong to no group.  The plan serves any
    number of products over the same rows."""
    dev = _need_gpu("group_rows", index)
    groups = int(groups)
    if groups < 1:
        raise ValueError("group_rows: at least one group")
    index = _integers("group_rows", "index", index)
    rows = index.numel()
    lib = _lib_handle()
    plan = torch.empty(rows + groups + 1 + 2 * lib.fl_group_tiles(rows, groups), dtype=torch.int32, device=dev)
    nbytes = lib.fl_group_rows_bytes(rows, groups)
    ws = _workspace(nbytes, dev)
    out = RowGroups(rows, groups, plan)
    _launch("group_rows", lib.fl_group_rows, dev, index.data_ptr(), rows, groups, *out._at, _ptr(ws), nbytes)
    return out


# ---------------------------------------------------------------------------
# Products


def _rows_of(t, cols):
    """t as [rows, cols] with contiguous columns (a copy where its strides allow no such view)."""
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), cols)
    return t if cols <= 1 or t.stride(1) == 1 else t.contiguous()


def _linear_op(x, weight, bias, residual, plan, act):
    M, K = x.shape
    N = weight.shape[-2]
    if plan is None:
        groups, w_group, order, offsets, tiles = 1, 0, None, None, None
    else:
        groups, w_group = plan.groups, weight.stride(0)
        order, offsets, tiles = plan._at
    return FlLinear(M, N, K, groups, x.data_ptr(), x.stride(0), weight.data_ptr(), weight.stride(-2), w_group,
                    None if bias is None else bias.data_ptr(), None if residual is None else residual.data_ptr(),
                    0 if residual is None else residual.stride(0), order, offsets, tiles, _TYPES[x.dtype], act,
                    int(bias is not None and bias.dtype is torch.float32), 0)


def _linear_forward(x, weight, bias, residual, plan, act, keep):
    """(y, the laid out x and weight, the activation's argument or None)."""
    dev = x.device
    N, K = weight.shape[-2:]
    y = torch.empty(x.shape[:-1] + (N,), dtype=x.dtype, device=dev)
    x = _rows_of(x, K)
    if K > 1 and weight.stride(-1) != 1:
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if residual is not None:
        residual = _rows_of(residual, N)
    pre = torch.empty((x.shape[0], N), dtype=torch.float32, device=dev) if keep else None
    op = _linear_op(x, weight, bias, residual, plan, act)
    lib = _lib_handle()
    nbytes = lib.fl_linear_forward_bytes(op)
    ws = _workspace(nbytes, dev)
    _launch("linear", lib.fl_linear_forward, dev, op, y.data_ptr(), _ptr(pre), _ptr(ws), nbytes)
    return y, x, weight, pre


class _LinearFunction(autograd.Function):
    """act(x W_g^T + b_g) + residual; plan None: one group."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, plan, act):
        keep = act != 0 and any(ctx.needs_input_grad[:3])
        y, x2, w2, pre = _linear_forward(x, weight, bias, residual, plan, act, keep)
        ctx.save_for_backward(x2, w2, pre)
        ctx.plan, ctx.act, ctx.shapes = plan, act, (x.shape, bias.dtype if bias is not None else None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, pre = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            dev, lib = x.device, _lib_handle()
            (shape, bias_dtype), g = ctx.shapes, grad.contiguous()
            if g.data_ptr() % 16:
                g = g.clone()
            op = _linear_op(x, weight, None, None, ctx.plan, ctx.act)
            if need_x:
                dx = torch.empty(shape, dtype=x.dtype, device=dev)
            if need_w:
                dw = torch.empty(weight.shape, dtype=x.dtype, device=dev)
            if need_b:
                db = torch.empty(weight.shape[:-1], dtype=bias_dtype, device=dev)
            nbytes = lib.fl_linear_backward_bytes(op, need_x, need_w, need_b)
            ws = _workspace(nbytes, dev)
            _launch("linear", lib.fl_linear_backward, dev, op, g.data_ptr(), _ptr(pre), _ptr(dx), _ptr(dw), _ptr(db),
                    bias_dtype is torch.float32, _ptr(ws), nbytes)
        return dx, dw, db, grad if need_r else None, None, None


def _product(what, x, plan, weight, bias, activation, residual):
    _need_gpu(what, x, weight, bias, residual, None if plan is None else plan._plan)
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError("%s: activation must be one of %s" % (what, ", ".join(map(repr, _ACTIVATIONS))))
    dtype, wshape, xshape = x.dtype, weight.shape, x.shape
    if dtype not in _TYPES:
        raise TypeError("%s: x must be float32, bfloat16 or float16" % what)
    if weight.dtype is not dtype or (residual is not None and residual.dtype is not dtype):
        raise TypeError("%s: x, weight and residual must be of one type" % what)
    if len(wshape) != (2 if plan is None else 3) or len(xshape) < 1:
        raise ValueError("%s: weight must be [%soutputs, inputs] and x [..., inputs]"
                         % (what, "" if plan is None else "groups, "))
    if xshape[-1] != wshape[-1]:
        raise ValueError("%s: x has %d inputs, weight %d" % (what, xshape[-1], wshape[-1]))
    if bias is not None:
        if bias.dtype is not dtype and bias.dtype is not torch.float32:
            raise TypeError("%s: bias must be of x's type or float32" % what)
        if bias.shape != wshape[:-1]:
            raise ValueError("%s: bias must be %s" % (what, list(wshape[:-1])))
    if residual is not None and residual.shape != xshape[:-1] + wshape[-2:-1]:
        raise ValueError("%s: residual must be %s" % (what, list(xshape[:-1] + wshape[-2:-1])))
    if plan is not None:
        if wshape[0] != plan.groups:
            raise ValueError("%s: weight has %d groups, the plan %d" % (what, wshape[0], plan.groups))
        if math.prod(xshape[:-1]) != plan.rows:
            raise ValueError("%s: x has %d rows, the plan %d" % (what, math.prod(xshape[:-1]), plan.rows))
    if _differentiated(x, weight, bias, residual):
        return _LinearFunction.apply(x, weight, bias, residual, plan, act)
    return _linear_forward(x, weight, bias, residual, plan, act, False)[0]


def linear(x, weight, bias=None, activation=None, residual=None):
    """``activation(x @ weight.T + bias) + residual`` in one pass.

    x [..., inputs], weight [outputs, inputs], bias [outputs] (x's type or
    float32), residual [..., outputs]; activation None, "relu", "gelu" (the
    erf form), "silu", "tanh" or "sigmoid".  Rows and weights may be strided;
    operands whose last dimension is not contiguous are copied.  Sums are
    float32 and the result is rounded once; with float32 operands every
    product is off by less than 2^-22 of itself, to either side (a float32
    product by up to 2^-24), and a sum which an infinity or NaN enters is NaN.
    Activations are evaluated to 2^-20 of 1 + |argument|.  For the backward the
    activation's argument is kept in float32; its gradient is rounded to the
    operands' type as an operand of two products, but not as a term of the
    bias's."""
    return _product("linear", x, None, weight, bias, activation, residual)


def relation_linear(x, groups, weight, bias=None, activation=None, residual=None):
    """``linear`` with weights of its own for every group of rows.

    Row i of x [..., inputs] takes weight[g] ([groups, outputs, inputs]) and
    bias[g] ([groups, outputs]) of its group g in ``groups``
    (``group_rows(relation, number of relations)``, as many rows as x has); a
    row of no group gives its residual (0 without one) and takes no part in
    the gradients.  Results are in x's row order."""
    if not isinstance(groups, RowGroups):
        raise TypeError("relation_linear: groups must come from group_rows")
    return _product("relation_linear", x, groups, weight, bias, activation, residual)


# ---------------------------------------------------------------------------
# Constraints


def pack_allowed(mask):
    """The bit table of a bool mask [..., n]: int32 [..., ceil(n / 32)],
    column 32 w + b in bit b of word w (what ``allowed`` takes)."""
    dev = _need_gpu("pack_allowed", mask)
    if mask.dtype != torch.bool or mask.dim() < 1:
        raise TypeError("pack_allowed: mask must be bool [..., columns]")
    n = mask.shape[-1]
    rows = math.prod(mask.shape[:-1])
    words = torch.empty(mask.shape[:-1] + ((n + 31) // 32,), dtype=torch.int32, device=dev)
    mask = mask.contiguous()
    _launch("pack_allowed", _lib_handle().fl_pack_bits, dev, mask.data_ptr(), rows, n, words.data_ptr())
    return words


def history_from_pairs(rows, ids, count):
    """The ``history`` (offsets, ids) of ``count`` rows from (row, id) pairs in
    any order, such as the known answers of ``build_filter_indices_csr``;
    pairs whose row is outside [0, count) are left out."""
    _need_gpu("history_from_pairs", rows, ids)
    if rows.dim() != 1 or rows.shape != ids.shape:
        raise ValueError("history_from_pairs: rows and ids must be 1D and equally long")
    ids, count = _integers("history_from_pairs", "ids", ids), int(count)
    if count < 0:
        raise ValueError("history_from_pairs: count must be nonnegative")
    plan = group_rows(rows, max(count, 1))
    return plan.offsets[:count + 1].long(), ids[plan.order.long()]


class _Constraints:
    """The checked arguments of one call, laid out."""

    __slots__ = ("rows", "cols", "inner", "allowed", "group", "history", "history_ptr", "scalars")

    def op(self, x, bias):
        a, h, g, p = self.allowed, self.history, self.group, self.history_ptr
        return FlLogits(x.data_ptr(), self.rows, self.cols, x.stride(0), self.inner,
                        None if a is None else a.data_ptr(), 0 if a is None else a.shape[0],
                        0 if a is None else a.shape[1], None if g is None else g.data_ptr(),
                        None if bias is None else bias.data_ptr(), 0 if bias is None else bias.shape[0],
                        None if h is None else h.data_ptr(), None if p is None else p.data_ptr(),
                        0 if h is None else h.shape[-1], *self.scalars)


def _spread(t, count):
    """One entry a coarse owner -> one a fine owner (count of them)."""
    return t if t.shape[0] == count else t.repeat_interleave(count // max(t.shape[0], 1), 0)


def _table(what, name, t, width, group):
    """A table [width] or [groups, width] as [groups, width]."""
    if t.dim() not in (1, 2) or t.shape[-1] != width:
        raise ValueError("%s: %s must be [%d] or [groups, %d]" % (what, name, width, width))
    if t.dim() == 1:
        t = t.reshape(1, width)
    if t.shape[0] != 1 and group is None:
        raise ValueError("%s: %s has %d rows; group says which of them a row takes" % (what, name, t.shape[0]))
    if t.shape[0] == 0:
        raise ValueError("%s: %s has no rows" % (what, name))
    return t if t.is_contiguous() else t.contiguous()


def _constraints(what, logits, allowed, group, bias, history, *scalars):
    past, offsets = history, None
    if isinstance(history, (tuple, list)):
        if len(history) != 2:
            raise ValueError("%s: a ragged history is (offsets, ids)" % what)
        offsets, past = history
    _need_gpu(what, logits, allowed, group, bias, past, offsets)
    if logits.dtype not in _TYPES:
        raise TypeError("%s: logits must be float32, bfloat16 or float16" % what)
    lead = logits.shape[:-1]
    if logits.dim() < 1:
        raise ValueError("%s: logits must be [..., columns]" % what)
    scalars = [float(v) for v in scalars]
    for name, v in zip(("repetition", "presence", "frequency", "temperature"), scalars):
        if not math.isfinite(v) or (v <= 0.0 and name in ("repetition", "temperature")):
            raise ValueError("%s: %s must be finite%s" % (what, name, "" if name[-4:] in ("ence", "ency") else
                                                          " and positive"))
    c = _Constraints()
    c.rows, c.cols = math.prod(lead), logits.shape[-1]

    def owners_of(shape, name):
        if shape != lead[:len(shape)]:
            raise ValueError("%s: %s is for rows %s, the logits have %s" % (what, name, list(shape), list(lead)))
        return math.prod(shape)

    owners = None
    if group is not None:
        owners = owners_of(group.shape, "group")
        group = _integers(what, "group", group)
        if group.dim() != 1:
            group = group.reshape(-1)
    if past is not None:
        past = _integers(what, "history", past)
        if offsets is not None:
            if past.dim() != 1 or offsets.dim() != 1 or offsets.numel() < 1:
                raise ValueError("%s: a ragged history is 1D offsets and 1D ids" % what)
            offsets = _integers(what, "history", offsets)
            listed = offsets.numel() - 1
            if listed not in [math.prod(lead[:k]) for k in range(len(lead) + 1)]:
                raise ValueError("%s: history is for %d rows, the logits have %s" % (what, listed, list(lead)))
        else:
            if past.dim() < 1:
                raise ValueError("%s: history must be [..., ids]" % what)
            listed = owners_of(past.shape[:-1], "history")
            if past.dim() != 2:
                past = past.reshape(listed, past.shape[-1])
        if owners is None or listed > owners:
            owners = listed
        if offsets is None:
            past = _spread(past, owners)
        elif listed != owners:
            raise ValueError("%s: a ragged history needs as many rows as group has" % what)
    if group is not None:
        group = _spread(group, owners)
    c.inner = max(c.rows // owners, 1) if owners else 1
    if allowed is not None:
        if allowed.dtype is torch.bool:
            if allowed.shape[-1:] != (c.cols,):
                raise ValueError("%s: allowed must be [..., %d]" % (what, c.cols))
            allowed = pack_allowed(allowed)
        elif allowed.dtype is not torch.int32:
            raise TypeError("%s: allowed must be a bool mask or pack_allowed's words" % what)
        allowed = _table(what, "allowed", allowed, (c.cols + 31) // 32, group)
    if bias is not None:
        if bias.dtype not in _TYPES:
            raise TypeError("%s: bias must be float32, bfloat16 or float16" % what)
        bias = _table(what, "bias", bias.float(), c.cols, group)
        if allowed is not None and 1 not in (allowed.shape[0], bias.shape[0]) and allowed.shape[0] != bias.shape[0]:
            raise ValueError("%s: allowed and bias have different numbers of groups" % what)
    c.allowed, c.group, c.history, c.history_ptr = allowed, group, past, offsets
    c.scalars = (*scalars, _TYPES[logits.dtype])
    return c, bias


def _logits_forward(c, logits, bias, softmax):
    """(output, the laid out logits)."""
    dev, lib = logits.device, _lib_handle()
    out = torch.empty(logits.shape, dtype=torch.float32 if softmax else logits.dtype, device=dev)
    x = _rows_of(logits, c.cols)
    op = c.op(x, bias)
    if softmax:
        nbytes = lib.fl_logits_softmax_bytes(op)
        ws = _workspace(nbytes, dev)
        _launch("hop_attention", lib.fl_logits_softmax, dev, op, out.data_ptr(), _ptr(ws), nbytes)
    else:
        _launch("constrain_logits", lib.fl_logits_constrain, dev, op, out.data_ptr())
    return out, x


class _LogitsFunction(autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, c, softmax):
        out, x = _logits_forward(c, logits, bias, softmax)
        signs = c.history is not None and c.scalars[0] != 1.0  # the slopes go by the sign of logits + bias
        ctx.save_for_backward(x if signs else None, bias, out if softmax else None, c.allowed, c.group, c.history,
                              c.history_ptr)
        ctx.c, ctx.softmax, ctx.dtype = c, softmax, logits.dtype
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, bias, w = ctx.saved_tensors[:3]
        c, lib, dev = ctx.c, _lib_handle(), grad.device
        need_x, need_b = ctx.needs_input_grad[:2]
        shape, grad = grad.shape, grad.contiguous()
        dx = torch.empty(shape, dtype=ctx.dtype, device=dev) if need_x else None
        db = torch.empty_like(bias) if need_b else None
        # without their signs the logits are not read: the gradient's rows stand for them
        op = c.op(x if x is not None else _rows_of(grad, c.cols), bias)
        nbytes = lib.fl_logits_grad_bytes(op, ctx.softmax, need_x, need_b)
        ws = _workspace(nbytes, dev)
        _launch("hop_attention" if ctx.softmax else "constrain_logits", lib.fl_logits_grad, dev, op, _ptr(w),
                grad.data_ptr(), _ptr(dx), _ptr(db), _ptr(ws), nbytes)
        return dx, db, None, None


def _apply(logits, c, bias, softmax):
    if _differentiated(logits, bias):
        return _LogitsFunction.apply(logits, bias, c, softmax)
    return _logits_forward(c, logits, bias, softmax)[0]


def constrain_logits(logits, allowed=None, group=None, bias=None, history=None, repetition=1.0, presence=0.0,
                     frequency=0.0, temperature=1.0, fill=-math.inf):
    """Constrained logits or scores [..., n], of the logits' type.

    Per column, with c = how often the row's history holds it::

        u = logits + bias
        if c: u = (u / repetition if u > 0 else u * repetition) - presence - frequency * c
        out = u / temperature where allowed, else fill

    allowed: a bool mask [n] or [groups, n], or its ``pack_allowed`` (keep
    that where the mask stays the same); bias [n] or [groups, n].  group: the
    table row of every row, integers of the logits' leading shape or of its
    first dimensions (a query's steps then share it).  A table of one row is
    every row's, whatever its group; a group outside a table of several has
    nothing allowed.  history: ids [..., h] for the logits' leading shape or
    its first dimensions, padded with ids outside [0, n), or (offsets, ids)
    with the ids offsets[i] .. offsets[i+1] of row i; a column is counted up
    to some 65,000 times.  The scalars are float32; repetition and temperature
    lie in [2^-126, 2^126].

    Masked logits are not read into anything: they may be infinite or NaN.
    Gradients reach logits and bias; masked columns have none."""
    return _apply(logits, *_constraints("constrain_logits", logits, allowed, group, bias, history, repetition, presence,
                                        frequency, temperature, fill), softmax=False)


def hop_attention(logits, allowed=None, group=None, bias=None, history=None, repetition=1.0, presence=0.0,
                  frequency=0.0, temperature=1.0):
    """A hop's attention: the softmax of ``constrain_logits`` over the allowed
    columns, float32 [..., n], with the same arguments.  Masked columns are
    exactly 0; a row with nothing left (no column allowed, or every allowed
    logit -inf) is all zeros and has no gradient.  A NaN or +inf among a row's
    allowed logits makes the row's other allowed weights NaN."""
    return _apply(logits, *_constraints("hop_attention", logits, allowed, group, bias, history, repetition, presence,
                                        frequency, temperature, 0.0), softmax=True)

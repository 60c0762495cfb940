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
four are differentiable (once: a second derivative raises), run on torch's
current stream, allocate with torch, and neither synchronise nor keep
anything between calls, so they can be captured into a graph.  A captured
backward needs leaves whose gradient graph was not begun outside the capture,
as everywhere in torch.
"""
import contextlib
import math

import torch
from torch import autograd
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import FlLinear, FlLogits, check, ptr, stream_handle

__all__ = ["RowGroups", "group_rows", "linear", "relation_linear", "pack_allowed", "history_from_pairs",
           "constrain_logits", "hop_attention"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "silu": 3, "tanh": 4, "sigmoid": 5}
_HERE = contextlib.nullcontext()


def _on(dev):
    """The device that a call's tensors are on, as the current one."""
    return _HERE if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


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


def _integers(what, name, t):
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

    __slots__ = ("rows", "groups", "order", "offsets", "tiles")

    def __init__(self, rows, groups, order, offsets, tiles):
        self.rows, self.groups, self.order, self.offsets, self.tiles = rows, groups, order, offsets, tiles


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
    lib = _lib.lib()
    ntiles = lib.fl_group_tiles(rows, groups)
    # one allocation: order, offsets, tiles
    buf = torch.empty(rows + groups + 1 + 2 * ntiles, dtype=torch.int32, device=dev)
    order, offsets, tiles = buf[:rows], buf[rows:rows + groups + 1], buf[rows + groups + 1:]
    nbytes = lib.fl_group_rows_bytes(rows, groups)
    ws = _workspace(nbytes, dev)
    with _on(dev):
        check(lib.fl_group_rows(stream_handle(dev), ptr(index), rows, groups, ptr(order), ptr(offsets), ptr(tiles),
                                ptr(ws), nbytes), "group_rows")
    return RowGroups(rows, groups, order, offsets, tiles)


# ---------------------------------------------------------------------------
# Products


def _rows_of(t, cols):
    """t as [rows, cols] with contiguous columns (a copy where its strides allow no such view)."""
    t = t.reshape(math.prod(t.shape[:-1]), cols)
    return t if cols <= 1 or t.stride(1) == 1 else t.contiguous()


def _linear_op(x, weight, bias, residual, plan, act):
    M, K = x.shape
    N = weight.shape[-2]
    grouped = plan is not None
    return FlLinear(M, N, K, plan.groups if grouped else 1, x.data_ptr(), x.stride(0), weight.data_ptr(),
                    weight.stride(-2), weight.stride(0) if grouped else 0,
                    bias.data_ptr() if bias is not None else None,
                    residual.data_ptr() if residual is not None else None,
                    residual.stride(0) if residual is not None else 0,
                    plan.order.data_ptr() if grouped else None, plan.offsets.data_ptr() if grouped else None,
                    plan.tiles.data_ptr() if grouped else None, _TYPES[x.dtype], act,
                    int(bias is not None and bias.dtype == torch.float32), 0)


def _linear_forward(x, weight, bias, residual, plan, act, keep):
    """(y, the activation's argument or None)."""
    dev = x.device
    y = torch.empty((x.shape[0], weight.shape[-2]), dtype=x.dtype, device=dev)
    pre = torch.empty_like(y) if keep else None
    op = _linear_op(x, weight, bias, residual, plan, act)
    with _on(dev):
        check(_lib.lib().fl_linear_forward(stream_handle(dev), op, ptr(y), ptr(pre)), "linear")
    return y, pre


class _LinearFunction(autograd.Function):
    """act(x W_g^T + b_g) + residual of 2D rows; plan None: one group."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, plan, act):
        slopes = act != 0 and any(ctx.needs_input_grad[:3])
        y, pre = _linear_forward(x, weight, bias, residual, plan, act, slopes)
        ctx.save_for_backward(x, weight, pre)
        ctx.plan, ctx.act = plan, act
        ctx.bias_dtype = bias.dtype if bias is not None else None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            dev, lib = x.device, _lib.lib()
            d = grad.contiguous()
            op = _linear_op(x, weight, None, None, ctx.plan, ctx.act)
            with _on(dev):
                st = stream_handle(dev)
                if pre is not None:
                    g, d = d, torch.empty_like(pre)
                    check(lib.fl_linear_act_grad(st, _TYPES[x.dtype], ctx.act, ptr(g), ptr(pre), d.numel(), ptr(d)),
                          "linear")
                if need[0]:
                    dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
                    check(lib.fl_linear_input_grad(st, op, ptr(d), ptr(dx)), "linear")
                if need[1]:
                    dw = torch.empty(weight.shape, dtype=weight.dtype, device=dev)
                    nbytes = lib.fl_linear_weight_grad_bytes(op)
                    ws = _workspace(nbytes, dev)
                    check(lib.fl_linear_weight_grad(st, op, ptr(d), ptr(dw), ptr(ws), nbytes), "linear")
                if need[2]:
                    db = torch.empty(weight.shape[:-1], dtype=ctx.bias_dtype, device=dev)
                    nbytes = lib.fl_linear_bias_grad_bytes(op)
                    ws = _workspace(nbytes, dev)
                    check(lib.fl_linear_bias_grad(st, op, ptr(d), ptr(db), int(db.dtype == torch.float32), ptr(ws),
                                                  nbytes), "linear")
        return dx, dw, db, grad if need[3] else None, None, None


def _product(what, x, plan, weight, bias, activation, residual):
    _need_gpu(what, x, weight, bias, residual, plan.order if plan is not None else None)
    if activation not in _ACTIVATIONS:
        raise ValueError("%s: activation must be one of %s" % (what, ", ".join(map(repr, _ACTIVATIONS))))
    if x.dtype not in _TYPES:
        raise TypeError("%s: x must be float32, bfloat16 or float16" % what)
    if weight.dtype != x.dtype or (residual is not None and residual.dtype != x.dtype):
        raise TypeError("%s: x, weight and residual must be of one type" % what)
    if bias is not None and bias.dtype not in (x.dtype, torch.float32):
        raise TypeError("%s: bias must be of x's type or float32" % what)
    dims = 2 if plan is None else 3
    if weight.dim() != dims or x.dim() < 1:
        raise ValueError("%s: weight must be [%soutputs, inputs] and x [..., inputs]" % (what, "groups, " * (dims - 2)))
    N, K = weight.shape[-2:]
    if x.shape[-1] != K:
        raise ValueError("%s: x has %d inputs, weight %d" % (what, x.shape[-1], K))
    if plan is not None and weight.shape[0] != plan.groups:
        raise ValueError("%s: weight has %d groups, the plan %d" % (what, weight.shape[0], plan.groups))
    if bias is not None and bias.shape != weight.shape[:-1]:
        raise ValueError("%s: bias must be %s" % (what, list(weight.shape[:-1])))
    shape = x.shape[:-1] + (N,)
    if residual is not None and residual.shape != shape:
        raise ValueError("%s: residual must be %s" % (what, list(shape)))
    x = _rows_of(x, K)
    if plan is not None and x.shape[0] != plan.rows:
        raise ValueError("%s: x has %d rows, the plan %d" % (what, x.shape[0], plan.rows))
    if K > 1 and weight.stride(-1) != 1:
        weight = weight.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    if residual is not None:
        residual = _rows_of(residual, N)
    act = _ACTIVATIONS[activation]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        y = _LinearFunction.apply(x, weight, bias, residual, plan, act)
    else:
        y = _linear_forward(x, weight, bias, residual, plan, act, False)[0]
    return y.view(shape)


def linear(x, weight, bias=None, activation=None, residual=None):
    """``activation(x @ weight.T + bias) + residual`` in one pass.

    x [..., inputs], weight [outputs, inputs], bias [outputs] (x's type or
    float32), residual [..., outputs]; activation None, "relu", "gelu" (the
    erf form), "silu", "tanh" or "sigmoid".  Rows and weights may be strided;
    operands whose last dimension is not contiguous are copied.  Sums are
    float32 and the result is rounded once; with float32 operands products
    are as exact as float32 ones, except that a sum which an infinity or NaN
    enters is NaN.  For the gradients of bfloat16 and float16 operands the
    activation's argument and its gradient are kept in their type."""
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
    with _on(dev):
        check(_lib.lib().fl_pack_bits(stream_handle(dev), ptr(mask), rows, n, ptr(words)), "pack_allowed")
    return words


def history_from_pairs(rows, ids, count):
    """The ``history`` (offsets, ids) of ``count`` rows from (row, id) pairs in
    any order, such as the known answers of ``build_filter_indices_csr``;
    pairs whose row is outside [0, count) are left out."""
    _need_gpu("history_from_pairs", rows, ids)
    if rows.dim() != 1 or rows.shape != ids.shape:
        raise ValueError("history_from_pairs: rows and ids must be 1D and equally long")
    ids = _integers("history_from_pairs", "ids", ids)
    plan = group_rows(rows, max(int(count), 1))
    return plan.offsets[:int(count) + 1].long(), ids[plan.order.long()]


class _Constraints:
    """The checked arguments of one call."""

    __slots__ = ("rows", "cols", "inner", "allowed", "group", "bias", "history", "history_ptr", "scalars")

    def op(self, x, bias):
        a, h = self.allowed, self.history
        return FlLogits(x.data_ptr() if x is not None else None, self.rows, self.cols,
                        x.stride(0) if x is not None else 0, self.inner,
                        a.data_ptr() if a is not None else None, a.shape[0] if a is not None else 0,
                        a.stride(0) if a is not None else 0,
                        self.group.data_ptr() if self.group is not None else None,
                        bias.data_ptr() if bias is not None else None, bias.shape[0] if bias is not None else 0,
                        h.data_ptr() if h is not None else None,
                        self.history_ptr.data_ptr() if self.history_ptr is not None else None,
                        h.shape[-1] if h is not None else 0, *self.scalars)


def _spread(t, count):
    """One entry a coarse owner -> one a fine owner (count of them)."""
    return t if t.shape[0] == count else t.repeat_interleave(count // max(t.shape[0], 1), 0)


def _constraints(what, logits, allowed, group, bias, history, repetition, presence, frequency, temperature, fill):
    past, offsets = history, None
    if isinstance(history, (tuple, list)):
        if len(history) != 2:
            raise ValueError("%s: a ragged history is (offsets, ids)" % what)
        offsets, past = history
    _need_gpu(what, logits, allowed, group, bias, past, offsets)
    if logits.dtype not in _TYPES:
        raise TypeError("%s: logits must be float32, bfloat16 or float16" % what)
    if logits.dim() < 1:
        raise ValueError("%s: logits must be [..., columns]" % what)
    for name, v, least in (("repetition", repetition, 0.0), ("temperature", temperature, 0.0),
                           ("presence", presence, None), ("frequency", frequency, None)):
        if not math.isfinite(v) or (least is not None and not v > least):
            raise ValueError("%s: %s must be %s" % (what, name, "finite" if least is None else "positive"))
    lead, n = logits.shape[:-1], logits.shape[-1]
    c = _Constraints()
    c.rows, c.cols = math.prod(lead), n

    def owners_of(shape, name):
        if tuple(shape) != tuple(lead[:len(shape)]):
            raise ValueError("%s: %s is for rows %s, the logits have %s" % (what, name, list(shape), list(lead)))
        return math.prod(shape)

    counts = []
    if group is not None:
        counts.append(owners_of(group.shape, "group"))
        group = _integers(what, "group", group).reshape(-1)
    if past is not None:
        past = _integers(what, "history", past)
        if offsets is not None:
            if past.dim() != 1 or offsets.dim() != 1 or offsets.numel() < 1:
                raise ValueError("%s: a ragged history is 1D offsets and 1D ids" % what)
            offsets = _integers(what, "history", offsets)
            owners = offsets.numel() - 1
            if owners not in [math.prod(lead[:k]) for k in range(len(lead) + 1)]:
                raise ValueError("%s: history is for %d rows, the logits have %s" % (what, owners, list(lead)))
        else:
            if past.dim() < 1:
                raise ValueError("%s: history must be [..., ids]" % what)
            owners = owners_of(past.shape[:-1], "history")
            past = past.reshape(owners, past.shape[-1])
        counts.append(owners)
    owners = max(counts) if counts else c.rows
    if group is not None:
        group = _spread(group, owners)
    if past is not None and offsets is None:
        past = _spread(past, owners)
    elif past is not None and offsets.numel() - 1 != owners:
        raise ValueError("%s: a ragged history needs as many rows as group has" % what)
    c.inner = max(c.rows // owners, 1) if owners else 1
    if allowed is not None:
        if allowed.dtype == torch.bool:
            if allowed.shape[-1:] != (n,):
                raise ValueError("%s: allowed must be [..., %d]" % (what, n))
            allowed = pack_allowed(allowed)
        elif allowed.dtype != torch.int32:
            raise TypeError("%s: allowed must be a bool mask or pack_allowed's words" % what)
        if allowed.dim() not in (1, 2) or allowed.shape[-1] != (n + 31) // 32:
            raise ValueError("%s: allowed must be [%d words] or [groups, %d words]" % ((what,) + ((n + 31) // 32,) * 2))
        allowed = allowed.reshape(-1, allowed.shape[-1]).contiguous()
    if bias is not None:
        if bias.dtype not in _TYPES:
            raise TypeError("%s: bias must be float32, bfloat16 or float16" % what)
        if bias.dim() not in (1, 2) or bias.shape[-1] != n:
            raise ValueError("%s: bias must be [%d] or [groups, %d]" % (what, n, n))
        bias = bias.float().reshape(-1, n).contiguous()
    for name, t in (("allowed", allowed), ("bias", bias)):
        if t is not None and t.shape[0] != 1 and group is None:
            raise ValueError("%s: %s has %d rows; group says which of them a row takes" % (what, name, t.shape[0]))
    if allowed is not None and bias is not None and 1 not in (allowed.shape[0], bias.shape[0]) and \
            allowed.shape[0] != bias.shape[0]:
        raise ValueError("%s: allowed and bias have different numbers of groups" % what)
    if (allowed is not None and allowed.shape[0] == 0) or (bias is not None and bias.shape[0] == 0):
        raise ValueError("%s: a table without rows" % what)
    c.allowed, c.group, c.history, c.history_ptr = allowed, group, past, offsets
    c.scalars = (repetition, presence, frequency, temperature, fill, _TYPES[logits.dtype])
    return c, bias, _rows_of(logits, n)


def _logits_forward(c, x, bias, softmax):
    dev, lib = x.device, _lib.lib()
    out = torch.empty((c.rows, c.cols), dtype=torch.float32 if softmax else x.dtype, device=dev)
    op = c.op(x, bias)
    with _on(dev):
        st = stream_handle(dev)
        if softmax:
            nbytes = lib.fl_logits_softmax_bytes(op)
            ws = _workspace(nbytes, dev)
            check(lib.fl_logits_softmax(st, op, ptr(out), ptr(ws), nbytes), "hop_attention")
        else:
            check(lib.fl_logits_constrain(st, op, ptr(out)), "constrain_logits")
    return out


class _LogitsFunction(autograd.Function):
    @staticmethod
    def forward(ctx, x, bias, c, softmax):
        out = _logits_forward(c, x, bias, softmax)
        signs = c.history is not None and c.scalars[0] != 1.0  # the slopes go by the sign of x + bias
        ctx.save_for_backward(x if signs else None, bias, out if softmax else None, c.allowed, c.group, c.history,
                              c.history_ptr)
        ctx.c, ctx.softmax, ctx.x = c, softmax, (x.dtype, x.device)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, bias, w = ctx.saved_tensors[:3]
        c, (dtype, dev) = ctx.c, ctx.x
        lib = _lib.lib()
        grad = grad.contiguous()
        need_x, need_b = ctx.needs_input_grad[:2]
        dx = torch.empty((c.rows, c.cols), dtype=dtype, device=dev) if need_x else None
        db = torch.empty_like(bias) if need_b else None
        plan = group_rows(c.group, bias.shape[0]) if need_b and bias.shape[0] > 1 else None
        # without their signs the logits are not read: any row stands for them
        op = c.op(x if x is not None else grad, bias)
        with _on(dev):
            nbytes = lib.fl_logits_grad_bytes(op, int(ctx.softmax), int(need_b))
            ws = _workspace(nbytes, dev)
            check(lib.fl_logits_grad(stream_handle(dev), op, ptr(w), ptr(grad),
                                     ptr(plan.order) if plan is not None else None,
                                     ptr(plan.offsets) if plan is not None else None, ptr(dx), ptr(db), ptr(ws),
                                     nbytes), "hop_attention" if ctx.softmax else "constrain_logits")
        return dx, db, None, None


def _apply(logits, c, bias, x, softmax):
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        out = _LogitsFunction.apply(x, bias, c, softmax)
    else:
        out = _logits_forward(c, x, bias, softmax)
    return out.view(logits.shape)


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
    first dimensions (a query's steps then share it); a group outside the
    tables has nothing allowed.  history: ids [..., h] for the logits' leading
    shape or its first dimensions, padded with ids outside [0, n), or
    (offsets, ids) with the ids offsets[i] .. offsets[i+1] of row i.

    Masked logits are not read into anything: they may be infinite or NaN.
    Gradients reach logits and bias; masked columns have none."""
    return _apply(logits, *_constraints("constrain_logits", logits, allowed, group, bias, history, float(repetition),
                                        float(presence), float(frequency), float(temperature), float(fill)),
                  softmax=False)


def hop_attention(logits, allowed=None, group=None, bias=None, history=None, repetition=1.0, presence=0.0,
                  frequency=0.0, temperature=1.0):
    """A hop's attention: the softmax of ``constrain_logits`` over the allowed
    columns, float32 [..., n], with the same arguments.  Masked columns are
    exactly 0; a row with nothing left (no column allowed, or every allowed
    logit -inf) is all zeros and has no gradient."""
    return _apply(logits, *_constraints("hop_attention", logits, allowed, group, bias, history, float(repetition),
                                        float(presence), float(frequency), float(temperature), 0.0), softmax=True)

"""The operators between a rule generator's hidden states, the hops and the answers, as measurable cases.

A case is a dict of plain values.  Its ``op`` says which public entry point one pass goes through:

  linear     rows [rows, inner] times weights [outer, inner], with bias, activation and residual in the same
             pass: a generator's layers, and the head that makes relation logits of its hidden states;
  grouped    the same with weights of its own for every head relation: the rows are grouped by their relation,
             then multiplied group by group;
  constrain  masks, biases and penalties for repeated ids on score rows: answers of a query batch under type
             constraints, entity priors and known answers;
  attention  the same on relation logits, with the softmax over what is allowed: the attention that a hop takes.

``train`` cases also return the gradients of everything a training step needs them for.  Sizes are those of the
repository's benchmark configurations (25 to 1645 relation operators, 3,000 to 4.6M entities, batches of 32 to 512
queries, 3 hops, 3 channels) or generic layer widths.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def _linear(rows, inner, outer, dtype="fp32", act="none", bias=True, residual=False, train=False):
    return dict(op="linear", rows=rows, inner=inner, outer=outer, dtype=dtype, act=act, bias=bias, residual=residual,
                train=train)


def _grouped(rows, groups, inner, outer, dtype="fp32", act="none", bias=True, residual=False, train=False, law=0.0):
    return dict(op="grouped", rows=rows, groups=groups, inner=inner, outer=outer, dtype=dtype, act=act, bias=bias,
                residual=residual, train=train, law=law)


def _constrain(rows, cols, groups=1, dtype="fp32", allow=0.5, known=0, bias="none", train=False):
    return dict(op="constrain", rows=rows, cols=cols, groups=groups, dtype=dtype, allow=allow, known=known, bias=bias,
                train=train)


def _attention(queries, steps, cols, groups=1, dtype="fp32", allow=0.5, past=0, bias="none", train=False, empty=False):
    return dict(op="attention", queries=queries, steps=steps, cols=cols, groups=groups, dtype=dtype, allow=allow,
                past=past, bias=bias, train=train, empty=empty)


def listed():
    def named(name, case):
        return dict(case, name=name)

    return [
        # relation logits of an evaluation batch: 32 queries x 3 hops, 475 relation operators
        named("head eval relational", _linear(96, 256, 475)),
        # the same head in a web-scale training step: 512 queries (256 and their inverses) x 3 hops, 1645 operators
        named("head web train", _linear(1536, 2048, 1645, train=True)),
        # a wide generator layer over many rows in half precision: the products' own rate
        named("layer bf16", _linear(8192, 2048, 2048, "bf16", "gelu", residual=True)),
        # the same kind of layer in training
        named("layer fp16 train", _linear(16384, 2048, 2048, "fp16", "silu", residual=True, train=True)),
        # per-relation heads of an evaluation batch: few rows, many relations, so mostly groups of one row
        named("relation heads eval", _grouped(96, 474, 128, 475, law=1.0)),
        # per-relation heads in training over the query batches of a ranking run, uniform relations
        named("relation heads train", _grouped(15000, 74, 128, 75, act="tanh", train=True)),
        # per-relation layers in half precision with skewed relations
        named("relation layers bf16 train", _grouped(16384, 24, 1024, 2048, "bf16", "gelu", train=True, law=0.5)),
        # the answers of an evaluation batch under type constraints, the known ones penalised
        named("answers medium", _constrain(32, 41_000, 22, known=40)),
        # the same over a web-scale graph's entities with an entity prior
        named("answers web", _constrain(32, 4_600_000, 64, allow=0.3, known=60, bias="row")),
        # scores in training: half precision, a trained prior for every query relation's entities
        named("scores large train", _constrain(509, 123_000, 74, "bf16", known=20, bias="table", train=True)),
        # attention of a handful of queries on a small graph: launches count
        named("attention small", _attention(32, 3, 25, 24, past=2, empty=True)),
        # attention of a web-scale training step: every query's 3 hops x 3 channels in one call
        named("attention web train", _attention(512, 9, 1645, 1644, past=2, bias="table", train=True)),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    op = rng.choice(["linear", "linear", "grouped", "grouped", "constrain", "attention"])
    dtype = rng.choice(["fp32", "fp32", "bf16", "fp16"])
    train = rng.random() < 0.5
    act = rng.choice(["none", "relu", "gelu", "silu", "tanh", "sigmoid"])
    if op == "linear":
        return _linear(_log_int(rng, 1, 16384), _log_int(rng, 64, 2048), _log_int(rng, 25, 2048), dtype, act,
                       rng.random() < 0.8, rng.random() < 0.3, train)
    if op == "grouped":
        groups = _log_int(rng, 2, 474)
        inner, outer = _log_int(rng, 64, 1024), _log_int(rng, 25, 1645)
        while groups * inner * outer > 60_000_000:
            groups = max(2, groups // 2)
        rows = _log_int(rng, 16, 16384)
        law = rng.choice([0.0, 0.5]) if rows * max(inner, outer) > 2_000_000 else rng.choice([0.0, 1.0])
        return _grouped(rows, groups, inner, outer, dtype, act, rng.random() < 0.8, rng.random() < 0.3, train, law)
    if op == "constrain":
        cols = _log_int(rng, 3_000, 4_600_000)
        rows = _log_int(rng, 1, max(2, min(512, 60_000_000 // cols)))
        groups = rng.randint(2, 74) if cols < 200_000 else rng.randint(1, 8)
        return _constrain(rows, cols, groups, dtype, rng.choice([0.02, 0.3, 0.9]), rng.choice([0, 5, 60]),
                          rng.choice(["none", "row", "table"] if cols < 200_000 else ["none", "row"]), train)
    cols = _log_int(rng, 25, 1645)
    return _attention(_log_int(rng, 1, 1024), rng.randint(1, 9), cols, rng.randint(2, 2 * cols), dtype,
                      rng.choice([0.05, 0.5, 1.0]), rng.randint(0, 3), rng.choice(["none", "row", "table"]), train,
                      rng.random() < 0.3)


# ---------------------------------------------------------------------------
# Inputs


def _words(mask):
    """One bit per column, 32 columns a word, column 32 w + j in bit j of word w: how a program keeps a mask table."""
    pad = (-mask.shape[1]) % 32
    m = torch.nn.functional.pad(mask, (0, pad)).view(mask.shape[0], -1, 32).long()
    w = (m << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _draw_index(rows, groups, law, g):
    p = torch.arange(1, groups + 1, device=DEV, dtype=torch.float64) ** -law
    p = p[torch.randperm(groups, generator=g, device=DEV)]
    return torch.searchsorted(torch.cumsum(p / p.sum(), 0), torch.rand(rows, generator=g, device=DEV,
                                                                       dtype=torch.float64)).clamp_(max=groups - 1)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    s = dict(case=case)
    if case["op"] in ("linear", "grouped"):
        M, K, N = case["rows"], case["inner"], case["outer"]
        G = (case["groups"],) if case["op"] == "grouped" else ()
        s["x"] = torch.tanh(normal(M, K)).to(t)  # hidden states of a recurrent generator
        s["weight"] = (normal(*G, N, K) / math.sqrt(K)).to(t)
        s["bias"] = (0.1 * normal(*G, N)).to(t) if case["bias"] else None
        s["residual"] = normal(M, N).to(t) if case["residual"] else None
        s["grad"] = (normal(M, N) / M * 16).to(t) if case["train"] else None  # a loss averages over its rows
        if G:
            s["index"] = _draw_index(M, G[0], case["law"], g)
            s["most"] = int(torch.bincount(s["index"], minlength=G[0]).max())
    else:
        n, G = case["cols"], case["groups"]
        if case["op"] == "constrain":
            owners, shape = case["rows"], (case["rows"], n)
            # popularity-like scores: a few large, most small
            x = torch.exp(1.5 * normal(*shape))
        else:
            owners, shape = case["queries"], (case["queries"], case["steps"], n)
            x = 2.0 * normal(*shape)
        s["logits"] = x.to(t)
        del x
        s["group"] = torch.randint(G, (owners,), generator=g, device=DEV)
        mask = torch.rand(G, n, generator=g, device=DEV) < case["allow"]
        if case["op"] == "attention":
            mask[:, -1] = True  # the identity operator stays
            if case["empty"]:
                mask[0] = False
        s["mask"], s["words"] = mask, _words(mask)
        b = case["bias"]
        s["bias"] = None if b == "none" else 0.5 * normal(n) if b == "row" else 0.5 * normal(G, n)
        s["history"] = None
        if case["op"] == "attention" and case["past"]:  # the operators taken in earlier hops, padded
            h = torch.randint(n, (owners, case["past"]), generator=g, device=DEV)
            s["history"] = torch.where(torch.rand(h.shape, generator=g, device=DEV) < 0.2, -1, h)
        if case["op"] == "constrain" and case["known"]:  # the known answers of every query, ragged
            count = torch.randint(2 * case["known"] + 1, (owners,), generator=g, device=DEV)
            off = torch.zeros(owners + 1, dtype=torch.int64, device=DEV)
            off[1:] = torch.cumsum(count, 0)
            total = int(off[-1])
            s["history"] = (off, torch.randint(n, (total,), generator=g, device=DEV))
        s["grad"] = normal(*shape).to(t if case["op"] == "constrain" else torch.float32) if case["train"] else None
    return s


PENALTY = dict(repetition=1.5, presence=0.25, frequency=0.125, temperature=0.75)


# ---------------------------------------------------------------------------
# The operators' plain forms


def _act(p, act):
    if act == "relu":
        return torch.where(p > 0, p, torch.zeros_like(p))
    if act == "gelu":
        return 0.5 * p * (1.0 + torch.erf(p * math.sqrt(0.5)))
    if act == "silu":
        return p / (1.0 + torch.exp(-p))
    if act == "tanh":
        return torch.tanh(p)
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-p))
    return p


def _slope(p, act):
    if act == "relu":
        return (p > 0).to(p.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(p * math.sqrt(0.5))) + p * torch.exp(-0.5 * p * p) / math.sqrt(2.0 * math.pi)
    if act == "silu":
        q = 1.0 / (1.0 + torch.exp(-p))
        return q * (1.0 + p * (1.0 - q))
    if act == "tanh":
        return 1.0 - torch.tanh(p) ** 2
    if act == "sigmoid":
        q = 1.0 / (1.0 + torch.exp(-p))
        return q * (1.0 - q)
    return torch.ones_like(p)


def _plain_linear(s):
    c = s["case"]
    t = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    p = x @ w.t()
    if s["bias"] is not None:
        p = p + s["bias"].float()
    y = _act(p, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(t)}
    if c["train"]:
        d = s["grad"].float() * _slope(p, c["act"])
        out["dx"], out["dweight"] = (d @ w).to(t), (d.t() @ x).to(t)
        if s["bias"] is not None:
            out["dbias"] = d.sum(0).to(t)
        if s["residual"] is not None:
            out["dresidual"] = s["grad"]
    return out


def _plain_grouped(s):
    c = s["case"]
    t = s["x"].dtype
    x, w, index = s["x"].float(), s["weight"].float(), s["index"]
    M, G, most = x.shape[0], c["groups"], s["most"]
    if M <= G and not c["train"]:  # fewer rows than weights: a copy of the weights for every row
        p = torch.bmm(w[index], x[:, :, None])[:, :, 0]
    else:  # every group padded to the largest one
        order = torch.argsort(index, stable=True)
        count = torch.zeros(G, dtype=torch.int64, device=x.device).index_add_(0, index, torch.ones_like(index))
        sorted_index = index[order]
        place = sorted_index * most + torch.arange(M, device=x.device) - (torch.cumsum(count, 0) - count)[sorted_index]
        xp = torch.zeros(G * most, c["inner"], device=x.device)
        xp[place] = x[order]
        xp = xp.view(G, most, c["inner"])
        yp = torch.bmm(xp, w.transpose(1, 2).contiguous()).view(G * most, c["outer"])
        p = torch.empty(M, c["outer"], device=x.device)
        p[order] = yp[place]
    if s["bias"] is not None:
        p = p + s["bias"].float()[index]
    y = _act(p, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(t)}
    if c["train"]:
        d = s["grad"].float() * _slope(p, c["act"])
        dp = torch.zeros(G * most, c["outer"], device=x.device)
        dp[place] = d[order]
        dp = dp.view(G, most, c["outer"])
        dx = torch.empty_like(x)
        dx[order] = torch.bmm(dp, w).view(G * most, c["inner"])[place]
        out["dx"], out["dweight"] = dx.to(t), torch.bmm(dp.transpose(1, 2).contiguous(), xp).to(t)
        if s["bias"] is not None:
            out["dbias"] = dp.sum(1).to(t)
        if s["residual"] is not None:
            out["dresidual"] = s["grad"]
    return out


def _per_row(s, table):
    """The rows' entries of a table that has one row, or one for every group."""
    x = s["logits"]
    if table.dim() == 1 or table.shape[0] == 1:
        return table.reshape(-1)
    rows = table[s["group"]]
    return rows if x.dim() == 2 else rows[:, None]


def _repeats(s):
    """How often each column is in its row's history, or None."""
    h, n = s["history"], s["case"]["cols"]
    if h is None:
        return None
    owners = s["logits"].shape[0]
    if isinstance(h, tuple):
        row = torch.repeat_interleave(torch.arange(owners, device=DEV), h[0][1:] - h[0][:-1], output_size=h[1].numel())
        count = torch.zeros(owners * n, device=DEV)
        return count.index_add_(0, row * n + h[1], torch.ones(h[1].numel(), device=DEV)).view(owners, n)
    count = torch.zeros(owners, n + 1, device=DEV)
    count.scatter_add_(1, torch.where(h < 0, n, h), torch.ones(h.shape, device=DEV))
    return count[:, None, :n]


def _plain_constrained(s):
    """(constrained values, allowed, slope of them in the logits), in 32 bits."""
    v = s["logits"].float()
    if s["bias"] is not None:
        v = v + _per_row(s, s["bias"])
    allowed = _per_row(s, s["mask"])
    tau, rho = PENALTY["temperature"], PENALTY["repetition"]
    count = _repeats(s)
    slope = torch.full((), 1.0 / tau, device=DEV)
    if count is not None:
        up = v > 0
        seen = count > 0
        slope = torch.where(seen, torch.where(up, 1.0 / rho, rho) / tau, slope)
        v = torch.where(seen, torch.where(up, v / rho, v * rho), v)
        v = v - (PENALTY["presence"] * seen.float() + PENALTY["frequency"] * count)
    return torch.where(allowed, v / tau, -math.inf), allowed, slope


def _bias_gradient(s, d):
    if s["bias"].dim() == 1:
        return d.sum(tuple(range(d.dim() - 1)))
    d = d if d.dim() == 2 else d.sum(1)
    return torch.zeros_like(s["bias"]).index_add_(0, s["group"], d)


def _plain_constrain(s):
    t = s["logits"].dtype
    v, allowed, slope = _plain_constrained(s)
    out = {"scores": v.to(t)}
    if s["grad"] is not None:
        d = torch.where(allowed, s["grad"].float() * slope, 0.0)
        out["dlogits"] = d.to(t)
        if s["bias"] is not None:
            out["dbias"] = _bias_gradient(s, d)
    return out


def _plain_attention(s):
    t = s["logits"].dtype
    v, allowed, slope = _plain_constrained(s)
    top = v.amax(-1, keepdim=True)
    e = torch.where(allowed, torch.exp(v - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = e.sum(-1, keepdim=True)
    w = e / torch.where(total == 0, 1.0, total)
    out = {"w": w}
    if s["grad"] is not None:
        d = w * (s["grad"] - (w * s["grad"]).sum(-1, keepdim=True)) * slope
        out["dlogits"] = d.to(t)
        if s["bias"] is not None:
            out["dbias"] = _bias_gradient(s, d)
    return out


PLAIN = {"linear": _plain_linear, "grouped": _plain_grouped, "constrain": _plain_constrain,
         "attention": _plain_attention}


# ---------------------------------------------------------------------------
# The framework's calls


def _own_products(s):
    from flashlog_amd import attention as fa
    c = s["case"]
    leaves = {k: s[k] for k in ("x", "weight", "bias", "residual") if s[k] is not None}
    if c["train"]:
        leaves = {k: v.detach().requires_grad_(True) for k, v in leaves.items()}
    act = None if c["act"] == "none" else c["act"]
    if c["op"] == "linear":
        y = fa.linear(leaves["x"], leaves["weight"], leaves.get("bias"), act, leaves.get("residual"))
    else:
        groups = fa.group_rows(s["index"], c["groups"])
        y = fa.relation_linear(leaves["x"], groups, leaves["weight"], leaves.get("bias"), act, leaves.get("residual"))
    out = {"y": y.detach()}
    if c["train"]:
        grads = torch.autograd.grad(y, list(leaves.values()), s["grad"])
        out.update({"d" + k: g for k, g in zip(leaves, grads)})
    return out


def _own_logits(s):
    from flashlog_amd import attention as fa
    c = s["case"]
    leaves = {k: s[k] for k in ("logits", "bias") if s[k] is not None}
    if c["train"]:
        leaves = {k: v.detach().requires_grad_(True) for k, v in leaves.items()}
    fn, name = (fa.constrain_logits, "scores") if c["op"] == "constrain" else (fa.hop_attention, "w")
    y = fn(leaves["logits"], allowed=s["words"], group=s["group"], bias=leaves.get("bias"), history=s["history"],
           **PENALTY)
    out = {name: y.detach()}
    if c["train"]:
        grads = torch.autograd.grad(y, list(leaves.values()), s["grad"])
        out.update({"d" + k: g for k, g in zip(leaves, grads)})
    return out


OWN = {"linear": _own_products, "grouped": _own_products, "constrain": _own_logits, "attention": _own_logits}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] in ("linear", "grouped"):
        M, K, N = case["rows"], case["inner"], case["outer"]
        G = min(case.get("groups", 1), M)
        weights, rows = G * N * (K + int(case["bias"])), M * (K + N * (1 + int(case["residual"])))
        moved = weights + rows
        if case["train"]:  # the output's gradient in, the operands' gradients out
            moved += M * N * (1 + int(case["residual"])) + M * K + case.get("groups", 1) * N * (K + int(case["bias"]))
        moved = moved * size + (8 * M if case["op"] == "grouped" else 0)
        return {"bytes": moved, "flops": 2 * M * K * N * (3 if case["train"] else 1)}
    n, G = case["cols"], case["groups"]
    if case["op"] == "constrain":
        owners = rows = case["rows"]
        ids, out = owners * case["known"], size
    else:
        owners, rows = case["queries"], case["queries"] * case["steps"]
        ids, out = owners * case["past"], 4
    G = min(G, owners)
    bias = 0 if case["bias"] == "none" else 4 * n * (1 if case["bias"] == "row" else G)
    moved = rows * n * (size + out) + G * n // 8 + bias + 8 * ids + 8 * owners
    flops = rows * n * (8 if case["op"] == "constrain" else 12)
    if case["train"]:
        whole = 0 if case["bias"] == "none" else 4 * n * (1 if case["bias"] == "row" else case["groups"])
        moved += rows * n * (out + size) + whole
        flops += rows * n * 6
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------
# The definitions in 64 bits


def _exact_act(p, act):
    """(value, derivative) of the activation."""
    one = torch.ones_like(p)
    if act == "relu":
        return p.clamp(min=0), torch.heaviside(p, torch.zeros_like(p))
    if act == "gelu":
        cdf = torch.special.ndtr(p)
        return p * cdf, cdf + p * torch.exp(-p.square() / 2) * (2 * math.pi) ** -0.5
    if act == "silu":
        q = torch.special.expit(p)
        return p * q, q * (one + p - p * q)
    if act == "tanh":
        y = torch.sinh(p) / torch.cosh(p)
        return y, one / torch.cosh(p).square()
    if act == "sigmoid":
        q = torch.special.expit(p)
        return q, q * torch.special.expit(-p)
    return p, one


def _exact_products(case, s):
    x, w = s["x"].double(), s["weight"].double()
    M, N = x.shape[0], case["outer"]
    b = s["bias"].double() if s["bias"] is not None else None
    parts = [(slice(None), w, b)]
    if case["op"] == "grouped":
        parts = [((s["index"] == k).nonzero()[:, 0], w[k], None if b is None else b[k]) for k in range(case["groups"])]
    y = torch.empty(M, N, dtype=torch.float64, device=DEV)
    out = {"y": y}
    if case["train"]:
        g = s["grad"].double()
        out["dx"] = torch.empty_like(x)
        dw, db = [], []
    for rows, wk, bk in parts:
        xr = x[rows]
        value, slope = _exact_act(torch.matmul(xr, wk.T) + (0 if bk is None else bk), case["act"])
        y[rows] = value + (0 if s["residual"] is None else s["residual"][rows].double())
        if case["train"]:
            d = g[rows] * slope
            out["dx"][rows] = torch.matmul(d, wk)
            dw.append(torch.matmul(d.T, xr))
            db.append(d.sum(0))
    if case["train"]:
        grouped = case["op"] == "grouped"
        out["dweight"] = torch.stack(dw) if grouped else dw[0]
        if b is not None:
            out["dbias"] = torch.stack(db) if grouped else db[0]
        if s["residual"] is not None:
            out["dresidual"] = g
    return out


def _exact_logits(case, s):
    n, owners = case["cols"], s["logits"].shape[0]
    rho, tau = PENALTY["repetition"], PENALTY["temperature"]
    y, grad_in, weights = [], [], []
    db = None
    if s["bias"] is not None:
        db = torch.zeros_like(s["bias"], dtype=torch.float64).reshape(-1, n)
    for o in range(owners):  # one query at a time
        k = int(s["group"][o])
        x = s["logits"][o].reshape(-1, n).double()
        kb = 0 if db is not None and db.shape[0] == 1 else k
        if db is not None:
            x = x + s["bias"].reshape(-1, n)[kb].double()
        seen = torch.zeros(n, dtype=torch.float64, device=DEV)
        if isinstance(s["history"], tuple):
            ids = s["history"][1][int(s["history"][0][o]):int(s["history"][0][o + 1])]
        else:
            ids = s["history"][o] if s["history"] is not None else seen.new_empty(0).long()
        ids, times = torch.unique(ids[ids >= 0], return_counts=True)
        seen[ids] = times.double()
        factor = torch.where(x > 0, 1 / rho, rho)
        factor = torch.where(seen > 0, factor, torch.ones_like(factor))
        v = (x * factor - (PENALTY["presence"] * (seen > 0) + PENALTY["frequency"] * seen)) / tau
        off = ~s["mask"][k]
        v = v.masked_fill(off, -math.inf)
        if case["op"] == "attention":
            w = torch.zeros_like(v) if bool(off.all()) else torch.softmax(v, -1)
            y.append(w)
            if case["train"]:
                g = s["grad"][o].reshape(-1, n).double()
                d = (w * g - w * (w * g).sum(-1, keepdim=True)) * factor / tau
        else:
            y.append(v)
            if case["train"]:
                d = (s["grad"][o].reshape(-1, n).double() * factor / tau).masked_fill(off, 0)
        if case["train"]:
            grad_in.append(d)
            if db is not None:
                db[kb] += d.sum(0)
    shape = s["logits"].shape
    out = {"scores" if case["op"] == "constrain" else "w": torch.stack(y).view(shape)}
    if case["train"]:
        out["dlogits"] = torch.stack(grad_in).view(shape)
        if db is not None:
            out["dbias"] = db.view(s["bias"].shape)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return (_exact_products if case["op"] in ("linear", "grouped") else _exact_logits)(case, s)

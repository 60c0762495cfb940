"""The operators that train what makes relation logits and entity scores, as measurable cases.

A case is a dict of plain values.  Its ``op`` says which public entry point one pass goes through:

  norm      layer normalisation of a generator's hidden states;
  entropy   softmax cross entropy of hidden states [rows, inner] over a vocabulary of relations or entities with
            embeddings [cols, inner], one target a row, the logits not kept;
  listed    the same product against a teacher's top answers: ids and teacher logits [rows, top];
  scores    distillation from a teacher's top answers on score rows [rows, cols] that a program has already, -inf where
            a constraint masks them.

``train`` cases also return the gradients of everything a training step needs them for.  Sizes are those of the
repository's benchmark configurations (25 to 1645 relation operators, 3,000 to 4.6M entities, batches of 32 to 512
queries, 3 hops) or generic layer widths.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-5


def _norm(rows, cols, dtype="fp32", wide=False, train=False):
    return dict(op="norm", rows=rows, cols=cols, dtype=dtype, wide=wide, train=train)


def _entropy(rows, inner, cols, dtype="fp32", bias=False, idle=0.0, train=False):
    return dict(op="entropy", rows=rows, inner=inner, cols=cols, dtype=dtype, bias=bias, idle=idle, train=train)


def _listed(rows, inner, cols, top, dtype="fp32", bias=False, tau=1.0, train=False):
    return dict(op="listed", rows=rows, inner=inner, cols=cols, top=top, dtype=dtype, bias=bias, tau=tau, train=train)


def _scores(rows, cols, top, dtype="fp32", allow=1.0, tau=1.0, train=False):
    return dict(op="scores", rows=rows, cols=cols, top=top, dtype=dtype, allow=allow, tau=tau, train=train)


def listed():
    def named(name, case):
        return dict(case, name=name)

    return [
        # hidden states of an evaluation batch, 32 queries x 3 hops: launches count
        named("norm eval", _norm(96, 256)),
        # a web-scale training step: 512 queries (256 and their inverses) x 3 hops
        named("norm web train", _norm(1536, 2048, train=True)),
        # a wide layer over many rows in half precision, its gain and shift kept in 32 bits
        named("norm bf16 train", _norm(16384, 2048, "bf16", wide=True, train=True)),
        # how well an evaluation batch predicts the next relation of a rule body
        named("relation loss eval", _entropy(96, 256, 475, bias=True)),
        # relations of rule bodies as targets in a web-scale training step
        named("relation loss web train", _entropy(1536, 2048, 1645, bias=True, train=True)),
        # entities as targets of many queries, a tenth of the batch padding
        named("entity loss bf16 train", _entropy(8192, 512, 41_000, "bf16", idle=0.1, train=True)),
        # entities of a web-scale graph as targets of one batch
        named("entity loss web train", _entropy(512, 128, 4_600_000, "bf16", train=True)),
        # a small batch learns from the answers of a rule model
        named("entity list train", _listed(128, 256, 41_000, 20, bias=True, tau=2.0, train=True)),
        # many queries learn from a larger model's top answers
        named("entity list fp16 train", _listed(4096, 1024, 123_000, 64, "fp16", tau=2.0, train=True)),
        # how near an evaluation batch's scores are to a teacher's
        named("scores list eval", _scores(32, 41_000, 20)),
        # propagated scores under type constraints in training, half precision
        named("scores list large train", _scores(509, 123_000, 64, "bf16", allow=0.5, tau=2.0, train=True)),
        # the same over a web-scale graph's entities
        named("scores list web train", _scores(32, 4_600_000, 64, allow=0.3, train=True)),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    op = rng.choice(["norm", "entropy", "entropy", "listed", "scores"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    train = rng.random() < 0.6
    if op == "norm":
        return _norm(_log_int(rng, 1, 16384), _log_int(rng, 25, 8192), dtype, rng.random() < 0.5, train)
    tau = rng.choice([1.0, 2.0, 0.5])
    top = _log_int(rng, 1, 100)
    if op == "scores":
        cols = _log_int(rng, 475, 4_600_000)
        rows = _log_int(rng, 1, max(2, min(4096, 60_000_000 // cols)))
        return _scores(rows, cols, top, dtype, rng.choice([0.05, 0.3, 1.0]), tau, train)
    inner, cols = _log_int(rng, 64, 2048), _log_int(rng, 25, 4_600_000)
    if rng.random() < 0.5:  # as widths mostly are
        inner -= inner % 8
    while inner * cols > 600_000_000:
        cols //= 2
    most = min(8192, 2_000_000_000 // cols, 400_000_000_000 // (cols * inner))
    rows = _log_int(rng, 1, max(2, most // (4 if dtype == "fp32" else 1)))
    if op == "entropy":
        return _entropy(rows, inner, cols, dtype, rng.random() < 0.5, rng.choice([0.0, 0.1, 0.5]), train)
    return _listed(rows, inner, cols, top, dtype, rng.random() < 0.5, tau, train)


# ---------------------------------------------------------------------------
# Inputs


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[case["dtype"]]
    M, n = case["rows"], case["cols"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    s = dict(case=case)
    if case["op"] == "norm":
        # what residual layers add up to: columns of different sizes, rows off 0
        s["x"] = (normal(M, n) * torch.exp(0.5 * normal(n)) + 0.3 * normal(M, 1)).to(t)
        wt = torch.float32 if case["wide"] else t
        s["weight"], s["bias"] = (1.0 + 0.2 * normal(n)).to(wt), (0.1 * normal(n)).to(wt)
        s["grad"] = (normal(M, n) * (16 / M)).to(t) if case["train"] else None
        return s
    if case["op"] == "scores":
        x = 2.0 * normal(M, n)
        if case["allow"] < 1.0:
            x = x.masked_fill_(uniform(M, n) >= case["allow"], -math.inf)
        s["logits"] = x.to(t)
        del x
    else:
        K = case["inner"]
        s["x"] = normal(M, K).to(t)  # normalised hidden states
        s["weight"] = torch.empty(n, K, dtype=t, device=DEV)
        for part in s["weight"].split(1 << 20):
            part.copy_(normal(*part.shape) * (2.5 / math.sqrt(K)))
        s["bias"] = normal(n).to(t) if case["bias"] else None
    if case["op"] == "entropy":
        target = (n * uniform(M) ** 2).long().clamp_(max=n - 1)  # some entities far more often than others
        s["target"] = torch.where(uniform(M) < case["idle"], -1, target)
    else:
        k = case["top"]
        ids = torch.randint(n, (M, k), generator=g, device=DEV)
        length = torch.where(uniform(M) < 0.2, (uniform(M) * k).long(), k)  # shorter lists are padded
        s["ids"] = torch.where(torch.arange(k, device=DEV) < length[:, None], ids, -1)
        s["teacher"] = (3.0 * normal(M, k)).sort(-1, descending=True)[0]
    s["grad"] = (0.5 + uniform(M)) / M if case["train"] else None  # a weighted mean of the rows' losses
    return s


# ---------------------------------------------------------------------------
# The operators' plain forms


def _plain_norm(s):
    t = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    n = x.shape[1]
    mean = x.sum(1, keepdim=True) / n
    c = x - mean
    r = 1.0 / torch.sqrt((c * c).sum(1, keepdim=True) / n + EPS)
    h = c * r
    out = {"y": (h * w + s["bias"].float()).to(t)}
    if s["grad"] is not None:
        g = s["grad"].float()
        gw = g * w
        out["dx"] = (r * (gw - gw.sum(1, keepdim=True) / n - h * ((gw * h).sum(1, keepdim=True) / n))).to(t)
        out["dweight"], out["dbias"] = (g * h).sum(0).to(s["weight"].dtype), g.sum(0).to(s["bias"].dtype)
    return out


def _log_sum(u):
    """(log of the sum of exp of every row, exp(u - it))."""
    top = u.amax(1, keepdim=True)
    e = torch.exp(u - top)
    total = e.sum(1, keepdim=True)
    return (top + torch.log(total))[:, 0], e.div_(total)


def _plain_logits(s):
    z = s["x"].float() @ s["weight"].float().t()
    return z if s["bias"] is None else z.add_(s["bias"].float())


def _product_gradients(s, d):
    t = s["x"].dtype
    out = {"dx": (d @ s["weight"].float()).to(t), "dweight": (d.t() @ s["x"].float()).to(t)}
    if s["bias"] is not None:
        out["dbias"] = d.sum(0).to(t)
    return out


def _plain_entropy(s):
    z, target = _plain_logits(s), s["target"]
    live = target >= 0
    at = torch.where(live, target, 0)
    zt = z.gather(1, at[:, None])[:, 0]
    lse, p = _log_sum(z)
    out = {"loss": torch.where(live, lse - zt, 0.0)}
    if s["grad"] is not None:
        p.scatter_add_(1, at[:, None], torch.full_like(zt, -1.0)[:, None])
        out.update(_product_gradients(s, p.mul_(torch.where(live, s["grad"], 0.0)[:, None])))
    return out


def _plain_list(s, z):
    """(losses, their gradient in z) of logits in 32 bits."""
    tau, ids = s["case"]["tau"], s["ids"]
    u = z / tau
    at = ids.clamp(min=0)
    ut = u.gather(1, at)
    valid = (ids >= 0) & (ut > -math.inf)
    live = valid.any(1)
    v = torch.where(valid, s["teacher"].float() / tau, -math.inf)
    top = torch.where(live, v.amax(1), 0.0)[:, None]
    e = torch.exp(v - top)
    total = torch.where(live, e.sum(1), 1.0)[:, None]
    q = e / total
    lse, p = _log_sum(u)
    apart = torch.where(valid, (v - top - torch.log(total)) - (ut - lse[:, None]), 0.0)
    loss = torch.where(live, tau * tau * (q * apart).sum(1), 0.0)
    if s["grad"] is None:
        return loss, None
    p.scatter_add_(1, at, -q)
    return loss, p.mul_(torch.where(live, tau * s["grad"], 0.0)[:, None])


def _plain_listed(s):
    loss, d = _plain_list(s, _plain_logits(s))
    return {"loss": loss} if d is None else {"loss": loss, **_product_gradients(s, d)}


def _plain_scores(s):
    loss, d = _plain_list(s, s["logits"].float())
    return {"loss": loss} if d is None else {"loss": loss, "dlogits": d.to(s["logits"].dtype)}


PLAIN = {"norm": _plain_norm, "entropy": _plain_entropy, "listed": _plain_listed, "scores": _plain_scores}


# ---------------------------------------------------------------------------
# The framework's calls


def _own(s):
    from flashlog_amd import attention, losses
    c = s["case"]
    names = {"norm": ("x", "weight", "bias"), "scores": ("logits",)}.get(c["op"], ("x", "weight", "bias"))
    leaves = {k: s[k] for k in names if s[k] is not None}
    if c["train"]:
        leaves = {k: v.detach().requires_grad_(True) for k, v in leaves.items()}
    if c["op"] == "norm":
        y = attention.layer_norm(leaves["x"], leaves["weight"], leaves["bias"], EPS)
    elif c["op"] == "entropy":
        y = losses.linear_cross_entropy(leaves["x"], leaves["weight"], s["target"], leaves.get("bias"))
    elif c["op"] == "listed":
        y = losses.linear_distillation(leaves["x"], leaves["weight"], s["ids"], s["teacher"], leaves.get("bias"),
                                       temperature=c["tau"])
    else:
        y = losses.distillation(leaves["logits"], s["ids"], s["teacher"], temperature=c["tau"])
    out = {"y" if c["op"] == "norm" else "loss": y.detach()}
    if c["train"]:
        grads = torch.autograd.grad(y, list(leaves.values()), s["grad"])
        out.update({"d" + k: g for k, g in zip(leaves, grads)})
    return out


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without


def work(case):
    size, M, n, train = SIZE[case["dtype"]], case["rows"], case["cols"], case["train"]
    if case["op"] == "norm":
        ws = 4 if case["wide"] else size
        return {"bytes": M * n * size * (4 if train else 2) + 2 * n * ws * (2 if train else 1),
                "flops": M * n * (20 if train else 8)}
    lists = 8 * M if case["op"] == "entropy" else 12 * M * case["top"]
    ends = 4 * M * (2 if train else 1)  # losses, their gradients
    if case["op"] == "scores":
        return {"bytes": M * n * size * (2 if train else 1) + lists + ends, "flops": M * n * (8 if train else 5)}
    K = case["inner"]
    operands = (M * K + n * K + n * int(case["bias"])) * size
    return {"bytes": operands * (2 if train else 1) + lists + ends, "flops": 2 * M * K * n * (3 if train else 1)}


# ---------------------------------------------------------------------------
# The definitions in 64 bits


def _exact_norm(s):
    x, w, b = (s[k].double() for k in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    scale = (var + EPS).rsqrt()
    h = (x - mean) * scale
    out = {"y": torch.addcmul(b, h, w)}
    if s["grad"] is not None:
        g = s["grad"].double()
        d = g * w
        out["dx"] = scale * (d - d.mean(1, keepdim=True) - h * (d * h).mean(1, keepdim=True))
        out["dweight"], out["dbias"] = torch.einsum("mn,mn->n", g, h), g.sum(0)
    return out


def _exact_weights(teacher, ids, z, n, tau):
    """(share of each listed id, the listed ids that count), a list at a time."""
    ok = (ids >= 0) & (ids < n)
    ok &= ~torch.isneginf(z.gather(1, ids.clamp(0, n - 1)))
    v = (teacher.double() / tau).masked_fill(~ok, -math.inf)
    return torch.nan_to_num(torch.softmax(v, 1), nan=0.0), ok


def _exact_rows(case, s, z, rows):
    """(losses, gradient in the logits) of some rows' logits in 64 bits."""
    n = z.shape[1]
    if case["op"] == "entropy":
        target = s["target"][rows]
        ids, ok = target[:, None], target[:, None] >= 0
        q, tau = ok.double(), 1.0
    else:
        ids, tau = s["ids"][rows], case["tau"]
        q, ok = _exact_weights(s["teacher"][rows], ids, z, n, tau)
    logp = torch.log_softmax(z / tau, 1)
    at = ids.clamp(min=0)
    loss = tau ** 2 * (torch.xlogy(q, q) - q * torch.where(ok, logp.gather(1, at), 0.0)).sum(1)
    if s["grad"] is None:
        return loss, None
    d = logp.exp_() * ok.any(1, keepdim=True)
    d.scatter_add_(1, at, -q)
    return loss, d.mul_(tau * s["grad"][rows].double()[:, None])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    M, n = case["rows"], case["cols"]
    step = max(1, 400_000_000 // n)
    loss, dl = [], []
    if case["op"] == "scores":
        for r in range(0, M, step):
            rows = slice(r, r + step)
            a, d = _exact_rows(case, s, s["logits"][rows].double(), rows)
            loss.append(a)
            dl.append(d)
        out = {"loss": torch.cat(loss)}
        return out if s["grad"] is None else {**out, "dlogits": torch.cat(dl)}
    x, w = s["x"].double(), s["weight"].double()
    b = 0.0 if s["bias"] is None else s["bias"].double()
    dx, dw, db = [], torch.zeros_like(w), torch.zeros(n, dtype=torch.float64, device=DEV)
    for r in range(0, M, step):
        rows = slice(r, r + step)
        a, d = _exact_rows(case, s, torch.matmul(x[rows], w.T) + b, rows)
        loss.append(a)
        if d is not None:
            dx.append(torch.matmul(d, w))
            dw += torch.matmul(d.T, x[rows])
            db += d.sum(0)
    out = {"loss": torch.cat(loss)}
    if s["grad"] is not None:
        out["dx"], out["dweight"] = torch.cat(dx), dw
        if s["bias"] is not None:
            out["dbias"] = db
    return out

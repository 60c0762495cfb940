"""linear_cross_entropy, linear_distillation and distillation against their
definitions in 64 bits.

Tolerances are bounds derived from the arithmetic.  With e = 2^-24 and u the
half step of an output's type: a logit z = x w + b is off by at most
(K + 16) e S, S the sum of its terms' magnitudes (16 covers the bias and, for
float32, the terms dropped below 2^-22; a given logit is exact); u = z / tau by
that over tau and 4 e |u|.  lse is off by the largest such error among the
columns, weighed by p, and by (80 + 2 |lse|) e for its sums, exponentials (off
by 2 e times 1 + the distance from the maximum) and logarithm.  p is off by
those errors and 8 e (1 + |u - lse|) relative to itself, a teacher's share q by
16 e (1 + the range of its list).  dz = c (p - Q) is rounded to the operands'
type or to half (u, and where it is held in half, at the scale of the largest |c|, 2^-38 of
that) and enters sums of n terms with (n + 16) e.  Operands that are held in half
at the scale of their largest (float32 as two planes, bfloat16 in training) lose
up to 2^-38 of that."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _losses():
    from flashlog_amd import losses
    return losses


def _tiny(t):
    return float(torch.finfo(t).smallest_normal) * torch.finfo(t).eps


def _rows(z, dz, ids, teacher, tau, g, t):
    """(loss, its bound, dz, its bound before rounding, coefficients) of rows of logits in 64 bits."""
    M, V = z.shape
    u = z / tau
    du = dz / tau + 4 * E * torch.nan_to_num(u.abs(), posinf=0)
    p = torch.softmax(u, 1)
    lse = torch.logsumexp(u, 1)
    left = ~torch.isneginf(u).all(1)
    p, lse = torch.where(left[:, None], p, 0.0), torch.where(left, lse, 0.0)
    far = torch.where(p > 0, (u - lse[:, None]).abs(), 0.0)
    dlse = (p * (du + 2 * E * (1 + far))).sum(1) + (80 + 2 * lse.abs()) * E
    dp = p * (du + dlse[:, None] + 8 * E * (1 + far))
    at = ids.clamp(0, V - 1)
    ut, dut = u.gather(1, at), du.gather(1, at)
    inside = (ids >= 0) & (ids < V)
    if teacher is None:
        q, dq, logq, ok = inside.double(), torch.zeros_like(ut), torch.zeros_like(ut), inside
    else:
        ok = inside & ~torch.isneginf(ut) & ~torch.isneginf(teacher.double())
        v = (teacher.double() / tau).masked_fill(~ok, -math.inf)
        top = v.amax(1, keepdim=True) if v.shape[1] else v.new_zeros(M, 1)
        logq = torch.where(ok, torch.log_softmax(v, 1), 0.0)
        q = torch.where(ok, logq.exp(), 0.0)
        dq = q * 16 * E * (1 + torch.where(ok, (v - top).abs() + v.abs(), 0.0))
    live = ok.any(1) & left
    q = torch.where(live[:, None], q, 0.0)
    term = torch.where(q > 0, logq - ut + lse[:, None], 0.0)
    loss = tau ** 2 * torch.where(live, (q * term).sum(1), 0.0)
    some = torch.where(q > 0, q * (dut + dlse[:, None] + 16 * E * (1 + logq.abs() + ut.abs() + lse.abs()[:, None]))
                       + dq * (1 + term.abs()), 0.0).sum(1)
    dloss = tau ** 2 * some + (q.shape[1] + 16) * E * tau ** 2 * (q * term).abs().sum(1)
    Q = torch.zeros_like(z).scatter_add_(1, at, q)
    dQ = torch.zeros_like(z).scatter_add_(1, at, torch.where(q > 0, dq + q.shape[1] * E * q, 0.0))
    c = torch.where(live, tau * g.double(), 0.0)[:, None]
    d = torch.where(c == 0, 0.0, c * (p - Q))
    dd = c.abs() * (dp + dQ) + 4 * E * d.abs()
    return loss, torch.where(live, dloss, 0.0), d, dd, c


def _held(got, value, bound, what):
    got, value, bound = got.double().cpu().reshape(value.shape), value.cpu(), bound.cpu()
    odd = ~torch.isfinite(value)
    assert torch.equal(torch.nan_to_num(got[odd], nan=5.0), torch.nan_to_num(value[odd], nan=5.0)), what
    over = ((got - value).abs() - bound)[~odd]
    assert not over.isnan().any(), what
    assert (over <= 0).all(), "%s: off by %.3g more than allowed" % (what, over.max())


def vocab_reference(x, w, b, ids, teacher, tau, g):
    """{name: (value, bound)} of the losses of rows that are a product."""
    t = x.dtype
    u = torch.finfo(t).eps / 2
    K, (V, M) = x.shape[1], (w.shape[0], x.shape[0])
    x, w = x.double(), w.double()
    z, mag = x @ w.T, x.abs() @ w.abs().T
    if b is not None:
        z, mag = z + b.double(), mag + torch.nan_to_num(b.double().abs(), posinf=0)
    live = ((ids >= 0) & (ids < V)).any(1, keepdim=True)
    xm, wm = (x.abs() * live).max() if x.numel() else 0.0, w.abs().max() if w.numel() else 0.0
    lost = 2.0 ** -38 * (xm * w.abs().sum(1)[None, :] + wm * x.abs().sum(1, keepdim=True))
    loss, dloss, d, dd, c = _rows(z, (K + 16) * E * mag + lost, ids, teacher, tau, g, t)
    if K:  # bfloat16's is held in half, half's of few rows with what rounding leaves
        u = 2.0 ** -22 if t is torch.float16 and M <= 64 else min(u, 2.0 ** -11)
    dd = dd + u * d.abs() + c.abs().max() * 2.0 ** -38 + _tiny(t)
    dd = torch.where(c == 0, 0.0, dd)
    out = {"loss": (loss, dloss * 1.01 + 1e-30)}
    for name, a, v, n in (("dx", d, w, V), ("dw", d.T, x, M)):
        out[name] = (a @ v, (dd if name == "dx" else dd.T) @ v.abs() + (n + 16) * E * (a.abs() @ v.abs())
                     + 2.0 ** -38 * (wm if name == "dx" else xm) * a.abs().sum(1, keepdim=True))
    if b is not None:
        out["db"] = (d.sum(0), dd.sum(0) + (M + 16) * E * d.abs().sum(0))
    for k in list(out)[1:]:
        tt = b.dtype if k == "db" else t
        out[k] = (out[k][0], (out[k][1] + torch.finfo(tt).eps / 2 * out[k][0].abs()) * 1.01 + _tiny(tt))
    return out


def _make(M, K, V, t, seed, k=None, bias=True, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).to(t)
    w = (torch.randn(V, K, generator=g) * spread / max(K, 1) ** 0.5).to(t)
    b = torch.randn(V, generator=g).to(t) if bias else None
    grad = torch.rand(M, generator=g) / M
    ids = torch.randint(-1 if V > 1 else 0, V, (M, 1 if k is None else k), generator=g)
    teacher = None if k is None else 2 * torch.randn(M, k, generator=g)
    return x, w, b, ids, teacher, grad


def _loss_of(x, w, b, ids, teacher, tau):
    if teacher is None:
        return _losses().linear_cross_entropy(x, w, ids[..., 0], b)
    return _losses().linear_distillation(x, w, ids, teacher.cuda(), b, temperature=tau)


def _run(x, w, b, ids, teacher, tau, g):
    dev = [v.cuda() for v in (x, w)] + ([b.cuda()] if b is not None else [])
    leaves = [v.detach().requires_grad_(True) for v in dev]
    bias = leaves[2] if b is not None else None
    loss = _loss_of(leaves[0], leaves[1], bias, ids.cuda(), teacher, tau)
    grads = torch.autograd.grad(loss, leaves, g.cuda().reshape(loss.shape))
    return {"loss": loss.detach(), **dict(zip(("dx", "dw", "db"), grads))}


def _check(x, w, b, ids, teacher, tau, g):
    ref = vocab_reference(x, w, b, ids, teacher, tau, g)
    out = _run(x, w, b, ids, teacher, tau, g)
    assert out["loss"].dtype is torch.float32 and set(out) == set(ref)
    for k, (value, bound) in ref.items():
        _held(out[k], value, bound, k)
    with torch.no_grad():  # other kernels: no backward follows
        ev = _loss_of(x.cuda(), w.cuda(), None if b is None else b.cuda(), ids.cuda(), teacher, tau)
    _held(ev, *ref["loss"], "loss without gradients")
    return out


SIZES = [(1, 1, 1), (1, 7, 2), (3, 64, 25), (5, 1, 300), (64, 40, 475), (65, 100, 257), (130, 256, 1645), (17, 33, 3001),
         (300, 72, 515), (2, 2048, 100), (1000, 8, 9), (96, 0, 12)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,V", SIZES)
def test_cross_entropy(M, K, V, t):
    x, w, b, ids, _, g = _make(M, K, V, t, M + 31 * K + 7 * V, bias=V % 2 == 1)
    _check(x, w, b, ids, None, 1.0, g)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,V,k,tau", [(1, 7, 2, 1, 1.0), (3, 64, 25, 40, 2.0), (64, 40, 475, 5, 0.5),
                                         (65, 100, 257, 64, 1.0), (130, 256, 1645, 20, 4.0), (17, 33, 3001, 65, 3.0),
                                         (2, 16, 5000, 1000, 1.0), (8, 24, 50, 0, 1.0)])
def test_linear_distillation(M, K, V, k, tau, t):
    x, w, b, ids, teacher, g = _make(M, K, V, t, M + K + V + k, k=k, bias=k % 2 == 0)
    _check(x, w, b, ids, teacher, tau, g)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,V", [(300, 256, 1000), (257, 512, 2049), (1000, 64, 4096), (520, 200, 3333),
                                   (2, 1024, 70000), (48, 600, 5000), (66, 520, 140000), (130, 256, 4100), (70, 512, 4096), (150, 200, 4500), (400, 100, 3400), (460, 64, 4600)])
def test_many_tiles(M, K, V, t):
    """Sizes of several tiles in every direction, odd ends among them."""
    x, w, b, ids, _, g = (v.cuda() if v is not None else None for v in _make(M, K, V, t, M + K + V))
    _check(x, w, b, ids, None, 1.0, g)


@pytest.mark.parametrize("t,M,K", [(torch.float32, 300, 16), (torch.bfloat16, 700, 8), (torch.float16, 700, 8),
                                   (torch.bfloat16, 128, 9), (torch.float16, 60, 9)])
def test_several_pieces_of_the_vocabulary(t, M, K):
    """More logits than a piece of 1 GB holds (in the last one a few columns), the bias's gradient among them."""
    of = 2 * M if t is torch.float16 and M <= 64 else M  # rows of the logits' gradient
    V = (1 << 30) // (4 if t is torch.float32 else 2) // of // 256 * 256 + 300 + 11
    x, w, b, ids, teacher, g = (v.cuda() if v is not None else None for v in _make(M, K, V, t, 5, k=9))
    ids[0, :3] = torch.tensor([V - 1, V - 12, V - 320])
    _check(x, w, b, ids, teacher, 2.0, g)


@pytest.mark.parametrize("t", TYPES)
def test_sharp_rows(t):
    """Rows whose target has nearly all of the mass, and far logits."""
    x, w, b, ids, _, g = _make(70, 32, 301, t, 9, spread=12.0)
    z = x.float() @ w.float().T + b.float()
    ids[::2, 0] = z.argmax(1)[::2]
    _check(x, w, b, ids, None, 1.0, g)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("step", [84.0, 200.0])
def test_columns_far_above_the_first(step, t):
    """Large products in which a part's later columns are e^84 (within float32's range) or e^200 times its first ones."""
    M, K, V = 300, 32, 40000
    x, w, _, ids, _, g = (v.cuda() if v is not None else None for v in _make(M, K, V, t, 19, bias=False))
    b = step * (torch.arange(V, device="cuda") // 256 % 2)
    ids[::2, 0] = 256 + ids[::2, 0] % 256
    _check(x, w, b, ids, None, 1.0, g)


def test_small_gradients_in_half():
    """Weights of the rows' losses far below half's smallest number, in all rows or in some."""
    x, w, b, ids, _, g = _make(40, 64, 500, torch.float16, 10, bias=False)
    for grad in (g * 1e-7, torch.where(torch.arange(40) % 2 == 0, g, g * 1e-6), g * 1e30, torch.zeros(40)):
        ref = vocab_reference(x, w, None, ids, None, 1.0, grad)
        out = _run(x, w, None, ids, None, 1.0, grad)
        for k in ("dx", "dw"):
            value, bound = ref[k]
            most = 65504.0  # what overflows half is infinite
            fits = value.abs() + bound < most
            _held(torch.where(fits, out[k].double().cpu(), 0.0), torch.where(fits, value, 0.0), bound, k)


@pytest.mark.parametrize("t", TYPES)
def test_fp32_bias(t):
    x, w, b, ids, teacher, g = _make(33, 48, 200, t, 11, k=4)
    out = _check(x, w, b.float() + 0.01, ids, teacher, 1.0, g)
    assert out["db"].dtype is torch.float32


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,V", [(40, 24, 150), (300, 128, 4000)])
def test_columns_that_the_bias_takes_out(M, K, V, t):
    x, w, b, ids, teacher, g = _make(M, K, V, t, 12, k=6)
    b[torch.randperm(V, generator=torch.Generator().manual_seed(1))[:2 * V // 3]] = -math.inf
    ids[3] = 0
    b[0] = -math.inf
    out = _check(x, w, b, ids, teacher, 1.0, g)  # listed ids that are out do not count
    assert (out["db"].cpu()[torch.isneginf(b)] == 0).all()
    assert out["loss"][3] == 0 and (out["dx"][3] == 0).all()
    # a target that is out: infinite loss, a finite gradient
    out = _check(x, w, b, ids[:, :1], None, 1.0, g)
    assert out["loss"][3] == math.inf
    # nothing is left
    b.fill_(-math.inf)
    out = _run(x, w, b, ids[:, :1], None, 1.0, g)
    assert all((v == 0).all() for v in out.values())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,V", [(50, 40, 90), (300, 128, 4000)])
def test_rows_without_a_target(M, K, V, t):
    x, w, b, ids, _, g = _make(M, K, V, t, 13)
    ids[:, 0] = torch.tensor([-1, V, 5, -100, 1 << 40])[torch.arange(M) % 5]
    out = _check(x, w, b, ids, None, 1.0, g)
    off = torch.arange(M) % 5 != 2
    # whatever such rows hold, as padded ones may, nothing else changes
    pad = torch.where(off[:, None], torch.finfo(t).max / 2, x)
    for k, v in _run(pad, w, b, ids, None, 1.0, g).items():
        assert torch.equal(v, out[k]), k
    assert (out["loss"].cpu()[off] == 0).all() and (out["dx"].cpu()[off] == 0).all()
    ids.fill_(-1)
    assert all((v == 0).all() for v in _run(x, w, b, ids, None, 1.0, g).values())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,V", [(9, 40, 90), (300, 128, 4000)])
def test_not_finite_rows_stay_apart(M, K, V, t):
    x, w, b, ids, _, g = _make(M, K, V, t, 14)
    ids.clamp_(min=0)
    bad = x.clone()
    bad[2, 3] = float("nan")
    good, out = _run(x, w, b, ids, None, 1.0, g), _run(bad, w, b, ids, None, 1.0, g)
    rows = [r for r in range(M) if r != 2]
    assert out["loss"][2].isnan() and out["dx"][2].isnan().all()
    for k in ("loss", "dx"):
        assert torch.equal(out[k][rows], good[k][rows])


@pytest.mark.parametrize("t", TYPES)
def test_operands_of_many_magnitudes(t):
    """Rows of x and of the weight over factors of 2^10, and operands of zeros."""
    x, w, b, ids, _, g = _make(300, 128, 4000, t, 17)
    x = x * 2.0 ** -(torch.arange(300) % 11)[:, None]
    w = w * 2.0 ** -(torch.arange(4000) % 11)[:, None]
    _check(x.to(t), w.to(t), b, ids, None, 1.0, g)
    for a, c in ((x * 0, w), (x, w * 0), (x * 0, w * 0)):
        _check(a.to(t), c.to(t), b, ids, None, 1.0, g)


@pytest.mark.parametrize("t", TYPES)
def test_saved_tensors_on_other_strides(t):
    """A hook may give the backward its operands on strides that the forward did not have."""
    M, K, V = 300, 128, 4000
    x, w, b, ids, _, g = _make(M, K, V, t, 18)
    ref = vocab_reference(x, w, b, ids, None, 1.0, g)

    def shifted(v):  # the same values on rows that begin 2 or 4 bytes behind 16
        if v.dim() != 2 or v.dtype is not t:
            return v
        base = v.new_zeros(v.shape[0], v.shape[1] + 9)
        base[:, 1:1 + v.shape[1]] = v
        return base[:, 1:1 + v.shape[1]]

    def straight(v):
        return v.clone(memory_format=torch.contiguous_format) if v.dtype is t else v

    for first, then in ((straight, shifted), (shifted, straight)):
        leaves = [v.cuda().requires_grad_(True) for v in (x, w, b)]
        with torch.autograd.graph.saved_tensors_hooks(lambda v: v, then):
            loss = _losses().linear_cross_entropy(first(leaves[0]), first(leaves[1]), ids[:, 0].cuda(), leaves[2])
        for k, v in zip(("dx", "dw", "db"), torch.autograd.grad(loss, leaves, g.cuda())):
            _held(v, *ref[k], k)


def test_no_rows():
    x = torch.zeros(0, 4, device="cuda", requires_grad=True)
    w = torch.zeros(6, 4, device="cuda", requires_grad=True)
    loss = _losses().linear_cross_entropy(x, w, torch.zeros(0, dtype=torch.long, device="cuda"))
    dx, dw = torch.autograd.grad(loss, (x, w), torch.zeros_like(loss))
    assert loss.shape == (0,) and dx.shape == (0, 4) and (dw == 0).all()


@pytest.mark.parametrize("t", TYPES)
def test_strides_shapes_and_alignment(t):
    x, w, b, ids, teacher, g = _make(12, 37, 64, t, 15, k=3)
    ref = vocab_reference(x, w, b, ids, teacher, 1.0, g)
    wide = torch.zeros(12, 80, dtype=t)
    wide[:, 5:42] = x
    rows = torch.zeros(64, 100, dtype=t)
    rows[:, 1:38] = w
    for xv in (wide.cuda()[:, 5:42], x.t().contiguous().cuda().t()):
        for wv in (rows.cuda()[:, 1:38], w.t().contiguous().cuda().t()):
            leaves = [xv.detach().requires_grad_(True), wv.detach().requires_grad_(True)]
            # three leading dimensions, int32 ids, a teacher of half precision's values
            loss = _losses().linear_distillation(leaves[0].reshape(2, 3, 2, 37), leaves[1],
                                                 ids.int().reshape(2, 3, 2, 3).cuda(),
                                                 teacher.reshape(2, 3, 2, 3).cuda(), b.cuda())
            assert loss.shape == (2, 3, 2)
            _held(loss, ref["loss"][0].reshape(2, 3, 2), ref["loss"][1].reshape(2, 3, 2), "loss")
            grad = g.reshape(2, 3, 2).transpose(0, 2).contiguous().cuda().transpose(0, 2)
            for k, v in zip(("dx", "dw"), torch.autograd.grad(loss, leaves, grad)):
                _held(v, *ref[k], k)
    one = _losses().linear_cross_entropy(x[0].cuda(), w.cuda(), ids[0, 0].cuda())
    assert one.shape == ()


def test_only_some_gradients():
    x, w, b, ids, _, g = _make(70, 65, 333, torch.bfloat16, 16)
    ref = vocab_reference(x, w, b, ids, None, 1.0, g)
    for names in (["dx"], ["dw"], ["db"], ["dx", "db"], ["dw", "db"]):
        leaves = {k: v.cuda().requires_grad_(k in names) for k, v in (("dx", x), ("dw", w), ("db", b))}
        loss = _losses().linear_cross_entropy(leaves["dx"], leaves["dw"], ids[:, 0].cuda(), leaves["db"])
        for k, v in zip(names, torch.autograd.grad(loss, [leaves[k] for k in names], g.cuda())):
            _held(v, *ref[k], k)


# ---------------------------------------------------------------------------
# Rows that are given


def scores_reference(z, ids, teacher, tau, g):
    t = z.dtype
    loss, dloss, d, dd, _ = _rows(z.double(), torch.zeros(z.shape, dtype=torch.float64), ids, teacher, tau, g, t)
    return {"loss": (loss, dloss * 1.01 + 1e-30),
            "dx": (d, (dd + torch.finfo(t).eps / 2 * d.abs()) * 1.01 + _tiny(t))}


def _run_scores(z, ids, teacher, tau, g):
    leaf = z.cuda().requires_grad_(True)
    loss = _losses().distillation(leaf, ids.cuda(), teacher.cuda(), temperature=tau)
    return {"loss": loss.detach(), "dx": torch.autograd.grad(loss, leaf, g.cuda())[0]}


def _make_scores(M, V, k, t, seed, allow=1.0):
    g = torch.Generator().manual_seed(seed)
    z = (3 * torch.randn(M, V, generator=g))
    z = torch.where(torch.rand(M, V, generator=g) < allow, z, -math.inf).to(t)
    ids = torch.randint(-2, V + 2, (M, k), generator=g)
    return z, ids, 2 * torch.randn(M, k, generator=g), torch.rand(M, generator=g)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,V,k,tau,allow", [(1, 1, 1, 1.0, 1.0), (3, 2, 5, 2.0, 0.5), (5, 25, 25, 1.0, 0.3),
                                             (32, 475, 20, 0.5, 0.5), (7, 2047, 64, 1.0, 1.0), (7, 2048, 65, 3.0, 0.9),
                                             (6, 2049, 3, 1.0, 0.1), (4, 41000, 100, 2.0, 0.5), (1, 300001, 4096, 1.0, 1.0),
                                             (300, 33, 0, 1.0, 1.0)])
def test_distillation(M, V, k, tau, allow, t):
    z, ids, teacher, g = _make_scores(M, V, k, t, M + V + k, allow)
    ref, out = scores_reference(z, ids, teacher, tau, g), _run_scores(z, ids, teacher, tau, g)
    for name, (value, bound) in ref.items():
        _held(out[name], value, bound, name)


def test_the_same_id_twice():
    z, ids, teacher, g = _make_scores(20, 3000, 12, torch.float32, 21)
    ids[:, 6:] = ids[:, :6]
    ids[5] = 7
    ref, out = scores_reference(z, ids, teacher, 1.0, g), _run_scores(z, ids, teacher, 1.0, g)
    for name, (value, bound) in ref.items():
        _held(out[name], value, bound, name)


def test_masked_empty_and_padded_rows():
    z, ids, teacher, g = _make_scores(8, 2500, 6, torch.float32, 22)
    z[0] = -math.inf                        # nothing is left
    z[1, ids[1].clamp(0, 2499)] = -math.inf  # nothing that is listed is left
    ids[2] = -1                             # nothing is listed
    teacher[3, :4] = -math.inf
    teacher[4] = -math.inf
    z[5, 1:] = torch.finfo(torch.float32).min
    ids[5] = 0
    ref, out = scores_reference(z, ids, teacher, 1.0, g), _run_scores(z, ids, teacher, 1.0, g)
    for name, (value, bound) in ref.items():
        _held(out[name], value, bound, name)
    for r in (0, 1, 2, 4):
        assert out["loss"][r] == 0 and (out["dx"][r] == 0).all()
    assert (out["dx"].cpu()[torch.isneginf(z)] == 0).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tau", [1.0, 0.5])
def test_masks_of_the_lowest_value(tau, t):
    """Masks that are finite: a row of nothing else is uniform, as its distances from the largest are 0."""
    z, ids, teacher, g = _make_scores(7, 4500, 9, t, 25)
    low, far = torch.finfo(t).min, -math.inf
    ids[1], ids[2] = 2 * torch.arange(9) + 1, 7
    z[0], z[1, ::2], z[2] = low, low, low
    z[2, 7] = 1.0
    same, list_ = z.clone(), teacher.clone()
    same[0], same[1, ::2], same[2] = 0.0, far, far  # in 64 bits: what differs by a constant or is as good as 0
    same[2, 7] = 1.0
    teacher[3], teacher[4, :4] = torch.finfo(torch.float32).min, torch.finfo(torch.float32).min
    list_[3], list_[4, :4] = 0.0, far
    ref, out = scores_reference(same, ids, list_, tau, g), _run_scores(z, ids, teacher, tau, g)
    for name, (value, bound) in ref.items():
        _held(out[name], value, bound, name)


def test_not_finite_scores():
    z, ids, teacher, g = _make_scores(9, 2500, 6, torch.float32, 23)
    ids.clamp_(0, 2499)
    good = _run_scores(z, ids, teacher, 1.0, g)
    bad, list_ = z.clone(), teacher.clone()
    bad[1, 2000], bad[4, 7] = float("nan"), math.inf
    bad[6] = float("nan")
    list_[7, 2] = float("nan")
    out = _run_scores(bad, ids, list_, 1.0, g)
    rows = [0, 2, 3, 5, 8]
    for k in out:
        assert torch.equal(out[k][rows], good[k][rows])
    assert out["loss"][[1, 4, 6, 7]].isnan().all() and out["dx"][[1, 6]].isnan().all()
    assert out["dx"][7, ids[7]].isnan().all()


def test_strided_scores():
    z, ids, teacher, g = _make_scores(12, 700, 5, torch.bfloat16, 24)
    ref = scores_reference(z, ids, teacher, 1.0, g)
    base = torch.zeros(12, 1000, dtype=torch.bfloat16)
    base[:, 3:703] = z
    leaf = base.cuda().requires_grad_(True)
    for view in (leaf[:, 3:703], leaf[:, 3:703].reshape(3, 4, 700)):
        shape = view.shape[:-1]
        loss = _losses().distillation(view, ids.reshape(*shape, 5).cuda(), teacher.reshape(*shape, 5).cuda())
        dx = torch.autograd.grad(loss, leaf, g.reshape(shape).cuda())[0]
        _held(loss, ref["loss"][0].reshape(shape), ref["loss"][1].reshape(shape), "loss")
        _held(dx[:, 3:703], *ref["dx"], "dx")
        assert (dx[:, :3] == 0).all()


def test_no_scores():
    for shape in ((0, 5), (3, 0)):
        z = torch.zeros(shape, device="cuda", requires_grad=True)
        ids = torch.zeros(shape[0], 2, dtype=torch.long, device="cuda")
        loss = _losses().distillation(z, ids, torch.zeros(shape[0], 2, device="cuda"))
        assert loss.shape == shape[:1] and (loss == 0).all()
        assert torch.autograd.grad(loss, z, torch.ones_like(loss))[0].shape == shape


def test_scores_behind_two_gigabytes():
    V = 4_600_000
    M = (1 << 31) // V + 2
    z = torch.zeros(M, V, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    z[-1] = torch.randn(V, generator=g, device="cuda").bfloat16()
    ids = torch.tensor([[0, V - 1]], device="cuda").expand(M, 2).contiguous()
    teacher = torch.zeros(M, 2, device="cuda")
    leaf = z.requires_grad_(True)
    loss = _losses().distillation(leaf, ids, teacher)
    dx = torch.autograd.grad(loss, leaf, torch.ones_like(loss))[0]
    ref = scores_reference(z[-1:].detach().cpu(), ids[-1:].cpu(), teacher[-1:].cpu(), 1.0, torch.ones(1))
    _held(loss[-1:], *ref["loss"], "loss")
    _held(dx[-1:], *ref["dx"], "dx")


# ---------------------------------------------------------------------------
# As a program calls them


def test_gradients_against_differences():
    """In one direction, central differences of the definitions in 64 bits."""
    x, w, b, ids, teacher, g = _make(6, 20, 40, torch.float32, 31, k=4)
    out, ref = _run(x, w, b, ids, teacher, 2.0, g), vocab_reference(x, w, b, ids, teacher, 2.0, g)
    gen = torch.Generator().manual_seed(2)
    for name, v in (("dx", x), ("dw", w), ("db", b)):
        way, step = torch.randn(v.shape, generator=gen).double(), 1e-5

        def value(at):
            a = {"dx": x.double(), "dw": w.double(), "db": b.double()}
            a[name] = a[name] + at * step * way
            z = a["dx"] @ a["dw"].T + a["db"]
            return (_rows(z, torch.zeros_like(z), ids, teacher, 2.0, g, torch.float32)[0] * g.double()).sum()

        slope = (value(1) - value(-1)) / (2 * step)
        got = (out[name].double().cpu() * way).sum()
        # differences: third derivatives times step^2 (1e-10) and 1e-16 / step of the sum; the gradient: its bound
        assert (slope - got).abs() <= (ref[name][1] * way.abs()).sum() + 1e-8, name


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V", [1200, 2200])
def test_same_bits_and_other_streams(V, t):
    x, w, b, ids, teacher, g = _make(500, 128, V, t, 32, k=7)
    z, sids, steacher, sg = _make_scores(20, 9000, 30, torch.float16, 33)
    first = [_run(x, w, b, ids, teacher, 1.0, g), _run_scores(z, sids, steacher, 1.0, sg)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [_run(x, w, b, ids, teacher, 1.0, g), _run_scores(z, sids, steacher, 1.0, sg)]
    side.synchronize()
    for a, c in zip(first, again):
        for k in a:
            assert torch.equal(a[k], c[k]), k


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,V", [(150, 72, 700), (300, 128, 4000)])
def test_captured_forward_and_backward(M, K, V, t):
    x, w, b, ids, teacher, g = (v.cuda() for v in _make(M, K, V, t, 34, k=5))
    z, sids, steacher, sg = (v.cuda() for v in _make_scores(10, 5000, 8, t, 35, 0.5))
    leaves = [v.detach().clone().requires_grad_(True) for v in (x, w, b, z)]

    def step(p):
        out = []
        for loss, of, grad in ((_losses().linear_distillation(p[0], p[1], ids, teacher, p[2], 2.0), p[:3], g),
                               (_losses().linear_cross_entropy(p[0], p[1], ids[:, 0]), p[:2], g),
                               (_losses().distillation(p[3], sids, steacher), p[3:], sg)):
            out += [loss, *torch.autograd.grad(loss, of, grad)]
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([v.detach().clone().requires_grad_(True) for v in leaves])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(leaves)
    for k in range(4):
        with torch.no_grad():
            leaves[0].copy_(x * (0.5 + k))
            leaves[3].copy_(z * (0.5 + k))
        torch.ones(1000, device="cuda").sum().item()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(held, step([v.detach().clone().requires_grad_(True) for v in leaves])):
            assert torch.equal(a, c)


def test_refusals():
    L = _losses()
    x, w = torch.zeros(2, 3, device="cuda"), torch.zeros(4, 3, device="cuda")
    t, ids, teacher = (torch.zeros(2, dtype=torch.long, device="cuda"),
                       torch.zeros(2, 5, dtype=torch.long, device="cuda"), torch.zeros(2, 5, device="cuda"))
    big = torch.zeros(2, 4097, device="cuda")
    for error, call in (
            (TypeError, lambda: L.linear_cross_entropy(x.double(), w.double(), t)),
            (TypeError, lambda: L.linear_cross_entropy(x, w.half(), t)),
            (TypeError, lambda: L.linear_cross_entropy(x, w, t.float())),
            (TypeError, lambda: L.linear_cross_entropy(x.half(), w.half(), t, w[:, 0].bfloat16())),
            (ValueError, lambda: L.linear_cross_entropy(x, w[:, :2], t)),
            (ValueError, lambda: L.linear_cross_entropy(x, w[0], t)),
            (ValueError, lambda: L.linear_cross_entropy(x, w[:0], t)),
            (ValueError, lambda: L.linear_cross_entropy(x, w, t[:1])),
            (ValueError, lambda: L.linear_cross_entropy(x, w, ids)),
            (ValueError, lambda: L.linear_cross_entropy(x, w, t, x[0])),
            (RuntimeError, lambda: L.linear_cross_entropy(x, w, t.cpu())),
            (ValueError, lambda: L.linear_distillation(x, w, t, teacher)),
            (ValueError, lambda: L.linear_distillation(x, w, ids, teacher[:, :4])),
            (ValueError, lambda: L.linear_distillation(x, w, ids, teacher, temperature=0.0)),
            (ValueError, lambda: L.linear_distillation(x, w, ids, teacher, temperature=math.inf)),
            (TypeError, lambda: L.linear_distillation(x, w, ids, teacher.double())),
            (ValueError, lambda: L.linear_distillation(x, w, ids, teacher.clone().requires_grad_(True))),
            (ValueError, lambda: L.distillation(x, big.long(), big)),
            (ValueError, lambda: L.distillation(x, ids[:1], teacher[:1])),
            (ValueError, lambda: L.distillation(x, ids, teacher, temperature=math.nan)),
            (TypeError, lambda: L.distillation(x.double(), ids, teacher)),
            (RuntimeError, lambda: L.distillation(x, ids.cpu(), teacher))):
        with pytest.raises(error):
            call()
    leaf = x.clone().requires_grad_(True)
    for loss in (L.linear_cross_entropy(leaf, w, t), L.distillation(leaf, ids, teacher)):
        first = torch.autograd.grad(loss.sum(), leaf, create_graph=True)[0]
        with pytest.raises(RuntimeError):
            torch.autograd.grad(first.sum(), leaf)


def test_a_generator_in_training():
    """layer_norm -> linear -> a relation loss and, on the same states, scores under constraints held to a teacher,
    against torch in 64 bits.  Bounds: every operator's outputs are within a few steps of 2^-24 of their magnitudes
    (sums of at most 300 terms), so the gradients, sums of products of them, within 2000 of those of the gradients'
    largest magnitudes."""
    from flashlog_amd import attention as fa
    L = _losses()
    g = torch.Generator().manual_seed(41)
    Q, D, R, n = 48, 64, 30, 300
    x, gain, shift = torch.randn(Q, D, generator=g), 1 + 0.1 * torch.randn(D, generator=g), torch.zeros(D)
    w1, b1 = torch.randn(D, D, generator=g) / D ** 0.5, torch.zeros(D)
    rel, ent = torch.randn(R, D, generator=g) / D ** 0.5, torch.randn(n, D, generator=g) / D ** 0.5
    target = torch.randint(-1, R, (Q,), generator=g)
    ids, teacher = torch.randint(0, n, (Q, 10), generator=g), torch.randn(Q, 10, generator=g)
    types, of = torch.rand(4, n, generator=g) < 0.6, torch.randint(4, (Q,), generator=g)

    def program(p, own):
        x, gain, shift, w1, b1, rel, ent = p
        if own:
            h = fa.linear(fa.layer_norm(x, gain, shift), w1, b1, "tanh", residual=x)
            scores = fa.constrain_logits(fa.linear(h, ent), allowed=types.cuda(), group=of.cuda())
            return (L.linear_cross_entropy(h, rel, target.cuda()).mean()
                    + L.distillation(scores, ids.cuda(), teacher.cuda(), temperature=2.0).mean())
        c = x - x.mean(1, keepdim=True)
        h = torch.tanh((c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt() * gain + shift) @ w1.T + b1) + x
        lp = torch.log_softmax(h @ rel.T, 1)
        first = torch.where(target >= 0, -lp.gather(1, target.clamp(min=0)[:, None])[:, 0], 0.0).mean()
        z = (h @ ent.T).masked_fill(~types[of], -math.inf) / 2
        ok = types[of].gather(1, ids)
        v = (teacher.double() / 2).masked_fill(~ok, -math.inf)
        live = ok.any(1)
        lq = torch.where(ok, torch.log_softmax(v, 1), 0.0)
        q = torch.where(ok, lq.exp(), 0.0)
        u = torch.where(ok, torch.log_softmax(z, 1).gather(1, ids), 0.0)
        return first + 4 * torch.where(live, (q * (lq - u)).sum(1), 0.0).mean()

    params = [x, gain, shift, w1, b1, rel, ent]
    mine = [v.cuda().requires_grad_(True) for v in params]
    want = [v.double().requires_grad_(True) for v in params]
    a, c = program(mine, True), program(want, False)
    assert abs(a.item() - c.item()) <= 2000 * E * abs(c.item())
    for p, q in zip(torch.autograd.grad(a, mine), torch.autograd.grad(c, want)):
        assert (p.double().cpu() - q).abs().max() <= 2000 * E * q.abs().max()

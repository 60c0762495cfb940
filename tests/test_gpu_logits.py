"""constrain_logits and hop_attention against their definitions in 64 bits.

Bounds, with e = 2^-24 and u the output type's half step: a constrained value
takes at most 8 roundings of terms no larger than
B = ((|x| + |b|) max(rho, 1/rho, 1) + presence + frequency c) / tau, so it is
off by at most 8 e B before its own rounding.  A weight w = exp(v - m) / s is
off by the factor of twice the values' error in v - m (the row's largest),
the sum's n e and 8 e.  The gradient's dot sum w g carries the weights' errors
and (n + 4) e of its terms' magnitudes."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _fa():
    from flashlog_amd import attention
    return attention


def _u(t):
    return torch.finfo(t).eps / 2, float(torch.finfo(t).smallest_normal) * torch.finfo(t).eps


def _case(lead, n, t, seed, groups=None, bias="none", allow=0.6, past=0, owners=1):
    """owners: how many of the leading dimensions name an owner."""
    g = torch.Generator().manual_seed(seed)
    c = dict(x=(2 * torch.randn(*lead, n, generator=g)).to(t), allowed=None, group=None, bias=None, history=None)
    own = lead[:owners]
    if groups:
        c["group"] = torch.randint(groups, own, generator=g)
    if allow is not None:
        c["allowed"] = torch.rand(groups or 1, n, generator=g) < allow
    if bias != "none":
        c["bias"] = torch.randn(*((groups, n) if bias == "table" else (n,)), generator=g)
    if past == "ragged":
        count = torch.randint(0, 9, (math.prod(own),), generator=g)
        off = torch.cat([torch.zeros(1, dtype=torch.long), count.cumsum(0)])
        c["history"] = (off, torch.randint(-1, n + 1, (int(off[-1]),), generator=g))
    elif past:
        c["history"] = torch.randint(-1, n, own + (past,), generator=g)
    return c


OPTIONS = dict(repetition=1.4, presence=0.3, frequency=0.2, temperature=0.8)


def _rows(c, opts):
    """Per row (as one flat list): value, bound, allowed, slope, sign margin, table row."""
    x = c["x"]
    n = x.shape[-1]
    lead = x.shape[:-1]
    rows = math.prod(lead)
    xf = x.double().reshape(rows, n)
    rho, tau = opts.get("repetition", 1.0), opts.get("temperature", 1.0)
    pres, freq = opts.get("presence", 0.0), opts.get("frequency", 0.0)

    def owner_of(count):
        return torch.arange(rows) // max(rows // count, 1) if count else torch.zeros(rows, dtype=torch.long)

    g = torch.zeros(rows, dtype=torch.long)
    if c["group"] is not None:
        g = c["group"].reshape(-1)[owner_of(c["group"].numel())]
    tables = [t for t in (c["allowed"], None if c["bias"] is None else c["bias"].reshape(-1, n)) if t is not None]
    out_of = torch.zeros(rows, dtype=torch.bool)
    for t in tables:
        if t.shape[0] > 1:
            out_of |= (g < 0) | (g >= t.shape[0])
    gs = torch.where(out_of, 0, g)
    pick = lambda t: t[gs if t.shape[0] > 1 else torch.zeros(rows, dtype=torch.long)]
    ok = pick(c["allowed"]).clone() if c["allowed"] is not None else torch.ones(rows, n, dtype=torch.bool)
    ok[out_of] = False
    b = pick(c["bias"].reshape(-1, n)).double() if c["bias"] is not None else torch.zeros(rows, n, dtype=torch.float64)
    cnt = torch.zeros(rows, n, dtype=torch.float64)
    h = c["history"]
    if h is not None:
        if isinstance(h, tuple):
            own = owner_of(h[0].numel() - 1)
            lists = [h[1][h[0][o]:h[0][o + 1]] for o in own]
        else:
            own = owner_of(math.prod(h.shape[:-1]))
            lists = [h.reshape(-1, h.shape[-1])[o] for o in own]
        for i, ids in enumerate(lists):
            for j in ids.tolist():
                if 0 <= j < n:
                    cnt[i, j] += 1
    s = xf + b
    seen = cnt > 0
    factor = torch.where(seen, torch.where(s > 0, 1 / rho, rho), torch.ones_like(s))
    v = (s * factor - torch.where(seen, pres + freq * cnt, torch.zeros_like(s))) / tau
    big = ((xf.abs() + b.abs()) * max(rho, 1 / rho, 1.0) + pres + freq * cnt) / tau
    return v, 8 * E * big, ok, factor / tau, gs, out_of


def _gpu(c):
    def go(t):
        return None if t is None else tuple(go(i) for i in t) if isinstance(t, tuple) else t.cuda()
    return {k: go(v) for k, v in c.items()}


def _check(c, opts, softmax, dtype_bits=True, seed=0):
    fa = _fa()
    d = _gpu(c)
    x = d["x"].requires_grad_(True)
    b = d["bias"].requires_grad_(True) if d["bias"] is not None else None
    fn = fa.hop_attention if softmax else fa.constrain_logits
    kw = dict(allowed=d["allowed"], group=d["group"], bias=b, history=d["history"], **opts)
    out = fn(x, **kw)
    t = x.dtype
    assert out.shape == x.shape and out.dtype == (torch.float32 if softmax else t)
    with torch.no_grad():
        assert torch.equal(fn(x, **kw), out.detach())
        if d["allowed"] is not None:
            kw["allowed"] = fa.pack_allowed(d["allowed"])
            assert torch.equal(fn(x, **kw), out.detach())
    n = x.shape[-1]
    v, dv, ok, slope, g, out_of = _rows(c, opts)
    rows = v.shape[0]
    gy = torch.randn(out.shape, generator=torch.Generator().manual_seed(seed + 1)).to(out.dtype)
    gd = gy.double().reshape(rows, n)
    got = out.detach().double().cpu().reshape(rows, n)
    u, tiny = _u(t)
    if softmax:
        vm = torch.where(ok, v, -math.inf)
        m = vm.amax(-1, keepdim=True)
        e = torch.where(ok, torch.exp(v - torch.where(m == -math.inf, 0.0, m)), 0.0)
        total = e.sum(-1, keepdim=True)
        w = e / torch.where(total == 0, 1.0, total)
        rel = 2 * torch.where(ok, dv, 0.0).amax(-1, keepdim=True) + 2 * E * torch.where(
            ok & (w > 0), (v - m).abs(), 0.0) + (n + 8) * E
        bound = w * rel * 1.01 + 2e-38
        assert (got[~ok] == 0).all()
        assert ((got - w).abs() <= bound).all()
        dot = (w * gd).sum(-1, keepdim=True)
        ddot = (bound * gd.abs()).sum(-1, keepdim=True) + (n + 4) * E * (w * gd.abs()).sum(-1, keepdim=True)
        dx = w * (gd - dot) * slope
        ddx = (bound * (gd - dot).abs() + w * (ddot + 2 * E * (gd.abs() + dot.abs()))) * slope + 4 * E * dx.abs()
    else:
        assert torch.equal(torch.isinf(got), ~ok)
        assert ((got - v).abs()[ok] <= (dv + u * v.abs() * 1.01 + tiny)[ok]).all()
        dx = torch.where(ok, gd * slope, 0.0)
        ddx = 4 * E * dx.abs()
    leaves = [x] + ([b] if b is not None else [])
    grads = torch.autograd.grad(out, leaves, gy.cuda())
    assert grads[0].dtype == t
    gx = grads[0].double().cpu().reshape(rows, n)
    # a column whose sign the rounding of x + bias may turn takes either slope
    rho = opts.get("repetition", 1.0)
    near = v.abs() * opts.get("temperature", 1.0) <= 4 * E * (1 + v.abs())
    assert near.sum() == 0 or rho == 1.0 or softmax or c["history"] is None
    assert ((gx - dx).abs() <= ddx + u * dx.abs() * 1.01 + tiny + 2e-38).all()
    assert (gx[~ok] == 0).all()
    if b is not None:
        bt = c["bias"].reshape(-1, n)
        want, bound = torch.zeros_like(bt, dtype=torch.float64), torch.zeros_like(bt, dtype=torch.float64)
        at = torch.where(out_of, 0, g) if bt.shape[0] > 1 else torch.zeros(rows, dtype=torch.long)
        live = dx.clone()
        want.index_add_(0, at, live)
        bound.index_add_(0, at, ddx + (rows + 4) * E * dx.abs())
        assert ((grads[1].double().cpu().reshape(bt.shape) - want).abs() <= bound * 1.01 + 1e-37).all()


LEADS = [((1,), 1), ((7,), 33), ((5, 3), 25), ((4, 3), 475), ((3,), 1024), ((2, 2), 1645), ((3,), 2049), ((2,), 8192)]


@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lead,n", LEADS)
def test_sizes(lead, n, t, softmax):
    _check(_case(lead, n, t, n, groups=4, bias="table", past=3), OPTIONS, softmax)


@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("t", TYPES)
def test_long_rows(t, softmax):
    """Rows longer than one workgroup holds."""
    _check(_case((3,), 8193, t, 1, groups=2, bias="table", past="ragged"), OPTIONS, softmax)
    _check(_case((2,), 41003, t, 2, bias="row", past="ragged"), OPTIONS, softmax)


@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("bias", ["none", "row", "table"])
@pytest.mark.parametrize("past", [0, 2, "ragged"])
@pytest.mark.parametrize("opts", [{}, OPTIONS, dict(repetition=0.5), dict(presence=1.0, temperature=2.0)])
def test_options(opts, past, bias, softmax):
    _check(_case((6, 4), 77, torch.float32, 3, groups=3, bias=bias, past=past), opts, softmax)


@pytest.mark.parametrize("softmax", [False, True])
def test_owners_of_either_dimension(softmax):
    c = _case((4, 5), 60, torch.float32, 4, groups=3, bias="table", past=2)
    c["group"] = torch.randint(3, (4, 5), generator=torch.Generator().manual_seed(5))  # finer than the history
    _check(c, OPTIONS, softmax)
    c = _case((4, 5), 60, torch.float32, 6, groups=3, past="ragged", owners=2)
    c["group"] = c["group"][:, 0].contiguous()  # coarser
    _check(c, OPTIONS, softmax)
    c = _case((20,), 60, torch.float32, 7, allow=None)
    _check(c, {}, softmax)


@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("n", [40, 300, 1500, 5000, 9000])
def test_many_rows_of_one_table_row(n, softmax):
    """The bias gradient's parts: rows of one group, and of a few uneven ones."""
    rows = 200 if n < 5000 else 40
    _check(_case((rows,), n, torch.float32, 8, bias="row"), OPTIONS, softmax)
    c = _case((rows,), n, torch.bfloat16, 9, groups=3, bias="table")
    c["group"][: rows // 2] = 1
    _check(c, OPTIONS, softmax)


@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("n", [50, 9000])
def test_rows_with_nothing_left(n, softmax):
    c = _case((8,), n, torch.float32, 10, groups=4, bias="table", past=2)
    c["allowed"][1] = False
    c["allowed"][2] = False
    c["allowed"][2, n - 1] = True  # one column
    c["group"] = torch.tensor([0, 1, 2, 3, -1, 4, 1 << 40, 2])  # three of no table row
    _check(c, OPTIONS, softmax)


@pytest.mark.parametrize("n", [50, 1200, 9000])
@pytest.mark.parametrize("t", TYPES)
def test_what_is_masked_is_not_read(n, t):
    """Infinities, NaN and the type's lowest value in masked places, in logits and in gradients."""
    fa = _fa()
    c = _case((6,), n, t, 11, allow=0.5)
    clean = _gpu(c)
    dirty = dict(clean, x=clean["x"].clone())
    off = ~clean["allowed"].expand(6, n)
    bad = torch.tensor([math.inf, -math.inf, math.nan, torch.finfo(t).min], device="cuda").to(t)
    dirty["x"][off] = bad[torch.arange(int(off.sum()), device="cuda") % 4]
    for fn in (fa.constrain_logits, fa.hop_attention):
        outs, grads = [], []
        for d in (clean, dirty):
            x = d["x"].detach().requires_grad_(True)
            y = fn(x, allowed=d["allowed"], temperature=0.5)
            g = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(y.dtype).cuda()
            if d is dirty:
                g[off] = math.nan
            outs.append(y.detach())
            grads.append(torch.autograd.grad(y, [x], g)[0])
        assert torch.equal(outs[0], outs[1]) and torch.equal(grads[0], grads[1])


@pytest.mark.parametrize("n", [30, 1500, 8500])
def test_infinite_and_lowest_logits(n):
    """Additive masks: -inf counts as nothing, the lowest value as a value."""
    fa = _fa()
    x = torch.randn(5, n, generator=torch.Generator().manual_seed(12))
    x[0] = -math.inf
    x[1] = torch.finfo(torch.float32).min
    x[2, : n // 2] = -math.inf
    x[3, : n // 2] = torch.finfo(torch.float32).min
    x[4, 3] = math.nan
    w = fa.hop_attention(x.cuda()).cpu().double()
    assert (w[0] == 0).all()
    assert (w[1] - 1 / n).abs().max() <= (n + 8) * E / n
    for r in (2, 3):
        want = torch.softmax(x[r].double(), -1)
        assert ((w[r] - want).abs() <= want * (n + 16) * E + 2e-38).all()
    assert torch.isnan(w[4]).all()
    xg = x.cuda().requires_grad_(True)
    (g,) = torch.autograd.grad(fa.hop_attention(xg)[:4].square().sum(), [xg])
    assert torch.isfinite(g[:4]).all() and (g[0] == 0).all()


def test_gradient_against_differences():
    """hop_attention's gradient against central differences of the 64-bit definition."""
    c = _case((4, 2), 40, torch.float32, 13, groups=3, bias="table", past=3)
    v, _, ok, _, _, _ = _rows(c, OPTIONS)
    gy = torch.randn(8, 40, generator=torch.Generator().manual_seed(14)).double()

    def loss(x):
        v, _, ok, _, _, _ = _rows(dict(c, x=x), OPTIONS)
        return float((torch.softmax(torch.where(ok, v, -math.inf), -1) * gy).sum())

    d = _gpu(c)
    x = d["x"].requires_grad_(True)
    y = _fa().hop_attention(x, allowed=d["allowed"], group=d["group"], bias=d["bias"], history=d["history"], **OPTIONS)
    (g,) = torch.autograd.grad(y, [x], gy.float().view(4, 2, 40).cuda())
    h = 1e-4
    base = c["x"].double()
    for i in range(0, 320, 7):
        up, down = base.clone().view(-1), base.clone().view(-1)
        up[i] += h
        down[i] -= h
        num = (loss(up.view(base.shape)) - loss(down.view(base.shape))) / (2 * h)
        assert abs(num - float(g.reshape(-1)[i])) <= 1e-5  # h^2 times a third derivative below 100


def test_fill_and_pack():
    fa = _fa()
    for n in (1, 31, 32, 33, 64, 65, 1645):
        mask = torch.rand(5, n, generator=torch.Generator().manual_seed(n)) < 0.5
        words = fa.pack_allowed(mask.cuda()).cpu().numpy().view(np.uint32)
        bits = (words[:, np.arange(n) // 32] >> (np.arange(n) % 32).astype(np.uint32)) & 1
        assert np.array_equal(bits.astype(bool), mask.numpy())
        x = torch.randn(5, n).cuda()
        y = fa.constrain_logits(x, allowed=mask.cuda(), group=torch.arange(5).cuda(), fill=-7.0)
        assert torch.equal(y, torch.where(mask.cuda(), x, torch.tensor(-7.0).cuda()))


def test_history_from_pairs():
    fa = _fa()
    rng = np.random.default_rng(0)
    rows, ids = rng.integers(-1, 12, 400), rng.integers(0, 50, 400)
    off, got = fa.history_from_pairs(torch.from_numpy(rows).cuda(), torch.from_numpy(ids).cuda(), 11)
    off, got = off.cpu().numpy(), got.cpu().numpy()
    for r in range(11):
        assert np.array_equal(got[off[r]:off[r + 1]], ids[rows == r])
    x = torch.rand(11, 50).cuda()
    y = fa.constrain_logits(x, history=(torch.from_numpy(off).cuda(), torch.from_numpy(got).cuda()), presence=1.0)
    seen = torch.zeros(11, 50, dtype=torch.bool)
    for r in range(11):
        seen[r, ids[rows == r]] = True
    assert torch.equal(y, x - seen.cuda().float())


def test_offsets_outside_the_ids_are_cut():
    """A ragged history whose offsets run backwards or past the list reads nothing beyond it."""
    fa = _fa()
    x = torch.ones(4, 30).cuda()
    off = torch.tensor([-5, 2, 1, 99, 3]).cuda()
    ids = torch.tensor([3, 4, 5]).cuda()
    y = fa.constrain_logits(x, history=(off, ids), presence=1.0).cpu()
    want = torch.ones(4, 30)
    want[0, [3, 4]] = 0
    want[2, [4, 5]] = 0
    assert torch.equal(y, want)


def test_strided_and_empty_rows():
    fa = _fa()
    wide = torch.randn(6, 90).cuda()
    mask = (torch.rand(80) < 0.5).cuda()
    part = wide[:, 5:85]
    assert torch.equal(fa.hop_attention(part, allowed=mask), fa.hop_attention(part.contiguous(), allowed=mask))
    turned = part.t().contiguous().t()
    assert torch.equal(fa.constrain_logits(turned, allowed=mask), fa.constrain_logits(part, allowed=mask))
    assert fa.hop_attention(torch.zeros(0, 7).cuda()).shape == (0, 7)
    assert fa.hop_attention(torch.zeros(3, 0).cuda()).shape == (3, 0)
    x = torch.zeros(0, 7).cuda().requires_grad_(True)
    b = torch.zeros(7).cuda().requires_grad_(True)
    gx, gb = torch.autograd.grad(fa.hop_attention(x, bias=b).sum(), [x, b])
    assert gx.shape == (0, 7) and (gb == 0).all()
    assert fa.hop_attention(torch.zeros(3, 4).cuda(), history=torch.zeros(3, 0, dtype=torch.long).cuda(),
                            repetition=2.0).allclose(torch.tensor(0.25).cuda())


def test_refusals():
    fa = _fa()
    x = torch.randn(4, 3, 10).cuda()
    i64 = lambda *s: torch.zeros(*s, dtype=torch.long).cuda()
    for fn in (fa.constrain_logits, fa.hop_attention):
        for exc, kw in [
            (ValueError, dict(temperature=0.0)), (ValueError, dict(temperature=math.nan)),
            (ValueError, dict(repetition=-1.0)), (ValueError, dict(presence=math.inf)),
            (ValueError, dict(allowed=torch.ones(9, dtype=torch.bool).cuda())),
            (ValueError, dict(allowed=torch.ones(2, 10, dtype=torch.bool).cuda())),
            (TypeError, dict(allowed=torch.ones(10).cuda())),
            (ValueError, dict(allowed=torch.ones(2, dtype=torch.int32).cuda())),
            (ValueError, dict(allowed=torch.ones(0, 10, dtype=torch.bool).cuda(), group=i64(4))),
            (ValueError, dict(bias=torch.zeros(9).cuda())), (ValueError, dict(bias=torch.zeros(2, 10).cuda())),
            (TypeError, dict(bias=i64(10))),
            (ValueError, dict(allowed=torch.ones(2, 10, dtype=torch.bool).cuda(), bias=torch.zeros(3, 10).cuda(),
                              group=i64(4))),
            (ValueError, dict(group=i64(5))), (TypeError, dict(group=torch.zeros(4).cuda())),
            (ValueError, dict(history=i64(5, 2))), (ValueError, dict(history=(i64(6), i64(2)))),
            (ValueError, dict(history=(i64(5), i64(2, 2)))), (ValueError, dict(history=(i64(5), i64(3), i64(3)))),
            (ValueError, dict(history=(i64(5), i64(3)), group=i64(4, 3))),
            (RuntimeError, dict(allowed=torch.ones(10, dtype=torch.bool))),
        ]:
            with pytest.raises(exc):
                fn(x, **kw)
        with pytest.raises(TypeError):
            fn(x.double())
        with pytest.raises(RuntimeError):
            fn(x.cpu())


def test_same_bits_and_graph():
    """Every run the same bits; captured forward and backward replayed on new inputs beside eager work."""
    fa = _fa()
    c = _gpu(_case((30, 4), 475, torch.float32, 15, groups=9, bias="table", past=3))
    words = fa.pack_allowed(c["allowed"])
    gy = torch.randn(30, 4, 475).cuda()

    def step(x, b, group, hist):
        x, b = x.detach().requires_grad_(True), b.detach().requires_grad_(True)
        w = fa.hop_attention(x, allowed=words, group=group, bias=b, history=hist, **OPTIONS)
        s = fa.constrain_logits(x, allowed=words, group=group, bias=b, history=hist, fill=0.0, **OPTIONS)
        return [w.detach(), s.detach(), *torch.autograd.grad(w, [x, b], gy), *torch.autograd.grad(s, [x, b], gy)]

    args = [c["x"], c["bias"], c["group"], c["history"]]
    first = step(*args)
    for _ in range(2):
        for p, q in zip(first, step(*args)):
            assert torch.equal(p, q)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*args)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = step(*args)
    for k in range(3):
        g = torch.Generator().manual_seed(40 + k)
        args[0].copy_(torch.randn(30, 4, 475, generator=g))
        args[2].copy_(torch.randint(-1, 10, (30,), generator=g))
        args[3].copy_(torch.randint(-1, 475, (30, 3), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(step(*args), out):
            assert torch.equal(p, q)


@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("t", TYPES)
def test_long_histories(t, softmax):
    """More ids than a byte counts: short rows, rows of several segments, an id many times over."""
    g = torch.Generator().manual_seed(50)
    for n in (30, 1645, 5000):
        c = _case((2, 3), n, t, 51, groups=2, bias="table")
        c["history"] = torch.randint(-2, n + 2, (2, 700), generator=g)
        c["history"][0, :400] = n // 2
        _check(c, dict(OPTIONS, frequency=0.01), softmax)


def test_a_history_that_outgrows_its_counters():
    """Past 65,000 repeats a column is counted no further, and its neighbours stay right."""
    fa = _fa()
    ids = torch.full((1, 150_000), 11)
    ids[0, :3] = torch.tensor([10, 12, 12])
    y = fa.constrain_logits(torch.zeros(1, 300).cuda(), history=ids.cuda(), frequency=1.0).cpu()[0]
    assert y[10] == -1 and y[12] == -2 and -65_100 <= y[11] <= -65_000
    y[[10, 11, 12]] = 0
    assert (y == 0).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n", [70, 3000])
def test_gradient_of_the_bias_alone(n, t):
    fa = _fa()
    c = _gpu(_case((40,), n, t, 60, groups=5, bias="table", past=2))
    gy = torch.randn(40, n).cuda()
    both, alone = [], []
    for keep in (True, False):
        x, b = c["x"].detach().requires_grad_(keep), c["bias"].detach().requires_grad_(True)
        kw = dict(allowed=c["allowed"], group=c["group"], bias=b, history=c["history"], **OPTIONS)
        for fn in (fa.hop_attention, fa.constrain_logits):
            y = fn(x, **kw)
            (both if keep else alone).append(torch.autograd.grad(y, [b], gy.to(y.dtype))[0])
    for p, q in zip(both, alone):
        assert torch.equal(p, q)


@pytest.mark.parametrize("t,rows", [(torch.float32, 35), (torch.bfloat16, 70), (torch.float16, 70)])
def test_outputs_larger_than_the_caches(t, rows):
    """Rows of an odd length whose output is stored past the caches, off the 16-byte boundaries."""
    c = _case((rows,), 250001, t, 21, groups=3, bias="table", past="ragged")
    _check(c, dict(presence=0.3, frequency=0.2, temperature=0.8), False)


def test_more_elements_than_32_bits_count():
    """Rows behind the 2^31st element; sums of ones are exact."""
    fa = _fa()
    rows, n = 480, 4_600_001
    x = torch.empty(rows, n, device="cuda").normal_().requires_grad_(True)
    ok = torch.rand(n, device="cuda") < 0.5
    bias = torch.randn(n, device="cuda").requires_grad_(True)
    out = fa.constrain_logits(x, allowed=ok, bias=bias)
    for i in (0, 300, rows - 1):
        assert torch.equal(out[i], torch.where(ok, x[i] + bias, -math.inf))
    dx, db = torch.autograd.grad(out, [x, bias], torch.ones_like(out))
    for i in (0, 300, rows - 1):
        assert torch.equal(dx[i], ok.float())
    assert torch.equal(db, ok.float() * rows)


@pytest.mark.parametrize("rows,inner,groups", [(70, 1, 3), (72, 8, 40), (69, 3, 20)])
def test_long_rows_by_their_bias(rows, inner, groups):
    """Large outputs with a table of biases: few, with steps of one owner, with owners of none, and too many to share."""
    c = _case((rows // inner, inner), 250001, torch.bfloat16, 22, groups=groups, bias="table", past=3)
    c["group"][::7] = groups
    _check(c, dict(presence=0.3, frequency=0.2, temperature=0.8), False)

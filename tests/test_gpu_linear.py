"""linear, relation_linear and group_rows against their definitions in 64
bits.

Tolerances are bounds, element by element, derived from the arithmetic.  With
u the operands' half step and e = 2^-24, a sum of K products in float32 is
off by at most (K + 16) e S, S the sum of the products' magnitudes (16 covers
the bias and, for float32 operands, the products dropped: below 3 * 2^-22 of
each).  An activation's slope is below 1.13 and its own evaluation off by at
most 16 e of 1 + |p|; every output is rounded once more (u).  The backward
keeps the activation's argument p and d = g act'(p) in the operands' type:
d is off by at most u |d| + |g| (2 u |p| + the error of p) (no second
derivative exceeds 1), and by |g| where relu's argument is nearer to 0 than
its error; then the same bound for the sums over d."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = [None, "relu", "gelu", "silu", "tanh", "sigmoid"]


def _fa():
    from flashlog_amd import attention
    return attention


def _half_step(t):
    return torch.finfo(t).eps / 2


def _tiny(t):
    return float(torch.finfo(t).smallest_normal) * torch.finfo(t).eps  # a subnormal step


def _act(p, act):
    """(value, slope) in 64 bits."""
    if act == "relu":
        return p.clamp(min=0), (p > 0).double()
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-p / 2 ** 0.5)
        return p * cdf, cdf + p * torch.exp(-p * p / 2) / (2 * np.pi) ** 0.5
    if act == "silu":
        q = torch.sigmoid(p)
        return p * q, q * (1 + p * (1 - q))
    if act == "tanh":
        return torch.tanh(p), 1 - torch.tanh(p) ** 2
    if act == "sigmoid":
        q = torch.sigmoid(p)
        return q, q * (1 - q)
    return p, torch.ones_like(p)


def _make(M, K, N, t, seed, groups=None, bias=True, residual=True, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    lead = () if groups is None else (groups,)
    x = torch.randn(M, K, generator=g).to(t)
    w = (torch.randn(*lead, N, K, generator=g) * scale / max(K, 1) ** 0.5).to(t)
    b = torch.randn(*lead, N, generator=g).to(t) if bias else None
    r = torch.randn(M, N, generator=g).to(t) if residual else None
    gy = torch.randn(M, N, generator=g).to(t)
    return x, w, b, r, gy


def _reference(x, w, b, r, gy, act, index=None):
    """Values and bounds: {name: (value, bound)} in 64 bits on the CPU."""
    t = x.dtype
    u, tiny = _half_step(t), _tiny(t)
    M, K = x.shape
    G = 1 if index is None else w.shape[0]
    w3 = w.double().reshape(G, -1, K)
    N = w3.shape[1]
    b3 = torch.zeros(G, N, dtype=torch.float64) if b is None else b.double().reshape(G, N)
    idx = torch.zeros(M, dtype=torch.long) if index is None else index
    x, gy = x.double(), gy.double()
    out = {k: torch.zeros(s, dtype=torch.float64) for k, s in
           (("y", (M, N)), ("dx", (M, K)), ("dw", (G, N, K)), ("db", (G, N)))}
    tol = {k: torch.zeros_like(v) for k, v in out.items()}
    for k in range(G):
        rows = (idx == k).nonzero()[:, 0]
        xr, wk = x[rows], w3[k]
        p = xr @ wk.T + b3[k]
        dp = (K + 16) * E * (xr.abs() @ wk.abs().T + b3[k].abs())
        v, slope = _act(p, act)
        out["y"][rows] = v
        tol["y"][rows] = 1.13 * dp + (16 * E * (1 + p.abs()) if act else 0)
        g = gy[rows]
        d = g * slope
        dd = torch.zeros_like(d)
        if act:
            dd = u * d.abs() + g.abs() * (2 * u * p.abs() + dp + 16 * E) + tiny
            if act == "relu":
                dd = torch.where(p.abs() <= dp, g.abs(), u * d.abs() + tiny)
        out["dx"][rows] = d @ wk
        tol["dx"][rows] = dd @ wk.abs() + (N + 16) * E * (d.abs() @ wk.abs())
        n = len(rows)
        out["dw"][k] = d.T @ xr
        tol["dw"][k] = dd.T @ xr.abs() + (n + 16) * E * (d.abs().T @ xr.abs())
        out["db"][k] = d.sum(0)
        tol["db"][k] = dd.sum(0) + (n + 16) * E * d.abs().sum(0)
    if r is not None:
        out["y"] += r.double()
        tol["y"] += E * out["y"].abs()
    shape = {"dw": w.shape, "db": w.shape[:-1]}
    return {k: (v.reshape(shape.get(k, v.shape)), (tol[k] + u * v.abs() * 1.01 + tiny).reshape(shape.get(k, v.shape)))
            for k, v in out.items()}


def _close(name, got, want, tol):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    assert torch.isfinite(got).all(), name
    bad = (got - want).abs() > tol
    assert not bad.any(), "%s: %d of %d off, worst %.3g of its bound" % (
        name, int(bad.sum()), bad.numel(), float(((got - want).abs() / tol).max()))


def _check(x, w, b, r, gy, act, index=None):
    fa = _fa()
    leaves = [t.cuda().requires_grad_(True) if t is not None else None for t in (x, w, b, r)]
    if index is None:
        call = lambda a: fa.linear(a[0], a[1], a[2], act, a[3])
    else:
        plan = fa.group_rows(index.cuda(), w.shape[0])
        call = lambda a: fa.relation_linear(a[0], plan, a[1], a[2], act, a[3])
    y = call(leaves)
    with torch.no_grad():
        assert torch.equal(call(leaves), y.detach())  # the same without a graph
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], gy.cuda())
    ref = _reference(x, w, b, r, gy, act, index)
    _close("y", y, *ref["y"])
    names = [n for n, t in zip(("dx", "dw", "db", "dr"), leaves) if t is not None]
    for n, g in zip(names, grads):
        if n == "dr":
            assert torch.equal(g.cpu(), gy)
        else:
            assert g.dtype == x.dtype
            _close(n, g, *ref[n])


SHAPES = [(1, 1, 1), (1, 64, 25), (3, 7, 5), (33, 100, 63), (96, 256, 475), (130, 65, 129), (257, 33, 260),
          (300, 512, 150)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_linear_shapes(shape, t):
    M, K, N = shape
    _check(*_make(M, K, N, t, M + K + N), act=None)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_linear_activations(act, t):
    _check(*_make(67, 48, 70, t, 3, scale=3.0), act=act)
    _check(*_make(67, 48, 70, t, 4, bias=False, residual=False), act=act)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", [(1100, 160, 1645), (4100, 140, 136), (2048, 1024, 75), (1, 2048, 1645)])
def test_linear_large_tiles(shape, t):
    """Enough rows and columns for the wide tiles, parts of the weight gradient's rows, one row of many inputs."""
    M, K, N = shape
    _check(*_make(M, K, N, t, 5), act="silu")


@pytest.mark.parametrize("t", TYPES[1:])
@pytest.mark.parametrize("shape", [(6100, 72, 2048), (6100, 2048, 72), (2000, 136, 2041), (2000, 2048, 264),
                                   (32800, 256, 200)])
def test_linear_half_precision_tiles(shape, t):
    """Shapes and alignments of the wide tiles: the forward, dx and dW of each, ends of K and of the columns."""
    M, K, N = shape
    _check(*_make(M, K, N, t, 15), act="relu")


@pytest.mark.parametrize("t", TYPES[1:])
@pytest.mark.parametrize("K,N", [(200, 1024), (264, 520)])
def test_relation_linear_half_precision_tiles(K, N, t):
    g = torch.Generator().manual_seed(1)
    index = torch.randint(-1, 4, (8200,), generator=g)
    index[2000:5000] = 3
    _check(*_make(8200, K, N, t, 16, groups=4), act="tanh", index=index)


def test_misaligned_gradient():
    """A contiguous gradient that begins inside a tensor, off the 16-byte boundaries."""
    fa = _fa()
    x, w, b, r, gy = _make(33000, 256, 200, torch.bfloat16, 17)
    flat = torch.zeros(33000 * 200 + 3, dtype=torch.bfloat16, device="cuda")
    flat[3:] = gy.cuda().view(-1)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = fa.linear(*leaves)
    for p, q in zip(torch.autograd.grad(y, leaves, flat[3:].view(33000, 200), retain_graph=True),
                    torch.autograd.grad(y, leaves, gy.cuda())):
        assert torch.equal(p, q)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,groups,K,N", [(1, 3, 8, 4), (96, 474, 32, 25), (50, 7, 100, 33), (700, 5, 130, 140),
                                             (513, 4, 129, 257)])
def test_relation_linear(rows, groups, K, N, t):
    g = torch.Generator().manual_seed(rows)
    index = torch.randint(groups, (rows,), generator=g)
    index[torch.rand(rows, generator=g) < 0.3] = groups // 2  # one large group; others may be empty
    _check(*_make(rows, K, N, t, 6, groups=groups), act="gelu", index=index)


@pytest.mark.parametrize("t", TYPES)
def test_relation_linear_rows_of_no_group(t):
    index = torch.tensor([2, -1, 0, 5, 2, 100, 0, 2, -7, 4] * 9)
    x, w, b, r, gy = _make(90, 40, 36, t, 7, groups=5)
    _check(x, w, b, r, gy, "sigmoid", index)
    fa = _fa()
    plan = fa.group_rows(index.cuda(), 5)
    y = fa.relation_linear(x.cuda(), plan, w.cuda(), b.cuda(), "sigmoid")
    assert (y.cpu()[(index < 0) | (index >= 5)] == 0).all()
    none = fa.group_rows(torch.full((90,), -1).cuda(), 5)
    wg = w.cuda().requires_grad_(True)
    xg = x.cuda().requires_grad_(True)
    y = fa.relation_linear(xg, none, wg, b.cuda(), "sigmoid", r.cuda())
    assert torch.equal(y.detach().cpu(), r)
    dx, dw = torch.autograd.grad(y, [xg, wg], gy.cuda())
    assert (dx == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("rows,groups", [(0, 3), (1, 1), (64, 5), (1000, 1644), (16384, 74), (16385, 74), (5000, 4095),
                                         (5000, 4096), (40000, 65534), (100_000, 2)])
def test_group_rows(rows, groups):
    rng = np.random.default_rng(rows + groups)
    index = rng.integers(-2, groups + 2, rows)
    plan = _fa().group_rows(torch.from_numpy(index).cuda(), groups)
    key = np.where((index < 0) | (index >= groups), groups, index)
    assert np.array_equal(plan.order.cpu().numpy(), np.argsort(key, kind="stable"))
    counts = np.bincount(key, minlength=groups + 1)
    assert np.array_equal(plan.offsets.cpu().numpy(), np.concatenate([[0], np.cumsum(counts)[:groups]]))
    # tiles: every place once, none across groups
    tiles = plan.tiles.cpu().numpy().reshape(-1, 2)
    tiles = tiles[tiles[:, 0] >= 0]
    begin = np.concatenate([[0], np.cumsum(counts)])
    from flashlog_amd import _lib
    block = _lib.lib().fl_group_block(rows, groups)
    want = [(g, p) for g in range(groups + 1) for p in range(begin[g], begin[g + 1], block)]
    assert tiles.tolist() == [list(map(int, t)) for t in want]


def test_index_types_and_shapes():
    fa = _fa()
    for t in (torch.int32, torch.int16, torch.int64, torch.uint8):
        plan = fa.group_rows(torch.tensor([[1, 0], [2, 1]], dtype=t).cuda(), 3)
        assert plan.order.tolist() == [1, 0, 3, 2]


@pytest.mark.parametrize("t", TYPES)
def test_strided_operands(t):
    """Rows and weights that are slices of larger tensors, transposed ones, and leading dimensions."""
    fa = _fa()
    x, w, b, r, gy = _make(42, 31, 29, t, 8)
    ref = _reference(x, w, b, r, gy, "tanh")
    wide = torch.zeros(42, 50, dtype=t).cuda()
    wide[:, 3:34] = x.cuda()
    wbig = torch.zeros(58, 40, dtype=t).cuda()
    wbig[::2, 1:32] = w.cuda()
    views = [(wide[:, 3:34], wbig[::2, 1:32]), (x.cuda().t().contiguous().t(), w.cuda().t().contiguous().t())]
    for xv, wv in views:
        xv, wv = xv.detach().requires_grad_(True), wv.detach().requires_grad_(True)
        rv = r.cuda().t().contiguous().t()
        y = fa.linear(xv.view(6, 7, 31) if xv.stride(1) == 1 else xv, wv, b.cuda(), "tanh",
                      rv.reshape(6, 7, 29) if xv.stride(1) == 1 else rv)
        _close("y", y.reshape(42, 29), *ref["y"])
        dx, dw = torch.autograd.grad(y, [xv, wv], gy.cuda().view(y.shape).transpose(0, 1).contiguous().transpose(0, 1))
        _close("dx", dx, *ref["dx"])
        _close("dw", dw, *ref["dw"])


def test_float32_bias_of_half_operands():
    fa = _fa()
    x, w, _, _, gy = _make(40, 30, 20, torch.bfloat16, 9)
    b = torch.randn(20, generator=torch.Generator().manual_seed(1))
    bg = b.cuda().requires_grad_(True)
    y = fa.linear(x.cuda(), w.cuda(), bg)
    (db,) = torch.autograd.grad(y, [bg], gy.cuda())
    assert db.dtype == torch.float32
    want = gy.double().sum(0)
    assert ((db.double().cpu() - want).abs() <= 56 * E * gy.double().abs().sum(0)).all()
    # an expanded gradient
    (db,) = torch.autograd.grad(fa.linear(x.cuda(), w.cuda(), bg).float().sum(), [bg])
    assert (db == 40).all()


@pytest.mark.parametrize("M,K,N", [(0, 5, 4), (5, 0, 4), (5, 4, 0)])
def test_empty(M, K, N):
    fa = _fa()
    x = torch.randn(M, K).cuda().requires_grad_(True)
    w = torch.randn(N, K).cuda().requires_grad_(True)
    b = torch.randn(N).cuda().requires_grad_(True)
    y = fa.linear(x, w, b, "silu")
    assert y.shape == (M, N)
    if K == 0:
        bb = b.detach().cpu()
        assert torch.allclose(y.detach().cpu(), torch.nn.functional.silu(bb).expand(M, N), rtol=1e-6)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.ones_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape and (dw == 0).all()
    plan = fa.group_rows(torch.zeros(M, dtype=torch.long).cuda(), 3)
    w3 = torch.randn(3, N, K).cuda().requires_grad_(True)
    y = fa.relation_linear(x, plan, w3)
    assert y.shape == (M, N)
    (dw,) = torch.autograd.grad(y, [w3], torch.ones_like(y))
    assert (dw == 0).all()


def test_magnitudes_of_float32():
    """Planes keep the exponent range: tiny, huge and mixed float32 values."""
    fa = _fa()
    g = torch.Generator().manual_seed(2)
    for sx, sw in ((1e-30, 1e10), (1e18, 1e15), (1e-10, 1e-15)):
        x, w = torch.randn(40, 50, generator=g) * sx, torch.randn(30, 50, generator=g) * sw
        y = fa.linear(x.cuda(), w.cuda()).double().cpu()
        want, s = x.double() @ w.double().T, x.double().abs() @ w.double().abs().T
        assert ((y - want).abs() <= 66 * E * s + 1e-37).all()


def test_non_finite_rows_stay_their_own():
    fa = _fa()
    x, w, b, _, _ = _make(200, 40, 150, torch.float32, 11)
    clean = fa.linear(x.cuda(), w.cuda(), b.cuda())
    x[17, 3], x[140, 5] = float("inf"), float("nan")
    y = fa.linear(x.cuda(), w.cuda(), b.cuda())
    keep = torch.ones(200, dtype=torch.bool)
    keep[[17, 140]] = False
    assert torch.equal(y[keep.cuda()], clean[keep.cuda()])
    assert not torch.isfinite(y[17]).any() and not torch.isfinite(y[140]).any()


def test_same_bits_every_time():
    fa = _fa()
    x, w, b, r, gy = _make(2000, 130, 75, torch.float32, 12, groups=9)
    index = torch.randint(9, (2000,), generator=torch.Generator().manual_seed(3)).cuda()
    runs = []
    for _ in range(3):
        leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
        y = fa.relation_linear(leaves[0], fa.group_rows(index, 9), leaves[1], leaves[2], "gelu")
        runs.append([y.detach()] + list(torch.autograd.grad(y, leaves, gy.cuda())))
    for other in runs[1:]:
        for a, b_ in zip(runs[0], other):
            assert torch.equal(a, b_)


def test_refusals():
    fa = _fa()
    x, w = torch.randn(4, 5).cuda(), torch.randn(3, 5).cuda()
    plan = fa.group_rows(torch.zeros(4, dtype=torch.long).cuda(), 2)
    for exc, call in [
        (RuntimeError, lambda: fa.linear(x.cpu(), w)),
        (RuntimeError, lambda: fa.linear(x, w, torch.zeros(3))),
        (TypeError, lambda: fa.linear(x.double(), w.double())),
        (TypeError, lambda: fa.linear(x, w.half())),
        (TypeError, lambda: fa.linear(x, w, torch.zeros(3, dtype=torch.half).cuda())),
        (ValueError, lambda: fa.linear(x, w[:, :4])),
        (ValueError, lambda: fa.linear(x, w[None])),
        (ValueError, lambda: fa.linear(x, w, torch.zeros(4).cuda())),
        (ValueError, lambda: fa.linear(x, w, activation="softmax")),
        (ValueError, lambda: fa.linear(x, w, residual=torch.zeros(4, 4).cuda())),
        (TypeError, lambda: fa.relation_linear(x, torch.zeros(4), w[None])),
        (ValueError, lambda: fa.relation_linear(x, plan, w)),
        (ValueError, lambda: fa.relation_linear(x, plan, w[None])),
        (ValueError, lambda: fa.relation_linear(x[:3], plan, torch.randn(2, 3, 5).cuda())),
        (TypeError, lambda: fa.group_rows(torch.zeros(4).cuda(), 2)),
        (ValueError, lambda: fa.group_rows(torch.zeros(4, dtype=torch.long).cuda(), 0)),
    ]:
        with pytest.raises(exc):
            call()
    xg = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(fa.linear(xg, w, activation="tanh").sum(), [xg], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_another_stream_and_graph():
    """A side stream, then captured and replayed with new inputs, forward and backward."""
    fa = _fa()
    x, w, b, r, gy = (t.cuda() for t in _make(300, 64, 75, torch.float32, 13, groups=6))
    index = torch.randint(6, (300,), generator=torch.Generator().manual_seed(4)).cuda()

    def step(x, w, b, gy, index):
        x, w, b = (t.detach().requires_grad_(True) for t in (x, w, b))
        y = fa.relation_linear(x, fa.group_rows(index, 6), w, b, "tanh")
        return [y.detach()] + list(torch.autograd.grad(y, [x, w, b], gy))

    want = step(x, w, b, gy, index)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, w, b, gy, index)
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(want, got):
        assert torch.equal(p, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, w, b, gy, index)
    for k in range(3):
        x.copy_(torch.randn(300, 64, generator=torch.Generator().manual_seed(20 + k)))
        index.copy_(torch.randint(-1, 7, (300,), generator=torch.Generator().manual_seed(30 + k)))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(step(x, w, b, gy, index), out):
            assert torch.equal(p, q)


@pytest.mark.parametrize("t", TYPES[1:])
@pytest.mark.parametrize("groups,rows,sort", [(11, 8200, False), (24, 12300, True)])
def test_relation_linear_groups_over_xcds(groups, rows, sort, t):
    """More groups than XCDs, not a multiple of them: skewed, with empty ones, in parts of the rows."""
    g = torch.Generator().manual_seed(2)
    index = (torch.rand(rows, generator=g) ** 2 * (groups + 1)).long() - 1
    index[index == 3] = 4
    index = index.sort().values if sort else index
    _check(*_make(rows, 264, 520, t, 18, groups=groups), act="silu", index=index)


def test_more_elements_than_32_bits_count():
    """Rows behind the 2^31st element of x, dx and the gradient: the last rows and the first, zeros between them."""
    fa = _fa()
    M, K, N = 1_100_000, 2048, 256
    x0, w, _, _, g0 = _make(128, K, N, torch.bfloat16, 19, bias=False, residual=False)
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    gy = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    ends = torch.cat([torch.arange(64), torch.arange(M - 64, M)]).cuda()
    x[ends], gy[ends] = x0.cuda(), g0.cuda()
    x.requires_grad_(True)
    wg = w.cuda().requires_grad_(True)
    y = fa.linear(x, wg)
    dx, dw = torch.autograd.grad(y, [x, wg], gy)
    ref = _reference(x0, w, None, None, g0, None, None)
    _close("y", y[ends], *ref["y"])
    _close("dx", dx[ends], *ref["dx"])
    _close("dw", dw, *ref["dw"])
    assert not y[64:M - 64].any() and not dx[64:M - 64].any()

"""layer_norm against its definition in 64 bits.

Tolerances are bounds, element by element, derived from the arithmetic.  With
e = 2^-24, u the half step of an output's type and d = N / 256 + 80 a bound of
the additions that any value of a row's sum goes through: the mean is off by at
most d e mean|x|, x - mean by that and its own rounding, the variance by
2 mean(|c| dc) + d e var, its root's reciprocal by half of that relative to
var + eps and 4 e, and so on through the formulas; sums over the rows go
through at most M + 16 additions."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _fa():
    from flashlog_amd import attention
    return attention


def _tiny(t):
    return float(torch.finfo(t).smallest_normal) * torch.finfo(t).eps


def _make(M, N, t, seed, wide=False, offset=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, N, generator=g) * 1.5 + offset * torch.randn(M, 1, generator=g)).to(t)
    wt = torch.float32 if wide else t
    w, b = (1 + 0.3 * torch.randn(N, generator=g)).to(wt), torch.randn(N, generator=g).to(wt)
    return x, w, b, torch.randn(M, N, generator=g).to(t)


def reference(x, w, b, gy, eps=1e-5):
    """{name: (value, bound)} in 64 bits."""
    t = x.dtype
    wt = t if w is None else w.dtype
    u, uw = torch.finfo(t).eps / 2, torch.finfo(wt).eps / 2
    x, gy = x.double(), gy.double()
    M, N = x.shape
    d = N / 256 + 80
    w = torch.ones(N, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()

    def mean(v):
        return v.mean(1, keepdim=True)

    mu = mean(x)
    c = x - mu
    dc = d * E * mean(x.abs()) + E * c.abs()
    var = mean(c * c)
    dvar = 2 * mean(c.abs() * dc) + mean(dc * dc) + d * E * var
    r = 1 / (var + eps).sqrt()
    rel = dvar / (2 * (var + eps)) + 4 * E
    h = c * r
    dh = dc * r + h.abs() * (rel + E)
    y = h * w + b
    v = gy * w
    m1, m2 = mean(v), mean(v * h)
    dm1 = (d + 2) * E * mean(v.abs())
    dm2 = mean(v.abs() * dh) + (d + 2) * E * mean((v * h).abs())
    part = v - m1 - h * m2
    dx = r * part
    ddx = r * (dm1 + dh * m2.abs() + h.abs() * dm2 + 4 * E * (v.abs() + m1.abs() + (h * m2).abs())) + rel * dx.abs()
    dw, db = (gy * h).sum(0), gy.sum(0)
    rows = (M + 16) * E
    out = {"y": (y, w.abs() * dh + 3 * E * ((h * w).abs() + b.abs()) + u * y.abs()),
           "dx": (dx, ddx + u * dx.abs()),
           "dw": (dw, (gy.abs() * dh).sum(0) + rows * (gy * h).abs().sum(0) + uw * dw.abs()),
           "db": (db, rows * gy.abs().sum(0) + uw * db.abs())}
    return {k: (p, 1.01 * q + _tiny(t if k in ("y", "dx") else wt)) for k, (p, q) in out.items()}


def _held(got, want, what):
    value, bound = want
    got = got.double().cpu().reshape(value.shape)
    assert torch.isfinite(got).all(), what
    over = (got - value.cpu()).abs() - bound.cpu()
    assert (over <= 0).all(), "%s: off by %.3g more than allowed" % (what, over.max())


def _run(x, w, b, gy, eps=1e-5):
    leaves = [v.cuda().requires_grad_(True) if v is not None else None for v in (x, w, b)]
    y = _fa().layer_norm(*leaves, eps)
    grads = torch.autograd.grad(y, [v for v in leaves if v is not None], gy.cuda().reshape(y.shape))
    named = dict(zip([n for n, v in zip(("dx", "dw", "db"), leaves) if v is not None], grads))
    return {"y": y.detach(), **named}


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N", [(1, 1), (1, 25), (3, 2), (5, 63), (4, 64), (7, 256), (130, 475), (96, 512), (2, 1000),
                                 (33, 1645), (300, 2048), (9, 2049), (5, 4096), (3, 5001), (2, 8192), (3, 8193),
                                 (40, 20000), (2500, 40)])
def test_against_the_definition(M, N, t):
    x, w, b, gy = _make(M, N, t, M * 7919 + N)
    ref = reference(x, w, b, gy)
    out = _run(x, w, b, gy)
    for k, v in out.items():
        _held(v, ref[k], k)


@pytest.mark.parametrize("t", TYPES[1:])
@pytest.mark.parametrize("M,N", [(37, 300), (5, 3001), (6, 9000)])
def test_wide_weights(M, N, t):
    x, w, b, gy = _make(M, N, t, 3, wide=True)
    ref, out = reference(x, w, b, gy), _run(x, w, b, gy)
    assert out["dw"].dtype is torch.float32 and out["y"].dtype is t
    for k, v in out.items():
        _held(v, ref[k], k)


@pytest.mark.parametrize("given", ["neither", "weight", "bias"])
def test_weight_and_bias_are_optional(given):
    x, w, b, gy = _make(21, 130, torch.float32, 5)
    w, b = w if given == "weight" else None, b if given == "bias" else None
    ref = reference(x, w, b, gy)
    for k, v in _run(x, w, b, gy).items():
        _held(v, ref[k], k)


def test_far_mean():
    """Values whose mean is far larger than their spread."""
    x, w, b, gy = _make(9, 700, torch.float32, 6)
    x = x + 1000.0
    ref = reference(x, w, b, gy)
    for k, v in _run(x, w, b, gy).items():
        _held(v, ref[k], k)


def test_constant_rows():
    x = torch.full((3, 200), 0.7)
    y = _fa().layer_norm(x.cuda(), eps=1e-5).cpu()
    # the mean of equal values is off by d e of them at most, over sqrt(eps)
    assert (y.abs() <= 81 * E * 0.7 / 1e-5 ** 0.5 * 1.01).all()


@pytest.mark.parametrize("t", TYPES)
def test_strides_and_alignment(t):
    x, w, b, gy = _make(12, 301, t, 8)
    ref = reference(x, w, b, gy)
    base = torch.zeros(12, 2 * 301 + 7, dtype=t)
    base[:, 3:304] = x
    views = [base.cuda()[:, 3:304], x.t().contiguous().cuda().t(), x.reshape(3, 4, 301).cuda()]
    for v in views:
        y = _fa().layer_norm(v, w.cuda(), b.cuda())
        assert y.shape == v.shape
        _held(y, ref["y"], "y")
    leaf = base.cuda().requires_grad_(True)
    y = _fa().layer_norm(leaf[:, 3:304], w.cuda(), b.cuda())
    # a gradient that is not contiguous
    g = torch.autograd.grad(y, leaf, gy.t().contiguous().cuda().t())[0]
    _held(g[:, 3:304], ref["dx"], "dx")
    assert (g[:, :3] == 0).all() and (g[:, 304:] == 0).all()


def test_no_rows_no_columns():
    w = torch.ones(5, device="cuda", requires_grad=True)
    x = torch.zeros(0, 5, device="cuda", requires_grad=True)
    y = _fa().layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 5) and (dw == 0).all()
    assert _fa().layer_norm(torch.zeros(3, 0, device="cuda")).shape == (3, 0)


def test_not_finite_rows_stay_apart():
    x, w, b, gy = _make(6, 600, torch.float32, 9)
    bad = x.clone()
    bad[1, 5], bad[4, 599] = float("nan"), float("inf")
    good, out = _run(x, w, b, gy), _run(bad, w, b, gy)
    rows = [0, 2, 3, 5]
    for k in ("y", "dx"):
        assert torch.equal(out[k][rows], good[k][rows]) and out[k][[1, 4]].isnan().all()


def test_only_some_gradients():
    x, w, b, gy = _make(50, 333, torch.bfloat16, 10)
    ref = reference(x, w, b, gy)
    for names in (["dx"], ["dw"], ["db"], ["dw", "db"], ["dx", "db"]):
        leaves = {k: v.cuda().requires_grad_(k in names) for k, v in (("dx", x), ("dw", w), ("db", b))}
        y = _fa().layer_norm(*leaves.values())
        for k, g in zip(names, torch.autograd.grad(y, [leaves[k] for k in names], gy.cuda())):
            _held(g, ref[k], k)


def test_same_bits_and_other_streams():
    x, w, b, gy = _make(3000, 1024, torch.bfloat16, 11)
    first = _run(x, w, b, gy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _run(x, w, b, gy)
    side.synchronize()
    for k in first:
        assert torch.equal(first[k], again[k])


def test_gradient_against_differences():
    """In one direction, central differences of the definition in 64 bits."""
    x, w, b, gy = _make(4, 37, torch.float32, 12)
    out = _run(x, w, b, gy)
    g = torch.Generator().manual_seed(1)
    for name, v in (("dx", x), ("dw", w), ("db", b)):
        way = torch.randn(v.shape, generator=g).double()
        step = 1e-5

        def value(at):
            a = {"dx": x.double(), "dw": w.double(), "db": b.double()}
            a[name] = a[name] + at * step * way
            c = a["dx"] - a["dx"].mean(1, keepdim=True)
            y = c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt() * a["dw"] + a["db"]
            return (y * gy.double()).sum()

        slope = (value(1) - value(-1)) / (2 * step)
        got = (out[name].double().cpu() * way).sum()
        # differences: third derivatives times step^2 (1e-10) and 1e-16 / step of the sum; the gradient: its bound
        bound = (reference(x, w, b, gy)[name][1] * way.abs()).sum() + 1e-7 * gy.abs().sum()
        assert (slope - got).abs() <= bound, name


def test_captured_forward_and_backward():
    x, w, b, gy = (v.cuda() for v in _make(200, 700, torch.bfloat16, 13))
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b)]

    def step():
        y = _fa().layer_norm(*leaves)
        return (y, *torch.autograd.grad(y, leaves, gy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        with torch.no_grad():
            leaves[0].copy_(x * (k + 1) + 0.1)
        torch.ones(1000, device="cuda").sum().item()
        graph.replay()
        torch.cuda.synchronize()
        fresh = [v.detach().clone().requires_grad_(True) for v in leaves]
        y = _fa().layer_norm(*fresh)
        for a, c in zip(held, (y, *torch.autograd.grad(y, fresh, gy))):
            assert torch.equal(a, c)


def test_rows_behind_two_gigabytes():
    """Elements behind the 2^31st."""
    N = 8192
    M = (1 << 31) // N + 3
    x = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    tail = torch.randn(4, N, generator=g, device="cuda").bfloat16()
    x[-4:] = tail
    y = _fa().layer_norm(x)
    ref = reference(tail.cpu(), None, None, tail.cpu())
    _held(y[-4:], ref["y"], "y")
    assert (y[:2] == 0).all()


def test_refusals():
    fa = _fa()
    x = torch.zeros(2, 3, device="cuda")
    for error, call in ((TypeError, lambda: fa.layer_norm(x.double())),
                        (TypeError, lambda: fa.layer_norm(x, x[0].half())),
                        (TypeError, lambda: fa.layer_norm(x.half(), x[0].half(), x[0])),
                        (ValueError, lambda: fa.layer_norm(x, x[0, :2])),
                        (ValueError, lambda: fa.layer_norm(x, x)),
                        (ValueError, lambda: fa.layer_norm(x, eps=-1.0)),
                        (ValueError, lambda: fa.layer_norm(x, eps=float("nan"))),
                        (ValueError, lambda: fa.layer_norm(x[0, 0])),
                        (RuntimeError, lambda: fa.layer_norm(x, x[0].cpu()))):
        with pytest.raises(error):
            call()
    leaf = x.clone().requires_grad_(True)
    first = torch.autograd.grad(fa.layer_norm(leaf).sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), leaf)

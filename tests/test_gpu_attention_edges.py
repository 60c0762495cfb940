"""Calls of the attention operators that their documentation allows at the
ends of their ranges: no rows, non-finite values beside masks and in
gradients, more work items than one dimension of a launch holds."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALVES = [torch.bfloat16, torch.float16]


def _fa():
    from flashlog_amd import attention
    return attention


@pytest.mark.parametrize("n", [7, 3000])
@pytest.mark.parametrize("softmax", [False, True])
def test_no_rows_with_tables(softmax, n):
    """An empty batch beside tables of several rows: empty outputs, a zero gradient for the biases."""
    fa = _fa()
    fn = fa.hop_attention if softmax else fa.constrain_logits
    group = torch.zeros(0, dtype=torch.long, device="cuda")
    allowed = torch.ones(3, n, dtype=torch.bool, device="cuda")
    for lead in ((0,), (0, 4)):
        x = torch.zeros(*lead, n, device="cuda", requires_grad=True)
        b = torch.randn(3, n, device="cuda", requires_grad=True)
        y = fn(x, allowed=allowed, group=group, bias=b)
        assert y.shape == x.shape
        gx, gb = torch.autograd.grad(y, [x, b], torch.ones_like(y))
        assert gx.shape == x.shape and gb.shape == b.shape and not gb.any()


def test_ranks_of_no_queries():
    from flashlog_amd import evaluation as ev
    hits = np.zeros(10)
    none = torch.zeros(0, dtype=torch.long, device="cuda")
    mrr = ev.calculate_hits_constrained(torch.zeros(0, 50, device="cuda"), [], (none, none), hits,
                                        allowed=torch.ones(3, 50, dtype=torch.bool, device="cuda"))
    assert mrr == 0 and not hits.any()


@pytest.mark.parametrize("groups", [1, 4095, 4096, 65534, (1 << 24) - 1])
def test_no_rows_in_many_groups(groups):
    """Every group of no rows begins at 0, however many passes more rows would take."""
    fa = _fa()
    none = torch.zeros(0, dtype=torch.long, device="cuda")
    plan = fa.group_rows(none, groups)
    assert plan.order.numel() == 0 and plan.tiles.numel() == 0
    assert plan.offsets.shape == (groups + 1,) and not plan.offsets.any()
    off, ids = fa.history_from_pairs(none, none, groups)
    assert off.shape == (groups + 1,) and not off.any() and ids.numel() == 0


def test_no_rows_beside_a_large_bias_table():
    fa = _fa()
    x = torch.zeros(0, 6, device="cuda", requires_grad=True)
    b = torch.randn(5000, 6, device="cuda", requires_grad=True)
    w = fa.hop_attention(x, group=torch.zeros(0, dtype=torch.long, device="cuda"), bias=b)
    gx, gb = torch.autograd.grad(w, [x, b], torch.ones_like(w))
    assert gx.shape == (0, 6) and gb.shape == b.shape and not gb.any()


def test_mask_of_more_than_2_to_the_32_entries():
    fa = _fa()
    rows, n = 65537, 65600
    base = torch.rand(n, device="cuda") < 0.5
    turn = torch.arange(rows, device="cuda") % 3 == 1
    words = fa.pack_allowed(base[None] ^ turn[:, None])
    assert words.shape == (rows, n // 32)
    for rest, row in ((~turn, base), (turn, ~base)):
        want = fa.pack_allowed(row)
        got = words[rest]
        assert (got == want).all()
    bits = (fa.pack_allowed(base)[:, None] >> torch.arange(32, device="cuda")) & 1
    assert torch.equal(bits.reshape(-1).bool(), base)


@pytest.mark.parametrize("softmax", [False, True])
def test_rows_of_more_than_2_to_the_32_work_items(softmax):
    """A wave a row: rows behind the 2^26th, forward and backward, with the sums of a bias."""
    fa = _fa()
    rows, n = (1 << 26) + 77, 3
    x = torch.zeros(rows, n, device="cuda")
    g = torch.Generator().manual_seed(3)
    at = torch.tensor([0, 5, 1 << 25, (1 << 26) - 1, 1 << 26, (1 << 26) + 1, rows - 1]).cuda()
    x[at] = torch.randn(len(at), n, generator=g).cuda()
    bias = torch.randn(n, generator=g).cuda()
    gy = torch.zeros(rows, n, device="cuda")
    gy[at] = torch.randn(len(at), n, generator=g).cuda()
    fn = fa.hop_attention if softmax else fa.constrain_logits

    def run(x, gy):
        x, b = x.detach().requires_grad_(True), bias.detach().requires_grad_(True)
        y = fn(x, bias=b)
        return [y.detach(), *torch.autograd.grad(y, [x, b], gy)]

    many, few = run(x, gy), run(x[at], gy[at])
    assert torch.equal(many[0][at], few[0]) and torch.equal(many[1][at], few[1])
    rest = fn(torch.zeros(1, n, device="cuda"), bias=bias)
    same = (many[0] == rest).all(1)
    same[at] = True
    assert same.all()
    assert int(torch.count_nonzero(many[1].any(1))) <= len(at)
    bound = 2 * (len(at) + 8) * E * few[1].double().abs().sum(0)
    assert ((many[2].double() - few[1].double().sum(0)).abs() <= bound).all()


@pytest.mark.parametrize("n", [30, 1500, 9000])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_masked_columns_are_zero_beside_bad_values(bad, n):
    """A NaN or an infinity among the allowed logits does not reach the masked columns."""
    fa = _fa()
    g = torch.Generator().manual_seed(n)
    x = torch.randn(4, n, generator=g).cuda()
    ok = (torch.rand(n, generator=g) < 0.5).cuda()
    ok[n // 2] = True
    x[1, n // 2] = bad
    w = fa.hop_attention(x, allowed=ok)
    assert (w[:, ~ok] == 0).all()
    assert torch.isnan(w[1, n // 2])
    clean = fa.hop_attention(x[[0, 2, 3]], allowed=ok)
    assert torch.equal(w[[0, 2, 3]], clean)


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad
    fa = _fa()
    x, w, b, r = torch.randn(4, 5).cuda(), torch.randn(3, 5).cuda(), torch.randn(3).cuda(), torch.randn(4, 3).cuda()
    plan = fa.group_rows(torch.zeros(4, dtype=torch.long).cuda(), 1)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: fa.linear(dual(x), w), lambda: fa.linear(x, dual(w)), lambda: fa.linear(x, w, dual(b)),
                 lambda: fa.linear(x, w, residual=dual(r)), lambda: fa.relation_linear(dual(x), plan, w[None]),
                 lambda: fa.constrain_logits(dual(x)), lambda: fa.constrain_logits(x, bias=dual(x[0].clone())),
                 lambda: fa.hop_attention(dual(x)), lambda: fa.hop_attention(x, bias=dual(x[0].clone()))]
        for call in calls:
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    call()
        assert fa.linear(x, w).shape == (4, 3)


def _slope(p, act):
    if act == "relu":
        return (p > 0).double()
    if act == "gelu":
        return 0.5 * torch.erfc(-p / 2 ** 0.5) + p * torch.exp(-p * p / 2) / (2 * math.pi) ** 0.5
    if act == "tanh":
        return 1 - torch.tanh(p) ** 2
    q = torch.sigmoid(p)
    return q * (1 + p * (1 - q))


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("act", ["relu", "gelu", "silu", "tanh"])
@pytest.mark.parametrize("M,N,groups", [(24, 512, None), (24, 70, None), (120, 520, 5), (200, 520, 5),
                                        (120, 70, 5)])
def test_bias_gradient_adds_unrounded_terms(M, N, groups, act, t):
    """A float32 bias of half-precision operands: neither the activation's argument nor d = g act'(p) is rounded to
    the operands' type on the way.  The bound has, besides the sum's own, only the argument's float32 error (no
    second derivative exceeds 1) and 16 e of the slope's evaluation."""
    K = 8
    fa = _fa()
    g = torch.Generator().manual_seed(N)
    G = groups or 1
    x, w = torch.randn(M, K, generator=g).to(t), (torch.randn(G, N, K, generator=g) / K ** 0.5).to(t)
    b, gy = torch.randn(G, N, generator=g), torch.randn(M, N, generator=g).to(t)
    index = torch.randint(-1, G, (M,), generator=g) if groups else torch.zeros(M, dtype=torch.long)
    index[index == 3] = 2  # an empty group
    leaf = b.cuda().requires_grad_(True)
    if groups:
        y = fa.relation_linear(x.cuda(), fa.group_rows(index.cuda(), G), w.cuda(), leaf, act)
    else:
        y = fa.linear(x.cuda(), w[0].cuda(), leaf[0], act)
    (db,) = torch.autograd.grad(y, [leaf], gy.cuda())
    for k in range(G):
        rows = (index == k).nonzero()[:, 0]
        xr, wk, gr = x[rows].double(), w[k].double(), gy[rows].double()
        p = xr @ wk.T + b[k].double()
        dp = (K + 16) * E * (xr.abs() @ wk.abs().T + b[k].abs().double())
        d = gr * _slope(p, act)
        off = gr.abs() * (dp + 16 * E)
        if act == "relu":
            off = torch.where(p.abs() <= dp, gr.abs(), 0.0)
        bound = off.sum(0) + (len(rows) + 16) * E * d.abs().sum(0)
        assert ((db[k].double().cpu() - d.sum(0)).abs() <= bound).all()


@pytest.mark.parametrize("n", [40, 9000])
def test_rows_with_nothing_left_have_no_gradient(n):
    """Nor have single columns of weight 0: what comes back for them may be anything."""
    fa = _fa()
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, n, generator=g)
    x[1] = -math.inf
    x[2, : n // 2] = -math.inf
    gy = torch.randn(4, n, generator=g)
    for bias in (None, torch.zeros(n)):
        clean = gy.clone()
        dirty = gy.clone()
        clean[2, : n // 2] = 0
        dirty[1] = torch.tensor([math.nan, math.inf, -math.inf, 1.0])[torch.arange(n) % 4]
        dirty[2, : n // 2] = math.nan
        out = []
        for up in (clean, dirty):
            leaves = [x.cuda().requires_grad_(True)] + ([] if bias is None else [bias.cuda().requires_grad_(True)])
            w = fa.hop_attention(leaves[0], bias=leaves[1] if bias is not None else None)
            out.append(torch.autograd.grad(w, leaves, up.cuda()))
        assert (out[1][0][1] == 0).all()
        for p, q in zip(*out):
            assert torch.equal(p, q)


def test_scalars_out_of_float32():
    fa = _fa()
    x = torch.zeros(2, 5).cuda()
    for kw in (dict(temperature=1e39), dict(temperature=1e-39), dict(repetition=1e39), dict(repetition=1e-40),
               dict(presence=1e39), dict(frequency=-1e39)):
        for fn in (fa.constrain_logits, fa.hop_attention):
            with pytest.raises(ValueError):
                fn(x, **kw)


def test_history_of_a_count_of_rows():
    fa = _fa()
    rows, ids = torch.tensor([0, 2, 0]).cuda(), torch.tensor([7, 8, 9]).cuda()
    for count in (-1, -2):
        with pytest.raises(ValueError):
            fa.history_from_pairs(rows, ids, count)
    off, got = fa.history_from_pairs(rows, ids, 0)
    assert off.tolist() == [0]
    assert fa.constrain_logits(torch.zeros(0, 20).cuda(), history=(off, got), presence=1.0).shape == (0, 20)
    off, got = fa.history_from_pairs(rows, ids, 1)
    assert off.tolist() == [0, 2] and got[:2].tolist() == [7, 9]


def test_products_of_float32():
    """Single products: what the planes drop is below 2^-22 of each (values whose lower planes are all ones are the
    worst), the last addition is off by at most a step of 2^-23, those before it by 2^-28 in all."""
    g = torch.Generator().manual_seed(8)
    low = torch.randint(1 << 23, (2048,), generator=g)
    low[:700] |= 0xFFFF
    low[:300] = 0xFFFF
    low[:300] += torch.arange(300) << 14
    bits = low | 127 << 23
    x = bits.to(torch.int32).view(torch.float32)
    big = torch.tensor([torch.finfo(torch.float32).max, -torch.finfo(torch.float32).max, 3.3961e38])
    y = _fa().linear(x[:, None].cuda(), x[:512, None].cuda()).double().cpu()
    want = x.double()[:, None] * x.double()[None, :512]
    assert ((y - want).abs() <= (2.0 ** -22 + 2.0 ** -23 + 2.0 ** -28) * want).all()
    assert torch.equal(_fa().linear(big[:, None].cuda(), torch.ones(1, 1).cuda())[:, 0].cpu(), big)


@pytest.mark.parametrize("t", HALVES)
def test_bias_gradient_of_groups_captured(t):
    """Activation's gradient and column sums of gathered rows in one pass: the same bits every time, and in a graph
    that is replayed on other rows and groups beside eager work."""
    fa = _fa()
    g = torch.Generator().manual_seed(6)
    x, w = torch.randn(400, 40, generator=g).to(t).cuda(), (torch.randn(6, 515, 40, generator=g) / 6).to(t).cuda()
    b, gy = torch.randn(6, 515, generator=g).cuda(), torch.randn(400, 515, generator=g).to(t).cuda()
    index = torch.randint(-1, 7, (400,), generator=g).cuda()

    def step():
        leaves = [v.detach().requires_grad_(True) for v in (x, w, b)]
        y = fa.relation_linear(leaves[0], fa.group_rows(index, 6), leaves[1], leaves[2], "gelu")
        return [y.detach(), *torch.autograd.grad(y, leaves, gy)]

    first = step()
    for _ in range(2):
        for p, q in zip(first, step()):
            assert torch.equal(p, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        h = torch.Generator().manual_seed(60 + k)
        x.copy_(torch.randn(400, 40, generator=h))
        index.copy_(torch.randint(-1, 7, (400,), generator=h))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(want, out):
            assert torch.equal(p, q)


def test_as_many_rows_as_a_plan_takes():
    """2^31 - 1 rows, all but three in one group: its tiles are counted past 2^31 - 256 rows too."""
    fa = _fa()
    rows = (1 << 31) - 1
    index = torch.zeros(rows, dtype=torch.long, device="cuda")
    index[[5, 1 << 30, rows - 1]] = -1
    plan = fa.group_rows(index, 1)
    del index
    assert plan.offsets.tolist() == [0, rows - 3]
    assert plan.order[-4:].tolist() == [rows - 2, 5, 1 << 30, rows - 1]
    assert plan.order[4:6].tolist() == [4, 6]
    tiles = plan.tiles.view(-1, 2)
    n = (rows - 3 + 255) // 256
    assert not tiles[:n, 0].any() and torch.equal(tiles[:n, 1].long(), 256 * torch.arange(n, device="cuda"))
    assert tiles[n:].tolist()[0] == [1, rows - 3] and (tiles[n + 1:, 0] == -1).all()

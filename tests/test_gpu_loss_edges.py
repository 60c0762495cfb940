"""Calls of the losses that the documentation allows at the ends of their ranges."""
import pytest
import torch

from test_gpu_losses import _held, _rows, _tiny

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _losses():
    from flashlog_amd import losses
    return losses


def _make(M, K, V, t, seed, k=1, bias=True, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).to(t)
    w = (torch.randn(V, K, generator=g) * spread / max(K, 1) ** 0.5).to(t)
    b = torch.randn(V, generator=g).to(t) if bias else None
    ids = torch.randint(0, V, (M, k), generator=g)
    return x, w, b, ids, 2 * torch.randn(M, k, generator=g), 0.5 + torch.rand(M, generator=g)


def _run(x, w, b, ids, teacher, g, tau=1.0):
    """{name: losses and gradients} of cross entropy (teacher None) or distillation."""
    leaves = [v.cuda().requires_grad_(True) for v in (x, w, b) if v is not None]
    bias = leaves[2] if b is not None else None
    if teacher is None:
        loss = _losses().linear_cross_entropy(leaves[0], leaves[1], ids[..., 0].cuda(), bias)
    else:
        loss = _losses().linear_distillation(leaves[0], leaves[1], ids.cuda(), teacher.cuda(), bias, temperature=tau)
    grads = torch.autograd.grad(loss, leaves, g.cuda())
    return {"loss": loss.detach(), **dict(zip(("dx", "dw", "db"), grads))}


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,V", [(8, 24, 41000), (64, 256, 41000), (300, 64, 41000), (3, 0, 41000)])
def test_no_ids_over_a_large_vocabulary(M, K, V, t):
    """Nothing is listed: losses of 0 without gradients, at every number of parts of the vocabulary."""
    x, w, b, ids, teacher, g = _make(M, K, V, t, 1, k=0)
    out = _run(x, w, b, ids, teacher, g)
    assert out["loss"].shape == (M,) and out["dx"].shape == x.shape and out["dw"].shape == w.shape
    assert all((v == 0).all() for v in out.values())
    with torch.no_grad():
        loss = _losses().linear_distillation(x.cuda(), w.cuda(), ids.cuda(), teacher.cuda())
    assert (loss == 0).all()


#: By the plain tiles and by the wide ones (float32 in training from 256 rows and 2^30 products of two values on,
#: bfloat16 always).
ROWS = [(9, 40, 90), (60, 64, 500), (300, 128, 4000), (136, 256, 4100), (300, 256, 14100)]


@pytest.mark.parametrize("M,K,V", ROWS)
@pytest.mark.parametrize("offset", [0.0, 100.0, -4000.0, 4000.0])
def test_shares_add_up_beside_a_common_offset(M, K, V, offset):
    """sum(p) - 1 of every row, as the sum of the bias's gradient.  A share is off by 8 e (1 + its distance from the
    largest) in the backward and once more in the forward's sum, of terms that are added by lanes (V / 16 at most one
    after the other), waves and parts (64 steps); the column sums have M terms."""
    x, w, b, ids, _, g = _make(M, K, V, torch.float32, 7)
    b = b + offset  # rounded: the reference takes what is left
    ref_z = x.double() @ w.double().T + b.double()
    p = torch.softmax(ref_z, 1)
    off = (p * 16 * E * (1 + ref_z.amax(1, keepdim=True) - ref_z)).sum(1) + (V / 16 + 64) * E
    out = _run(x, w, b, ids, None, g)
    bound = (g * off).sum() + (M + 16) * E * 2 * g.sum()
    assert out["db"].double().sum().abs().item() <= bound.item()


def _reference(x, w, b, ids, g):
    """{name: (value, bound)} of cross entropy in 64 bits.  As in test_gpu_losses, but that nothing is lost relative to
    another row's or another column's values: what float32 holds is off by 2^-23 of itself; what 16-bit types hold of a
    row's p - q by 2^-11 of itself or 2^-39, and of weight's gradient's other operand 2^-38 of its largest value."""
    t, (M, K) = x.dtype, x.shape
    x, w = x.double(), w.double()
    z, mag = x @ w.T, x.abs() @ w.abs().T
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    loss, dloss, d, dd, c = _rows(z, (K + 16) * E * mag, ids, None, 1.0, g, t)
    if t is torch.float32:
        dd = dd + 2.0 ** -23 * d.abs() + _tiny(t)
        lost = 0.0
    else:
        dd = dd + 2.0 ** -11 * d.abs() + 2.0 ** -39 * c.abs()
        share = torch.where(c == 0, 0.0, d / torch.where(c == 0, 1.0, c)).abs()
        lost = 2.0 ** -38 * 2 * (c.abs() * (x.abs().amax(1, keepdim=True) if K else 0.0)).max() * share.sum(0)[:, None]
    out = {"loss": (loss, dloss * 1.01 + 1e-30)}
    for name, a, da, v, n in (("dx", d, dd, w, w.shape[0]), ("dw", d.T, dd.T, x, M)):
        out[name] = (a @ v, da @ v.abs() + (n + 16) * E * (a.abs() @ v.abs()) + (lost if name == "dw" else 0.0))
    if b is not None:
        out["db"] = (d.sum(0), dd.sum(0) + (M + 16) * E * d.abs().sum(0))
    for k in list(out)[1:]:
        tt = b.dtype if k == "db" else t
        out[k] = (out[k][0], (out[k][1] + torch.finfo(tt).eps / 2 * out[k][0].abs()) * 1.01 + _tiny(tt))
    return out


def _check(x, w, b, ids, g):
    ref, out = _reference(x, w, b, ids, g), _run(x, w, b, ids, None, g)
    for k, (value, bound) in ref.items():
        _held(out[k], value, bound, k)



@pytest.mark.parametrize("M,K,V", ROWS)
@pytest.mark.parametrize("spread", [2.0, 6.0])
def test_small_terms_in_float32(M, K, V, spread):
    """Softmax terms down to 2^-60, in rows whose losses weigh 1 and 2^-30: every entry is a float32 one."""
    x, w, b, ids, _, g = _make(M, K, V, torch.float32, 2, spread=spread)
    _check(x, w, b, ids, torch.where(torch.arange(M) % 3 == 0, g, g * 2.0 ** -30))


@pytest.mark.parametrize("M,K,V", ROWS)
def test_large_rows_beside_others_in_float32(M, K, V):
    """A row of x, then a row of the weight, 2^26 times the others' size."""
    x, w, b, ids, _, g = _make(M, K, V, torch.float32, 3)
    big = x.clone()
    big[5] *= 2.0 ** 26
    _check(big, w, b, ids, g)
    far = w.clone()
    far[7] *= 2.0 ** 26
    _check(x, far, b, ids, g)


@pytest.mark.parametrize("M,K,V", [(257, 520, 8100), (1100, 72, 14000), (256, 1030, 4150), (2000, 300, 1900)])
def test_wide_products_in_float32(M, K, V):
    """Several tiles in every direction, odd ends among them."""
    x, w, b, ids, _, g = _make(M, K, V, torch.float32, 11)
    ids[::7] = -1
    _check(x, w, b, ids, g)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,V", ROWS)
def test_weights_of_losses_stay_with_their_rows(M, K, V, t):
    """The gradient of one row's loss, of any size, changes no bit of another row's dx."""
    x, w, b, ids, _, g = _make(M, K, V, t, 4)
    one = _run(x, w, b, ids, None, g)
    rows = torch.arange(M) != 2
    for factor in (2.0 ** 45, 2.0 ** -45, -3.0, 0.0):
        other = _run(x, w, b, ids, None, torch.where(rows, g, g * factor))
        assert torch.equal(other["dx"][rows], one["dx"][rows]), factor


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K,V", ROWS)
def test_gradients_of_losses_of_different_weights(M, K, V, t):
    """Rows' losses weigh 1 and 2^-45 (half: 2^14 and 2^-10): every row's dx is within its own row's bound."""
    x, w, b, ids, _, g = _make(M, K, V, t, 5)
    large, small = (2.0 ** 14, 2.0 ** -10) if t is torch.float16 else (1.0, 2.0 ** -45)
    g = torch.where(torch.arange(M) % 3 == 0, g * large, g * small)
    ref, out = _reference(x, w, b.float(), ids, g), _run(x, w, b.float(), ids, None, g)
    for k in ("loss", "dx", "db"):
        _held(out[k], *ref[k], k)
    fits = ref["dw"][0].abs() + ref["dw"][1] < torch.finfo(t).max  # half: what overflows is infinite
    _held(torch.where(fits, out["dw"].double().cpu(), 0.0), torch.where(fits, ref["dw"][0], 0.0), ref["dw"][1], "dw")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,V", ROWS)
def test_sizes_of_rows_stay_with_them(M, K, V, t):
    """One row of x, of any size, changes no bit of another row's loss and dx."""
    x, w, b, ids, _, g = _make(M, K, V, t, 6)
    one = _run(x, w, b, ids, None, g)
    rows = torch.arange(M) != 2
    for factor in ((2.0 ** 10, 2.0 ** -10) if t is torch.float16 else (2.0 ** 50, 2.0 ** 10, 2.0 ** -50)):
        y = torch.where(rows[:, None], x, x * factor)
        other = _run(y, w, b, ids, None, g)
        for k in ("loss", "dx"):
            assert torch.equal(other[k][rows], one[k][rows]), (k, factor)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M", [3, 70])
def test_no_inputs(M, t):
    """The logits are the bias: its gradient is all there is."""
    x, w, b, ids, _, g = _make(M, 0, 300, t, 8)
    _check(x, w, b.float(), ids, g)


@pytest.mark.parametrize("t", TYPES)
def test_more_than_a_million_inputs(t):
    """x is 0 but for some inputs at both ends, so that the others add nothing and lose nothing."""
    M, K, V = 3, (1 << 20) + 72, 5
    some = torch.cat((torch.arange(40), torch.arange(K - 40, K)))
    x, w, b, ids, _, g = _make(M, len(some), V, t, 9)
    long_x = torch.zeros(M, K, dtype=t)
    long_x[:, some] = x
    long_w = torch.randn(V, K, generator=torch.Generator().manual_seed(10)).to(t)
    long_w[:, some] = w
    ref, out = _reference(x, w, b, ids, g), _run(long_x, long_w, b, ids, None, g)
    for k, (value, bound) in ref.items():
        got = out[k][:, some] if k in ("dx", "dw") else out[k]
        _held(got, value, bound, k)
    assert (out["dw"][:, 40:K - 40] == 0).all()


@pytest.mark.parametrize("t", TYPES)
def test_masked_columns_beside_what_is_not_finite(t):
    """Their gradient is 0 in rows with a NaN or an infinity, and where the loss's own gradient is one."""
    g = torch.Generator().manual_seed(12)
    z = torch.randn(5, 3000, generator=g).to(t)
    masked = torch.rand(5, 3000, generator=g) < 0.5
    ids = torch.randint(0, 3000, (5, 9), generator=g)
    z[masked] = -float("inf")
    z[0, ~masked[0]] = float("nan")
    z[1, ids[1, 0]] = float("inf")
    masked[1, ids[1, 0]] = False
    grad = torch.tensor([1.0, 1.0, float("inf"), float("nan"), 1.0])
    leaf = z.cuda().requires_grad_(True)
    loss = _losses().distillation(leaf, ids.cuda(), torch.randn(5, 9, generator=g).cuda())
    dx = torch.autograd.grad(loss, leaf, grad.cuda())[0].cpu()
    assert (dx[masked] == 0).all()
    assert dx[0][~masked[0]].isnan().all() and dx[4].isfinite().all() and (dx[4] != 0).any()


def test_bfloat16_rows_of_the_most_inputs():
    """2^23 of them, in so many rows of the weight that a tile's offsets reach the end of 32 bits."""
    M, K, V = 2, 1 << 23, 300
    some = torch.cat((torch.arange(40), torch.arange(K - 40, K)))
    x, w, b, ids, _, g = _make(M, len(some), V, torch.bfloat16, 13)
    ids[0] = V - 1
    long_x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    long_x[:, some] = x.cuda()
    long_w = torch.full((V, K), 0.5, dtype=torch.bfloat16, device="cuda")
    long_w[:, some] = w.cuda()
    ref, out = _reference(x, w, b, ids, g), _run(long_x, long_w, b, ids, None, g)
    for k, (value, bound) in ref.items():
        got = out[k][:, some] if k in ("dx", "dw") else out[k]
        _held(got, value, bound, k)
    # where x is 0: a weight of 1/2 times the sum of a row's gradients, which is 0 within their bound
    d = torch.softmax(x.double() @ w.double().T + b.double(), 1).scatter_add_(1, ids, -torch.ones(M, 1).double())
    bound = 0.5 * g.double() * (2.0 ** -11 + 2.0 ** -16) * d.abs().sum(1) + 2.0 ** -39 * V
    assert (out["dx"][:, 40:K - 40].abs().amax(1).double().cpu() <= bound * (1 + 2.0 ** -8)).all()
    assert (out["dw"][:, 40:K - 40] == 0).all()

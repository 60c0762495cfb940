"""Calls of the losses that the documentation allows at the ends of their ranges."""
import pytest
import torch

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


#: By the plain tiles and by the wide ones (float32 in training from 129 rows on, bfloat16 always).
ROWS = [(9, 40, 90), (60, 64, 500), (300, 128, 4000), (136, 256, 4100)]


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

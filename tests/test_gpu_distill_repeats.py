"""Teacher entries that name a column several times: the same bits from run to run, and the oracle's values."""
import pytest
import torch

import distill
from oracle import distill as od

pytestmark = pytest.mark.gpu


def _case(T, V, k, cols, dt):
    """k entries on `cols` columns of each row, whose logits carry most of the sum and span many magnitudes, so that an
    order of their sum shows in its last bits."""
    g = torch.Generator().manual_seed(V + k)
    z = torch.randn(T, V, generator=g)
    idx = torch.stack([torch.randperm(V, generator=g)[:cols][torch.randint(0, cols, (k,), generator=g)] for _ in range(T)])
    z.scatter_(1, idx, 8 + 3 * torch.randn(T, k, generator=g))
    return z.to(dt), idx.to(torch.int32), torch.randn(T, k, generator=g) * 2


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,k,cols", [(600, 5000, 1000, 300), (40, 70001, 1024, 400), (600, 40000, 500, 7), (8, 600, 70, 64)])
def test_results_do_not_change_from_run_to_run(gpu, T, V, k, cols, dt):
    z, idx, t = _case(T, V, k, cols, dt)
    zg, idx, t = z.to(gpu).requires_grad_(True), idx.to(gpu), t.to(gpu)
    lse = torch.logsumexp(t, 1) + 0.5
    for extra in (dict(), dict(teacher_lse=lse)):
        loss, grad = distill.topk_kl_rows(zg.detach(), idx, t, **extra)
        for _ in range(12):
            l2, g2 = distill.topk_kl_rows(zg.detach(), idx, t, **extra)
            assert torch.equal(loss, l2) and torch.equal(grad, g2)
        kept = []
        for _ in range(4):
            zg.grad = None
            out = distill.topk_kl(zg, idx, t, **extra)
            out.sum().backward()
            kept.append((out.detach(), zg.grad))
        assert all(torch.equal(a, kept[0][0]) and torch.equal(b, kept[0][1]) for a, b in kept)


@pytest.mark.parametrize("T,V,k,cols", [(5, 5000, 1000, 300), (3, 70001, 1024, 400)])
def test_against_the_oracle(gpu, T, V, k, cols):
    z, idx, t = _case(T, V, k, cols, torch.float32)
    lse = torch.logsumexp(t, 1) + 0.5
    loss, grad = distill.topk_kl_rows(z.to(gpu), idx.to(gpu), t.to(gpu), teacher_lse=lse.to(gpu))
    rl, rg = od.rows(z, idx, t, None, 1.0, lse)
    # sums of k + V terms around exponentials of differences up to 32: 2^-18 of the loss's terms, 2^-17 of q and p
    assert ((loss.double().cpu() - rl).abs() <= 2.0 ** -18 * (32 + rl.abs())).all()
    assert ((grad.double().cpu() - rg).abs() <= 2.0 ** -17 * (rg.abs() + 2.0 ** -6)).all()

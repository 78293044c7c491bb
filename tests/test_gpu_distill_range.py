"""The loss of teacher entries, and of a teacher's rest, on columns that the student masks by its type's lowest value: as
large as the formula says, finite where fp32 holds it."""
import pytest
import torch

import distill
from oracle import distill as od

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tau", [0.2, 0.7, 1.0, 4.0])
@pytest.mark.parametrize("T,V", [(6, 50), (6, 70001), (300, 5000)])
def test_entries_on_masked_columns(gpu, T, V, tau, dt):
    g = torch.Generator().manual_seed(V)
    k = 5
    z = torch.randn(T, V, generator=g).to(dt)
    idx = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(T)])
    t = torch.randn(T, k, generator=g)
    low = torch.finfo(dt).min
    z[0, idx[0, 0]] = low               # one entry
    z[1, idx[1, :3]] = low              # some
    z[2, idx[2]] = low                  # all of them
    keep = z[3, idx[3]].clone()
    z[3] = low                          # everything outside: the rest's mass
    z[3, idx[3]] = keep
    z[4, idx[4, 1]] = -float("inf")
    for lse in (None, torch.logsumexp(t / tau, 1) + 0.7):
        loss, grad = distill.topk_kl_rows(z.to(gpu), idx.to(gpu), t.to(gpu), None, tau, None if lse is None else lse.to(gpu))
        with torch.no_grad():
            again = distill.topk_kl(z.to(gpu), idx.to(gpu), t.to(gpu), tau, None if lse is None else lse.to(gpu))
        ref, _ = od.rows(z[:6], idx[:6], t[:6], None, tau, lse)
        for got in (loss, again):
            got = got[:6].double().cpu()
            ok = (got - ref).abs() <= 2.0 ** -16 * (ref.abs() + 40)  # sums of k terms, logits and logarithms up to 20
            ok |= (ref > 3.4e38) & (got == float("inf"))
            assert ok.all(), (got, ref)
        assert not torch.isnan(grad).any()

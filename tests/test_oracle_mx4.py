"""CPU checks of the 4-bit operators' oracles: known MX values and ties, the closed forms of the exponents, and gradients
against central differences."""
import math

import pytest
import torch

from oracle import distill as od
from oracle import mx, mx4


def test_e2m1_known_values():
    x = torch.zeros(4, 32)
    x[0, :8] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])  # ties go to the even code
    x[1, :3] = torch.tensor([6.1, 3.0, -0.2])  # just above 6: the scale is 2
    x[2, 0] = 2.0 ** -126
    x[3, :2] = torch.tensor([math.inf, 1.0])
    v = mx4.values(x, "e2m1")
    assert v[0, :8].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]
    assert v[1, :3].tolist() == [6.0, 3.0, 0.0] and math.copysign(1, v[1, 2].item()) == -1
    assert v[2, 0].item() == 2.0 ** -126
    assert v[3, :2].tolist() == [6.0 * 2.0 ** 127, 0.0]
    x[0, 31] = math.nan
    assert torch.isnan(mx4.values(x, "e2m1")[0]).all() and not torch.isnan(mx4.values(x, "e2m1")[1:]).any()


def test_e4m3_agrees_with_the_8bit_oracle():
    x = torch.randn(128, 256, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    q, s = mx.quant(x)
    assert torch.equal(mx4.values(x, "e4m3"), mx.dequant(q, s, 128, 256).double())


@pytest.mark.parametrize("fn", ["silu", "gelu"])
def test_gate_derivative_against_differences(fn):
    g = torch.linspace(-9, 9, 181, dtype=torch.float64)
    d = 1e-6
    num = (mx4.gate(fn, g + d)[0] - mx4.gate(fn, g - d)[0]) / (2 * d)
    # central differences: d² / 6 times a third derivative below 2, and rounding 2^-52 · 9 / d
    assert (num - mx4.gate(fn, g)[1]).abs().max() < 1e-8


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("tau", [0.7, 1.0, 3.0])
def test_distill_gradient_against_differences(rest, tau):
    gen = torch.Generator().manual_seed(3)
    V, k = 23, 5
    z = torch.randn(1, V, generator=gen, dtype=torch.float64) * 2
    idx = torch.tensor([[4, 17, -1, 4, 9]])  # padding and an entry that comes twice
    t = torch.randn(1, k, generator=gen, dtype=torch.float64)
    lse = torch.tensor([torch.logsumexp(t[0] / tau, 0).item() + 0.4]) if rest else None
    _, g = od.rows(z, idx, t, None, tau, lse)
    d = 1e-6
    for j in range(V):
        zp, zm = z.clone(), z.clone()
        zp[0, j] += d
        zm[0, j] -= d
        num = (od.rows(zp, idx, t, None, tau, lse)[0] - od.rows(zm, idx, t, None, tau, lse)[0]) / (2 * d)
        assert abs(num.item() - g[0, j].item()) < 1e-7, j  # rounding 2^-52 · 30 / d and d² / 6 times third derivatives


def test_distill_is_the_divergence_of_distributions():
    gen = torch.Generator().manual_seed(4)
    z, t = torch.randn(3, 11, generator=gen, dtype=torch.float64), torch.randn(3, 11, generator=gen, dtype=torch.float64)
    idx = torch.arange(11).expand(3, 11)  # every token: the full divergence, with and without the bucket
    ref = (t.softmax(1) * (t.log_softmax(1) - z.log_softmax(1))).sum(1)
    assert torch.allclose(od.rows(z, idx, t)[0], ref, atol=1e-12)
    assert torch.allclose(od.rows(z, idx, t, lse=t.logsumexp(1))[0], ref, atol=1e-12)


def test_distill_of_the_lowest_value_everywhere_is_uniform():
    z = torch.full((1, 203), torch.finfo(torch.float32).min)
    loss, g = od.rows(z, torch.tensor([[3]]), torch.tensor([[0.5]]))
    assert abs(loss.item() - math.log(203)) < 1e-12
    assert abs(g[0, 0].item() - 1 / 203) < 1e-15 and abs(g[0, 3].item() - (1 / 203 - 1)) < 1e-15

"""Tighter bounds for the gated block than those of test_gpu_mx4.py and test_gpu_mx4_model.py: its input gradient from gates
that are known to the last bit, element by element, and its forms for few rows against the operands' own values."""
import pytest
import torch

import mxfp4
from oracle import mx4
from test_gpu_mx4 import EPS, _randn, _sum_bound

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _span(v, err, fmt):
    """(MX values of v, how far they can move when each v moves by err): codes move only where v lies that near a tie."""
    q = mx4.values(v, fmt)
    return q, torch.maximum((mx4.values(v + err, fmt) - q).abs(), (mx4.values(v - err, fmt) - q).abs())


@pytest.mark.parametrize("act", ["e4m3", "e2m1"])
@pytest.mark.parametrize("fn", ["silu", "gelu"])
@pytest.mark.parametrize("M,N,K", [(1, 32, 64), (33, 31, 40), (150, 200, 256), (64, 257, 130)])
def test_input_gradient_from_known_gates(gpu, M, N, K, fn, act):
    """With x = 0 the kept [g | u] are the addend itself.  dg and du are off by some fp32 roundings of dh u and dh g
    (2^-18 of them with the hardware exponential), which moves the codes near a tie and no others."""
    wg, wu = _randn(1, N, K, std=K ** -0.5).to(BF), _randn(2, N, K, std=K ** -0.5).to(BF)
    add, dh = _randn(3, M, 2 * N, std=1.5).to(BF), _randn(4, M, N).to(BF)
    x = torch.zeros(M, K, dtype=BF, device=gpu, requires_grad=True)
    mxfp4.mx4_gated(x, mxfp4.GatedWeight(wg.to(gpu), wu.to(gpu)), add=add.to(gpu), fn=fn, act=act).backward(dh.to(gpu))
    g, u, d = add[:, :N].double(), add[:, N:].double(), dh.double()
    f, df = mx4.gate(fn, g)
    qg, eg = _span(d * u * df, 2.0 ** -18 * (d * u).abs() * (1 + g.abs()), act)
    qu, eu = _span(d * f, 2.0 ** -18 * (d * g).abs(), act)
    tg, tu = mx4.values(wg.t(), "e2m1"), mx4.values(wu.t(), "e2m1")
    dx = qg @ tg.t() + qu @ tu.t()
    mag = qg.abs() @ tg.abs().t() + qu.abs() @ tu.abs().t()
    moved = eg @ tg.abs().t() + eu @ tu.abs().t()
    bound = EPS[BF] * (dx.abs() + moved) + _sum_bound(act, 2 * N) * mag + moved
    assert (moved <= 0.2 * mag + 1e-30).all()  # the bound is one of a few codes
    assert ((x.grad.double().cpu() - dx).abs() <= bound + 1e-30).all()


@pytest.mark.parametrize("act", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M", [1, 8, 16, 17, 33, 64, 65])
@pytest.mark.parametrize("N,K", [(96, 4096), (50, 1000), (2048, 256)])
def test_few_and_thin_rows_of_the_gated_block(gpu, M, N, K, act):
    """h = silu(g) u of each row count's kernel against g and u from the operands' values in float64, the bound of
    test_gpu_mx4_shapes.py: |silu'| <= 1.13."""
    x = _randn(M, M, K).to(BF).to(gpu)
    ws = [_randn(N + i, N, K, std=K ** -0.5).to(BF).to(gpu) for i in range(2)]
    a = mxfp4.mx4_dequant(mxfp4.mx4_quant(x, fmt=act)).double()
    b = [mxfp4.mx4_dequant(mxfp4.mx4_quant(w)).double() for w in ws]
    g, u = a @ b[0].t(), a @ b[1].t()
    dg, du = (_sum_bound(act, K) * (a.abs() @ w.abs().t()) for w in b)
    f = g * torch.sigmoid(g)
    bound = 2.0 ** -8 * (f * u).abs() + 1.13 * dg * (u.abs() + du) + du * f.abs() + 2.0 ** -20 * (f * u).abs() + 1e-30
    G = mxfp4.GatedWeight(*ws)
    for saved in (False, True):
        h = mxfp4.mx4_gated(x.clone().requires_grad_(saved), G, act=act).detach().double()
        assert ((h - f * u).abs() <= bound).all(), ((h - f * u).abs() / bound).max()

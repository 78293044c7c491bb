"""The 4-bit operators at the ends of their types' ranges, against the formulas in float64."""
import pytest
import torch

import mxfp4
from oracle import mx4

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("act", ["e4m3", "e2m1"])
@pytest.mark.parametrize("fn", ["silu", "gelu"])
def test_gates_far_out(gpu, fn, act):
    """Gates of every magnitude that bf16 holds, through the addend of a block whose product is 0: past some tens the
    derivative is 1 or 0 and dg is dh u or 0, du = dh f is dh g or 0.  2^-7 covers the rounding of du and dg and of the kept
    values' products; below 2^-100 a sigmoid may be flushed."""
    mags = torch.tensor([0.0, 0.5, 3.0, 15.0, 16.5, 30.0, 90.0, 1e3, 1e6, 1e12, 1.3e13, 1e15, 2e19, 1e25, 1e30, 3e38]).to(BF)
    g = torch.cat([mags, -mags])  # 32 columns, one scale block
    N, K, M = 32, 64, 40
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(1)).to(BF).to(gpu)
    W = mxfp4.GatedWeight(w, w)
    x = torch.zeros(M, K, dtype=BF, device=gpu, requires_grad=True)
    add = torch.cat([g, torch.ones(N, dtype=BF)]).expand(M, 2 * N).contiguous().to(gpu).requires_grad_(True)
    dh = torch.full((M, N), 0.5, dtype=BF, device=gpu)
    h = mxfp4.mx4_gated(x, W, add=add, fn=fn, act=act)
    h.backward(dh)
    gd = g.double()
    f, df = mx4.gate(fn, gd)
    if fn == "gelu":  # the formula's own powers: exact limits past 1e3
        df = torch.where(gd > 1e3, torch.ones_like(df), torch.where(gd < -1e3, torch.zeros_like(df), df))
    for got, want in ((h[0], f), (h[-1], f), (add.grad[0, :N], 0.5 * df), (add.grad[-1, :N], 0.5 * df),
                      (add.grad[7, N:], 0.5 * f)):
        got = got.detach().double().cpu()
        assert ((got - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -100).all(), (got - want, got, want)
    assert not torch.isnan(x.grad).any()


def test_a_nan_gate_stays_nan(gpu):
    N, K = 32, 64
    w = torch.zeros(N, K, dtype=BF, device=gpu)
    add = torch.zeros(3, 2 * N, dtype=BF, device=gpu)
    add[1, 5] = float("nan")
    for fn in ("silu", "gelu"):
        a = add.clone().requires_grad_(True)
        h = mxfp4.mx4_gated(torch.zeros(3, K, dtype=BF, device=gpu), mxfp4.GatedWeight(w, w), add=a, fn=fn)
        h.sum().backward()
        bad = torch.isnan(a.grad)
        assert torch.isnan(h[1, 5]) and bad[1, 5] and bad[1, N + 5] and int(bad.sum()) == 2


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("dt", [BF, torch.float32])
def test_blocks_at_the_least_scale(gpu, dt, fmt):
    """Blocks around the largest value times 2^-127 and far below, denormals among them: the scale is 2^-127 at the least
    and codes are of v 2^127, in both axes and in the kernels that quantize their rows themselves."""
    g = torch.Generator().manual_seed(2)
    x = torch.zeros(40, 256, dtype=torch.float64)
    for i in range(40):  # from 2^-110 down to the least denormals
        x[i] = torch.randn(256, generator=g, dtype=torch.float64) * 2.0 ** (-110 - i)
    x[39, :32] = 448 * 2.0 ** -127
    x[38, :32] = 448 * 2.0 ** -127 * torch.linspace(0, 1, 32, dtype=torch.float64)
    x[37, :32] = 6 * 2.0 ** -127 * torch.linspace(-1, 1, 32, dtype=torch.float64)
    x = x.float().to(dt)
    m, mt = mxfp4.mx4_quant(x.to(gpu), fmt=fmt, both=True)
    for got, ref in ((m, x), (mt, x.t())):
        v = mxfp4.mx4_dequant(got).double().cpu()
        assert torch.equal(v, mx4.values(ref, fmt)), int((v != mx4.values(ref, fmt)).sum())


def test_products_of_rows_at_the_least_scale(gpu):
    """Rows of 2^-120 against weights of 2^100: what the quantizer keeps of them comes out of the product in both formats,
    of few rows and of many."""
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(40, 256, generator=g) * 2.0 ** -121).to(BF)
    w = (torch.randn(64, 256, generator=g) * 2.0 ** 100).to(BF)
    W = mxfp4.Weight(w.to(gpu))
    for act in ("e4m3", "e2m1"):
        ref, mag = mx4.linear(x, w, act)
        for rows in (40, 5):
            y = mxfp4.mx4_linear(x[:rows].to(gpu), W, act=act).double().cpu()
            assert ((y - ref[:rows]).abs() <= 2.0 ** -8 * ref[:rows].abs() + 2.0 ** -12 * mag[:rows]).all()

"""Every workgroup shape of the 4-bit products, ragged on both sides and at one, two and many K tiles, against the operands'
own values (mx4_dequant, tested by itself) multiplied in float64.  tests/test_mx4_host.py holds each size to its shape.

Bounds, as in test_gpu_mx4.py: a sum of K terms in fp32, the instruction's dropped low bits in E4M3, and the rounding of the
output; the gated block's from those of g and u through h = fn(g) u, |fn'| <= 1.13.
"""
import pytest
import torch

import mxfp4
from test_gpu_mx4 import _randn, _sum_bound

pytestmark = pytest.mark.gpu
BF = torch.bfloat16

PLAIN = {("thin", "e4m3"): [(17, 96, 200), (32, 40, 700)], ("thin", "e2m1"): [(17, 96, 200), (64, 30, 300), (33, 300, 1100)],
         ("64x64", "e4m3"): [(70, 130, 384), (300, 520, 128), (2049, 2050, 400), (65, 64, 1100)],
         ("64x64", "e2m1"): [(65, 64, 1100), (500, 1030, 150), (1200, 4200, 260)],
         ("64x128", "e4m3"): [(900, 2000, 390), (1500, 2100, 130)], ("64x128", "e2m1"): [(70, 130, 384), (2050, 2100, 300)],
         ("128x128", "e4m3"): [(1300, 2100, 900), (2500, 4200, 130)], ("128x128", "e2m1"): [(1500, 2100, 520), (2500, 4200, 130)],
         ("256x128", "e4m3"): [(4100, 4200, 256), (2500, 6200, 130)], ("256x128", "e2m1"): [(6000, 4200, 200)]}
GATED = {("thin", "e4m3"): [(30, 40, 256)], ("thin", "e2m1"): [(60, 40, 256)],
         ("64x128", "e4m3"): [(70, 130, 384), (1300, 2100, 900)], ("64x128", "e2m1"): [(70, 130, 384), (1200, 4200, 260)],
         ("128x128", "e4m3"): [(1025, 6200, 640), (2100, 4200, 260)], ("128x128", "e2m1"): [(1500, 2100, 520)],
         ("256x128", "e4m3"): [(2500, 4200, 130)], ("256x128", "e2m1"): [(5000, 2100, 300)]}


def _cases(table):
    return [(shape, act, *size) for (shape, act), sizes in table.items() for size in sizes]


def _operands(gpu, M, N, K, act, weights):
    x = _randn(M, M, K).to(BF).to(gpu)
    ws = [_randn(N + i, N, K, std=0.1).to(BF).to(gpu) for i in range(weights)]
    a = mxfp4.mx4_dequant(mxfp4.mx4_quant(x, fmt=act)).double()
    return x, ws, a, [mxfp4.mx4_dequant(mxfp4.mx4_quant(w)).double() for w in ws]


@pytest.mark.parametrize("shape,act,M,N,K", _cases(PLAIN))
def test_linear(gpu, shape, act, M, N, K):
    x, (w,), a, (b,) = _operands(gpu, M, N, K, act, 1)
    y = mxfp4.mx4_linear(x, mxfp4.Weight(w, transpose=False), act=act).double()
    ref, mag = a @ b.t(), a.abs() @ b.abs().t()
    assert ((y - ref).abs() <= 2.0 ** -8 * ref.abs() + _sum_bound(act, K) * mag).all()


@pytest.mark.parametrize("saved", [False, True])
@pytest.mark.parametrize("shape,act,M,N,K", _cases(GATED))
def test_gated(gpu, shape, act, M, N, K, saved):
    x, (wg, wu), a, (bg, bu) = _operands(gpu, M, N, K, act, 2)
    h = mxfp4.mx4_gated(x.requires_grad_(saved), mxfp4.GatedWeight(wg, wu), act=act).detach().double()
    g, u = a @ bg.t(), a @ bu.t()
    dg, du = (_sum_bound(act, K) * (a.abs() @ b.abs().t()) for b in (bg, bu))
    f = g * torch.sigmoid(g)
    bound = 2.0 ** -8 * (f * u).abs() + 1.13 * dg * (u.abs() + du) + du * f.abs() + 2.0 ** -20 * (f * u).abs() + 1e-30
    assert ((h - f * u).abs() <= bound).all()

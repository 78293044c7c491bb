"""What the products' sums keep, as include/mxfp4_ops.h states it: E2M1 products are exact before the fp32 sums; E4M3 ones
are added in groups of 16 consecutive k, in which every term loses what lies below 2^-13 of the largest one (taken as the
product of the operands' powers of two)."""
import pytest
import torch

import mxfp4
from test_gpu_mx4 import _randn

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _operands(gpu, x, w, act):
    a, b = mxfp4.mx4_quant(x.to(gpu), fmt=act), mxfp4.mx4_quant(w.to(gpu))
    return a, b, mxfp4.mx4_dequant(a).double(), mxfp4.mx4_dequant(b).double()


def _lost(A, B):
    """Bound of what the groups lose: 16 terms, each 2^-13 of 2^(eA + eB) <= |a| |b|, where an operand below its format's
    least normal number counts as that: 2^-6 of E4M3 and 1 of E2M1, at the block's scale (at most amax / 224 and amax / 3)."""
    def up(X, least):
        R, C = X.shape
        blk = torch.nn.functional.pad(X, (0, -C % 32)).abs().reshape(R, -1, 32)
        floor = blk.amax(2, keepdim=True) * least
        return torch.where(blk > 0, torch.maximum(blk, floor), blk).reshape(R, -1, 16)
    a, b = up(A, 2.0 ** -6 / 224), up(B, 1 / 3)
    return sum(16 * 2.0 ** -13 * (a[:, None, i] * b[None, :, i]).amax(2) for i in range(a.shape[1]))


@pytest.mark.parametrize("spread", [0.0, 2.0, 4.0])
@pytest.mark.parametrize("M,N,K", [(3, 40, 32), (16, 64, 300), (40, 130, 1000)])
def test_e4m3_sums(gpu, M, N, K, spread):
    x = _randn(1, M, K) * torch.exp(spread * _randn(2, M, K))
    a, b, A, B = _operands(gpu, x.to(BF), _randn(3, N, K).to(BF), "e4m3")
    ref, mag = A @ B.t(), A.abs() @ B.abs().t()
    bound = _lost(A, B) + K * 2.0 ** -23 * mag
    err = (mxfp4.mx4_mm(a, b, dtype=F32).double() - ref).abs()
    assert (err <= bound).all(), (err / bound).max()
    W = mxfp4.Weight(_randn(3, N, K).to(BF).to(gpu))
    y = mxfp4.mx4_linear(x.to(BF).to(gpu), W).double()  # the kernel for few rows up to 16
    assert ((y - ref).abs() <= bound + 2.0 ** -8 * ref.abs()).all()
    if not spread:  # 5e-6 was measured
        assert err.pow(2).mean().sqrt() <= 2.0 ** -16 * ref.pow(2).mean().sqrt()


@pytest.mark.parametrize("M,N,K", [(3, 40, 32), (16, 64, 300), (200, 130, 2048)])
def test_e2m1_sums_are_exact_while_fp32_holds_them(gpu, M, N, K):
    a, b, A, B = _operands(gpu, _randn(1, M, K), _randn(3, N, K), "e2m1")
    ref = A @ B.t()
    assert torch.equal(mxfp4.mx4_mm(a, b, dtype=F32).double(), ref) and torch.equal(ref, ref.float().double())

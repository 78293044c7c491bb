"""Matrices of more than a million rows: what mx4_quant takes, mx4_dequant gives back."""
import pytest
import torch

import mxfp4
from oracle import mx4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("R", [16 * 65535, 16 * 65535 + 1, 2 * 16 * 65535 + 33])
def test_values_of_tall_matrices(gpu, R, fmt):
    x = torch.randn(R, 32, generator=torch.Generator(device=gpu).manual_seed(R), device=gpu).to(torch.bfloat16)
    v = mxfp4.mx4_dequant(mxfp4.mx4_quant(x, fmt=fmt), torch.bfloat16)
    assert v.shape == x.shape
    step = 16 * 60000  # rows are quantized by themselves
    for r in range(0, R, step):
        assert torch.equal(v[r:r + step], mxfp4.mx4_dequant(mxfp4.mx4_quant(x[r:r + step], fmt=fmt), torch.bfloat16)), r
    for lo in (0, 1048448 - 20, 1048560 - 20, R - 40):  # the values themselves
        assert torch.equal(v[lo:lo + 40].double().cpu(), mx4.values(x[lo:lo + 40].cpu(), fmt)), lo

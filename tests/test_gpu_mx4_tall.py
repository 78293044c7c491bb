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
    for rows in (x[:40], x[-40:]), (x[1048550:1048600],) * 2:
        for part in rows:
            lo = (part.data_ptr() - x.data_ptr()) // 64
            assert torch.equal(v[lo:lo + len(part)].double().cpu(), mx4.values(part.cpu(), fmt))

"""Layers that mxfp4.enable_mxfp4 took, under autocast: inputs of the other 16-bit type are cast as linears cast them."""
import pytest
import torch

import distill_mxfp4
import mxfp4
import workloads

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("off", [(), ("up_proj",), ("gate_proj", "down_proj"), ("gate_proj", "up_proj", "down_proj")])
@pytest.mark.parametrize("given,cast", [(HF, BF), (BF, HF), (torch.float32, HF)])
def test_mlp_with_adapters(gpu, given, cast, off):
    m = distill_mxfp4.Model(1, 160, 288, 64, 8, True).to(gpu)
    mod = m.model.layers[0].mlp
    assert mxfp4.enable_mxfp4(m) == 3
    for n in off:
        getattr(mod, n).disable_adapters = True
    for rows in (30, 3):
        x = torch.randn(rows, 160, generator=torch.Generator().manual_seed(1)).to(given).to(gpu).requires_grad_(True)
        with torch.autocast("cuda", cast):
            y = mod(x)
        y.float().sum().backward()
        assert y.dtype == cast and x.grad.dtype == given and x.grad.abs().max() > 0
        assert torch.equal(y, mod(x.detach().to(cast)))


@pytest.mark.parametrize("given,cast", [(HF, BF), (BF, HF), (torch.float32, BF), (BF, BF)])
def test_linear(gpu, given, cast):
    m = workloads.build_attn(128, 128, 64, 8, 8, device=gpu)
    q = m.model.layers[0].self_attn.q_proj
    x = torch.randn(20, 128, generator=torch.Generator().manual_seed(2)).to(given).to(gpu)
    with torch.autocast("cuda", cast):
        want = q.base_layer(x).dtype
    mxfp4.enable_mxfp4(m)
    with torch.autocast("cuda", cast):
        y = q.base_layer(x)
        assert q(x).dtype == want
    assert y.dtype == want == cast and torch.equal(y, q.base_layer(x.to(cast)))

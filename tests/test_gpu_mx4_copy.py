"""A model whose layers enable_mxfp4 took can be copied, as one that enable_mxfp8 took can: the frozen weights are shared."""
import copy

import pytest
import torch

import distill_mxfp4
import mxfp4

pytestmark = pytest.mark.gpu


def test_deepcopy(gpu):
    m = distill_mxfp4.Model(2, 160, 288, 64, 8, True).to(gpu)
    mxfp4.enable_mxfp4(m)
    tok = torch.arange(20, device=gpu), torch.arange(1, 21, device=gpu)
    with torch.no_grad():
        want = m(*tok)
        c = copy.deepcopy(m)
        assert torch.equal(c(*tok), want)
        a, b = (t.model.layers[0].mlp for t in (m, c))
        assert b.forward.__self__ is b and b._mx4_gated[0] is a._mx4_gated[0]
        for p in b.parameters():
            if p.requires_grad:
                p.mul_(2)
        assert not torch.equal(c(*tok), want) and torch.equal(m(*tok), want)
        mxfp4.disable_mxfp4(c)
        assert torch.equal(m(*tok), want)
        assert b.down_proj.base_layer.weight.shape == (160, 288) and a.down_proj.base_layer.weight.shape == (0,)

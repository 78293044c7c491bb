"""4-bit models under the framework's grouped path on the GPU: group_linear and shared_prefix._mlp give what the layers
give when they are called by themselves."""
import pytest
import torch
from torch import nn

import distill_mxfp4
import fused_linear
import mxfp4
import shared_prefix
import workloads

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def test_group_linear_over_four_bit_linears(gpu):
    m = workloads.build_attn(256, 256, 128, 16, 32, device=gpu)
    attn = m.model.layers[0].self_attn
    assert mxfp4.enable_mxfp4(m) == 4
    thin = nn.Linear(256, 16, bias=False, device=gpu, dtype=BF).requires_grad_(False)
    x = torch.randn(2, 20, 256, generator=torch.Generator().manual_seed(1)).to(BF).to(gpu).requires_grad_(True)
    mods = (attn.q_proj, attn.k_proj, attn.v_proj, thin)
    with torch.autocast("cuda", BF):
        outs, want = fused_linear.group_linear(x, mods), [p(x) for p in mods]
        assert [o.shape[-1] for o in outs] == [256, 128, 128, 16]
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        plain = fused_linear.group_linear(x, (attn.k_proj.base_layer, thin))
        assert torch.equal(plain[0], attn.k_proj.base_layer(x)) and torch.equal(plain[1], thin(x))
        o = fused_linear.group_linear(outs[0], (attn.o_proj,), defer=True)[0]
        assert torch.equal(fused_linear.residual_add(x, o), x + attn.o_proj(outs[0]))
    sum(t.float().sum() for t in outs).backward()
    assert x.grad.abs().max() > 0 and attn.q_proj.lora_A["default"].weight.grad.abs().max() > 0


def test_shared_prefix_mlp_over_four_bit_weights(gpu):
    m = distill_mxfp4.Model(1, 160, 288, 64, 8, True).to(gpu)
    mlp = m.model.layers[0].mlp
    x = torch.randn(30, 160, generator=torch.Generator().manual_seed(2)).to(BF).to(gpu)
    assert mxfp4.enable_mxfp4(m) == 3
    with torch.autocast("cuda", BF):
        assert torch.equal(shared_prefix._mlp(mlp, x), mlp(x))
    mxfp4.disable_mxfp4(m)
    mlp.gate_proj.lora_dropout["default"] = nn.Dropout(0.1).eval()  # an MLP that enable_mxfp4 does not take whole
    assert mxfp4.enable_mxfp4(m) == 3 and "_mx4_gated" not in mlp.__dict__
    mlp.gate_proj.lora_dropout["default"] = nn.Identity()
    with torch.autocast("cuda", BF):
        got, want = shared_prefix._mlp(mlp, x).float(), mlp(x).float()
        # silu(g) u in one rounding or in two, then a product of 288 terms
        assert (got - want).abs().max() <= 2.0 ** -5 * want.abs().max()

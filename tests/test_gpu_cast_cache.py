"""GPU counterpart of test_cast_cache_host.py: the packed weight forms of a group and the fused MLP's belong to the
adapters they were made from."""
import gc

import pytest
import torch

import fused_linear
import fused_mlp
import mxfp8
import workloads

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def test_adapters_that_share_a_and_not_b(gpu):
    g = torch.Generator().manual_seed(4)
    m = workloads.build_attn(256, 128, 128, 16, 32, device=gpu)
    attn = m.model.layers[0].self_attn
    one, two = attn.k_proj, attn.v_proj
    two.lora_A["default"].weight = one.lora_A["default"].weight
    x = torch.randn(40, 256, generator=g).to(BF).to(gpu)
    with torch.no_grad(), torch.autocast("cuda", BF):
        for proj in (one, two):
            got, want = fused_linear.group_linear(x, [proj])[0].float(), proj(x).float()
            # the adapter's own part is of the size of the output: bf16 roundings of either order are not
            assert (got - want).abs().max() <= 2.0 ** -6 * want.abs().max()


def test_fused_mlps_one_after_the_other_without_a_new_step(gpu):
    """The same weights, adapters of another model each time: a stale copy would give the model before's output."""
    for k in range(6):
        model, inps = workloads.build_model(1, T=64, layers=1, device=gpu)
        mxfp8.enable_mxfp8(model)
        mlp = model.layers[0].mlp
        with torch.no_grad():
            for proj in (mlp.gate_proj, mlp.up_proj, mlp.down_proj):
                proj.lora_B["default"].weight.mul_(float(k))
            x = inps[0]["x"].to(gpu)
            got = fused_mlp.mlp(mlp, x)
            fused_linear.new_step()
            want = fused_mlp.mlp(mlp, x)
        assert torch.equal(got, want), k
        del model, mlp, proj, inps, got, want
        gc.collect()

"""Linears whose weights mxfp4.enable_mxfp4 holds in 4 bits inside the grouped path: called by themselves, never taken for
linears of no outputs.  The 4-bit product runs on the GPU alone; here a stand-in forward tells who was called."""
import types

import torch

import fused_linear
import shared_prefix
import workloads
from test_group_host import _frozen, _lora


def _four_bit(lin):
    """What enable_mxfp4 leaves of a linear, with a product that the CPU has."""
    w = lin.weight.data.clone()
    lin._mx4 = (None, "e4m3")
    lin.weight.data = torch.empty((0,), dtype=w.dtype)
    lin.forward = types.MethodType(lambda self, x: x @ w.t(), lin)
    return w


def test_a_four_bit_linear_beside_a_thin_one():
    g = torch.Generator().manual_seed(1)
    lin, thin, x = _frozen(128, 64, g), _frozen(16, 64, g), torch.randn(5, 64, generator=g)
    w = _four_bit(lin)
    assert fused_linear._part(lin) is None
    a, b = fused_linear.group_linear(x, (lin, thin))
    assert torch.equal(a, x @ w.t()) and torch.equal(b, thin(x))


def test_a_four_bit_linear_with_adapters():
    g = torch.Generator().manual_seed(2)
    mods = [_lora(128, 64, 8, g), _lora(64, 64, 8, g)]
    x = torch.randn(5, 64, generator=g)
    want = [m(x) for m in mods]
    for m in mods:
        _four_bit(m.base_layer)
        assert fused_linear._part(m) is None and fused_linear._adapted(m)[0] is m.base_layer
    for a, b in zip(fused_linear.group_linear(x, mods), want):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)
    y = fused_linear.group_linear(x, mods[:1], defer=True)[0]
    assert not isinstance(y, fused_linear.Deferred)
    torch.testing.assert_close(fused_linear.residual_add(want[0], y), 2 * want[0], rtol=1e-5, atol=1e-5)


def test_an_mlp_taken_whole_is_called_as_it_is():
    model, inps = workloads.build_model(1, T=4, layers=1, device="cpu")
    mlp = model.layers[0].mlp
    mlp._mx4_gated = ()
    mlp.forward = types.MethodType(lambda self, x: x + 1, mlp)
    for name in ("gate_proj", "up_proj", "down_proj"):
        _four_bit(getattr(mlp, name).base_layer)
    x = inps[0]["x"].float()
    assert torch.equal(shared_prefix._mlp(mlp, x), x + 1)

"""GPU tests of the 4-bit operators inside a model: enable_mxfp4 and its MLP against the oracle, adapters' gradients, what is
put back, the distillation example, and the products' behaviour under autograd."""
import pytest
import torch

import _native
import distill
import distill_mxfp4
import mxfp4
import workloads
from oracle import mx4

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _model(gpu, layers=1, d=160, ffn=288, rank=8):
    return distill_mxfp4.Model(layers, d, ffn, 64, rank, True).to(gpu)


def test_enable_mxfp4_mlp_against_the_oracle_and_back(gpu):
    m = _model(gpu)
    mod = m.model.layers[0].mlp
    base = {n: getattr(mod, n).base_layer.weight.detach().clone() for n in ("gate_proj", "up_proj", "down_proj")}
    lora = {n: (getattr(mod, n).lora_A["default"].weight, getattr(mod, n).lora_B["default"].weight, getattr(mod, n).scaling["default"])
            for n in base}
    x = torch.randn(50, 160, generator=torch.Generator().manual_seed(1)).to(BF)
    with torch.autocast("cuda", BF):
        before = mod(x.to(gpu))
    assert mxfp4.enable_mxfp4(m) == 3
    xg = x.to(gpu).requires_grad_(True)
    y = mod(xg)
    y.float().sum().backward()
    with pytest.raises(RuntimeError):
        mod.gate_proj(xg)  # held by the block
    ad = lambda n, t: ((t @ lora[n][0].detach().to(BF).t()) @ lora[n][1].detach().to(BF).t()) * lora[n][2]  # noqa: E731
    with torch.no_grad():
        add = torch.cat([ad("gate_proj", x.to(gpu)), ad("up_proj", x.to(gpu))], -1)
        h = mxfp4.mx4_gated(x.to(gpu), mxfp4.GatedWeight(base["gate_proj"], base["up_proj"]), add=add)
        ref = mxfp4.mx4_linear(h, mxfp4.Weight(base["down_proj"])) + ad("down_proj", h)
    assert torch.equal(y, ref)
    r = mx4.gated(x, base["gate_proj"].cpu(), base["up_proj"].cpu(), "e4m3", "silu", add.cpu())
    assert ((h.double().cpu() - r["h"]).abs() <= 2.0 ** -7 * r["h"].abs() + 2.0 ** -7 * r["h"].abs().max()).all()
    for n in base:
        for p in lora[n][:2]:
            assert p.grad is not None and p.grad.abs().max() > 0
    assert xg.grad.abs().max() > 0
    for n in base:
        getattr(mod, n).disable_adapters = True
    with torch.no_grad():
        h = mxfp4.mx4_gated(x.to(gpu), mxfp4.GatedWeight(base["gate_proj"], base["up_proj"]))
        assert torch.equal(mod(x.to(gpu)), mxfp4.mx4_linear(h, mxfp4.Weight(base["down_proj"])))
    mod.up_proj.disable_adapters = False
    mod.up_proj.merged = True
    with pytest.raises(ValueError):
        mod(x.to(gpu))
    mod.up_proj.merged = mod.gate_proj.disable_adapters = mod.down_proj.disable_adapters = False
    mxfp4.disable_mxfp4(m)
    for n in base:
        assert torch.equal(getattr(mod, n).base_layer.weight, base[n])
    with torch.autocast("cuda", BF):
        assert torch.equal(mod(x.to(gpu)), before)


def test_enable_mxfp4_refusals_and_plain_linears(gpu):
    m = workloads.build_attn(128, 128, 64, 8, 8, device=gpu)
    with pytest.raises(ValueError):
        mxfp4.enable_mxfp4(m, act="fp4")
    q = m.model.layers[0].self_attn.q_proj
    w = q.base_layer.weight.detach().clone()
    assert mxfp4.enable_mxfp4(m, act="e2m1") == 4
    with pytest.raises(ValueError):
        mxfp4.enable_mxfp4(m)  # twice
    x = torch.randn(20, 128, generator=torch.Generator().manual_seed(2)).to(BF).to(gpu)
    assert torch.equal(q.base_layer(x), mxfp4.mx4_linear(x, mxfp4.Weight(w), act="e2m1"))
    mxfp4.disable_mxfp4(m)
    assert torch.equal(q.base_layer.weight, w) and "forward" not in q.base_layer.__dict__


def test_distillation_example_learns(gpu):
    r = distill_mxfp4.run(steps=80, tokens=512, d=256, ffn=640, vocab=1000, log=lambda *a: None)
    assert r["linears"] == 6 and r["start"] > 0.01
    # what the adapters hold is learnable, the quantization's full-rank noise is not
    assert r["end"] < 0.8 * r["start"], (r["start"], r["end"])
    s, held = r["student"], r["held"]
    with torch.no_grad():
        many = s(held[0][:40], held[1][:40]).float()
        for rows in (1, 5, 16):  # single-token forms against the batch: other order of the sums, then bf16 through two layers
            few = s(held[0][:rows], held[1][:rows]).float()
            assert (few - many[:rows]).abs().max() <= 0.05 * many[:rows].abs().max()
    assert len(s.answer([1, 2], 4)) == 6


@pytest.mark.parametrize("act", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M", [8, 16, 17, 33, 64, 65])
@pytest.mark.parametrize("N,K", [(96, 4096), (50, 1024), (2048, 256)])
def test_few_and_thin_rows_agree_with_the_tiles(gpu, M, N, K, act):
    """Each row count's kernel against mx4_mm's tiles on the same operands (an fp32 result, then rounded): sums of K terms in
    another order, K 2^-24 (E4M3: 2^-12) of the sum of magnitudes, and one unit of bf16."""
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(BF).to(gpu)
    w = (torch.randn(N, K, generator=torch.Generator().manual_seed(N)) * 0.1).to(BF).to(gpu)
    got = mxfp4.mx4_linear(x, mxfp4.Weight(w), act=act).float()
    a, b = mxfp4.mx4_quant(x, fmt=act), mxfp4.mx4_quant(w)
    ref = mxfp4.mx4_mm(a, b, dtype=torch.float32)
    mag = mxfp4.mx4_dequant(a).abs() @ mxfp4.mx4_dequant(b).abs().t()
    bound = 2.0 ** -8 * ref.abs() + (2.0 ** -12 if act == "e4m3" else K * 2.0 ** -24) * mag
    assert ((got - ref).abs() <= bound).all()
    G = mxfp4.GatedWeight(w, w.flip(0))
    with torch.no_grad():
        h = mxfp4.mx4_gated(x, G, act=act)
    hg = mxfp4.mx4_gated(x.clone().requires_grad_(True), G, act=act)  # the tiles: something is saved
    top = mag.max() * mag.max()
    assert ((h - hg).float().abs() <= 2.0 ** -7 * hg.float().abs() + 2.0 ** -11 * top).all()


def test_double_backward_and_graph_rules(gpu):
    x = torch.randn(30, 64, generator=torch.Generator().manual_seed(1)).to(BF).to(gpu).requires_grad_(True)
    W = mxfp4.Weight(torch.randn(96, 64, generator=torch.Generator().manual_seed(2)).to(BF).to(gpu))
    dy = torch.randn(30, 96, generator=torch.Generator().manual_seed(3)).to(BF).to(gpu).requires_grad_(True)
    y = mxfp4.mx4_linear(x, W)
    dx, = torch.autograd.grad(y, x, dy, create_graph=True)
    v = torch.randn(30, 64, generator=torch.Generator().manual_seed(4)).to(BF).to(gpu)
    ddy, = torch.autograd.grad(dx, dy, v)  # the gradient of a product with Wᵀ is one with W
    assert torch.equal(ddy, mxfp4.mx4_linear(v, W).detach())
    G = mxfp4.GatedWeight(W_(gpu, 5), W_(gpu, 6))
    h = mxfp4.mx4_gated(x, G)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(h, x, torch.ones_like(h), create_graph=True)
    h = mxfp4.mx4_gated(x, G)
    h.sum().backward()
    with pytest.raises(RuntimeError):
        h.sum().backward()  # what it kept is gone
    z = torch.randn(4, 50, device=gpu, requires_grad=True)
    idx = torch.zeros(4, 1, dtype=torch.int32, device=gpu)
    loss = distill.topk_kl(z, idx, torch.zeros(4, 1, device=gpu))
    z.data.add_(0)
    with torch.no_grad():
        z.mul_(1.0)  # the logits changed: the saved statistics are not theirs
    with pytest.raises(RuntimeError):
        loss.sum().backward()


def W_(gpu, seed):
    return torch.randn(96, 64, generator=torch.Generator().manual_seed(seed)).to(BF).to(gpu)


def test_saved_tensors_pass_through_hooks(gpu):
    x = torch.randn(40, 64, generator=torch.Generator().manual_seed(1)).to(BF).to(gpu).requires_grad_(True)
    G = mxfp4.GatedWeight(W_(gpu, 2), W_(gpu, 3))
    mxfp4.mx4_gated(x, G).sum().backward()
    ref, x.grad = x.grad.clone(), None
    seen = []

    def pack(t):
        seen.append(t.shape)
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(gpu)):
        h = mxfp4.mx4_gated(x, G)
    h.sum().backward()
    assert seen and torch.equal(x.grad, ref)


def test_gradients_of_another_type_and_refused_types(gpu):
    x = torch.randn(20, 64, device=gpu).to(BF).requires_grad_(True)
    W = mxfp4.Weight(W_(gpu, 1))
    dy = torch.randn(20, 96, device=gpu)
    mxfp4.mx4_linear(x, W).backward(dy)  # autograd rounds it to the output's type
    got, x.grad = x.grad, None
    mxfp4.mx4_linear(x, W).backward(dy.to(BF))
    assert torch.equal(got, x.grad)
    with pytest.raises(_native.NativeError):
        mxfp4.mx4_linear(x.double(), W)


def test_enabled_layers_cast_under_autocast_as_linears_do(gpu):
    m = _model(gpu)
    mod = m.model.layers[0].mlp
    mxfp4.enable_mxfp4(m)
    x = torch.randn(30, 160, generator=torch.Generator().manual_seed(1)).to(gpu).requires_grad_(True)
    with torch.autocast("cuda", BF):
        y = mod(x)
    y.sum().backward()
    assert y.dtype == BF and x.grad.dtype == torch.float32
    assert torch.equal(y, mod(x.detach().to(BF)))
    with pytest.raises(_native.NativeError):
        mod(x)  # fp32 and no autocast
    a = workloads.build_attn(128, 128, 64, 8, 8, device=gpu)
    mxfp4.enable_mxfp4(a)
    q = a.model.layers[0].self_attn.q_proj.base_layer
    with torch.autocast("cuda", torch.float16):
        assert q(torch.randn(3, 128, device=gpu)).dtype == torch.float16

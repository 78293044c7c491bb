"""Frozen weights in MXFP4 (E2M1 codes, one E8M0 scale per 32 elements) on MI355X: quantization, the linear layer, the
gated feed-forward block, and their single-token forms.

The 4-bit counterpart of mxfp8: a frozen weight takes 17/32 byte an element and axis, and its products run on the scaled
matrix instructions with activations in 8 bits (act="e4m3", their rate is the 8-bit one) or 4 (act="e2m1", up to twice
that).  Everything runs in the hand-written kernels of libmxfp8_mlp.so; a CPU tensor is an error.

    W = mxfp4.Weight(linear.weight)            # once: both axes, [N, K]
    y = mxfp4.mx4_linear(x, W)                 # [.., N]; autograd gives dx, the weight is frozen
    G = mxfp4.GatedWeight(gate.weight, up.weight)
    h = mxfp4.mx4_gated(x, G)                  # silu(x Wgᵀ) * (x Wuᵀ)
    mxfp4.enable_mxfp4(model)                  # or a whole model's frozen linears and gated MLPs, adapters kept

Block scale: with amax the largest magnitude of the block and max = 6 (E2M1) or 448 (E4M3), the least power of two e with
amax <= max e (so nothing is clipped), 2^-127 at the least; codes round to nearest, ties to even.  A NaN makes its block
NaN; an infinity takes the format's largest value times 2^127.  Sums are fp32, with one rounding to the output's type.
With act="e2m1" the products that they add are exact.  With act="e4m3" the matrix instruction adds groups of 16 in fewer
bits: every term loses what lies below 2^-13 of the group's largest, 5e-6 of a result (rms) for normally distributed
values and 7e-5 for values spread over a block's whole range, so some outputs round to a neighbour of what fp32 sums give.
"""
import types

import torch
from torch import nn

import _native
import mxfp8
from fused_linear import _adapted

E2M1, E4M3 = 4, 8
_FMT = {"e2m1": E2M1, "e4m3": E4M3}
_FN = {"silu": 0, "gelu": 1}
_PLAIN = 0  # rows of an operand in their own order (include/mxfp4_ops.h)


def _fmt(name):
    if name not in _FMT:
        raise ValueError(f"unknown format {name!r}: one of {sorted(_FMT)}")
    return _FMT[name]


class MX:
    """A matrix [rows, cols] in MX form: codes q and E8M0 scales s in the blocked layouts of include/mxfp4_ops.h."""

    __slots__ = ("q", "s", "rows", "cols", "fmt")

    def __init__(self, q, s, rows, cols, fmt):
        self.q, self.s, self.rows, self.cols, self.fmt = q, s, rows, cols, fmt

    @property
    def shape(self):
        return (self.rows, self.cols)

    @property
    def nbytes(self):
        return self.q.numel() + self.s.numel()


def mx4_quant(x, fmt="e2m1", both=False):
    """x [R, C] (bf16, f16 or f32, any strides) -> MX along its columns; with both also MX of xᵀ [C, R] along x's rows,
    from the same read."""
    f = _fmt(fmt)
    if not both:
        return MX(*_native.host4().quant(x, f, _PLAIN), *x.shape, f)
    q, s, qt, st = _native.host4().quant_both(x, f, _PLAIN)
    R, C = x.shape
    return MX(q, s, R, C, f), MX(qt, st, C, R, f)


def mx4_dequant(m, dtype=torch.float32):
    """The values that an MX matrix stands for (exact in bf16 and f32; f16 as far as its exponents reach)."""
    return _native.host4().dequant(m.q, m.s, m.rows, m.cols, m.fmt, dtype)


def mx4_mm(a, b, dtype=torch.bfloat16):
    """a [M, K] · b [N, K]ᵀ of two MX matrices, b in E2M1 -> [M, N]."""
    if a.cols != b.cols or b.fmt != E2M1:
        raise ValueError(f"mx4_mm: {a.shape} by {b.shape} transposed, the second in e2m1")
    return _native.host4().gemm(a.q, a.s, a.fmt, b.q, b.s, _PLAIN, a.rows, b.rows, a.cols, dtype)


class Weight:
    """A frozen linear weight [N, K] in MXFP4 along K (forward) and along N (input gradient).  transpose=False keeps the
    first alone, for programs that never differentiate."""

    __slots__ = ("handle",)

    def __init__(self, w, transpose=True):
        self.handle = _native.host4().Weight(w, transpose)

    def __deepcopy__(self, memo):
        return self  # frozen: a copied model shares it

    @property
    def shape(self):
        return (self.handle.N, self.handle.K)

    @property
    def nbytes(self):
        return self.handle.nbytes


class GatedWeight:
    """The frozen gate and up weights [N, K] of a gated block: one operand along K, with gate and up rows next to each
    other, and one of [W_gate; W_up]ᵀ along N."""

    __slots__ = ("handle",)

    def __init__(self, w_gate, w_up):
        self.handle = _native.host4().Gated(w_gate, w_up)

    def __deepcopy__(self, memo):
        return self

    @property
    def shape(self):
        return (self.handle.N, self.handle.K)

    @property
    def nbytes(self):
        return self.handle.nbytes


def mx4_linear(x, w, act="e4m3"):
    """y = MX(x) · MX(W)ᵀ for x [.., K] in bf16 or f16 -> [.., N]; backward dx = MX(dy) · MX(Wᵀ)ᵀ with dy in the same
    format.  Up to 16 rows take one launch, quantization included."""
    return _native.host4().linear(w.handle, x, _FMT.get(act) or _fmt(act))


def mx4_gated(x, w, add=None, fn="silu", act="e4m3"):
    """h = fn(g) * u with [g | u] = MX(x) · MX([W_gate; W_up])ᵀ + add, for x [.., K] in bf16 or f16 -> [.., N]; fn "silu"
    or "gelu" (tanh form).  add: [.., 2 N] of x's type, or anything that broadcasts to it (a bias, adapters' output).
    Backward: dg and du from [g | u] kept in x's type, dx = MX(dg) · MX(W_gateᵀ)ᵀ + MX(du) · MX(W_upᵀ)ᵀ, d add = [dg | du].
    Without gradients up to 16 rows take one launch, quantization included, and nothing is kept."""
    if fn not in _FN:
        raise ValueError(f"unknown gate function {fn!r}: one of {sorted(_FN)}")
    return _native.host4().gated(w.handle, x, add, _FN[fn], _FMT.get(act) or _fmt(act))


# ---------------------------------------------------------------- a model's frozen linears
_SILU, _GELU = ("SiLU", "SiLUActivation"), ("GELUTanh", "PytorchGELUTanh")


def _gate_name(mlp):
    """The gate function of a gated MLP module, or None for one that mx4_gated does not have."""
    f = getattr(mlp, "act_fn", None)
    name = type(f).__name__
    if name in _SILU:
        return "silu"
    return "gelu" if name in _GELU or (isinstance(f, nn.GELU) and f.approximate == "tanh") else None


def _lora(proj):
    """fused_linear._adapted, and the base layer alone where the adapters are switched off for a while."""
    part = _adapted(proj)
    off = part is None and getattr(proj, "disable_adapters", False) and not proj.merged
    return (proj.base_layer, None, None, 1.0) if off else part


def _adapter(x, part):
    """An adapter's output s (x Aᵀ) Bᵀ in x's type, or None."""
    _, A, B, s = part
    return None if A is None else ((x @ A.to(x.dtype).t()) @ B.to(x.dtype).t()) * s


def _autocast(x):
    """x as a linear under autocast takes it: every floating type but float64 in autocast's."""
    on = x.is_cuda and x.is_floating_point() and x.dtype != torch.float64 and torch.is_autocast_enabled("cuda")
    return x.to(torch.get_autocast_dtype("cuda")) if on else x


def mlp(mod, x):
    """down(fn(gate(x)) * up(x)) of a gated MLP that enable_mxfp4 took: one gated block over the gate and up weights with
    their adapters' outputs added before the gate, and one linear."""
    G, D, fn, act = mod._mx4_gated
    parts = [_lora(getattr(mod, n)) for n in ("gate_proj", "up_proj", "down_proj")]
    if None in parts:
        raise ValueError("mxfp4.mlp: gate, up and down take plain frozen linears or one LoRA adapter without dropout, unmerged")
    x = _autocast(x)
    g, u = _adapter(x, parts[0]), _adapter(x, parts[1])
    add = None
    if g is not None or u is not None:
        zero = x.new_zeros(())
        wide = (*x.shape[:-1], G.shape[0])
        add = torch.cat([zero.expand(wide) if t is None else t for t in (g, u)], -1)
    h = mx4_gated(x, G, add=add, fn=fn, act=act)
    y = mx4_linear(h, D, act=act)
    d = _adapter(h, parts[2])
    return y if d is None else y + d


def _linear_forward(self, x):
    W, act = self._mx4
    if W is None:
        raise RuntimeError("this projection is held by its MLP's gated block (mxfp4.enable_mxfp4) and has no call of its own")
    return mx4_linear(_autocast(x), W, act=act)


def _patch(mod, forward):
    """Route mod's calls through `forward`; what its own `forward` attribute was, if it had one, waits in _mx4_forward."""
    mod._mx4_forward = mod.__dict__.get("forward")
    mod.forward = types.MethodType(forward, mod)


def _unpatch(mod):
    own = mod.__dict__.pop("_mx4_forward")
    del mod.forward
    if own is not None:
        mod.forward = own


def enable_mxfp4(model, act="e4m3"):
    """Quantize every frozen base linear of the decoder layers (those of mxfp8.enable_mxfp8: any shape here, no bias) to
    MXFP4 along both axes, move the weights to host memory and route the layers' forward through mx4_linear.  An MLP with
    gate_proj, up_proj, down_proj and a SiLU or tanh-GELU act_fn runs as `mlp` instead, if its adapters let it: hooks on the
    MLP run, hooks on its three projections do not, and gate_proj and up_proj cannot be called by themselves.  LoRA wrappers
    keep working: their base layer is what changes.  A call that fails leaves the model as it was.  Returns the number of
    linears."""
    _fmt(act)  # refuses an unknown name before anything is touched
    found = {id(lin): lin for _, lin in mxfp8._base_linears(model)}
    for lin in found.values():
        if lin.bias is not None or mxfp8.is_mx(lin) or "_mx4" in lin.__dict__:
            raise ValueError("enable_mxfp4: linears without bias that are not quantized yet")
    try:
        _enable(model, found, act)
    except BaseException:
        disable_mxfp4(model)
        raise
    torch.cuda.empty_cache()
    return len(found)


def _enable(model, found, act):
    held = {}
    for mod in model.modules():
        projs = [getattr(mod, n, None) for n in ("gate_proj", "up_proj", "down_proj")]
        if None in projs or _gate_name(mod) is None or None in [_lora(p) for p in projs]:
            continue
        base = [getattr(p, "base_layer", p) for p in projs]
        if all(id(b) in found for b in base) and base[0].weight.shape == base[1].weight.shape \
                and base[0].weight.dtype == base[1].weight.dtype:
            G, D = GatedWeight(base[0].weight, base[1].weight), Weight(base[2].weight)
            mod._mx4_gated = (G, D, _gate_name(mod), act)
            _patch(mod, mlp)
            held.update({id(base[0]): None, id(base[1]): None, id(base[2]): D})
    for lin in found.values():
        w = lin.weight.data
        W, cpu = held[id(lin)] if id(lin) in held else Weight(w), w.to("cpu", copy=True)
        lin._mx4, lin._mx4_cpu = (W, act), cpu
        lin.weight.data = torch.empty((0,), dtype=w.dtype, device=w.device)
        _patch(lin, _linear_forward)


def disable_mxfp4(model):
    """Put the weights back on their device and take the 4-bit copies and the patched forwards away."""
    for mod in model.modules():
        if "_mx4_gated" in mod.__dict__:
            del mod._mx4_gated
            _unpatch(mod)
        if "_mx4" in mod.__dict__:
            mod.weight.data = mod._mx4_cpu.to(mod.weight.device)
            del mod._mx4, mod._mx4_cpu
            _unpatch(mod)
    torch.cuda.empty_cache()

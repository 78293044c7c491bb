"""Frozen weights in MXFP4 (E2M1 codes, one E8M0 scale per 32 elements) on MI355X: quantization, the linear layer, the
gated feed-forward block, and their single-token forms.

The 4-bit counterpart of mxfp8: a frozen weight takes 17/32 byte an element and axis, and its products run on the scaled
matrix instructions with activations in 8 bits (act="e4m3", their rate is the 8-bit one) or 4 (act="e2m1", up to twice
that).  Everything runs in the hand-written kernels of libmxfp8_mlp.so; a CPU tensor is an error.

    W = mxfp4.Weight(linear.weight)            # once: both axes, [N, K]
    y = mxfp4.mx4_linear(x, W)                 # [.., N]; autograd gives dx, the weight is frozen
    G = mxfp4.GatedWeight(gate.weight, up.weight)
    h = mxfp4.mx4_gated(x, G)                  # silu(x Wgᵀ) * (x Wuᵀ)

Block scale: with amax the largest magnitude of the block and max = 6 (E2M1) or 448 (E4M3), the least power of two e with
amax <= max e (so nothing is clipped), 2^-127 at the least; codes round to nearest, ties to even.  A NaN makes its block
NaN; an infinity takes the format's largest value times 2^127.  Sums are fp32, with one rounding to the output's type.
"""
import torch

import _native

E2M1, E4M3 = 4, 8
_FMT = {"e2m1": E2M1, "e4m3": E4M3}
_FN = {"silu": 0, "gelu": 1}
_PLAIN, _PI = 0, 1  # row orders of an operand (include/mxfp4_ops.h)


def _fmt(name):
    if name not in _FMT:
        raise ValueError(f"unknown format {name!r}: one of {sorted(_FMT)}")
    return _FMT[name]


class MX:
    """A matrix [rows, cols] in MX form: codes q and E8M0 scales s in the blocked layouts of include/mxfp4_ops.h."""

    __slots__ = ("q", "s", "rows", "cols", "fmt", "order")

    def __init__(self, q, s, rows, cols, fmt, order=_PLAIN):
        self.q, self.s, self.rows, self.cols, self.fmt, self.order = q, s, rows, cols, fmt, order

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
    st = _native.stream_of(x, "mx4_quant")
    R, C = x.shape
    if not both:
        return MX(*_native.host4().quant(x.detach(), f, _PLAIN, st), R, C, f)
    q, s, qt, stt = _native.host4().quant_both(x.detach(), f, _PLAIN, st)
    return MX(q, s, R, C, f), MX(qt, stt, C, R, f)


def mx4_dequant(m, dtype=torch.float32):
    """The values that an MX matrix stands for (exact in bf16 and f32; f16 as far as its exponents reach)."""
    if m.order != _PLAIN:
        raise ValueError("mx4_dequant: a weight's own operand has its rows in another order")
    return _native.host4().dequant(m.q, m.s, m.rows, m.cols, m.fmt, dtype, _native.stream_of(m.q, "mx4_dequant"))


def mx4_mm(a, b, dtype=torch.bfloat16):
    """a [M, K] · b [N, K]ᵀ of two MX matrices, b in E2M1 -> [M, N]."""
    if a.cols != b.cols or b.fmt != E2M1 or a.order != _PLAIN:
        raise ValueError(f"mx4_mm: {a.shape} by {b.shape} transposed, the second in e2m1")
    return _native.host4().gemm(a.q, a.s, a.fmt, b.q, b.s, b.order, a.rows, b.rows, a.cols, dtype,
                                _native.stream_of(a.q, "mx4_mm"))


class Weight:
    """A frozen linear weight [N, K] in MXFP4 along K (forward) and along N (input gradient).  transpose=False keeps the
    first alone, for programs that never differentiate."""

    def __init__(self, w, transpose=True):
        w = w.detach()
        if w.dim() != 2 or w.numel() == 0:
            raise ValueError(f"Weight: a matrix, not {tuple(w.shape)}")
        self.N, self.K = w.shape
        st = _native.stream_of(w, "Weight")
        if transpose:
            self.q, self.s, self.qt, self.st = _native.host4().quant_both(w, E2M1, _PI, st)
        else:
            self.q, self.s = _native.host4().quant(w, E2M1, _PI, st)
            self.qt = self.st = None


class GatedWeight:
    """The frozen gate and up weights [N, K] of a gated block: one operand along K, with gate and up rows next to each
    other, and one of [W_gate; W_up]ᵀ along N."""

    def __init__(self, w_gate, w_up):
        self.N, self.K = w_gate.shape
        self.q, self.s, self.qt, self.st = _native.host4().quant_gate_up(
            w_gate.detach(), w_up.detach(), _native.stream_of(w_gate, "GatedWeight"))


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, fmt):
        ctx.w, ctx.fmt = w, fmt
        return _native.host4().linear(x, w.q, w.s, w.N, w.K, fmt, _native.stream_of(x, "mx4_linear"))

    @staticmethod
    def backward(ctx, dy):
        w = ctx.w
        dx = _native.host4().linear(dy, w.qt, w.st, w.K, w.N, ctx.fmt, _native.stream_of(dy, "mx4_linear"))
        return dx, None, None


def mx4_linear(x, w, act="e4m3"):
    """y = MX(x) · MX(W)ᵀ for x [.., K] in bf16 or f16 -> [.., N]; backward dx = MX(dy) · MX(Wᵀ)ᵀ with dy in the same
    format.  Up to 16 rows take one launch, quantization included."""
    f = _FMT.get(act) or _fmt(act)
    if torch.is_grad_enabled() and x.requires_grad:
        if w.qt is None:
            raise ValueError("mx4_linear: this weight was made without its transpose, it has no input gradient")
        return _Linear.apply(x, w, f)
    return _native.host4().linear(x, w.q, w.s, w.N, w.K, f, _native.stream_of(x, "mx4_linear"))


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, add, w, fn, fmt):
        ctx.w, ctx.fn, ctx.fmt, ctx.x_shape = w, fn, fmt, x.shape
        h, gu = _native.host4().gated(x, w.q, w.s, w.N, w.K, add, fn, fmt, True, _native.stream_of(x, "mx4_gated"))
        ctx.save_for_backward(gu)
        return h

    @staticmethod
    def backward(ctx, dh):
        w, (gu,) = ctx.w, ctx.saved_tensors
        need_x, need_add = ctx.needs_input_grad[:2]
        dx, dgu = _native.host4().gated_bwd(gu, dh, w.qt, w.st, w.N, w.K, ctx.fn, ctx.fmt, need_x, need_add,
                                            _native.stream_of(dh, "mx4_gated"))
        lead = ctx.x_shape[:-1]
        return dx.view(ctx.x_shape) if need_x else None, dgu.view(*lead, 2 * w.N) if need_add else None, None, None, None


def mx4_gated(x, w, add=None, fn="silu", act="e4m3"):
    """h = fn(g) * u with [g | u] = MX(x) · MX([W_gate; W_up])ᵀ + add, for x [.., K] in bf16 or f16 -> [.., N]; fn "silu"
    or "gelu" (tanh form).  add: [.., 2 N] of x's type, or anything that broadcasts to it (a bias, adapters' output).
    Backward: dg and du from [g | u] kept in x's type, dx = MX(dg) · MX(W_gateᵀ)ᵀ + MX(du) · MX(W_upᵀ)ᵀ, d add = [dg | du].
    Without gradients up to 16 rows take one launch, quantization included, and nothing is kept."""
    f = _FMT.get(act) or _fmt(act)
    if fn not in _FN:
        raise ValueError(f"unknown gate function {fn!r}: one of {sorted(_FN)}")
    grad = torch.is_grad_enabled() and (x.requires_grad or (add is not None and add.requires_grad))
    if add is not None:
        add = add.expand(*x.shape[:-1], 2 * w.N)  # autograd sums the gradient of what is broadcast
    if grad:
        return _Gated.apply(x, add, w, _FN[fn], f)
    return _native.host4().gated(x, w.q, w.s, w.N, w.K, add, _FN[fn], f, False, _native.stream_of(x, "mx4_gated"))[0]

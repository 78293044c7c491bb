"""CPU oracle of the 4-bit operators in float64: MX values by search among the format's values, products, the gated block
with its gradients, written from the definitions and apart from the kernels."""
import math

import torch

E2M1_VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
# 0, the subnormals, then four exponent bits by three mantissa bits without the NaN pattern
E4M3_VALUES = [m / 512 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1]
VALUES = {"e2m1": E2M1_VALUES, "e4m3": E4M3_VALUES}


def block_exponents(x, fmt):
    """E8M0 exponents (unbiased; nan for a block with a NaN, 127 for one with an infinity) of x [R, C]: float64 [R, C/32]."""
    top = VALUES[fmt][-1]
    R, C = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -C % 32)).reshape(R, -1, 32)
    amax = b.abs().amax(2)  # propagates NaN
    e = torch.full_like(amax, -127.0)
    for k in range(-127, 128):  # the least e with amax <= top 2^e
        e = torch.where(amax > top * 2.0 ** (k - 1), torch.full_like(e, float(k)), e)
    e = torch.where(torch.isinf(amax), torch.full_like(e, 127.0), e)
    return torch.where(torch.isnan(amax), amax, e), b


def values(x, fmt):
    """float64 [R, C]: the values that the MX form of x stands for."""
    R, C = x.shape
    e, b = block_exponents(x, fmt)
    v = torch.tensor(VALUES[fmt], dtype=torch.float64)
    scale = torch.pow(torch.tensor(2.0, dtype=torch.float64), torch.nan_to_num(e))[:, :, None]
    r = (b / scale).clamp(-v[-1].item(), v[-1].item())
    d = (r.abs()[..., None] - v).abs()
    near = d.min(-1, keepdim=True).values
    # of two equally near values the one with the even code
    idx = torch.arange(len(v))
    rank = torch.where(d == near, idx % 2, torch.full_like(idx, 2))
    code = rank.argmin(-1)
    out = torch.copysign(v[code], b) * scale
    out = torch.where(torch.isnan(e)[:, :, None], torch.full_like(out, math.nan), out)
    return out.reshape(R, -1)[:, :C]


def linear(x, w, act):
    """(y, Σ|terms|) of MX(x) · MX(W)ᵀ."""
    a, b = values(x, act), values(w, "e2m1")
    return a @ b.t(), a.abs() @ b.abs().t()


def gate(fn, g):
    """(fn(g), fn'(g)): silu, or gelu in its tanh form."""
    if fn == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s + g * s * (1 - s)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t ** 2) * c * (1 + 3 * 0.044715 * g ** 2)


def gated(x, wg, wu, act, fn, add=None):
    """dict of g, u (unrounded), h and the sums of |terms| of g and u."""
    N = wg.shape[0]
    gu, mag = linear(x, torch.cat([wg, wu]), act)
    if add is not None:
        gu = gu + add.double()
    g, u = gu[:, :N], gu[:, N:]
    return dict(g=g, u=u, h=gate(fn, g)[0] * u, mag=mag)


def gated_backward(g, u, dh, wg, wu, act, fn):
    """(dx, dg, du, MX values of dg and du) from the g and u that are kept (already in the activations' type)."""
    f, df = gate(fn, g)
    dg, du = dh.double() * u * df, dh.double() * f
    qg, qu = values(dg, act), values(du, act)
    return qg @ values(wg.t(), "e2m1").t() + qu @ values(wu.t(), "e2m1").t(), dg, du, (qg, qu)

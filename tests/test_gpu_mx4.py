"""GPU tests of the MXFP4 operators against the float64 oracle: values of quantized tensors are equal, products and the
gated block stay within bounds derived from the formats.

Bounds.  With S = Σ |terms| of an output element, fp32 sums of K exact E2M1 products are off by at most K 2^-24 S; the
matrix instruction drops low bits of the small E4M3 products of a step, 2^-13 of its largest term where it was measured, so
2^-12 S covers E4M3.  An output rounded to bf16 (f16) adds 2^-8 (2^-11) of itself, half a unit and the double rounding.
What follows a second quantization may see a code land on the neighbouring value, half a unit (2^-4 of a value in E4M3, 1/4
in E2M1) for the few values that lie within the fp32 error of a tie: up to four such codes a row are allowed for.
"""
import pytest
import torch

import mxfp4
from oracle import mx4

pytestmark = pytest.mark.gpu

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -23}
ACT = {"e4m3": 2.0 ** -12, "e2m1": None}
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _randn(seed, *shape, std=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std


def _sum_bound(act, K):
    return ACT[act] if ACT[act] else K * 2.0 ** -24


def _close(got, ref, bound, what=""):
    got = got.detach().double().cpu()
    bad = (got - ref).abs() > bound
    assert not bad.any() and not torch.isnan(got).any(), (what, int(bad.sum()), ((got - ref).abs() / bound).max().item())


# ---------------------------------------------------------------- quantization
@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("R,C", [(1, 32), (3, 1), (1, 128), (33, 130), (129, 257), (20, 40), (256, 384)])
def test_quant_values(gpu, R, C, dt, fmt):
    x = (_randn(R * 1000 + C, R, C) * torch.exp(2 * _randn(5, R, 1))).to(dt)
    m, mt = mxfp4.mx4_quant(x.to(gpu), fmt=fmt, both=True)
    one = mxfp4.mx4_quant(x.to(gpu), fmt=fmt)
    for got, ref in ((m, x), (one, x), (mt, x.t())):
        v = mxfp4.mx4_dequant(got).cpu()
        assert torch.equal(v.double(), mx4.values(ref, fmt)), (got.shape, fmt)
        assert torch.equal(mxfp4.mx4_dequant(got, BF).cpu().float(), v)


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_quant_edges(gpu, fmt):
    """Ties, powers of two times the largest value, zeros, denormals, infinities and NaN, each in its own block."""
    top = 6.0 if fmt == "e2m1" else 448.0
    x = torch.zeros(9, 64)
    x[0, :8] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    x[1, 0] = top * 2.0 ** 20
    x[2, 0] = top * 2.0 ** 20 * (1 + 2.0 ** -20)
    x[3, :4] = torch.tensor([3e38, -3.4e38, 1.0, 1e30])
    x[4, :4] = torch.tensor([1e-38, -1e-37, 3e-38, 1e-40])
    x[5, 32:36] = torch.tensor([float("inf"), 1.0, -5.0, 1e38])
    x[6, 40] = float("nan")
    x[7, :] = -0.0
    x[8, :] = torch.finfo(F32).min
    got, gott = mxfp4.mx4_quant(x.to(gpu), fmt=fmt, both=True)
    for m, r in ((got, x), (gott, x.t())):
        v, ref = mxfp4.mx4_dequant(m).cpu(), mx4.values(r, fmt)
        assert torch.equal(torch.isnan(v), torch.isnan(ref))
        big = ref.abs() > torch.finfo(F32).max  # 6 * 2^127: infinite in fp32
        assert torch.equal(torch.isinf(v), big)
        # E4M3 blocks with the least scale hold zeros (as mxfp8.mx_quant's): values below 448 * 2^-127
        ok = ~torch.isnan(ref) & ~big & ~((ref.abs() < 448 * 2.0 ** -127) if fmt == "e4m3" else torch.zeros_like(big))
        assert torch.equal(v.double()[ok], ref[ok])


def test_quant_strided_and_transposed_inputs(gpu):
    base = _randn(1, 70, 300).to(BF).to(gpu)
    for x in (base[:, 7:203], base[::3, :96], base.t(), base[5:6].expand(40, 300), base[:, ::2]):
        v = mxfp4.mx4_dequant(mxfp4.mx4_quant(x)).cpu()
        assert torch.equal(v.double(), mx4.values(x.cpu(), "e2m1"))
    for R, C in ((0, 64), (5, 0)):
        assert mxfp4.mx4_dequant(mxfp4.mx4_quant(base.new_empty(R, C))).shape == (R, C)


# ---------------------------------------------------------------- products
SHAPES = [(1, 1, 1), (1, 33, 40), (2, 64, 128), (16, 96, 2200), (17, 31, 100), (33, 130, 129), (64, 64, 256), (100, 300, 384),
          (130, 257, 640), (260, 520, 128)]


@pytest.mark.parametrize("act", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(gpu, M, N, K, act):
    x, w, dy = _randn(M, M, K).to(BF), _randn(N, N, K, std=0.1).to(BF), _randn(K, M, N).to(BF)
    W = mxfp4.Weight(w.to(gpu))
    xg = x.to(gpu).requires_grad_(True)
    y = mxfp4.mx4_linear(xg, W, act=act)
    y.backward(dy.to(gpu))
    ref, mag = mx4.linear(x, w, act)
    _close(y, ref, EPS[BF] * ref.abs() + _sum_bound(act, K) * mag, "y")
    ref, mag = mx4.linear(dy, w.t(), act)
    _close(xg.grad, ref, EPS[BF] * ref.abs() + _sum_bound(act, N) * mag, "dx")
    with torch.no_grad():
        assert torch.equal(mxfp4.mx4_linear(xg, W, act=act), y)


@pytest.mark.parametrize("act", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K", [(2050, 2100, 300), (4100, 4200, 256)])
def test_linear_every_tile_shape(gpu, M, N, K, act):
    """Sizes that reach the larger tiles, ragged on both sides; the reference is made on the GPU in float64."""
    x, w = _randn(1, M, K).to(BF), _randn(2, N, K, std=0.1).to(BF)
    y = mxfp4.mx4_linear(x.to(gpu), mxfp4.Weight(w.to(gpu)), act=act)
    a, b = mx4_gpu(x, act, gpu), mx4_gpu(w, "e2m1", gpu)
    ref, mag = (a @ b.t()).cpu(), (a.abs() @ b.abs().t()).cpu()
    _close(y, ref, EPS[BF] * ref.abs() + _sum_bound(act, K) * mag)


def mx4_gpu(x, fmt, gpu):
    """The oracle's values in slices (its search holds every value of the format for every element)."""
    return torch.cat([mx4.values(x[i:i + 256], fmt) for i in range(0, x.shape[0], 256)]).to(gpu)


@pytest.mark.parametrize("dt", [BF, HF, F32])
def test_mm_of_two_quantized_matrices(gpu, dt):
    for M, N, K, act in ((5, 7, 33, "e2m1"), (140, 200, 300, "e4m3"), (300, 64, 129, "e2m1")):
        a, b = _randn(1, M, K), _randn(2, N, K)
        got = mxfp4.mx4_mm(mxfp4.mx4_quant(a.to(gpu), fmt=act), mxfp4.mx4_quant(b.to(gpu)), dtype=dt)
        av, bv = mx4.values(a, act), mx4.values(b, "e2m1")
        ref, mag = av @ bv.t(), av.abs() @ bv.abs().t()
        _close(got, ref, EPS[dt] * ref.abs() + _sum_bound(act, K) * mag + (2.0 ** -24 if dt == HF else 0))


def test_linear_leading_dimensions_strides_and_f16(gpu):
    w = _randn(1, 96, 160, std=0.1)
    W = mxfp4.Weight(w.to(HF).to(gpu))
    x = _randn(2, 3, 50, 320).to(HF).to(gpu)[:, ::2, 7:167]
    for act in ("e4m3", "e2m1"):
        y = mxfp4.mx4_linear(x, W, act=act)
        assert y.shape == (3, 25, 96) and y.dtype == HF
        ref, mag = mx4.linear(x.cpu().reshape(-1, 160), w.to(HF), act)
        _close(y.reshape(-1, 96), ref, EPS[HF] * ref.abs() + _sum_bound(act, 160) * mag + 2.0 ** -24)
        few = mxfp4.mx4_linear(x[1, :7], W, act=act)
        _close(few, ref[25:32], EPS[HF] * ref[25:32].abs() + _sum_bound(act, 160) * mag[25:32] + 2.0 ** -24)
    assert mxfp4.mx4_linear(x[:0], W).shape == (0, 25, 96)
    one = mxfp4.mx4_linear(x[0, 0], W)
    assert one.shape == (96,) and torch.equal(one, mxfp4.mx4_linear(x[0, :1], W)[0])


def test_nan_and_infinity_stay_in_their_rows(gpu):
    x = _randn(1, 40, 256).to(BF)
    x[3, 100], x[30, 5] = float("nan"), float("inf")
    w = _randn(2, 64, 256).to(BF)
    W = mxfp4.Weight(w.to(gpu))
    for rows in (40, 10):
        for act in ("e4m3", "e2m1"):
            y = mxfp4.mx4_linear(x[:rows].to(gpu), W, act=act).cpu()
            assert torch.isnan(y[3]).all()
            keep = [i for i in range(rows) if i not in (3, 30)]
            ref, mag = mx4.linear(x[keep], w, act)
            _close(y[keep], ref, EPS[BF] * ref.abs() + _sum_bound(act, 256) * mag)


def test_results_do_not_change_from_call_to_call_or_stream_to_stream(gpu):
    x, W = _randn(1, 300, 512).to(BF).to(gpu), mxfp4.Weight(_randn(2, 700, 512).to(BF).to(gpu))
    G = mxfp4.GatedWeight(_randn(3, 700, 512).to(BF).to(gpu), _randn(4, 700, 512).to(BF).to(gpu))
    y, h = mxfp4.mx4_linear(x, W), mxfp4.mx4_gated(x, G)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            y2, h2 = mxfp4.mx4_linear(x, W), mxfp4.mx4_gated(x, G)
    side.synchronize()
    assert torch.equal(y, y2) and torch.equal(h, h2)


# ---------------------------------------------------------------- the gated block
@pytest.mark.parametrize("act", ["e4m3", "e2m1"])
@pytest.mark.parametrize("fn", ["silu", "gelu"])
@pytest.mark.parametrize("M,N,K,add", [(1, 32, 64, False), (5, 70, 100, True), (16, 128, 2048, False), (33, 31, 40, True),
                                       (150, 200, 256, True), (64, 257, 130, False)])
def test_gated(gpu, M, N, K, add, fn, act):
    x = _randn(M, M, K).to(BF)
    wg, wu = _randn(1, N, K, std=K ** -0.5).to(BF), _randn(2, N, K, std=K ** -0.5).to(BF)
    ad = _randn(3, M, 2 * N, std=0.5).to(BF) if add else None
    dh = _randn(4, M, N).to(BF)
    G = mxfp4.GatedWeight(wg.to(gpu), wu.to(gpu))
    xg = x.to(gpu).requires_grad_(True)
    ag = ad.to(gpu).requires_grad_(True) if add else None
    h = mxfp4.mx4_gated(xg, G, add=ag, fn=fn, act=act)
    h.backward(dh.to(gpu))
    r = mx4.gated(x, wg, wu, act, fn, ad)
    sb = _sum_bound(act, K)
    f, df = mx4.gate(fn, r["g"])
    # errors of g and u through h = f(g) u, and 2^-20 of the hardware exp2, reciprocal and products
    hb = (EPS[BF] + 2.0 ** -20) * r["h"].abs() + sb * (r["mag"][:, :N] * (df * r["u"]).abs() + r["mag"][:, N:] * f.abs()) \
        + 2 * sb * sb * r["mag"][:, :N] * r["mag"][:, N:]
    _close(h, r["h"], hb + 1e-30, "h")
    with torch.no_grad():  # up to 16 rows: the one-launch form, other order of the sums
        _close(mxfp4.mx4_gated(xg, G, add=ag, fn=fn, act=act), r["h"], hb + 1e-30, "h without gradients")
    g, u = r["g"].float().to(BF).double(), r["u"].float().to(BF).double()
    dx, dg, du, (qg, qu) = mx4.gated_backward(g, u, dh, wg, wu, act, fn)
    if add:
        # from the products that the instruction gives (small g and u carry its dropped bits); they may still round the
        # other way to the kept type: one unit of bf16 each, through the derivatives (|f''| <= 1.2 for both gates)
        got = ag.grad.double().cpu()
        acc = mxfp4.mx4_mm(mxfp4.mx4_quant(x.to(gpu), fmt=act), mxfp4.mx4_quant(torch.cat([wg, wu]).to(gpu)), dtype=F32)
        acc = (acc.cpu() + ad.float()).to(BF).double()
        g, u = acc[:, :N], acc[:, N:]
        fk, dfk = mx4.gate(fn, g)
        ref = torch.cat([dh.double() * u * dfk, dh.double() * fk], 1)
        dd = dh.double().abs()
        db = torch.cat([dd * 2.0 ** -7 * (u.abs() * dfk.abs() + 1.2 * u.abs() * g.abs()), dd * 2.0 ** -7 * g.abs() * 1.2], 1)
        _close(got, ref, (EPS[BF] + 2.0 ** -18) * ref.abs() + db + 1e-30, "dadd")
    tg, tu = mx4.values(wg.t(), "e2m1"), mx4.values(wu.t(), "e2m1")
    mag = qg.abs() @ tg.abs().t() + qu.abs() @ tu.abs().t()
    unit = 2.0 ** -3 if act == "e4m3" else 0.5
    top = (torch.cat([qg, qu], 1).abs().amax(1, keepdim=True) * torch.cat([tg, tu], 1).abs().amax(1)[None])
    _close(xg.grad, dx, EPS[BF] * dx.abs() + _sum_bound(act, 2 * N) * mag + 4 * unit * top + 1e-30, "dx")
    err = (xg.grad.double().cpu() - dx).pow(2).mean().sqrt() / dx.pow(2).mean().sqrt()
    assert err < 0.01, err  # bf16 alone is 0.0017; a few codes of the neighbouring value add to it


def test_gated_broadcast_addend_gets_the_summed_gradient(gpu):
    M, N, K = 40, 64, 128
    x = _randn(1, 2, M // 2, K).to(BF).to(gpu)
    G = mxfp4.GatedWeight(_randn(2, N, K, std=0.1).to(BF).to(gpu), _randn(3, N, K, std=0.1).to(BF).to(gpu))
    bias = _randn(4, 2 * N).to(BF).to(gpu).requires_grad_(True)
    full = bias.detach().expand(2, M // 2, 2 * N).contiguous().requires_grad_(True)
    dh = _randn(5, 2, M // 2, N).to(BF).to(gpu)
    h = mxfp4.mx4_gated(x, G, add=bias)
    h2 = mxfp4.mx4_gated(x, G, add=full)
    assert h.shape == (2, M // 2, N) and torch.equal(h, h2)
    h.backward(dh)
    h2.backward(dh)
    ref = full.grad.double().sum((0, 1))
    _close(bias.grad, ref.cpu(), (2.0 ** -8 * ref.abs() + 1e-6).cpu())


def test_gated_addend_gradient_against_differences(gpu):
    """d h / d add by central differences of the float64 formula (nothing is quantized between the addend and h)."""
    M, N, K = 6, 32, 64
    x, wg, wu = _randn(1, M, K).to(BF), _randn(2, N, K, std=0.1).to(BF), _randn(3, N, K, std=0.1).to(BF)
    add, dh = _randn(4, M, 2 * N).to(BF), _randn(5, M, N).to(BF)
    for fn in ("silu", "gelu"):
        ag = add.to(gpu).requires_grad_(True)
        h = mxfp4.mx4_gated(x.to(gpu), mxfp4.GatedWeight(wg.to(gpu), wu.to(gpu)), add=ag, fn=fn)
        h.backward(dh.to(gpu))
        d = 1e-5
        for half in (0, 1):
            step = torch.zeros(1, 2 * N, dtype=torch.float64)
            step[:, half * N:(half + 1) * N] = d
            hi = mx4.gated(x, wg, wu, "e4m3", fn, add.double() + step)["h"]
            lo = mx4.gated(x, wg, wu, "e4m3", fn, add.double() - step)["h"]
            num = (hi - lo) / (2 * d) * dh.double()
            # g and u are kept in bf16: 2^-8 of values up to 4, through derivatives up to 1.2, and the output's rounding
            bound = 2.0 ** -8 * num.abs() + dh.double().abs() * 2.0 ** -8 * 8
            _close(ag.grad[:, half * N:(half + 1) * N], num, bound)


def test_gated_without_gradient_of_x(gpu):
    x = _randn(1, 20, 64).to(BF).to(gpu)
    G = mxfp4.GatedWeight(_randn(2, 32, 64).to(BF).to(gpu), _randn(3, 32, 64).to(BF).to(gpu))
    add = torch.zeros(20, 64, dtype=BF, device=gpu, requires_grad=True)
    h = mxfp4.mx4_gated(x, G, add=add)
    h.sum().backward()  # a broadcast upstream gradient
    assert add.grad.shape == (20, 64) and x.grad is None
    assert mxfp4.mx4_gated(x[:0], G).shape == (0, 32)


def test_refusals(gpu):
    import _native
    W = mxfp4.Weight(torch.zeros(64, 128, dtype=BF, device=gpu))
    G = mxfp4.GatedWeight(torch.zeros(64, 128, dtype=BF, device=gpu), torch.zeros(64, 128, dtype=BF, device=gpu))
    x = torch.zeros(4, 128, dtype=BF, device=gpu)
    for bad in (x[:, :64], x.float(), x.cpu(), x.long()):
        with pytest.raises(_native.NativeError):
            mxfp4.mx4_linear(bad, W)
        with pytest.raises(_native.NativeError):
            mxfp4.mx4_gated(bad, G)
    with pytest.raises((RuntimeError, _native.NativeError)):
        mxfp4.mx4_gated(x, G, add=x[:, :64])
    with pytest.raises(_native.NativeError):
        mxfp4.mx4_gated(x, G, add=torch.zeros(4, 128, device=gpu))
    with pytest.raises(_native.NativeError):
        mxfp4.GatedWeight(torch.zeros(64, 128, dtype=BF, device=gpu), torch.zeros(32, 128, dtype=BF, device=gpu))
    with pytest.raises(ValueError):
        mxfp4.mx4_linear(x, W, act="bf16")
    with pytest.raises(ValueError):
        mxfp4.Weight(torch.zeros(0, 128, dtype=BF, device=gpu))
    with pytest.raises(ValueError):
        mxfp4.mx4_linear(x.clone().requires_grad_(True), mxfp4.Weight(torch.zeros(64, 128, dtype=BF, device=gpu), transpose=False))
    a, b = mxfp4.mx4_quant(x), mxfp4.mx4_quant(x[:, :64])
    with pytest.raises(ValueError):
        mxfp4.mx4_mm(a, b)
    with pytest.raises(ValueError):
        mxfp4.mx4_mm(a, mxfp4.mx4_quant(x, fmt="e4m3"))


def test_graph_replays(gpu):
    x = _randn(1, 200, 256).to(BF).to(gpu)
    one = _randn(2, 1, 256).to(BF).to(gpu)
    G = mxfp4.GatedWeight(_randn(3, 320, 256).to(BF).to(gpu), _randn(4, 320, 256).to(BF).to(gpu))
    W = mxfp4.Weight(_randn(5, 256, 320).to(BF).to(gpu))

    def f(a, b):
        with torch.no_grad():
            return mxfp4.mx4_linear(mxfp4.mx4_gated(a, G), W), mxfp4.mx4_linear(mxfp4.mx4_gated(b, G), W)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f(x, one)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f(x, one)
    for k in range(3):
        nx, no = _randn(10 + k, 200, 256).to(BF).to(gpu), _randn(20 + k, 1, 256).to(BF).to(gpu)
        ref = f(nx, no)
        x.copy_(nx)
        one.copy_(no)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1]), k

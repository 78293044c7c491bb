"""GPU tests of the distillation loss against the float64 oracle.

Bounds.  A row's loss is sums of at most V fp32 terms around logs of hardware exponentials: 2^-18 of the sum of |p log p|
and |p log q| covers k + log V roundings and the exponent's error (|z - m| / tau 2^-23 each).  A gradient is q - p of
magnitude at most 1, times weight and tau: 2^-17 of q and p, and the rounding of its type.
"""
import math

import pytest
import torch

import _native
import distill
from oracle import distill as od

pytestmark = pytest.mark.gpu

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10, torch.float32: 2.0 ** -22}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24, torch.float32: 1e-38}
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _case(seed, T, V, k, tau, rest, dt):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(T, V, generator=g) * 2).to(dt)
    idx = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(T)]) if T else torch.zeros(0, k, dtype=torch.int64)
    t = torch.randn(T, k, generator=g) * 2
    lse = (torch.logsumexp(t / tau, 1) + 0.3) if rest else None
    w = torch.rand(T, generator=g)
    return z, idx, t, lse, w


def _check(got, z, idx, t, w, tau, lse):
    loss, grad = got
    rl, rg = od.rows(z, idx, t, w, tau, lse)
    loss, g = loss.double().cpu(), grad.double().cpu()
    span = 1 + (z.double().amax(1) - z.double().amin(1)).nan_to_num(0, 0, 0).clamp(max=1e3) / tau
    lb = 2.0 ** -18 * tau * tau * (span + rl.abs().nan_to_num(0, 0, 0)) * 2
    ok = (loss - rl).abs() <= lb
    ok |= (rl == math.inf) & (loss == math.inf)
    assert ok.all(), (loss, rl)
    gb = EPS[grad.dtype] * rg.abs() + 2.0 ** -17 * tau * w[:, None].double() * span[:, None] * (rg.abs() / (tau * w[:, None].double()).clamp(min=1e-30) + 2.0 ** -6) + TINY[grad.dtype]
    assert ((g - rg).abs() <= gb).all(), ((g - rg).abs() / gb).max()


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("T,V,k,tau", [(1, 1, 1, 1.0), (3, 7, 2, 0.5), (5, 1000, 8, 1.0), (2, 33001, 20, 2.0), (1, 70003, 64, 1.0),
                                       (9, 4097, 100, 4.0), (2, 2048, 1024, 1.0)])
def test_rows(gpu, T, V, k, tau, dt, rest):
    z, idx, t, lse, w = _case(V + k, T, V, k, tau, rest, dt)
    got = distill.topk_kl_rows(z.to(gpu), idx.to(torch.int32).to(gpu), t.to(gpu), w.to(gpu), tau, None if lse is None else lse.to(gpu))
    _check(got, z, idx, t, w, tau, lse)


@pytest.mark.parametrize("rest", [False, True])
def test_many_rows_take_one_workgroup_each(gpu, rest):
    z, idx, t, lse, w = _case(7, 1100, 515, 6, 1.0, rest, BF)
    got = distill.topk_kl_rows(z.to(gpu), idx.to(gpu), t.to(gpu), w.to(gpu), 1.0, None if lse is None else lse.to(gpu))
    _check(got, z, idx, t, w, 1.0, lse)


@pytest.mark.parametrize("T", [3, 1100])
@pytest.mark.parametrize("rest", [False, True])
def test_padding_repeats_and_masks(gpu, T, rest):
    """Rows without a teacher, padded and repeated entries, teacher logits of -inf, logits of -inf and of the lowest value,
    rows of weight 0 that hold NaN, rows whose mask leaves nothing."""
    V, k = 203, 6
    z, idx, t, lse, w = _case(11, 12, V, k, 1.0, rest, F32)
    idx[0] = -1                                   # no teacher
    z[0, 5] = float("nan")
    idx[1, 2:] = torch.tensor([-1, V, V + 100, -7])  # outside the vocabulary
    idx[2] = idx[2, 0]                            # one column six times
    t[3, 1:] = -math.inf                          # padding by mass
    z[4, :] = -math.inf                           # a mask that leaves nothing
    z[5, :] = torch.finfo(F32).min                # the lowest value everywhere: uniform
    z[6, idx[6, 0]] = -math.inf                   # the teacher wants what the student cannot give
    w[7] = 0
    z[7, 3] = float("inf")
    z[8, :100] = torch.finfo(F32).min             # half a row masked by the lowest value
    z[9, 100:] = -math.inf                        # and by -inf, entries among the rest
    idx[9] = torch.arange(6)
    t[10] = -math.inf
    if T == 1100:  # the same rows in a launch that splits nothing
        rep = lambda a: None if a is None else a.repeat(92, *([1] * (a.dim() - 1)))  # noqa: E731
    else:
        rep = lambda a: a  # noqa: E731
    dev = lambda a: None if a is None else rep(a).to(gpu)  # noqa: E731
    loss, grad = distill.topk_kl_rows(dev(z), dev(idx), dev(t), dev(w), 1.0, dev(lse))
    _, rg = od.rows(z, idx, t, w, 1.0, lse)
    rl, _ = od.rows(z, idx, t, w, 1.0, lse)
    for r0 in range(0, loss.numel(), 12):
        lo, g = loss[r0:r0 + 12].double().cpu(), grad[r0:r0 + 12].double().cpu()
        for i in range(12):
            if i == 7:  # its loss is NaN: an infinite logit with a teacher
                assert torch.isnan(lo[i]) and (g[i] == 0).all()
                continue
            if rl[i] == math.inf:
                assert lo[i] == math.inf, i
            else:
                assert abs(lo[i] - rl[i]) <= 1e-5 * (1 + abs(rl[i])), (i, lo[i], rl[i])
            assert (g[i] - rg[i]).abs().max() <= 2.0 ** -18 * (1 + rg[i].abs().max()), (i, (g[i] - rg[i]).abs().max())
        assert lo[0] == 0 and (g[0] == 0).all() and lo[10] == 0 and (g[4] == 0).all()


def test_nan_logits_make_their_row_nan_only(gpu):
    z, idx, t, _, w = _case(3, 4, 600, 5, 1.0, False, BF)
    z[2, 17] = float("nan")
    loss, g = distill.topk_kl_rows(z.to(gpu), idx.to(gpu), t.to(gpu), w.to(gpu))
    assert torch.isnan(loss[2]) and torch.isnan(g[2]).all()
    keep = [0, 1, 3]
    _check((loss[keep], g[keep]), z[keep], idx[keep], t[keep], w[keep], 1.0, None)


@pytest.mark.parametrize("T,V", [(4, 40001), (1100, 515)])
def test_in_place_strided_and_odd_alignment(gpu, T, V):
    """The gradient over the logits, rows with a longer stride, bases off the 16-byte grid, gradients at another
    alignment than the logits."""
    z, idx, t, _, w = _case(5, T, V, 7, 1.0, False, BF)
    args = (idx.to(torch.int32).to(gpu), t.to(gpu), w.to(gpu))
    loss, ref = distill.topk_kl_rows(z.to(gpu), *args)
    buf = torch.zeros(T, V + 9, dtype=BF, device=gpu)
    for off in (0, 1, 5):
        zs = buf.zero_()[:, off:off + V]
        zs.copy_(z)
        l1, g1 = distill.topk_kl_rows(zs, *args)
        out = torch.zeros(T, V + 3, dtype=BF, device=gpu)[:, 2:2 + V]
        l2, g2 = distill.topk_kl_rows(zs, *args, out=out)
        assert g2.data_ptr() == out.data_ptr()
        l3, g3 = distill.topk_kl_rows(zs, *args, out=zs)  # in place, last
        assert g3.data_ptr() == zs.data_ptr()
        # the order of the sums goes by alignment: equal up to fp32 rounding, one unit of bf16
        for a, b in ((l1, g1), (l2, g2), (l3, g3)):
            assert (a - loss).abs().max() <= 1e-5 * (1 + loss.abs().max())
            assert (b.float() - ref.float()).abs().max() <= 2.0 ** -7 * ref.float().abs().max()
        assert torch.equal(g1, g2) and torch.equal(g1, g3)
        assert not buf[:, :off].any() and not buf[:, off + V:].any()  # nothing beside the rows


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("T,V", [(3, 20001), (1030, 300)])
def test_autograd_agrees_with_the_one_call_form(gpu, T, V, rest):
    z, idx, t, lse, w = _case(9, T, V, 5, 2.0, rest, F32)
    idx[1] = -1
    dev = lambda a: None if a is None else a.to(gpu)  # noqa: E731
    zg = z.to(gpu).requires_grad_(True)
    loss = distill.topk_kl(zg, dev(idx), dev(t), 2.0, dev(lse))
    (loss * w.to(gpu)).sum().backward()
    l1, g1 = distill.topk_kl_rows(z.to(gpu), dev(idx), dev(t), dev(w), 2.0, dev(lse))
    assert (loss - l1).abs().max() <= 1e-5 * (1 + l1.abs().max())
    assert (zg.grad - g1).abs().max() <= 1e-5 * g1.abs().max()
    with torch.no_grad():
        l2 = distill.topk_kl(zg, dev(idx), dev(t), 2.0, dev(lse))
    assert (l2 - l1).abs().max() <= 1e-5 * (1 + l1.abs().max())
    _check((l1, g1), z, idx, t, w, 2.0, lse)


def test_gradient_against_differences(gpu):
    """Differences of the float64 loss, entry by entry, at a few columns."""
    V, k, tau = 50, 4, 1.5
    z, idx, t, lse, _ = _case(13, 2, V, k, tau, True, F32)
    _, g = distill.topk_kl_rows(z.to(gpu), idx.to(gpu), t.to(gpu), None, tau, lse.to(gpu))
    d = 1e-4
    for j in [0, 7, 49] + idx[0].tolist():
        zp, zm = z.double().clone(), z.double().clone()
        zp[:, j] += d
        zm[:, j] -= d
        num = (od.rows(zp, idx, t, None, tau, lse)[0] - od.rows(zm, idx, t, None, tau, lse)[0]) / (2 * d)
        assert (num - g[:, j].double().cpu()).abs().max() < 1e-5  # d² / 6 and 2^-17 of values up to tau


def test_whole_vocabulary_and_empty(gpu):
    V = 17
    z, _, _, _, w = _case(1, 3, V, 4, 1.0, False, F32)
    t = torch.randn(3, V, generator=torch.Generator().manual_seed(2))
    idx = torch.arange(V).expand(3, V).contiguous()
    ref = (t.softmax(1) * (t.log_softmax(1) - z.log_softmax(1))).sum(1)
    for lse in (None, t.logsumexp(1).to(gpu)):
        loss, _ = distill.topk_kl_rows(z.to(gpu), idx.to(gpu), t.to(gpu), w.to(gpu), 1.0, lse)
        assert (loss.cpu() - ref).abs().max() < 1e-5
    loss, g = distill.topk_kl_rows(z[:0].to(gpu), idx[:0].to(gpu), t[:0].to(gpu))
    assert loss.shape == (0,) and g.shape == (0, V)


def test_refusals(gpu):
    import _native
    z, idx, t, _, w = _case(1, 4, 100, 3, 1.0, False, BF)
    z, idx, t, w = z.to(gpu), idx.to(gpu), t.to(gpu), w.to(gpu)
    bad = [lambda: distill.topk_kl_rows(z.double(), idx, t), lambda: distill.topk_kl_rows(z, idx.float(), t),
           lambda: distill.topk_kl_rows(z, idx[:2], t[:2]), lambda: distill.topk_kl_rows(z, idx, t[:, :2]),
           lambda: distill.topk_kl_rows(z, idx, t, w[:3]), lambda: distill.topk_kl_rows(z, idx, t, temperature=0.0),
           lambda: distill.topk_kl_rows(z, idx, t, out=z.float()), lambda: distill.topk_kl_rows(z[0], idx, t),
           lambda: distill.topk_kl_rows(z.t().contiguous().t(), idx, t), lambda: distill.topk_kl_rows(z, idx.cpu(), t),
           lambda: distill.topk_kl_rows(z, idx[:, :0], t[:, :0]), lambda: distill.topk_kl_rows(z, idx, t, out=z[:, :50]),
           lambda: distill.topk_kl_rows(z[:1].expand(4, 100), idx, t, out=z[:1].expand(4, 100))]
    for f in bad:
        with pytest.raises(_native.NativeError):
            f()


def test_graph_replays(gpu):
    z, idx, t, _, w = _case(1, 5, 30000, 9, 1.0, False, BF)
    zg, idx, t, w = z.to(gpu), idx.to(gpu), t.to(gpu), w.to(gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        distill.topk_kl_rows(zg, idx, t, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, g = distill.topk_kl_rows(zg, idx, t, w)
    for k in range(3):
        new = (torch.randn(5, 30000, generator=torch.Generator().manual_seed(k)) * 2).to(BF).to(gpu)
        ref = distill.topk_kl_rows(new, idx, t, w)
        zg.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, ref[0]) and torch.equal(g, ref[1]), k


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dt,T,V", [(BF, 70, 1), (BF, 70, 5), (BF, 70, 40), (BF, 70, 63), (BF, 70, 64), (BF, 70, 71), (BF, 70, 200),
                                    (HF, 70, 9000), (F32, 40, 30), (F32, 40, 33), (F32, 40, 5001)])
def test_rows_that_begin_anywhere_in_a_line(gpu, dt, T, V, rest):
    """Rows an odd number of elements apart: every place in a 128-byte line is some row's first; the gradient in place, at the
    same places of other rows' lines, and at other places."""
    z, idx, t, lse, w = _case(V, T, V, min(V, 6), 1.0, rest, dt)
    ld = V + (2 if V % 2 else 1)
    wide = torch.zeros(T, ld, dtype=dt, device=gpu)
    wide[:, :V] = z.to(gpu)
    args = idx.to(gpu), t.to(gpu), w.to(gpu), 1.0, None if lse is None else lse.to(gpu)
    for shift in (0, 16 // wide.element_size(), 1):
        flat = torch.zeros(T * ld + shift, dtype=dt, device=gpu)
        out = flat[shift:].view(T, ld)[:, :V]
        _check(distill.topk_kl_rows(wide[:, :V], *args, out=out), z, idx, t, w, 1.0, lse)
    got = distill.topk_kl_rows(wide[:, :V], *args, out=wide[:, :V])
    _check(got, z, idx, t, w, 1.0, lse)
    assert not wide[:, V:].any()


@pytest.mark.parametrize("shift", [0, 1, 8, 37])
def test_split_rows_that_begin_anywhere_in_a_line(gpu, shift):
    T, V = 3, 70001
    z, idx, t, lse, w = _case(3, T, V, 64, 1.0, True, BF)
    idx[:, :4] = torch.tensor([0, 1, V - 2, V - 1])  # ends of the row, whichever vector or scalar holds them
    idx[:, 4:] = 2 + idx[:, 4:] % 900 * 77  # some more than once
    flat = torch.zeros(T * V + 64, dtype=BF, device=gpu)
    zz = flat[shift:shift + T * V].view(T, V)
    zz.copy_(z)
    got = distill.topk_kl_rows(zz, idx.to(gpu), t.to(gpu), w.to(gpu), 1.0, lse.to(gpu))
    _check(got, z, idx, t, w, 1.0, lse)


def test_a_buffer_over_the_logits_is_their_own_or_apart(gpu):
    """In place or beside the logits; a buffer that overlaps them otherwise is refused, and autograd sees the write."""
    z, idx, t, _, w = _case(2, 5, 40, 3, 1.0, False, BF)
    args = idx.to(gpu), t.to(gpu), w.to(gpu)
    buf = torch.zeros(6, 100, dtype=BF, device=gpu)
    zz = buf[:5, :40]
    zz.copy_(z)
    ref = distill.topk_kl_rows(zz, *args)[1]
    beside = buf[:5, 40:80]
    assert torch.equal(distill.topk_kl_rows(zz, *args, out=beside)[1], ref)
    for bad in (buf[1:, :40], buf[:5, 39:79], buf.view(-1)[:200].view(5, 40), buf.view(-1)[99:499].view(5, 80)[:, :40]):
        with pytest.raises(_native.NativeError, match="overlap"):
            distill.topk_kl_rows(zz, *args, out=bad)
    flat = torch.zeros(400, dtype=BF, device=gpu)  # one after the other
    flat[:200] = z.to(gpu).view(-1)
    distill.topk_kl_rows(flat[:200].view(5, 40), *args, out=flat[200:].view(5, 40))
    x = z.to(gpu).requires_grad_(True)
    y = torch.tanh(x)  # keeps its result
    distill.topk_kl_rows(y.detach(), *args, out=y.detach())
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()

"""The native calls of the 4-bit operators and the loss run without the interpreter's lock, as those of the 8-bit path do
(test_gpu_threads.py has the method)."""
import pytest
import torch

import _native
import test_gpu_threads as base

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _calls(gpu):
    h = _native.host4()
    x, one = torch.randn(40, 128, device=gpu).to(BF), torch.randn(1, 128, device=gpu).to(BF)
    w = torch.randn(64, 128, device=gpu).to(BF)
    W, G = h.Weight(w, True), h.Gated(w, w)
    q, s = h.quant(x, 8, 0)
    bq, bs = h.quant(w, 4, 0)
    z, idx, t = torch.randn(4, 1000, device=gpu), torch.zeros(4, 2, dtype=torch.int32, device=gpu), torch.zeros(4, 2, device=gpu)
    return {"quant": lambda: h.quant(x, 4, 0), "quant_both": lambda: h.quant_both(x, 4, 0),
            "dequant": lambda: h.dequant(q, s, 40, 128, 8, torch.float32),
            "gemm": lambda: h.gemm(q, s, 8, bq, bs, 0, 40, 64, 128, BF), "linear": lambda: h.linear(W, x, 8),
            "few": lambda: h.linear(W, one, 8), "gated": lambda: h.gated(G, x, None, 0, 4),
            "weight": lambda: h.Weight(w, False), "topk_kl": lambda: h.topk_kl(z, idx, t, 1.0, None),
            "topk_kl_rows": lambda: h.topk_kl_rows(z, idx, t, None, 1.0, None, None)}


@pytest.mark.parametrize("name", ["quant", "quant_both", "dequant", "gemm", "linear", "few", "gated", "weight", "topk_kl",
                                  "topk_kl_rows"])
def test_other_threads_run_during_native_calls(name, gpu, monkeypatch):
    monkeypatch.setattr(base, "_calls", _calls)
    base.test_other_threads_run_during_native_calls(name, gpu)

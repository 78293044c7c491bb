"""The native calls refuse rank-r operands that the kernels would read past, before anything is launched."""
import pytest
import torch

import _native
import mxfp8
from test_native_host import K, N, R, T, _bf, _codes

ONE = torch.zeros(8, dtype=torch.uint8)


def _quant(w):
    return _native.host().quant_lora(_bf(T, K), w, 1.0, True, 0)


def _gemm(P, Q):
    return _native.host().gemm(_codes(T, K), ONE, _codes(N, K), ONE, None, P, Q, 1.0, 3, T, 0)


def _seg(P, Q, rcols=(0, 16)):
    return _native.host().gemm_seg(_codes(T, K), ONE, _codes(N, K), ONE, [128, N - 128], P, Q, 1.0, 3, T, list(rcols), 16, 0)


def _tn(P, Q):
    job = (_bf(T, K), _bf(T, 32), torch.zeros(32, K), 1.0, False)
    return _native.host().gemm_tn(_codes(T, K), ONE, _codes(N, K), ONE, P, Q, 1.0, 3, T, [job], torch.zeros(1 << 16), 0)


BAD = [lambda: _quant(_bf(16, K - 128)), lambda: _quant(_bf(16, 2 * K)[:, :K]), lambda: _quant(torch.zeros(16, K)),
       lambda: _quant(_bf(K)), lambda: _gemm(_bf(T - 1, 16), _bf(N, 16)), lambda: _gemm(_bf(T, 16), _bf(N - 128, 16)),
       lambda: _gemm(_bf(T, 16), _bf(N, 8)), lambda: _gemm(_bf(T, 16), None), lambda: _gemm(_bf(T, 16), torch.zeros(N, 16)),
       lambda: _seg(_bf(T, 16), _bf(N, 32)), lambda: _seg(_bf(T, 32), _bf(N, 32), (0, 32)), lambda: _tn(_bf(T, 32), _bf(K, 32)),
       lambda: _native.lora_nt(_bf(T, K), _bf(16, N), _bf(T, 16)),
       lambda: _native.quant_lora(_bf(T, K), ONE, ONE, _bf(16, N), _bf(T, 16)),
       lambda: mxfp8.mx_quant_lora_tp(_bf(T, K), _bf(16, N), _bf(T, 32)),
       lambda: _native.host().mlp_graph(_bf(T, K), _bf(2 * R, 2 * K), _codes(2 * N, K), ONE, N, 0)]


@pytest.mark.parametrize("k", range(len(BAD)))
def test_operands_of_other_sizes_are_refused(k):
    with pytest.raises((RuntimeError, _native.NativeError), match="operands of other sizes|w of "):
        BAD[k]()


def test_fitting_operands_pass_the_checks():
    for call in (lambda: _quant(_bf(16, K)), lambda: _gemm(_bf(T, 16), _bf(N, 16)), lambda: _gemm(_bf(T, 48)[:, 16:32], _bf(N, 16)),
                 lambda: _gemm(None, None), lambda: _seg(_bf(T, 32), _bf(N, 32)), lambda: _seg(None, None, ()),
                 lambda: _tn(_bf(T, 32), _bf(N, 32))):
        with pytest.raises(_native.NativeError, match="must be on the GPU"):
            call()

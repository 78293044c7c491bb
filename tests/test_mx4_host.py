"""CPU checks of the 4-bit operators' boundary: every function of include/mxfp4_ops.h is exported, arguments are refused
before anything is launched, and host plans."""
import ctypes
import os
import re

import pytest
import torch

import _native
import distill
import mxfp4
import test_gpu_mx4_shapes as shapes

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "mxfp4_ops.h")
P = ctypes.c_void_p(1 << 20)  # never dereferenced: the checks fail first
I = ctypes.c_int64  # noqa: E741


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_native.LIB_PATH):
        pytest.skip("libmxfp8_mlp.so not built")
    L = _native.load()
    for name in ("mxfp4_gated_saved_elems", "distill_parts", "distill_workspace_size"):
        getattr(L, name).restype = ctypes.c_int64
    return L


def _declared():
    txt = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return re.findall(r"^\s*(?:int|int64_t)\s+((?:mxfp4|distill)_\w+)\s*\(", txt, flags=re.M)


def test_library_exports_every_declared_symbol(lib):
    names = _declared()
    assert len(names) == 12 and all(hasattr(lib, n) for n in names), names
    assert lib.mxfp4_abi_version() == _native.OPS_ABI_VERSION
    assert f"#define MXFP4_OPS_ABI_VERSION {_native.OPS_ABI_VERSION}" in open(HEADER).read()


def _refused(lib, rc, text):
    assert rc == -1 and text.encode() in lib.mxfp8_last_error(), lib.mxfp8_last_error()


def test_refusals(lib):
    def quant(x=P, type=0, rows=4, cols=64, ld=64, fmt=4, q=P, s=P, order=0, qt=None, st=None, ot=0, t0=0, tt=0):  # noqa: A002
        return lib.mxfp4_quant(x, I(type), I(rows), I(cols), I(ld), I(fmt), q, s, I(order), qt, st, I(ot), I(t0), I(tt), None)
    _refused(lib, quant(type=3), "element type")
    _refused(lib, quant(fmt=5), "format")
    _refused(lib, quant(s=None), "null")
    _refused(lib, quant(order=4), "order")
    _refused(lib, quant(rows=-1), "shape")
    _refused(lib, quant(q=ctypes.c_void_p(8)), "misaligned")
    _refused(lib, quant(qt=P, st=P, t0=1, tt=1), "column tiles")
    assert quant(rows=0) == 0 and quant(cols=0) == 0

    def gemm(a=P, fmt=4, order=1, M=4, N=64, K=128, c=P, ldc=64, type=0):  # noqa: A002
        return lib.mxfp4_gemm(a, P, I(fmt), P, P, I(order), I(M), I(N), I(K), c, I(ldc), I(type), None)
    _refused(lib, gemm(K=96), "shape")
    _refused(lib, gemm(N=0), "shape")
    _refused(lib, gemm(order=2), "order")
    _refused(lib, gemm(ldc=63), "output")
    _refused(lib, gemm(a=None), "null")
    _refused(lib, gemm(type=7), "element type")
    _refused(lib, gemm(fmt=0), "format")
    assert gemm(M=0) == 0

    def gated(type=0, fn=0, add=None, ld_add=0, ldh=64, gu=None):  # noqa: A002
        return lib.mxfp4_gated(P, P, I(4), P, P, I(4), I(64), I(128), add, I(ld_add), I(fn), P, I(ldh), gu, I(type), None)
    _refused(lib, gated(type=2), "bf16 or f16")
    _refused(lib, gated(fn=2), "gate function")
    _refused(lib, gated(add=P, ld_add=100), "addend")
    _refused(lib, gated(ldh=10), "output")
    _refused(lib, gated(gu=ctypes.c_void_p(8)), "output")

    def bwd(type=0, fmt=4, ld=64, fn=0, dh=P):  # noqa: A002
        return lib.mxfp4_gated_bwd(P, dh, I(ld), I(4), I(64), I(fn), I(type), I(fmt), P, P, None, None)
    _refused(lib, bwd(type=2), "bf16 or f16")
    _refused(lib, bwd(fmt=1), "format")
    _refused(lib, bwd(ld=3), "stride")
    _refused(lib, bwd(dh=None), "null")
    _refused(lib, bwd(fn=5), "gate function")

    def few(M=1, fmt=8, type=0, ldc=64):  # noqa: A002
        return lib.mxfp4_few(P, I(128), I(fmt), P, P, I(M), I(64), I(128), P, I(ldc), I(type), None)
    _refused(lib, few(M=17), "at most 16 rows")
    _refused(lib, few(fmt=2), "format")
    _refused(lib, few(type=2), "bf16 or f16")
    _refused(lib, few(ldc=2), "stride")
    _refused(lib, lib.mxfp4_few_gated(P, I(128), I(8), P, P, I(1), I(64), I(128), None, I(0), I(3), P, I(64), I(0), None),
             "gate function")

    def kl(V=100, ib=4, k=8, tau=1.0, parts=1, stages=3, z=P, grad=None, ldg=0, ws=None, type=0, lse=None):  # noqa: A002
        return lib.distill_topk_kl(z, I(type), I(V), I(4), I(V), P, I(ib), I(k), P, I(k), I(k), ctypes.c_float(tau), lse,
                                   None, P, grad, I(ldg), I(parts), I(stages), ws, None)
    _refused(lib, kl(V=0), "shape")
    _refused(lib, kl(ib=2), "indices")
    _refused(lib, kl(k=0), "teacher entries")
    _refused(lib, kl(k=1025), "teacher entries")
    _refused(lib, kl(tau=0.0), "temperature")
    _refused(lib, kl(tau=float("nan")), "temperature")
    _refused(lib, kl(parts=2), "null")
    _refused(lib, kl(parts=0), "plan")
    _refused(lib, kl(stages=4), "plan")
    _refused(lib, kl(grad=P, ldg=99), "stride")
    _refused(lib, kl(type=5), "element type")
    _refused(lib, kl(V=1 << 20), "too few parts")


def test_plans(lib):
    assert lib.mxfp4_gated_saved_elems(I(33), I(65)) == 2 * 3 * 2048
    parts = lambda T, V: lib.distill_parts(I(T), I(V), I(0))  # noqa: E731
    assert parts(4096, 65536) == 1 and parts(1, 1000) == 1 and parts(1, 65536) > 1
    for T in (1, 7, 300, 5000):
        for V in (1, 1000, 248001, 1 << 22):
            p = parts(T, V)
            assert 1 <= p <= 256 and -(-V // p) <= 1 << 18
    assert lib.distill_workspace_size(I(3), I(5), I(2)) == 3 * 2 * 8 + 3 * 5 * 8


def test_sizes_of_the_shape_tests_take_their_shapes(lib):
    for table, gated in ((shapes.PLAIN, False), (shapes.GATED, True)):
        for (shape, act), sizes in table.items():
            for size in sizes:
                assert _native.mx4_shape(*size, act, gated) == shape, (size, act, gated)
                if gated:  # what is saved keeps the launch from the kernel for few rows, and changes nothing else
                    assert _native.mx4_shape(*size, act, True, saved=True) == ("64x128" if shape == "thin" else shape)
        assert {a for _, a in table} == {"e4m3", "e2m1"}
    assert {s for s, _ in shapes.PLAIN} == {"thin", "64x64", "64x128", "128x128", "256x128"}
    assert {s for s, _ in shapes.GATED} == {"thin", "64x128", "128x128", "256x128"}
    with pytest.raises(_native.NativeError):
        _native.mx4_shape(0, 1, 1)


def test_cpu_tensors_and_names_are_refused():
    x = torch.zeros(4, 64)
    with pytest.raises(_native.NativeError):
        mxfp4.mx4_quant(x)
    with pytest.raises(_native.NativeError):
        mxfp4.Weight(x)
    with pytest.raises(_native.NativeError):
        distill.topk_kl(x, torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, 1))
    with pytest.raises(ValueError):
        mxfp4.mx4_quant(x, fmt="e3m2")
    with pytest.raises(ValueError):
        mxfp4.mx4_gated(x, None, fn="relu")

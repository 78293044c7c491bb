"""More rows than a launch has threads for are refused before anything is launched, in the stages called apart too."""
import ctypes

import pytest

from test_mx4_host import I, P, lib  # noqa: F401  (lib is a fixture)


@pytest.mark.parametrize("T,V,type,parts,stages", [  # threads of a workgroup times rows and parts reach 2^32
    (1 << 24, 100, 0, 1, 3), (1 << 23, 100, 0, 1, 1), (1 << 23, 100, 0, 1, 2), (1 << 23, 20000, 1, 1, 3),
    (1 << 22, 65536, 0, 1, 3), (1 << 22, 40000, 2, 1, 3), (1 << 18, 1 << 20, 0, 32, 3)])
def test_rows_past_a_launch(lib, T, V, type, parts, stages):  # noqa: F811
    rc = lib.distill_topk_kl(P, I(type), I(V), I(T), I(V), P, I(4), I(8), P, I(8), I(8), ctypes.c_float(1.0), None, None, P,
                             None, I(0), I(parts), I(stages), P, None)
    assert rc == -1 and b"threads" in lib.mxfp8_last_error()

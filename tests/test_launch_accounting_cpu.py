"""Kernel launches counted per extension call, on a stand-in of the extension module."""

from types import SimpleNamespace

import pytest

from mvp_engine.ops import _ext


@pytest.mark.parametrize("name,args,result,kernels", [
    ("gemm", (1, 2), None, 1), ("flash_attn_bwd", (), None, 3), ("gemm_fp8", (), None, 1),
    ("linear_fp8_fwd", ("x", "w", None, None, True, True, 0), [], 3),
    ("linear_fp8_fwd", ("x", "w", "w8", "sw8", True, True, 0), [], 2),
    ("linear_fp8_bwd", ("dy", "xt", "sxt", "wt", "swt", False, None, 0), [], 3),
    ("linear_fp8_bwd", ("dy", None, None, "wt", "swt", False, None, 0), [], 2),
    ("linear_fp8_bwd", ("dy", "xt", "sxt", None, None, False, "acc", 0), [], 2),
    ("orthogonalize", ("x", "out", 5), 17, 17), ("orthogonalize", ("x", "out", 2), 8, 8),
    ("muon_step_", ([], [], []), 34, 34), ("num_things", (), 9, 0)])
def test_kernels_of_a_call(name, args, result, kernels):
    calls = []
    ext = _ext._Counting(SimpleNamespace(**{name: lambda *a, **kw: calls.append(a) or result}))
    getattr(ext, name)(*args)  # not counted
    _ext.start_counting()
    for _ in range(3):
        assert getattr(ext, name)(*args) is result
    assert _ext.stop_counting() == 3 * kernels
    assert calls == [args] * 4

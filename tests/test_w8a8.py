"""CPU tests of the 8-bit product and its quantizer: what they refuse, before anything is launched."""
from __future__ import annotations

import pytest

from test_kv_pages import _aligned


def _product(gx, **change):
    a = dict(weights=_aligned(4096), weight_scales=_aligned(4096), codes=_aligned(4096), scales=_aligned(4096), output=_aligned(4096),
             kind=gx.TYPE_F32, rows=16, columns=64, tokens=2, workspace=None, bytes=0)
    a.update(change)
    at = lambda x: x if x is None or isinstance(x, int) else x.ctypes.data  # noqa: E731
    return gx.lib().gfxinfer_launch_w8a8_gemm(at(a["weights"]), at(a["weight_scales"]), at(a["codes"]), at(a["scales"]), at(a["output"]),
                                              a["kind"], a["rows"], a["columns"], a["tokens"], at(a["workspace"]), a["bytes"], None)


@pytest.mark.parametrize("change", [
    dict(weights=None), dict(weight_scales=None), dict(codes=None), dict(scales=None), dict(output=None), dict(rows=0),
    dict(rows=(1 << 24) + 1), dict(columns=0), dict(columns=24), dict(columns=1 << 17), dict(tokens=0), dict(tokens=(1 << 24) + 1),
    dict(weights=_aligned(4096).ctypes.data + 8), dict(codes=_aligned(4096).ctypes.data + 4),
    dict(output=_aligned(4096).ctypes.data + 8), dict(scales=_aligned(4096).ctypes.data + 2),
    dict(rows=1 << 24, columns=16, tokens=1 << 24),           # more tiles than a launch has workgroups
    dict(tokens=300, rows=256, columns=8192), dict(tokens=300, rows=256, columns=8192, workspace=_aligned(64), bytes=64)])
def test_bad_products_are_refused(gx, change):
    assert _product(gx, **change) == gx.INVALID_ARGUMENT
    assert gx.last_error()


def test_other_types_are_unsupported(gx):
    assert _product(gx, kind=gx.TYPE_BF16) == gx.UNSUPPORTED
    assert gx.lib().gfxinfer_launch_quantize_rows_i8(_aligned(256).ctypes.data, 3, 1, 16, 16, _aligned(256).ctypes.data,
                                                     _aligned(256).ctypes.data, None) == gx.UNSUPPORTED


def test_workspace_sizes(gx):
    assert gx.w8a8_gemm_workspace_bytes(16, 64, 1) == 0                    # few tokens need none
    assert gx.w8a8_gemm_workspace_bytes(256, 8192, 300) > 0                # K is divided
    for bad in ((0, 64, 1), (16, 63, 1), (16, 64, 0), (16, 1 << 17, 300)):
        assert gx.w8a8_gemm_workspace_bytes(*bad) == 0


@pytest.mark.parametrize("change", [
    dict(input=None), dict(codes=None), dict(scales=None), dict(rows=0), dict(rows=(1 << 24) + 1), dict(columns=8), dict(columns=1 << 17),
    dict(stride=56), dict(stride=68), dict(input=_aligned(4096).ctypes.data + 8), dict(codes=_aligned(4096).ctypes.data + 8)])
def test_bad_rows_are_refused(gx, change):
    a = dict(input=_aligned(4096), rows=2, columns=64, stride=64, codes=_aligned(4096), scales=_aligned(4096))
    a.update(change)
    at = lambda x: x if x is None or isinstance(x, int) else x.ctypes.data  # noqa: E731
    assert gx.lib().gfxinfer_launch_quantize_rows_i8(at(a["input"]), gx.TYPE_F16, a["rows"], a["columns"], a["stride"], at(a["codes"]),
                                                     at(a["scales"]), None) == gx.INVALID_ARGUMENT
    assert gx.last_error()

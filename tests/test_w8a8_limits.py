"""The largest calls of the 8-bit product and its quantizer: what a launch holds (less than 2^32 threads along a dimension)."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import say
from test_kv_pages import _aligned

SCALE = np.float32(1) / np.float32(127)


@pytest.mark.parametrize("rows,tokens", [
    (1 << 20, 1 << 19),                                       # 2^23 tiles of 256 x 256
    (1 << 24, 1 << 15), (1 << 15, 1 << 24), (1 << 24, 1 << 24),
])
def test_products_of_more_tiles_than_a_launch_holds_are_refused(gx, rows, tokens):
    x = _aligned(64).ctypes.data
    for kind in (gx.TYPE_F16, gx.TYPE_F32):
        assert gx.lib().gfxinfer_launch_w8a8_gemm(x, x, x, x, x, kind, rows, 16, tokens, None, 0, None) == gx.INVALID_ARGUMENT
        assert "launch" in gx.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,columns", [((1 << 24), 16), ((1 << 20) + 3, 16), ((1 << 20) + 2, 8208)])
def test_as_many_rows_as_documented(device, gx, rows, columns):
    """Rows in all parts of the range equal the definition; the others, zeros, have codes of 0 and the smallest scale."""
    import torch
    say("many rows", rows, columns)
    rng = np.random.default_rng(rows)
    at = sorted({0, 1, (1 << 20) - 1, 1 << 20, rows - 2, rows - 1} | set(rng.integers(0, rows, 50).tolist()))
    some = (rng.standard_normal((len(at), columns))).astype(np.float16)
    x = torch.zeros(rows, columns, dtype=torch.float16, device="cuda")
    place = torch.tensor(at, device="cuda")
    x[place] = torch.from_numpy(some).cuda()
    codes = torch.full((rows, columns), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((rows,), 99.0, device="cuda")
    gx.launch_quantize_rows_i8(x, codes, scales)
    torch.cuda.synchronize()
    scale = (np.abs(some.astype(np.float32)).max(1) * SCALE).astype(np.float32)
    want = np.rint(some.astype(np.float64) / scale[:, None].astype(np.float64)).astype(np.int8)
    assert np.array_equal(scales[place].cpu().numpy(), scale) and np.array_equal(codes[place].cpu().numpy(), want)
    codes[place], scales[place] = 0, 2.0 ** -126
    assert int(torch.count_nonzero(codes.view(torch.int64))) == 0 and bool((scales == 2.0 ** -126).all())

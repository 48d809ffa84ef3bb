"""The 8-bit product and its quantizer on the GPU, bit for bit: the integer sums are exact, and the scales are applied as
float(sum) * (scale * weight_scale) in fp32, rounded once more for an fp16 output."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import dev, host, say

pytestmark = pytest.mark.gpu
SCALE = np.float32(1) / np.float32(127)


def _codes_of(x):
    """(codes, scales) by the definition: the quotient in 64 bits, where next to a half nothing is lost."""
    x = x.astype(np.float32)
    bad = ~np.isfinite(x).all(1)
    scale = np.maximum(np.abs(np.where(bad[:, None], 0, x)).max(1) * SCALE, np.float32(2.0 ** -126)).astype(np.float32)
    codes = np.clip(np.rint(np.where(bad[:, None], 0, x).astype(np.float64) / scale[:, None].astype(np.float64)), -127, 127)
    return codes.astype(np.int8), np.where(bad, np.float32(np.nan), scale)


def _tensor(x, kind):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).cuda().to(getattr(torch, kind))


def _quantize(gx, x):
    import torch
    codes = torch.full((x.shape[0] + 1, x.shape[1]), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((x.shape[0] + 1,), 99.0, device="cuda")
    gx.launch_quantize_rows_i8(x, codes, scales)
    c, s = host(codes), host(scales)
    assert np.all(c[-1] == 99) and s[-1] == 99.0                           # rows behind the last one stay
    return c[:-1], s[:-1]


@pytest.mark.parametrize("kind", ["float16", "float32", "bfloat16"])
@pytest.mark.parametrize("rows,columns", [(1, 16), (3, 48), (1, 5120), (5, 2064), (130, 1040), (2, 16384), (2, 16400), (3, 32784), (1, 131056)])
def test_codes_equal_the_definition(device, gx, kind, rows, columns):
    rng = np.random.default_rng(rows * 7 + columns)
    say("row quantizer", kind, rows, columns)
    x = _tensor(rng.standard_normal((rows, columns)) * np.exp(rng.standard_normal(columns)), kind)
    codes, scales = _quantize(gx, x)
    want, wanted_scales = _codes_of(host(x.float()))
    assert np.array_equal(scales, wanted_scales)
    assert np.array_equal(codes, want)


def test_codes_next_to_a_half(device, gx):
    """Quotients whose fp32 rounding is a half although they lie beside it, and true halves, which go to even."""
    rng = np.random.default_rng(11)
    top = np.float32(rng.uniform(0.5, 2.0))
    scale = np.float32(top * SCALE)
    half = ((np.arange(-126, 126) + 0.5) * np.float64(scale)).astype(np.float32)
    x = np.concatenate([half, np.nextafter(half, np.float32(9)), np.nextafter(half, np.float32(-9)), [top, 0, -0.0, -top]]).astype(np.float32)
    x = np.resize(x, (len(x) + 15) // 16 * 16)[None]
    ties = np.array([[127.0] + [k + 0.5 for k in range(-8, 7)]], np.float32)   # scale 1: exact halves
    for rows in (x, ties):
        q = rows.astype(np.float32) / (np.abs(rows).max() * SCALE)
        assert np.any(np.abs(q - np.trunc(q)) == 0.5)
        codes, scales = _quantize(gx, _tensor(rows, "float32"))
        want, wanted_scales = _codes_of(rows)
        assert np.array_equal(codes, want) and np.array_equal(scales, wanted_scales)


def test_strange_rows(device, gx):
    """Zeros, the smallest numbers, infinities and NaN; a row's scale does not depend on the others."""
    x = np.zeros((6, 2048), np.float32)
    x[1] = 1e-44
    x[2, 1500] = np.inf
    x[3, 7] = np.nan
    x[4] = np.float32(3.4e38)
    x[5] = np.linspace(-1, 1, 2048)
    codes, scales = _quantize(gx, _tensor(x, "float32"))
    want, wanted_scales = _codes_of(x)
    assert np.array_equal(codes, want)
    assert np.array_equal(scales, wanted_scales, equal_nan=True)


def test_rows_at_a_pitch(device, gx):
    import torch
    wide = torch.randn(9, 400, device="cuda").half()
    codes, scales = _quantize(gx, wide[:, 16:272])
    want, wanted_scales = _codes_of(host(wide[:, 16:272].float()))
    assert np.array_equal(codes, want) and np.array_equal(scales, wanted_scales)


def _product(gx, w, ws, a, s, half, guard=3):
    import torch
    tokens, rows = a.shape[0], w.shape[0]
    # One allocation with guard elements behind the result: the last row's neighbours stay.
    flat = torch.full((tokens * rows + guard,), 7.0, dtype=torch.float16 if half else torch.float32, device="cuda")
    need = gx.w8a8_gemm_workspace_bytes(rows, w.shape[1], tokens)
    work = torch.full((max(need, 16),), 0x7f, dtype=torch.uint8, device="cuda")
    gx.launch_w8a8_gemm(dev(w), dev(ws), dev(a), dev(s), flat[:tokens * rows].view(tokens, rows), work)
    got = host(flat)
    assert np.all(got[tokens * rows:] == 7.0)
    return got[:tokens * rows].reshape(tokens, rows)


def _want(w, ws, a, s, half):
    total = (a.astype(np.float64) @ w.astype(np.float64).T).astype(np.int64)
    y = total.astype(np.float32) * (s[:, None] * ws[None, :])
    return y.astype(np.float16) if half else y


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("tokens,rows,columns", [
    (1, 1, 16), (1, 5, 64), (1, 5120, 5120), (2, 33, 80), (15, 48, 1040), (16, 100, 4096), (17, 31, 528), (32, 64, 2048), (33, 250, 512),
    (64, 513, 272), (65, 40, 16), (65, 200, 144), (100, 129, 1168), (128, 128, 128), (129, 257, 384), (200, 1000, 8192), (300, 256, 8208),
    (509, 640, 17408), (513, 8200, 96), (4100, 4352, 112), (2049, 8193, 400)])
def test_products_equal_the_definition(device, gx, half, tokens, rows, columns):
    rng = np.random.default_rng(tokens * 31 + rows + columns)
    say("8-bit product", tokens, rows, columns, half)
    a, w = (rng.integers(-128, 128, (x, columns), dtype=np.int8) for x in (tokens, rows))
    s, ws = ((rng.random(x) + 0.5).astype(np.float32) * np.float32(1e-3 if half else 1.0) for x in (tokens, rows))
    assert np.array_equal(_product(gx, w, ws, a, s, half), _want(w, ws, a, s, half))


@pytest.mark.parametrize("tokens,rows,columns", [
    (65, 1999, 528), (65, 1999, 4112), (65, 17001, 1040), (65, 7000, 8208), (1000, 7000, 528), (65, 17001, 8208), (2000, 5000, 656),
    (4096, 4096, 144), (300, 33025, 272), (400, 33025, 272), (50, 33025, 2064), (17, 5001, 16400), (9, 5001, 16400), (4, 77, 1040), (5, 77, 1040)])
def test_every_tile_shape(device, gx, tokens, rows, columns):
    """Small, middle and large tiles, in one piece and with K divided among workgroups, most with a ragged edge; whole rounds of
    the largest tiles alone and with other tiles behind them."""
    rng = np.random.default_rng(tokens + rows + columns)
    say("8-bit product", tokens, rows, columns)
    a, w = (rng.integers(-128, 128, (x, columns), dtype=np.int8) for x in (tokens, rows))
    s, ws = ((rng.random(x) + 0.5).astype(np.float32) for x in (tokens, rows))
    assert np.array_equal(_product(gx, w, ws, a, s, False), _want(w, ws, a, s, False))


@pytest.mark.parametrize("tokens", [1, 64, 70])
def test_the_largest_sums(device, gx, tokens):
    """All codes -128 at the longest K: 128 * 128 * 131056 is the largest sum a call can make, below 2^31."""
    columns = 131056
    a, w = np.full((tokens, columns), -128, np.int8), np.full((20, columns), -128, np.int8)
    w[3] = 127
    s, ws = np.ones(tokens, np.float32), np.ones(20, np.float32)
    assert np.array_equal(_product(gx, w, ws, a, s, False), _want(w, ws, a, s, False))


def test_nan_scales_reach_their_row_only(device, gx):
    rng = np.random.default_rng(5)
    a, w = rng.integers(-127, 128, (70, 256), dtype=np.int8), rng.integers(-127, 128, (300, 256), dtype=np.int8)
    s, ws = np.ones(70, np.float32), np.ones(300, np.float32)
    s[9], a[9] = np.nan, 0
    got = _product(gx, w, ws, a, s, False)
    assert np.isnan(got[9]).all() and np.array_equal(np.delete(got, 9, 0), np.delete(_want(w, ws, a, s, False), 9, 0))


@pytest.mark.parametrize("tokens", [5, 300])
def test_captured_products_replay(device, gx, tokens):
    """Quantizer and product recorded once, replayed over inputs that change, with eager work between."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    w = torch.randint(-127, 128, (384, 2048), generator=g, device="cuda").to(torch.int8)
    ws, x = normal(384).abs(), normal(tokens, 2048).half()
    codes, scales = torch.empty(tokens, 2048, dtype=torch.int8, device="cuda"), torch.empty(tokens, device="cuda")
    out, work = torch.empty(tokens, 384, device="cuda"), torch.empty(max(16, gx.w8a8_gemm_workspace_bytes(384, 2048, tokens)), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        gx.launch_quantize_rows_i8(x, codes, scales)
        gx.launch_w8a8_gemm(w, ws, codes, scales, out, work)
    for _ in range(3):
        x.copy_(normal(tokens, 2048))
        graph.replay()
        torch.cuda.synchronize()
        c, s = _codes_of(host(x.float()))
        assert np.array_equal(host(out), _want(host(w), host(ws), c, s, False))


def test_operands_of_the_wrappers_are_checked(device, gx):
    import torch
    w, ws = torch.zeros(32, 64, dtype=torch.int8, device="cuda"), torch.zeros(32, device="cuda")
    a, s, y = torch.zeros(2, 64, dtype=torch.int8, device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(2, 32, device="cuda")
    gx.launch_w8a8_gemm(w, ws, a, s, y, None)
    for bad in (lambda: gx.launch_w8a8_gemm(w.cpu(), ws, a, s, y, None), lambda: gx.launch_w8a8_gemm(w, ws.half(), a, s, y, None),
                lambda: gx.launch_w8a8_gemm(w, ws, a[:, :48], s, y, None), lambda: gx.launch_w8a8_gemm(w, ws, a, s, y.bfloat16(), None),
                lambda: gx.launch_w8a8_gemm(w.T, ws, a, s, y, None), lambda: gx.launch_w8a8_gemm(w, ws[:31], a, s, y, None),
                lambda: gx.launch_quantize_rows_i8(y.int(), a, s), lambda: gx.launch_quantize_rows_i8(y.T, a, s),
                lambda: gx.launch_quantize_rows_i8(y.cpu(), a, s), lambda: gx.launch_quantize_rows_i8(y, a[:1, :48], s)):
        with pytest.raises(ValueError):
            bad()

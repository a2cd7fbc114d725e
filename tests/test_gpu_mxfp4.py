"""MXFP4 matrices on the GPU: quantisation and back against the CPU definition
(oracle/mxfp4.py) bit for bit, products against 64-bit sums of the decoded values.

Products: every a * b of two e2m1 values and their scales is exact in fp32, the sums are
fp32. A sum of K products is a chain of K / 128 instructions, each adding 128 products; with
one step of 2^-23 for each instruction and for each of a tree's 7 levels, and 8 more for the
sums of waves, a result is off by at most (K / 128 + 15) 2^-23 sum |a b|, and by half a step
of its type when it is rounded.
"""

import pytest
import torch

from oracle import mxfp4
from tokserve_amd.kernels import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
CODES, SCALES = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def _bytes(x: torch.Tensor) -> torch.Tensor:
    return x.view(torch.uint8).cpu()


def _rows(rows, cols, dtype, seed, spread=12):
    """Rows whose blocks span many magnitudes, with zeros and values on the rounding borders."""

    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols // 32, 32, generator=g)
    x = x * 2.0 ** torch.randint(-spread, spread, (rows, cols // 32, 1), generator=g).float()
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.5, 0.0, -0.0, -0.25, -5.0])
    pick = torch.randint(0, len(borders), x.shape, generator=g)
    on = torch.rand(x.shape, generator=g) < 0.2
    x = torch.where(on, borders[pick], x)
    return x.view(rows, cols).to(dtype)


def _special(dtype):
    """Blocks of a row that test the scale rule (in a dtype's range)."""

    x = torch.zeros(10, 32)
    x[0] = torch.linspace(-1, 1, 32)
    x[1] = 0.0
    x[2, 3] = float("nan")
    x[3, 31] = float("-inf")
    x[4] = torch.finfo(dtype).tiny * torch.linspace(-4, 4, 32)
    x[5] = torch.finfo(dtype).max * torch.linspace(-1, 1, 32)
    x[6, 0] = torch.finfo(dtype).smallest_normal / 4  # a subnormal alone
    x[7] = -6.0
    x[8, 5] = 2.0 ** -9
    x[9] = torch.linspace(3.9, 4.1, 32)
    return x.reshape(1, -1).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (33, 2048), (1000, 160), (5, 11264)])
def test_quantize_is_exact(device, dtype, rows, cols) -> None:
    x = _rows(rows, cols, dtype, rows + cols)
    codes, scales = ops.mxfp4_quantize(x.to(device))
    want_codes, want_scales = mxfp4.quantize(x)
    assert codes.dtype == torch.float4_e2m1fn_x2 and scales.dtype == torch.float8_e8m0fnu
    assert torch.equal(_bytes(scales), want_scales)
    assert torch.equal(_bytes(codes), want_codes)
    for out in DTYPES:
        back = ops.mxfp4_dequantize(codes, scales, out)
        assert torch.equal(back.cpu(), mxfp4.values(want_codes, want_scales).to(out))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_of_special_blocks(device, dtype) -> None:
    x = _special(dtype)
    codes, scales = ops.mxfp4_quantize(x.to(device))
    want_codes, want_scales = mxfp4.quantize(x)
    assert torch.equal(_bytes(scales), want_scales)
    assert torch.equal(_bytes(codes), want_codes)
    back = ops.mxfp4_dequantize(codes, scales, torch.float32).cpu()
    want = mxfp4.values(want_codes, want_scales).float()
    assert torch.isnan(want).sum() == 64
    torch.testing.assert_close(back, want, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_strided_and_unaligned_rows(device, dtype) -> None:
    wide = _rows(7, 256, dtype, 3).to(device)
    for x in (wide[:, 64:128], wide[:, 1:33], wide[::2], wide.t().contiguous().t()[:, :96],
              wide.view(7, 4, 64)[:, 1:3]):
        codes, scales = ops.mxfp4_quantize(x)
        want_codes, want_scales = mxfp4.quantize(x.cpu().contiguous())
        assert torch.equal(_bytes(codes), want_codes) and torch.equal(_bytes(scales), want_scales)
        out = torch.empty((x.numel() // x.shape[-1], x.shape[-1] + 3), dtype=dtype, device=device)
        rows = out[:, 1:-2]  # neither its rows nor its base in 16-byte steps
        flat = (codes.view(rows.shape[0], -1), scales.view(rows.shape[0], -1))
        ops.mxfp4_dequantize(*flat, dtype, out=rows)
        assert torch.equal(rows.cpu(), mxfp4.values(want_codes, want_scales).to(dtype)
                           .view(rows.shape))


def _check_product(got, a, b, dtype):
    """got against the 64-bit product of the decoded a (M, K) and b (N, K)."""

    exact, size = a @ b.t(), a.abs() @ b.abs().t()
    limit = (a.shape[1] / 128 + 15) * 2.0 ** -23 * size + torch.finfo(dtype).eps / 2 * exact.abs()
    error = (got.cpu().double() - exact).abs()
    assert got.dtype == dtype and got.shape == exact.shape
    assert bool((error <= limit + torch.finfo(dtype).tiny).all()), (error / limit.clamp(min=1e-30)).max()


SHAPES = [(1, 1, 32), (1, 2560, 2048), (2, 17, 96), (15, 33, 512), (16, 16, 544), (17, 100, 1024),
          (33, 130, 2048), (48, 300, 5632), (64, 64, 480), (65, 129, 1024), (127, 260, 608),
          (128, 256, 256), (200, 1000, 96), (257, 513, 1280), (300, 2048, 512), (1030, 770, 736)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_and_matmul(device, dtype, m, n, k) -> None:
    x = _rows(m, k, dtype, m + k, spread=4)
    w = _rows(n, k, torch.float32, n + k, spread=3)
    w_codes, w_scales = ops.mxfp4_quantize(w.to(device))
    out = ops.mxfp4_linear(x.to(device), w_codes, w_scales)
    a = mxfp4.values(*mxfp4.quantize(x))
    b = mxfp4.values(*mxfp4.quantize(w))
    _check_product(out, a, b, dtype)
    x_codes, x_scales = ops.mxfp4_quantize(x.to(device))
    assert torch.equal(ops.mxfp4_matmul(x_codes, x_scales, w_codes, w_scales, dtype), out)


@pytest.mark.parametrize("m", [5, 40, 300])
def test_product_of_nan_and_empty_blocks(device, m) -> None:
    """A NaN block makes its rows NaN and no others; blocks of zeros add nothing."""

    x = _rows(m, 256, torch.float32, 1, spread=2)
    w = _rows(70, 256, torch.float32, 2, spread=2)
    x[3, 40] = float("nan")
    x[1] = 0.0
    w[10, 200] = float("inf")
    w[20, :64] = 0.0
    out = ops.mxfp4_linear(x.to(device), *ops.mxfp4_quantize(w.to(device))).cpu()
    nan = torch.zeros(m, 70, dtype=torch.bool)
    nan[3], nan[:, 10] = True, True
    assert torch.equal(torch.isnan(out), nan)
    a, b = mxfp4.values(*mxfp4.quantize(x)), mxfp4.values(*mxfp4.quantize(w))
    keep_m, keep_n = torch.arange(m) != 3, torch.arange(70) != 10
    _check_product(out[keep_m][:, keep_n], a[keep_m], b[keep_n], torch.float32)


@pytest.mark.parametrize("m", [3, 48, 270])
def test_product_into_a_view_and_of_strided_inputs(device, m) -> None:
    """Rows of a wider output are written and nothing beside them."""

    x = _rows(m, 576, torch.bfloat16, 5, spread=2).to(device)[:, 32:544]
    w = _rows(90, 512, torch.float32, 6, spread=2)
    codes, scales = ops.mxfp4_quantize(w.to(device))
    wide = torch.full((m + 2, 97), 7.0, dtype=torch.bfloat16, device=device)
    ops.mxfp4_linear(x, codes, scales, out=wide[1:-1, 3:93])
    a = mxfp4.values(*mxfp4.quantize(x.cpu().contiguous()))
    _check_product(wide[1:-1, 3:93], a, mxfp4.values(*mxfp4.quantize(w)), torch.bfloat16)
    wide[1:-1, 3:93] = 7.0
    assert bool((wide == 7.0).all())


def test_products_of_no_rows_and_batches(device) -> None:
    w = _rows(40, 64, torch.float32, 6)
    codes, scales = ops.mxfp4_quantize(w.to(device))
    assert ops.mxfp4_linear(torch.empty(0, 64, device=device), codes, scales).shape == (0, 40)
    empty = ops.mxfp4_quantize(torch.empty(0, 64, device=device))
    assert ops.mxfp4_matmul(*empty, codes, scales, torch.float16).shape == (0, 40)
    assert ops.mxfp4_dequantize(*empty, torch.float16).shape == (0, 64)
    x = _rows(6, 64, torch.float32, 7).view(2, 3, 64).to(device)
    out = ops.mxfp4_linear(x, codes, scales)
    assert out.shape == (2, 3, 40)
    assert torch.equal(out.view(6, 40), ops.mxfp4_linear(x.view(6, 64), codes, scales))
    assert torch.equal(ops.mxfp4_linear(x[1, 2], codes, scales), out[1, 2])


@pytest.mark.parametrize("m", [4, 50, 600])
def test_linear_on_another_stream_in_a_graph_and_with_a_workspace(device, m) -> None:
    """The same results eagerly, on a side stream with a caller's workspace, and from a
    replayed graph with other work between its replays."""

    w = ops.mxfp4_quantize(_rows(700, 1056, torch.float32, 8).to(device))
    x = _rows(m, 1056, torch.bfloat16, 9, spread=3).to(device)
    other = _rows(m, 1056, torch.bfloat16, 10, spread=3).to(device)
    want, want_other = ops.mxfp4_linear(x, *w), ops.mxfp4_linear(other, *w)
    size = ops.mxfp4_linear_workspace_bytes(m, 700, 1056)
    space = torch.empty(max(size, 1), dtype=torch.uint8, device=device)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.mxfp4_linear(x, *w, workspace=space)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.mxfp4_linear(static, *w)
    for source, expected in ((x, want), (other, want_other), (x, want)):
        static.copy_(source)
        graph.replay()
        ops.mxfp4_linear(other, *w)
        torch.cuda.synchronize()
        assert torch.equal(out, expected)


def test_refused_products(device) -> None:
    x = torch.randn(4, 64, device=device)
    codes, scales = ops.mxfp4_quantize(torch.randn(40, 64, device=device))
    with pytest.raises(ValueError, match="workspace"):
        ops.mxfp4_linear(x, codes, scales, workspace=torch.empty(8, dtype=torch.uint8,
                                                                 device=device))
    with pytest.raises(ValueError, match="requires HIP device"):
        ops.mxfp4_linear(x, codes, scales, out=torch.empty(4, 40))


def test_refused_matrices(device) -> None:
    """The refusals of tests/test_mxfp4_host.py, by the operators themselves."""

    def on(*shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=torch.uint8 if dtype.itemsize == 1 else dtype,
                           device=device).view(dtype)

    codes, scales = on(4, 32, dtype=CODES), on(4, 2, dtype=SCALES)
    with pytest.raises(ValueError, match="multiple of 32"):
        ops.mxfp4_quantize(on(4, 48))
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        ops.mxfp4_quantize(on(4, 64, dtype=torch.int32))
    with pytest.raises(TypeError, match="float4_e2m1fn_x2"):
        ops.mxfp4_dequantize(on(4, 32, dtype=torch.uint8), scales, torch.float32)
    with pytest.raises(TypeError, match="out must be float32"):
        ops.mxfp4_dequantize(codes, scales, torch.float64)
    with pytest.raises(ValueError, match="one entry per 32"):
        ops.mxfp4_dequantize(codes, on(4, 1, dtype=SCALES), torch.float32)
    with pytest.raises(ValueError, match="contiguous"):
        ops.mxfp4_dequantize(on(8, 32, dtype=CODES)[::2], scales, torch.float32)
    with pytest.raises(ValueError, match="the inputs' K"):
        ops.mxfp4_linear(on(3, 32), codes, scales)
    with pytest.raises(ValueError, match="have A's K"):
        ops.mxfp4_matmul(codes, scales, on(4, 16, dtype=CODES), on(4, 1, dtype=SCALES),
                         torch.float32)
    with pytest.raises(ValueError, match="at least one row"):
        ops.mxfp4_linear(on(3, 64), on(0, 32, dtype=CODES), on(0, 2, dtype=SCALES))
    with pytest.raises(ValueError, match="out must have shape"):
        ops.mxfp4_linear(on(3, 64), codes, scales, out=on(3, 5))
    with pytest.raises(ValueError, match="the inputs' dtype"):
        ops.mxfp4_linear(on(3, 64), codes, scales, out=on(3, 4, dtype=torch.float16))
    with pytest.raises(ValueError, match="the given dtype"):
        ops.mxfp4_dequantize(codes, scales, torch.float16, out=on(4, 64))
    with pytest.raises(ValueError, match="go together"):
        ops.mxfp4_quantize(on(4, 64), codes=codes)
    with pytest.raises(ValueError, match="shape \\(..., K / 2\\)"):
        ops.mxfp4_quantize(on(3, 64), codes=codes, scales=scales)
    with pytest.raises(ValueError, match="must be contiguous"):
        ops.mxfp4_linear(on(3, 2, 64), codes, scales, out=on(3, 2, 8)[..., :4])
    with pytest.raises(ValueError, match="workspace must be"):
        ops.mxfp4_linear(on(3, 64), codes, scales, workspace=on(100))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(65, 64, 2048), (100, 130, 2080), (128, 257, 5632), (190, 72, 2592),
                                   (66, 1000, 4128), (40, 8200, 1056), (64, 8192, 2048)])
def test_products_of_a_long_depth_or_many_columns(device, dtype, m, n, k) -> None:
    """The projection and the two calls may sum in different orders here: each by itself."""

    x = _rows(m, k, dtype, m + k, spread=4)
    w = _rows(n, k, torch.float32, n + k, spread=3)
    w_codes, w_scales = ops.mxfp4_quantize(w.to(device))
    a = mxfp4.values(*mxfp4.quantize(x))
    b = mxfp4.values(*mxfp4.quantize(w))
    _check_product(ops.mxfp4_linear(x.to(device), w_codes, w_scales), a, b, dtype)
    x_codes, x_scales = ops.mxfp4_quantize(x.to(device))
    _check_product(ops.mxfp4_matmul(x_codes, x_scales, w_codes, w_scales, dtype), a, b, dtype)


@pytest.mark.parametrize("m,k", [(70, 2080), (200, 5632)])
def test_nan_blocks_of_a_long_depth(device, m, k) -> None:
    """A NaN block makes its row (of A) or column (of B) NaN and nothing else."""

    x = _rows(m, k, torch.float32, 3, spread=2)
    w = _rows(96, k, torch.float32, 4, spread=2)
    x[5, k - 1] = float("nan")
    w[90, 1024] = float("inf")
    out = ops.mxfp4_linear(x.to(device), *ops.mxfp4_quantize(w.to(device))).cpu()
    bad = torch.zeros(m, 96, dtype=torch.bool)
    bad[5] = True
    bad[:, 90] = True
    assert torch.equal(out.isnan(), bad)


@pytest.mark.parametrize("m,n,k", [(1, 500, 2048), (40, 96, 544), (70, 130, 2080), (300, 200, 1024)])
def test_projections_on_two_streams(device, m, n, k) -> None:
    """Calls at once, each with scratch memory of its own, and with a workspace for each."""

    w = ops.mxfp4_quantize(_rows(n, k, torch.float32, 1, spread=3).to(device))
    inputs = [_rows(m, k, torch.bfloat16, s, spread=3).to(device) for s in (2, 3)]
    want = [ops.mxfp4_linear(x, *w) for x in inputs]
    size = ops.mxfp4_linear_workspace_bytes(m, n, k)
    spaces = [torch.empty(size + 16, dtype=torch.uint8, device=device) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for turn in range(12):
        i = turn % 2
        with torch.cuda.stream(streams[i]):
            results.append((i, ops.mxfp4_linear(inputs[i], *w,
                                                workspace=spaces[i] if turn % 4 < 2 else None)))
    torch.cuda.synchronize()
    for i, got in results:
        assert torch.equal(got, want[i])

"""int8_linear against the product in doubles: sizes that end inside every tile, extreme codes, unaligned views, graphs."""
import ctypes

import pytest
import torch

from block_reference import assert_close, int8_linear
from torch_dist_ext_amd import _capi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tde(cuda_device):
    import torch_dist_ext_amd
    return torch_dist_ext_amd


def make(tokens, k, n, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-127, 128, (tokens, k), generator=g).to(torch.int8)
    weight = torch.randint(-128, 128, (n, k), generator=g).to(torch.int8)
    scales = torch.rand(tokens, generator=g) * 0.02 + 0.001
    weight_scales = torch.rand(n, generator=g) * 0.002 + 0.0001
    return codes, scales, weight, weight_scales, torch.randn(n, generator=g) if bias else None


def run(tde, args, dtype):
    return tde.int8_linear(*[None if x is None else x.cuda() for x in args], dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("tokens,k,n", [
    (1, 1, 1), (1, 16, 1), (1, 4096, 65), (2, 127, 3), (3, 1024, 1280), (4, 8192, 7), (5, 64, 130), (8, 520, 33), (9, 2048, 257), (16, 1000, 127),
    (17, 33, 128), (31, 128, 129), (32, 5000, 100), (33, 129, 256), (48, 5120, 300), (64, 144, 64), (65, 260, 511), (100, 4100, 96),
    (127, 384, 200), (128, 128, 128), (129, 127, 255), (200, 640, 1000), (255, 1024, 513), (257, 1160, 260), (300, 2056, 1030), (513, 260, 259),
    (1030, 520, 770),
])
def test_sizes(tde, tokens, k, n, dtype):
    args = make(tokens, k, n, seed=tokens * 7 + k + n, bias=(tokens + n) % 2 == 0)
    got = run(tde, args, dtype)
    assert got.dtype == dtype
    assert_close(got, *int8_linear(*args, dtype), "%dx%dx%d" % (tokens, k, n))


@pytest.mark.parametrize("tokens", [1, 40, 150])
@pytest.mark.parametrize("code,weight", [(-128, -128), (127, -128), (127, 127)])
def test_largest_sums_stay_exact(tde, tokens, code, weight):
    """131071 products of 2^14: the sum is just below 2^31."""
    k, n = _capi.INT8_MAX_K, 5
    codes = torch.full((tokens, k), code, dtype=torch.int8)
    w = torch.full((n, k), weight, dtype=torch.int8)
    w[1, ::2] = 0
    args = (codes, torch.ones(tokens), w, torch.ones(n), None)
    assert_close(run(tde, args, torch.float32), *int8_linear(*args, torch.float32))


@pytest.mark.parametrize("tokens,k,n", [(1, 64, 40), (20, 300, 64), (130, 512, 140)])
def test_scales_that_are_not_finite_stay_in_their_row_and_channel(tde, tokens, k, n):
    codes, scales, weight, ws, _ = make(tokens, k, n, 3, bias=False)
    want, bound = int8_linear(codes, scales, weight, ws, None, torch.bfloat16)
    scales, ws = scales.clone(), ws.clone()
    scales[tokens - 1], ws[n // 2], ws[n - 1] = float("nan"), float("inf"), float("nan")
    got = run(tde, (codes, scales, weight, ws, None), torch.bfloat16).cpu()
    assert torch.isnan(got[tokens - 1]).all() and torch.isnan(got[:, n - 1]).all()
    keep = torch.ones(n, dtype=torch.bool)
    keep[n // 2] = keep[n - 1] = False
    rows = torch.arange(tokens) != tokens - 1
    assert_close(got[rows][:, keep], want[rows][:, keep], bound[rows][:, keep])
    assert not torch.isfinite(got[:, n // 2]).any() or bool((want[:, n // 2] == 0).any())


def test_leading_dimensions_and_views_that_begin_anywhere(tde):
    codes, scales, weight, ws, bias = make(6 * 35, 200, 90, 11)
    want, bound = int8_linear(codes, scales, weight, ws, bias, torch.float16)
    for skip in (1, 2, 3, 5, 8, 13):
        c = torch.empty(codes.numel() + 64, dtype=torch.int8, device="cuda")[skip:skip + codes.numel()].view(6, 35, 200)
        w = torch.empty(weight.numel() + 64, dtype=torch.int8, device="cuda")[skip + 1:skip + 1 + weight.numel()].view(90, 200)
        c.copy_(codes.view(6, 35, 200))
        w.copy_(weight)
        got = tde.int8_linear(c, scales.cuda().view(6, 35), w, ws.cuda(), bias.cuda(), torch.float16)
        assert got.shape == (6, 35, 90)
        assert_close(got.view(-1, 90), want, bound, "skip %d" % skip)


@pytest.mark.parametrize("tokens,k,n", [(0, 64, 32), (3, 64, 0)])
def test_nothing_to_do(tde, tokens, k, n):
    assert run(tde, make(tokens, k, n, 1), torch.bfloat16).shape == (tokens, n)


@pytest.mark.parametrize("tokens,n", [(1, 37), (7, 130), (33, 200), (140, 133), (300, 258)])
def test_nothing_is_written_outside_the_output(tde, tokens, n):
    """Through the C entry point, between two bands of bytes that have to stay."""
    codes, scales, weight, ws, _ = [x if x is None else x.cuda() for x in make(tokens, 96, n, 5, bias=False)]
    band = 4096
    for dtype, code in ((torch.bfloat16, _capi.BF16), (torch.float32, _capi.F32)):
        size = tokens * n * torch.finfo(dtype).bits // 8
        buf = torch.full((band + size + band,), 0x5A, dtype=torch.uint8, device="cuda")
        p = _capi.Int8Product(tokens=tokens, k=96, n=n, out_dtype=code, codes=codes.data_ptr(), weight=weight.data_ptr(), scales=scales.data_ptr(),
                              weight_scales=ws.data_ptr(), out=buf.data_ptr() + band)
        _capi.check(_capi.load().tde_int8_linear(ctypes.byref(p), torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        host = buf.cpu()
        assert bool((host[:band] == 0x5A).all()) and bool((host[band + size:] == 0x5A).all())
        got = host[band:band + size].view(dtype).view(tokens, n)
        assert_close(got, *int8_linear(codes.cpu(), scales.cpu(), weight.cpu(), ws.cpu(), None, dtype))


def test_replayed_graphs_and_another_stream(tde):
    for tokens, k, n in ((1, 1024, 96), (16, 4096, 128), (200, 256, 300)):
        args = [None if x is None else x.cuda() for x in make(tokens, k, n, 21)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = tde.int8_linear(*args, torch.bfloat16)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph, twin = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = tde.int8_linear(*args, torch.bfloat16)
        with torch.cuda.graph(twin):
            out2 = tde.int8_linear(*args, torch.bfloat16)
        for replay in range(3):
            fresh = make(tokens, k, n, 30 + replay)
            args[0].copy_(fresh[0])
            want = tde.int8_linear(*args, torch.bfloat16)
            graph.replay()
            twin.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(out2, want)
            assert_close(out, *int8_linear(*[x if x is None else x.cpu() for x in args], torch.bfloat16))
        assert eager.shape == out.shape

"""Calls of the 8-bit floating point operators and of counter-based dropout that a user may make beside the ordinary ones:
beside other kernels on the device, into parts of larger buffers, of views that the dispatcher would resolve, with states
that change, over sums long enough to show how they are added."""

import pytest
import torch

pytestmark = pytest.mark.gpu

E4 = torch.float8_e4m3fn


def _x(g, R, C):
    """Normal numbers with rows of different size."""
    x = torch.randn(R, C, generator=g, device=g.device)
    return x * torch.exp2(torch.randint(-4, 5, (R, 1), generator=g, device=g.device).float())


def test_products_beside_other_tensor_core_kernels(dev):
    """Products cut over clusters and of whole tiles, on one stream, while another stream multiplies with a library's tensor-core
    kernels: both give what they give alone."""
    from approxtorch_b200.backend import ops
    g = torch.Generator(dev).manual_seed(3)
    sizes = [(1, 4096, 4096), (37, 1000, 4096), (100, 5500, 2048), (300, 1000, 700), (1300, 1300, 3000)]
    held = [(ops.fp8_quantize_rows(_x(g, M, K)), ops.fp8_quantize_blocks(_x(g, N, K), transposed=False)) for M, N, K in sizes]
    mats = [torch.randn(n, n, generator=g, device=dev).bfloat16() for n in (512, 1024, 2048)]
    want = [ops.fp8_gemm(*a, *b) for a, b in held]
    want_mats = [m @ m for m in mats]
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    got, got_mats = [], []
    for _ in range(10):
        with torch.cuda.stream(one):
            got.append([ops.fp8_gemm(*a, *b) for a, b in held])
        with torch.cuda.stream(two):
            got_mats.append([m @ m for m in mats])
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(p, q) for p, q in zip(out, want))
    for out in got_mats:
        assert all(torch.equal(p, q) for p, q in zip(out, want_mats))

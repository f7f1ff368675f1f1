"""GPU parity of the block-scaled 8-bit floating point operators against the 64-bit oracle.

Quantised numbers and scales are compared exactly: division by a power of two is exact and the rounding is the nearest
one.  Products: the tensor core adds K exact products in fp32 in some order, each addition off by at most one unit in the
last place (2^-23 of the running sum, which no partial sum's magnitude exceeds sum |a b|), so an element is off by at most
K 2^-23 sum|a b|, plus two roundings of the epilogue (alpha, bias: 2^-24 each) and half a step of the result's type."""

import numpy as np
import pytest
import torch

from oracle import fp8_oracle as fo

pytestmark = pytest.mark.gpu

F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _x(rng, R, C, dt="fp32"):
    """Normal numbers with rows and columns of very different size."""
    x = rng.standard_normal((R, C)) * np.exp2(rng.integers(-6, 6, (R, 1))) * np.exp2(rng.integers(-4, 4, (1, C)))
    return torch.from_numpy(x.astype(np.float32)).to(DT[dt])


def _d(t):
    return t.detach().double().cpu().numpy()


def _bytes(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


def _scales(t):
    b = _bytes(t)
    return np.where(b == 255, np.nan, np.exp2(b.astype(np.float64) - 127))


def _check_quantised(q, s, x64, fmt, block_rows):
    rq, rs = fo.quantise(x64, fmt, block_rows)
    np.testing.assert_array_equal(_scales(s), rs)
    np.testing.assert_array_equal(_d(q.contiguous().float()), rq)


SHAPES = [(1, 1), (1, 4096), (3, 127), (128, 128), (129, 130), (200, 2048), (257, 1000), (1000, 33)]


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("R,C", SHAPES)
def test_quantise_every_layout(dev, R, C, dt, fmt):
    from approxtorch_b200.backend import ops
    x = _x(np.random.default_rng(R * 1000 + C), R, C, dt).to(dev)
    x64 = _d(x)
    q, s = ops.fp8_quantize_rows(x, F8[fmt])
    assert q.dtype == F8[fmt] and s.dtype == torch.float8_e8m0fnu and q.shape == (R, C) and s.shape == (R, -(-C // 128))
    _check_quantised(q, s, x64, fmt, 1)
    q2, s2, qt, st = ops.fp8_quantize_both(x, F8[fmt])
    assert np.array_equal(_bytes(q2), _bytes(q)) and np.array_equal(_bytes(s2), _bytes(s))
    _check_quantised(qt, st, x64.T, fmt, 1)
    q3, s3, qt3, st3 = ops.fp8_quantize_blocks(x, F8[fmt])
    _check_quantised(q3, s3, x64, fmt, 128)
    assert np.array_equal(_bytes(qt3), _bytes(q3).T) and np.array_equal(_bytes(st3), _bytes(s3).T)
    q4, s4 = ops.fp8_quantize_blocks(x, F8[fmt], transposed=False)
    assert np.array_equal(_bytes(q4), _bytes(q3)) and np.array_equal(_bytes(s4), _bytes(s3))


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
def test_quantise_strided_and_unaligned_inputs(dev, dt):
    from approxtorch_b200.backend import ops
    base = _x(np.random.default_rng(5), 300, 520, dt).to(dev)
    for x in (base[:, :500], base[:, 1:258], base[::2, 8:264], base.t(), base[:, ::2], base[7:8], base[:1].expand(130, 520),
              base.flatten()[3:3 + 131 * 129].view(131, 129)):
        ref = x.contiguous()
        for f in (ops.fp8_quantize_rows, ops.fp8_quantize_both, ops.fp8_quantize_blocks):
            for got, want in zip(f(x), f(ref)):
                assert np.array_equal(_bytes(got), _bytes(want))
        _check_quantised(*ops.fp8_quantize_rows(x), _d(x), "e4m3", 1)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_quantise_edges_of_the_range(dev, fmt):
    """Zeros, subnormals, the largest numbers, borders between two scales, ties, infinities and NaN."""
    from approxtorch_b200.backend import ops
    F = fo.FORMATS[fmt][0]
    x = np.zeros((16, 256), np.float32)
    x[1, :] = 1e-44                                        # subnormal: the scale stops at 2^-126
    x[2, 5] = np.finfo(np.float32).max
    x[3, 7] = F                                            # exactly the largest: scale 1
    x[4, 7] = np.nextafter(np.float32(F), np.float32(np.inf))   # just above: scale 2
    x[5, :128] = np.linspace(-F, F, 128)
    x[6, :128] = np.float32(2.0) ** -np.arange(128)
    x[7, 0], x[7, 1] = 256.0, 17 / 16                      # a tie between 1 and 1.125 where the scale is 1
    x[7, 2:66] = np.arange(64) / 32 + 1
    x[8, 3] = np.nan
    x[9, 130] = np.inf
    x[10, 0], x[10, 200] = -np.inf, np.nan
    x[11, :] = -0.0
    x[12, 0] = 2.0 ** -126
    t = torch.from_numpy(x).to(dev)
    _check_quantised(*ops.fp8_quantize_rows(t, F8[fmt]), x, fmt, 1)
    q, s, qt, st = ops.fp8_quantize_both(t, F8[fmt])
    _check_quantised(q, s, x, fmt, 1)
    _check_quantised(qt, st, x.T, fmt, 1)
    _check_quantised(*ops.fp8_quantize_blocks(t, F8[fmt])[:2], x, fmt, 128)


def test_quantise_with_dropout_masks_without_looking(dev):
    from approxtorch_b200.backend import ops
    seed, offset = -987654321987654321, 1 << 33
    state = torch.tensor([seed, offset], dtype=torch.int64, device=dev)
    for R, C, p in ((5, 128, 0.5), (130, 257, 0.1), (64, 1001, 0.9), (33, 300, 1.0), (128, 136, 1e-9)):
        x = _x(np.random.default_rng(C), R, C).to(dev)
        keep = fo.keep_mask((R, C), p, seed, offset)
        x[torch.from_numpy(~keep).to(dev)] = float("nan")              # dropped places may hold anything
        x64 = np.where(keep, _d(x), 0.0)
        _check_quantised(*ops.fp8_quantize_rows(x, drop_p=p, rng=state), x64, "e4m3", 1)
        q, s, qt, st = ops.fp8_quantize_both(x, drop_p=p, rng=state)
        _check_quantised(q, s, x64, "e4m3", 1)
        _check_quantised(qt, st, x64.T, "e4m3", 1)


# ---------------------------------------------------------------------------------------------------- products
def _held(rng, R, K, fmt, block_rows, dev):
    from approxtorch_b200.backend import ops
    x = _x(rng, R, K).to(dev)
    if block_rows == 128:
        return ops.fp8_quantize_blocks(x, F8[fmt], transposed=False)
    return ops.fp8_quantize_rows(x, F8[fmt])


def _off(y, ref, mag, K, out):
    half = torch.finfo(DT[out]).eps / 2
    tol = (K * 2.0 ** -23 + 2 * 2.0 ** -24) * mag
    tol = tol + half * (np.abs(ref) + tol) + float(torch.finfo(DT[out]).smallest_normal) * half * 2
    err = np.abs(_d(y) - ref)
    assert (err <= tol).all(), (err / tol).max()


def _check_product(a, b, y, bias, alpha, out):
    ref, mag = fo.product(_d(a[0].contiguous().float()), _scales(a[1]), _d(b[0].contiguous().float()), _scales(b[1]),
                          None if bias is None else _d(bias), alpha)
    assert y.dtype == DT[out] and tuple(y.shape) == ref.shape
    _off(y, ref, mag, a[0].shape[1], out)


PRODUCTS = [(1, 1, 1), (1, 256, 128), (1, 1000, 2048), (2, 130, 127), (7, 4096, 1024), (16, 64, 4096), (17, 100, 300), (64, 512, 640),
            (65, 48, 129), (128, 128, 512), (129, 193, 515), (200, 1000, 2048), (513, 257, 1100), (1000, 777, 96), (1500, 2000, 384)]


@pytest.mark.parametrize("out", ["fp32", "bf16"])
@pytest.mark.parametrize("b_rows", [1, 128])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product(dev, M, N, K, b_rows, out):
    from approxtorch_b200.backend import ops, _C
    rng = np.random.default_rng(M + 7 * N + 13 * K)
    a, b = _held(rng, M, K, "e4m3", 1, dev), _held(rng, N, K, "e4m3", b_rows, dev)
    bias = torch.from_numpy(rng.standard_normal(N).astype(np.float32)).to(dev) if (M + N) % 2 else None
    y = ops.fp8_gemm(*a, *b, bias=bias, alpha=1.25, out_dtype=DT[out])
    _check_product(a, b, y, bias, 1.25, out)


@pytest.mark.parametrize("fa,fb", [("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("M,N,K", [(3, 200, 260), (150, 200, 260)])
def test_product_of_mixed_formats_and_block_scales_on_both_sides(dev, M, N, K, fa, fb):
    from approxtorch_b200.backend import ops
    rng = np.random.default_rng(3)
    a, b = _held(rng, M, K, fa, 128, dev), _held(rng, N, K, fb, 128, dev)
    _check_product(a, b, ops.fp8_gemm(*a, *b, out_dtype=torch.float16, alpha=2.0 ** -14), None, 2.0 ** -14, "fp16")


@pytest.mark.parametrize("M", [5, 140])
def test_product_takes_operands_as_they_lie(dev, M):
    """Pitches, bases and orders that the kernel cannot read directly give the same bits as the plain layout."""
    from approxtorch_b200.backend import ops
    rng = np.random.default_rng(11)
    N, K = 150, 300
    a, b = _held(rng, M, K, "e4m3", 1, dev), _held(rng, N, K, "e4m3", 1, dev)
    want = ops.fp8_gemm(*a, *b, out_dtype=torch.float32)
    u8 = lambda t: t.view(torch.uint8)     # noqa: E731

    def pitched(t, pitch, off):
        buf = torch.full((t.shape[0] * pitch + off + 64,), 200, dtype=torch.uint8, device=dev)
        v = buf[off:off + t.shape[0] * pitch].view(t.shape[0], pitch)[:, :t.shape[1]]
        v.copy_(u8(t))
        return v.view(t.dtype)
    for pitch, off in ((K, 0), (K + 4, 0), (320, 1), (304, 16)):
        a2 = pitched(a[0], pitch, off)
        assert torch.equal(ops.fp8_gemm(a2, a[1], *b, out_dtype=torch.float32), want)
    colmajor = torch.empty(K, M, dtype=torch.uint8, device=dev)
    colmajor.copy_(u8(a[0]).t())
    assert torch.equal(ops.fp8_gemm(colmajor.view(torch.float8_e4m3fn).t(), a[1], *b, out_dtype=torch.float32), want)
    for pitch, off in ((3, 0), (4, 1), (5, 3), (8, 4)):
        assert torch.equal(ops.fp8_gemm(a[0], pitched(a[1], pitch, off), *b, out_dtype=torch.float32), want)
    tight = u8(a[1]).contiguous().flatten().clone().view(M, 3)       # no room behind the last row
    assert torch.equal(ops.fp8_gemm(a[0], tight, *b, out_dtype=torch.float32), want)
    st = torch.empty(3, M, dtype=torch.uint8, device=dev)
    st.copy_(u8(a[1]).t())
    assert torch.equal(ops.fp8_gemm(a[0], st.t(), *b, out_dtype=torch.float32), want)


def test_product_edges(dev):
    from approxtorch_b200.backend import ops
    f8, z = torch.float8_e4m3fn, lambda *s, dt=torch.uint8: torch.zeros(s, dtype=dt, device=dev)     # noqa: E731
    bias = torch.arange(5, dtype=torch.float32, device=dev)
    # nothing to add up: the bias alone
    y = ops.fp8_gemm(z(3, 0).view(f8), z(3, 0), z(5, 0).view(f8), z(5, 0), bias=bias, out_dtype=torch.float32)
    assert torch.equal(y, bias.expand(3, 5))
    assert ops.fp8_gemm(z(0, 8).view(f8), z(0, 1), z(5, 8).view(f8), z(5, 1)).shape == (0, 5)
    assert ops.fp8_gemm(z(3, 8).view(f8), z(3, 1), z(0, 8).view(f8), z(0, 1)).shape == (3, 0)
    # a NaN block poisons its row and no other; infinities of the input arrive as NaN
    rng = np.random.default_rng(2)
    x = _x(rng, 140, 256).to(dev)
    x[130, 200] = float("inf")
    x[2, 3] = float("nan")
    a, b = ops.fp8_quantize_rows(x), _held(rng, 70, 256, "e4m3", 128, dev)
    y = ops.fp8_gemm(*a, *b, out_dtype=torch.float32)
    bad = torch.isnan(y).all(dim=1)
    assert bad.nonzero().flatten().tolist() == [2, 130] and not torch.isnan(y[~bad]).any()
    # extreme scales: 2^-126 on one side, 2^100 on the other
    a = (torch.full((130, 128), 448.0, device=dev).to(f8), torch.full((130, 1), 1, dtype=torch.uint8, device=dev))
    b = (torch.full((9, 128), 1.0, device=dev).to(f8), torch.full((9, 1), 227, dtype=torch.uint8, device=dev))
    assert torch.equal(ops.fp8_gemm(*a, *b, out_dtype=torch.float32), torch.full((130, 9), 448.0 * 128 * 2.0 ** -26, device=dev))


@pytest.mark.parametrize("M", [4, 200])
def test_product_with_masked_result(dev, M):
    from approxtorch_b200.backend import ops
    rng = np.random.default_rng(8)
    state = torch.tensor([77, 3], dtype=torch.int64, device=dev)
    for N in (256, 131):
        a, b = _held(rng, M, 384, "e4m3", 1, dev), _held(rng, N, 384, "e4m3", 1, dev)
        y = ops.fp8_gemm(*a, *b, out_dtype=torch.float32)
        keep = torch.from_numpy(fo.keep_mask((M, N), 0.3, 77, 3)).to(dev)
        got = ops.fp8_gemm(*a, *b, out_dtype=torch.float32, drop_p=0.3, rng=state)
        assert torch.equal(got, torch.where(keep, y, 0.0))


def test_results_repeat_bit_for_bit_and_no_wait_ran_out(dev):
    import ctypes
    from approxtorch_b200.backend import ops, _C
    rng = np.random.default_rng(4)
    for M, N, K in ((1, 1024, 4096), (20, 300, 4096), (700, 900, 1300)):
        a, b = _held(rng, M, K, "e4m3", 1, dev), _held(rng, N, K, "e4m3", 128, dev)
        ys = [ops.fp8_gemm(*a, *b, out_dtype=torch.float32) for _ in range(6)]
        assert all(torch.equal(y, ys[0]) for y in ys)
    status = ctypes.c_int(-1)
    assert _C.lib.atb_fp8_status(ctypes.byref(status)) == 0 and status.value == 0


def test_refusals_on_the_device(dev):
    from approxtorch_b200.backend import ops
    f8 = torch.float8_e4m3fn
    q, s = ops.fp8_quantize_rows(torch.randn(4, 200, device=dev))
    for call in (lambda: ops.fp8_gemm(q, s[:3], q, s), lambda: ops.fp8_gemm(q, s[:, :1], q, s), lambda: ops.fp8_gemm(q, s, q[:, :100], s[:, :1]),
                 lambda: ops.fp8_gemm(q.float(), s, q, s), lambda: ops.fp8_gemm(q, s.float(), q, s), lambda: ops.fp8_gemm(q, s, q, s, out_dtype=f8),
                 lambda: ops.fp8_gemm(q, s, q, s, bias=torch.zeros(5, device=dev)), lambda: ops.fp8_gemm(q, s, q, s, bias=torch.zeros(4)),
                 lambda: ops.fp8_gemm(q, s, q, s, drop_p=0.5), lambda: ops.fp8_gemm(q[0], s, q, s),
                 lambda: ops.fp8_quantize_rows(torch.zeros(3, device=dev)), lambda: ops.fp8_quantize_rows(torch.zeros(3, 3, device=dev, dtype=torch.float64)),
                 lambda: ops.fp8_quantize_rows(torch.zeros(3, 3, device=dev), torch.float16),
                 lambda: ops.fp8_quantize_rows(torch.zeros(3, 3, device=dev), drop_p=0.5),
                 lambda: ops.fp8_quantize_rows(torch.zeros(3, 3, device=dev), drop_p=0.5, rng=torch.zeros(2, dtype=torch.int64)),
                 lambda: ops.fp8_quantize_rows(torch.zeros(3, 3, device=dev), drop_p=0.5, rng=torch.zeros(3, dtype=torch.int64, device=dev))):
        with pytest.raises(RuntimeError):
            call()


def test_captured_and_replayed_on_a_side_stream(dev):
    from approxtorch_b200.backend import ops
    x, w = torch.randn(96, 640, device=dev), torch.randn(200, 640, device=dev)
    wq = ops.fp8_quantize_blocks(w, transposed=False)

    def chain():
        return ops.fp8_gemm(*ops.fp8_quantize_rows(x), *wq, out_dtype=torch.float32)
    want = chain()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(chain(), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = chain()
    x.copy_(torch.randn_like(x))
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, chain()) and not torch.equal(y, want)

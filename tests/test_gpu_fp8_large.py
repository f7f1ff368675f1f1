"""The block-scaled product and its neighbours where launches take their other forms: many tiles, many waves, long
reductions, matrices beyond 32-bit offsets, concurrent streams, pitched results.  References are 64-bit products on the GPU
of the operands' decoded values; tolerances as in test_gpu_fp8.py (K 2^-23 of the magnitudes, two roundings of the
epilogue, half a step of the result's type)."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import fp8_oracle as fo

pytestmark = pytest.mark.gpu

E4 = torch.float8_e4m3fn


def _x(g, R, C):
    """Normal numbers with rows of different size."""
    x = torch.randn(R, C, generator=g, device=g.device)
    return x * torch.exp2(torch.randint(-4, 5, (R, 1), generator=g, device=g.device).float())


def _decoded(q, s):
    """Values of an operand in 64 bits, from the bytes of its scales."""
    rows = 1 if s.shape[0] == q.shape[0] else 128
    e = s.contiguous().view(torch.uint8).double() - 127
    s64 = torch.exp2(e).repeat_interleave(rows, 0)[:q.shape[0]].repeat_interleave(128, 1)[:, :q.shape[1]]
    return q.contiguous().float().double() * s64


def _check(y, a, b, bias=None, alpha=1.0, keep=None):
    da, db = _decoded(*a), _decoded(*b)
    K, half = da.shape[1], torch.finfo(y.dtype).eps / 2
    ref, mag = alpha * (da @ db.t()), abs(alpha) * (da.abs() @ db.abs().t())
    if bias is not None:
        ref, mag = ref + bias.double(), mag + bias.double().abs()
    if keep is not None:
        ref = torch.where(keep, ref, 0.0)
    tol = (K * 2.0 ** -23 + 2 * 2.0 ** -24) * mag
    # half a step of the result: eps / 2 of the value, and below the smallest normal number, where the steps stay as they are
    # (fp16: 2^-24 apart below 2^-14), eps / 2 of that number (2^-11 2^-14 = 2^-25, half of 2^-24)
    tol = tol + half * (ref.abs() + tol) + half * torch.finfo(y.dtype).smallest_normal
    worst = ((y.double() - ref).abs() / tol.clamp(min=1e-300)).max().item()
    assert worst <= 1.0, worst


def _operands(dev, M, N, K, b_rows, seed=0):
    from approxtorch_b200.backend import ops
    g = torch.Generator(dev).manual_seed(seed + M + 3 * N + 5 * K)
    a, w = ops.fp8_quantize_rows(_x(g, M, K)), _x(g, N, K)
    return a, (ops.fp8_quantize_blocks(w, transposed=False) if b_rows == 128 else ops.fp8_quantize_rows(w))


# several waves of 256-column tiles on overlapping accumulators, of narrower tiles, single blocks, few rows or columns
MANY = [(2600, 2700, 700), (5000, 2100, 130), (2304, 4096, 1024), (4100, 300, 900), (300, 4100, 900), (20000, 33, 260), (33, 20000, 260),
        (1, 40000, 200), (1300, 1300, 3000), (129, 9000, 4200)]


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", MANY)
def test_product_of_many_tiles(dev, M, N, K, out):
    from approxtorch_b200.backend import ops
    a, b = _operands(dev, M, N, K, 128 if (M + K) % 3 else 1)
    bias = torch.randn(N, device=dev)
    _check(ops.fp8_gemm(*a, *b, bias=bias, alpha=2.0 ** -9, out_dtype=out), a, b, bias, 2.0 ** -9)


@pytest.mark.parametrize("M,N,K", [(300, 500, 2049), (300, 500, 20000), (2600, 1500, 5000), (17, 700, 33000), (1, 300, 100000), (3, 200, 200000),
                                   (700, 64, 65536)])
def test_product_over_long_reductions(dev, M, N, K):
    """Beyond 2048 steps an fp32 result is added up from partial sums of 1024: K 2^-23 still bounds it, and a constant
    product, whose running sum grows with every step, has to come out within 2^-18 (an accumulator that cuts what does not fit
    loses up to 2^-24 of the running sum in every one of the 32 additions between two roundings: 32 2^-24 = 2^-19, twice)."""
    from approxtorch_b200.backend import ops
    a, b = _operands(dev, M, N, K, 1)
    _check(ops.fp8_gemm(*a, *b, out_dtype=torch.float32), a, b)
    _check(ops.fp8_gemm(*a, *b, alpha=2.0 ** -12, out_dtype=torch.bfloat16), a, b, None, 2.0 ** -12)
    ones = (torch.full((M, K), 1.125, device=dev).to(E4), torch.full((M, -(-K // 128)), 127, dtype=torch.uint8, device=dev))
    onesb = (torch.full((N, K), 1.375, device=dev).to(E4), torch.full((N, -(-K // 128)), 127, dtype=torch.uint8, device=dev))
    y = ops.fp8_gemm(*ones, *onesb, out_dtype=torch.float32)
    assert ((y - 1.125 * 1.375 * K).abs() <= 2.0 ** -18 * 1.125 * 1.375 * K).all()


@pytest.mark.parametrize("M,N,K", [(700, 1000, 400), (9, 1001, 2000), (1300, 517, 2600)])
def test_masked_product_of_many_tiles(dev, M, N, K):
    from approxtorch_b200.backend import ops
    a, b = _operands(dev, M, N, K, 1)
    keep = torch.from_numpy(fo.keep_mask((M, N), 0.35, 5, 1 << 40)).to(dev)
    state = torch.tensor([5, 1 << 40], dtype=torch.int64, device=dev)
    y = ops.fp8_gemm(*a, *b, out_dtype=torch.float32, drop_p=0.35, rng=state)
    assert (y[~keep] == 0).all()
    _check(y, a, b, keep=keep)


def test_operands_beyond_32_bit_offsets(dev):
    """A of 4.9 GB: rows past 4 GiB give what they give by themselves."""
    from approxtorch_b200.backend import ops
    M, N, K = 75000, 24, 65536
    a = torch.randint(0, 120, (M, K), dtype=torch.uint8, device=dev).view(E4)        # finite, non-negative
    sa = torch.randint(120, 130, (M, K // 128), dtype=torch.uint8, device=dev)
    b = torch.randint(0, 120, (N, K), dtype=torch.uint8, device=dev).view(E4)
    sb = torch.full((N, K // 128), 118, dtype=torch.uint8, device=dev)
    y = ops.fp8_gemm(a, sa, b, sb, alpha=2.0 ** -10)
    for first in (0, 40000, M - 300):
        part = slice(first, first + 300)
        _check(y[part], (a[part], sa[part]), (b, sb), alpha=2.0 ** -10)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,C,pitch,off", [(130, 257, 257, 0), (300, 1001, 1001, 0), (129, 136, 136, 0), (129, 136, 137, 3), (17, 264, 300, 8), (257, 129, 136, 8),
                                           (128, 127, 128, 1), (3, 5, 5, 0)])
def test_quantiser_draws_wherever_rows_start(dev, R, C, pitch, off, dt):
    """Dropout inside the quantiser for rows on and off 16-byte boundaries: both layouts against the oracle, bit for bit."""
    from approxtorch_b200.backend import ops
    g = torch.Generator(dev).manual_seed(R + C)
    x = torch.randn(off + R * pitch + 8, generator=g, device=dev).to(dt)[off:off + R * pitch].view(R, pitch)[:, :C]
    state = torch.tensor([-5, 1 << 50], dtype=torch.int64, device=dev)
    keep = fo.keep_mask((R, C), 0.4, -5, 1 << 50)
    x64 = np.where(keep, x.double().cpu().numpy(), 0.0)
    out = ops.fp8_quantize_both(x, drop_p=0.4, rng=state)
    rows = ops.fp8_quantize_rows(x, drop_p=0.4, rng=state)
    assert all(torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)) for a, b in zip(rows, out))
    for q, s, ref in ((*out[:2], x64), (*out[2:], x64.T)):
        rq, rs = fo.quantise(ref)
        np.testing.assert_array_equal(q.contiguous().float().double().cpu().numpy(), rq)
        np.testing.assert_array_equal(np.exp2(s.contiguous().view(torch.uint8).cpu().numpy().astype(np.float64) - 127), rs)


def test_result_beyond_32_bit_offsets(dev):
    """A result of 4.6e9 elements: rows past 2^32 elements."""
    from approxtorch_b200.backend import ops
    M, N, K = 70000, 65600, 130
    a, b = _operands(dev, M, N, K, 1)
    bias = torch.randn(N, device=dev)
    y = ops.fp8_gemm(*a, *b, bias=bias)
    for part in (slice(0, 100), slice(65500, 65600), slice(M - 100, M)):
        _check(y[part], (a[0][part], a[1][part]), b, bias)


def test_one_sum_of_seconds(dev):
    """2^30 steps into one element take seconds; no wait of the kernel may run out over them.  960 ones among zeros, their
    sum exact in bf16."""
    from approxtorch_b200.backend import _C, ops
    K = (1 << 30) - 5
    a = torch.zeros((1, K + 5), dtype=torch.uint8, device=dev)
    a[0, torch.randperm(K // 997, device=dev)[:959] * 997] = 0x38
    a[0, K - 1] = 0x38
    a = a.view(E4)[:, :K]
    s = torch.full((1, -(-K // 128)), 127, dtype=torch.uint8, device=dev)
    assert ops.fp8_gemm(a, s, a, s).item() == 960.0
    status = ctypes.c_int(-1)
    assert _C.lib.atb_fp8_status(ctypes.byref(status)) == 0 and status.value == 0


def test_quantiser_beyond_32_bit_offsets(dev):
    from approxtorch_b200.backend import ops
    R, C = 36000, 65544                                    # 2.36e9 elements of bf16, rows past 2^31 elements
    x = torch.empty(R, C, dtype=torch.bfloat16, device=dev)
    for i in range(0, R, 6000):
        x[i:i + 6000].normal_()
    state = torch.tensor([31, 7], dtype=torch.int64, device=dev)
    q, s, qt, st = ops.fp8_quantize_both(x, drop_p=0.25, rng=state)
    for r in (0, 32767, R - 1):
        keep = fo.kept(np.arange(r * C, (r + 1) * C, dtype=np.uint64), 0.25, 31, 7)
        rq, rs = fo.quantise(np.where(keep, x[r].double().cpu().numpy(), 0.0)[None])
        np.testing.assert_array_equal(q[r].float().double().cpu().numpy()[None], rq)
        np.testing.assert_array_equal(np.exp2(s[r].view(torch.uint8).cpu().numpy().astype(np.float64) - 127)[None], rs)
    for c in (0, C - 1):
        keep = fo.kept(np.arange(R, dtype=np.uint64) * np.uint64(C) + np.uint64(c), 0.25, 31, 7)
        rq, rs = fo.quantise(np.where(keep, x[:, c].double().cpu().numpy(), 0.0)[None])
        np.testing.assert_array_equal(qt[c].float().double().cpu().numpy()[None], rq)
        np.testing.assert_array_equal(np.exp2(st[c].view(torch.uint8).cpu().numpy().astype(np.float64) - 127)[None], rs)


def test_many_rows_of_the_quantiser(dev):
    """More than 65535 tiles of rows."""
    from approxtorch_b200.backend import ops
    x = torch.randn(65536 * 128 + 77, 3, device=dev)
    q, s = ops.fp8_quantize_rows(x)
    for part in (slice(0, 50), slice(len(x) - 100, len(x))):
        rq, rs = fo.quantise(x[part].double().cpu().numpy())
        np.testing.assert_array_equal(q[part].float().double().cpu().numpy(), rq)
        np.testing.assert_array_equal(np.exp2(s[part].contiguous().view(torch.uint8).cpu().numpy().astype(np.float64) - 127), rs)


def _call(M, N, K, a, b, y, ldy, out_code, bias=None):
    from approxtorch_b200.backend import _C
    p = lambda t: None if t is None else t.data_ptr()        # noqa: E731
    return _C.lib.atb_fp8_gemm(p(a[0]), 5, a[0].stride(0), p(a[1]), a[1].stride(0), 1, p(b[0]), 5, b[0].stride(0), p(b[1]), b[1].stride(0), 1,
                               p(bias), 1.0, y, out_code, ldy, M, N, K, 0, None, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("M,N,K", [(5, 200, 600), (40, 33, 600), (300, 193, 300), (700, 1000, 2600)])
def test_c_entry_writes_its_rows_and_nothing_else(dev, M, N, K):
    """A pitched result inside a larger buffer: what lies around it stays."""
    from approxtorch_b200.backend import ops
    a, b = _operands(dev, M, N, K, 1)
    want = ops.fp8_gemm(*a, *b, out_dtype=torch.float32)
    for ldy, first in ((N, 0), (N + 1, 3), (-(-N // 4) * 4 + 8, 4)):
        buf = torch.full((first + M * ldy + 64,), -77.0, device=dev)
        assert _call(M, N, K, a, b, buf.data_ptr() + 4 * first, ldy, 0) == 0
        inside = torch.zeros_like(buf, dtype=torch.bool)
        rows = torch.as_strided(inside, (M, N), (ldy, 1), first)
        rows.fill_(True)
        assert torch.equal(torch.as_strided(buf, (M, N), (ldy, 1), first), want)
        assert (buf[~inside] == -77.0).all()


def test_c_quantiser_writes_its_rows_and_nothing_else(dev):
    from approxtorch_b200.backend import _C
    for R, C in ((5, 130), (130, 70), (129, 257)):
        x = torch.randn(R, C, device=dev)
        ldq, lds, ldqt, ldst = -(-C // 16) * 16 + 32, -(-C // 128) + 3, -(-R // 16) * 16 + 16, -(-R // 128) + 2
        bufs = [torch.full((n + 64,), 0xEE, dtype=torch.uint8, device=dev) for n in (R * ldq, R * lds, C * ldqt, C * ldst)]
        assert _C.lib.atb_fp8_quantize(x.data_ptr(), 0, R, C, C, 5, 1, bufs[0].data_ptr(), ldq, bufs[1].data_ptr(), lds, bufs[2].data_ptr(), ldqt,
                                       bufs[3].data_ptr(), ldst, None, 0, None, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
        for buf, rows, pitch, width in ((bufs[0], R, ldq, C), (bufs[1], R, lds, -(-C // 128)), (bufs[2], C, ldqt, R), (bufs[3], C, ldst, -(-R // 128))):
            assert (buf[rows * pitch:] == 0xEE).all()
            body = buf[:rows * pitch].view(rows, pitch)
            edge = -(-width // 16) * 16 if buf is bufs[0] or buf is bufs[2] else width        # padding to 16 bytes may be written
            tail = body[:, -(-width // 128) * 128 if buf is bufs[0] or buf is bufs[2] else edge:]
            assert (tail == 0xEE).all()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_dropout_of_inputs_that_start_anywhere(dev, dt):
    """The same elements give the same result wherever they lie, in the loop over many groups, a last group and a short one."""
    from approxtorch_b200.backend import ops
    state = torch.tensor([4, 9], dtype=torch.int64, device=dev)
    for n in (2 ** 24 + 5, 4099, 9, 8, 7, 1):
        x = torch.randn(n, device=dev).to(dt)
        want = ops.dropout(x, 0.3, state)
        for first in (1, 2, 3, 5):
            buf = torch.full((n + 8,), float("nan"), device=dev, dtype=dt)
            buf[first:first + n] = x
            assert torch.equal(ops.dropout(buf[first:first + n], 0.3, state), want)


@pytest.mark.parametrize("fmt", [torch.float8_e4m3fn, torch.float8_e5m2], ids=["e4m3", "e5m2"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,C,pitch", [(2500, 2056, 2056), (128, 128 * 301, 128 * 301), (128 * 331 - 7, 120, 136), (9000, 1000, 1024)])
def test_both_layouts_of_more_tiles_than_resident_blocks(dev, R, C, pitch, dt, fmt):
    """Blocks that go from tile to tile write what a block a tile would: equal to the two images made one at a time."""
    from approxtorch_b200.backend import _C, ops
    g = torch.Generator(dev).manual_seed(5)
    x = torch.full((R, pitch), float("nan"), device=dev, dtype=dt)[:, :C]
    x.copy_(_x(g, R, C))
    x[R // 2, C // 3], x[R - 1, C - 1], x[0, 5] = float("inf"), float("nan"), 0.0
    q, s, qt, st = ops.fp8_quantize_both(x, fmt)
    for got, want in zip((q, s, qt, st), (*ops.fp8_quantize_rows(x, fmt), *ops.fp8_quantize_rows(x.t().contiguous(), fmt))):
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
    # column sums over each 128 rows: 128 values added in fp32, off by at most 127 half steps of the magnitudes' sum
    x[R // 2, C // 3], x[R - 1, C - 1] = 1.0, 2.0
    nb, up = -(-R // 128), lambda v: -(-v // 16) * 16                        # noqa: E731
    sums = torch.full((nb * C + 16,), -7.0, device=dev)
    bufs = [torch.empty(n, dtype=torch.uint8, device=dev) for n in (R * up(C), R * up(-(-C // 128)), C * up(R), C * up(nb))]
    code = 3 if dt == torch.bfloat16 else 4
    assert _C.lib.atb_fp8_quantize(x.data_ptr(), code, R, C, pitch, 5 if fmt == E4 else 6, 1, bufs[0].data_ptr(), up(C), bufs[1].data_ptr(),
                                   up(-(-C // 128)), bufs[2].data_ptr(), up(R), bufs[3].data_ptr(), up(nb), sums.data_ptr(), 0, None,
                                   ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    xd = torch.zeros(nb * 128, C, dtype=torch.float64, device=dev)
    xd[:R] = x.double()
    xd = xd.view(nb, 128, C)
    assert (sums[nb * C:] == -7.0).all()
    assert ((sums[:nb * C].view(nb, C).double() - xd.sum(1)).abs() <= 127 * 2.0 ** -24 * xd.abs().sum(1)).all()
    want = ops.fp8_quantize_both(x, fmt)
    for buf, w in zip(bufs, want):
        rows, width = w.shape
        assert torch.equal(buf.view(rows, up(width))[:, :width], w.view(torch.uint8))


@pytest.mark.parametrize("R,C,dt", [(5, 130, torch.float32), (200, 72, torch.bfloat16), (129, 257, torch.float16), (2600, 2048, torch.bfloat16)])
def test_c_quantiser_makes_the_transposed_image_alone(dev, R, C, dt):
    from approxtorch_b200.backend import _C, ops
    x = torch.randn(R, C, device=dev).to(dt)
    want = ops.fp8_quantize_both(x)[2:]
    ldqt, ldst = -(-R // 16) * 16, -(-R // 128)
    qt = torch.empty(C, ldqt, dtype=torch.uint8, device=dev)
    st = torch.empty(C, ldst, dtype=torch.uint8, device=dev)
    code = {torch.float32: 0, torch.bfloat16: 3, torch.float16: 4}[dt]
    assert _C.lib.atb_fp8_quantize(x.data_ptr(), code, R, C, C, 5, 1, None, 0, None, 0, qt.data_ptr(), ldqt, st.data_ptr(), ldst, None, 0,
                                   None, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    assert torch.equal(qt[:, :R], want[0].view(torch.uint8)) and torch.equal(st, want[1].view(torch.uint8))


def test_linear_fp8_gradients_without_an_input_gradient(dev):
    """A first layer: the weight and bias gradients are those of a layer whose input wants one too."""
    import approxtorch_b200 as at
    for M, N, K, dt in ((140, 50, 96, torch.float32), (2560, 2048, 256, torch.bfloat16)):
        x, go = torch.randn(M, K, device=dev).to(dt), torch.randn(M, N, device=dev).to(dt)
        w, b = torch.randn(N, K, device=dev, requires_grad=True), torch.randn(N, device=dev, requires_grad=True)
        got = torch.autograd.grad(at.nn.gemm_fp8.linear_fp8(x, w, b), (w, b), go)
        want = torch.autograd.grad(at.nn.gemm_fp8.linear_fp8(x.clone().requires_grad_(True), w, b), (w, b), go)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_streams_at_once(dev):
    """Products, quantisers and dropout of two streams in flight together give what they give alone."""
    from approxtorch_b200.backend import ops
    sizes = [(1, 4096, 2048), (300, 1000, 700), (2600, 2000, 600), (40, 3000, 5000), (900, 900, 3000)]
    g = torch.Generator(dev).manual_seed(9)
    inputs = [(_x(g, M, K), _x(g, N, K)) for M, N, K in sizes]
    state = torch.tensor([1, 1], dtype=torch.int64, device=dev)

    def work(i):
        x, w = inputs[i]
        a, b = ops.fp8_quantize_both(x, drop_p=0.2, rng=state), ops.fp8_quantize_blocks(w)
        return (ops.fp8_gemm(*a[:2], *b[:2], out_dtype=torch.float32), ops.fp8_gemm(*a[:2], *b[:2]), ops.dropout(x, 0.3, state), a[2].view(torch.uint8))
    want = [work(i) for i in range(len(sizes))]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for rep in range(6):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                for i in range(len(sizes)) if k == 0 else reversed(range(len(sizes))):
                    got.append((i, work(i)))
    torch.cuda.synchronize()
    for i, out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def test_two_graphs_replayed_together(dev):
    from approxtorch_b200.backend import ops
    g = torch.Generator(dev).manual_seed(1)
    nets = []
    for M, N, K in ((600, 800, 900), (5, 2000, 4000)):
        x, w = _x(g, M, K), _x(g, N, K)
        ops.fp8_gemm(*ops.fp8_quantize_rows(x), *ops.fp8_quantize_blocks(w, transposed=False))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.fp8_gemm(*ops.fp8_quantize_rows(x), *ops.fp8_quantize_blocks(w, transposed=False))
        nets.append((x, w, graph, y))
    for rep in range(5):
        for x, _, _, _ in nets:
            x.normal_(generator=g)
        torch.cuda.synchronize()
        for s, (_, _, graph, _) in zip((torch.cuda.Stream(), torch.cuda.Stream()), nets):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for x, w, _, y in nets:
            assert torch.equal(y, ops.fp8_gemm(*ops.fp8_quantize_rows(x), *ops.fp8_quantize_blocks(w, transposed=False)))


def test_a_kernel_right_behind_another_sees_its_writes(dev):
    """Launches may overlap the one before; every link of a chain without a pause has to see what the last one wrote, and
    must not write where the last one still reads."""
    from approxtorch_b200.backend import ops
    g = torch.Generator(dev).manual_seed(4)
    w = ops.fp8_quantize_blocks(_x(g, 512, 512) / 16, transposed=False)
    state = torch.tensor([3, 0], dtype=torch.int64, device=dev)
    for M in (1, 130, 3000):
        x0 = _x(g, M, 512)

        def chain(wait):
            x = x0
            for i in range(12):
                taken = ops.dropout_advance(state)
                q = ops.fp8_quantize_rows(x, drop_p=0.1, rng=taken)
                wait()
                y = ops.fp8_gemm(*q, *w, out_dtype=torch.float32)
                wait()
                x = ops.dropout(y, 0.2, taken) if i % 2 else y * 1.0
                wait()
            return x
        state[1] = 0
        want = chain(torch.cuda.synchronize)
        for _ in range(4):
            state[1] = 0
            assert torch.equal(chain(lambda: None), want)


def test_linear_fp8_takes_what_autograd_hands_it(dev):
    import approxtorch_b200 as at
    lin = at.nn.gemm_fp8.linear_fp8
    g = torch.Generator(dev).manual_seed(2)
    x, w, b = _x(g, 140, 96).requires_grad_(True), _x(g, 50, 96).requires_grad_(True), torch.randn(50, device=dev, requires_grad=True)
    go = torch.randn(140, 50, device=dev)
    want = torch.autograd.grad(lin(x, w, b), (x, w, b), go)
    # strided, expanded and permuted gradients
    wide = torch.empty(140, 80, device=dev)
    wide[:, 7:57] = go
    for grad in (wide[:, 7:57], go.t().contiguous().t()):
        for got, ref in zip(torch.autograd.grad(lin(x, w, b), (x, w, b), grad), want):
            assert torch.equal(got, ref)
    sums = torch.autograd.grad(lin(x, w, b).sum(), (x, w, b))
    ones = torch.autograd.grad(lin(x, w, b), (x, w, b), torch.ones(140, 50, device=dev))
    assert all(torch.equal(p, q) for p, q in zip(sums, ones))
    # one gradient at a time
    y = lin(x, w, b)
    for i, leaf in enumerate((x, w, b)):
        got, = torch.autograd.grad(y, leaf, go, retain_graph=True)
        torch.testing.assert_close(got, want[i], rtol=2 ** -20, atol=2 ** -20 * want[i].abs().max().item())
    # leading dimensions, a single vector, half-precision parameters, no bias
    x3 = x.detach().view(7, 20, 96).requires_grad_(True)
    got = torch.autograd.grad(lin(x3, w, b), (x3, w), go.view(7, 20, 50))
    assert torch.equal(got[0].view(140, 96), want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(lin(x[3].detach(), w, b), lin(x[3:4].detach(), w, b)[0])
    wb, bb = w.detach().bfloat16().requires_grad_(True), b.detach().half().requires_grad_(True)
    xb = x.detach().bfloat16().requires_grad_(True)
    grads = torch.autograd.grad(lin(xb, wb, bb), (xb, wb, bb), go.bfloat16())
    assert [t.dtype for t in grads] == [torch.bfloat16, torch.bfloat16, torch.float16]
    assert torch.equal(lin(x, w), lin(x, w, torch.zeros(50, device=dev)))
    with torch.no_grad():
        assert not lin(x, w, b).requires_grad
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(lin(x, w, b), (x,), go, create_graph=True)
    for bad in (lambda: lin(x, w[:, :90], b), lambda: lin(x, w, b[:40]), lambda: lin(x, w, b, drop_p=0.5), lambda: lin(x.double(), w, b),
                lambda: lin(x, w.double(), b), lambda: lin(x, w.cpu(), b), lambda: lin(x, w[:0], None)):
        with pytest.raises(RuntimeError):
            bad()


def test_linear_fp8_with_everything_dropped(dev):
    """p = 1: the product is over nothing, whatever x holds; the gradients of x and W are zero."""
    import approxtorch_b200 as at
    state = torch.tensor([1, 1], dtype=torch.int64, device=dev)
    x = torch.full((150, 200), float("inf"), device=dev, requires_grad=True)
    w, b = torch.randn(70, 200, device=dev, requires_grad=True), torch.randn(70, device=dev, requires_grad=True)
    y = at.nn.gemm_fp8.linear_fp8(x, w, b, drop_p=1.0, rng=state)
    assert torch.equal(y, b.expand(150, 70))
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert (gx == 0).all() and (gw == 0).all() and (gb == 150).all()


def test_layers_recomputed_with_a_given_state(dev):
    """Activation checkpointing runs the forward twice; with the state handed in, results and gradients are those of one run."""
    import approxtorch_b200 as at
    from torch.utils.checkpoint import checkpoint
    drop, lin = at.nn.CounterDropout(0.4, seed=5).to(dev), at.nn.Linear_fp8(96, 50, dropout=0.3, seed=6).to(dev)
    x, go = torch.randn(140, 96, device=dev, requires_grad=True), torch.randn(140, 50, device=dev)
    r1, r2 = at.backend.ops.dropout_advance(drop.rng), at.backend.ops.dropout_advance(lin.rng)
    run = lambda t: lin(drop(t, r1), r2)                                     # noqa: E731
    leaves = (x, lin.weight, lin.bias)
    y = run(x)
    want = torch.autograd.grad(y, leaves, go)
    for reentrant in (False, True):
        z = checkpoint(run, x, use_reentrant=reentrant)
        assert torch.equal(z, y)
        for t in leaves:
            t.grad = None
        z.backward(go)
        assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))
    assert drop.rng.tolist() == [5, 1] and lin.rng.tolist() == [6, 1]        # a given state leaves the layer's own as it is
    with torch.autograd.graph.save_on_cpu():
        z = run(x)
    assert all(torch.equal(g, w) for g, w in zip(torch.autograd.grad(z, leaves, go), want))
    with torch.inference_mode():
        assert torch.equal(run(x), y)


def test_captured_backward_beside_an_eager_graph_is_refused(dev):
    """While a result computed on the default stream holds the leaves' gradient nodes, capturing their backward pass raises;
    once it is let go the same capture works."""
    import approxtorch_b200 as at
    state = torch.tensor([3, 0], dtype=torch.int64, device=dev)
    x, w, go = torch.randn(64, 96, device=dev), torch.randn(50, 96, device=dev, requires_grad=True), torch.randn(64, 50, device=dev)
    for run, leaf, g in ((lambda: at.nn.gemm_fp8.linear_fp8(x, w), w, go),
                         (lambda: at.nn.dropout.counter_dropout(w, 0.5, state), w, torch.randn_like(w))):
        want, = torch.autograd.grad(run(), leaf, g)
        alive = run()
        with pytest.raises(RuntimeError, match="let go of all results"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(run(), leaf, g)
        torch.cuda.synchronize()
        assert torch.equal(torch.autograd.grad(alive, leaf, g)[0], want)     # the eager one is whole
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(run(), leaf, g)
        graph.replay()
        assert torch.equal(got, want)


def test_dropout_differentiates_twice(dev):
    import approxtorch_b200 as at
    state = torch.tensor([8, 8], dtype=torch.int64, device=dev)
    x = torch.randn(300, device=dev, requires_grad=True)
    gx, = torch.autograd.grad(at.nn.dropout.counter_dropout(x, 0.5, state).square().sum(), x, create_graph=True)
    ggx, = torch.autograd.grad(gx.sum(), x)
    keep = torch.from_numpy(fo.keep_mask((300,), 0.5, 8, 8)).to(dev)
    assert torch.equal(ggx, torch.where(keep, 8.0, 0.0))      # d2/dx2 (2 x)^2 where kept


def test_small_training_run(dev):
    """A head of dropout and two 8-bit layers under SGD beside an approximate convolution: it runs, every parameter gets a
    finite gradient, the masks move on."""
    import approxtorch_b200 as at
    from oracle import lut_oracle as lo
    torch.manual_seed(0)
    lut = torch.from_numpy(lo.lut_exact_signed().reshape(-1)).float().to(dev)
    net = torch.nn.Sequential(at.nn.Conv2d_int8(3, 16, 3, lut, padding=1, bias=True), torch.nn.ReLU(), torch.nn.AdaptiveAvgPool2d(4),
                              torch.nn.Flatten(), at.nn.Linear_fp8(256, 64, dropout=0.2, seed=1), torch.nn.ReLU(),
                              at.nn.CounterDropout(0.1, seed=2), at.nn.Linear_fp8(64, 10)).to(dev)
    opt = torch.optim.SGD(net.parameters(), lr=0.01)
    x, t = torch.randn(48, 3, 12, 12, device=dev), torch.randint(0, 10, (48,), device=dev)
    for _ in range(3):
        opt.zero_grad()
        torch.nn.functional.cross_entropy(net(x), t).backward()
        for p in net.parameters():
            assert p.grad is not None and torch.isfinite(p.grad).all()
        opt.step()
    assert net[4].rng.tolist() == [1, 3] and net[6].rng.tolist() == [2, 3]

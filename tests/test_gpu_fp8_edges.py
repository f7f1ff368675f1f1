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


@pytest.mark.parametrize("code,dt", [(0, torch.float32), (3, torch.bfloat16), (4, torch.float16)])
@pytest.mark.parametrize("R,C", [(5, 130), (130, 70), (129, 257), (200, 72), (300, 1001), (2500, 2056)])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_c_quantiser_leaves_a_wider_buffer_around_its_rows(dev, R, C, block_rows, dt, code):
    """Images in column ranges of wider buffers: a row is written up to the next multiple of 16 bytes and no further."""
    import ctypes
    from approxtorch_b200.backend import _C, ops
    x = torch.randn(R, C, device=dev).to(dt)
    x[R // 2, C // 2] = float("inf")                         # a block of NaN bytes
    want = ops.fp8_quantize_both(x) if block_rows == 1 else ops.fp8_quantize_blocks(x)
    up = lambda v, to: -(-v // to) * to                      # noqa: E731
    spread = 1 if block_rows == 1 else 128
    shapes = [(R, C, 16), (-(-R // spread), -(-C // 128), 1), (C, R, 16), (-(-C // spread), -(-R // 128), 1)]
    bufs = [torch.full((rows, up(cols, 16) + 192), 0xEE, dtype=torch.uint8, device=dev) for rows, cols, _ in shapes]
    args = [v for b in bufs for v in (b.data_ptr() + 32, b.stride(0))]
    assert _C.lib.atb_fp8_quantize(x.data_ptr(), code, R, C, C, 5, block_rows, *args, None, 0, None,
                                   ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    for buf, (rows, cols, to), ref in zip(bufs, shapes, want):
        before, inside, after = buf[:, :32], buf[:, 32:32 + cols], buf[:, 32 + up(cols, to):]
        assert torch.equal(inside, ref.view(torch.uint8))
        assert before.numel() and after.shape[1] >= 160 and (before == 0xEE).all() and (after == 0xEE).all()


# forms of the product: cut over a cluster and not, whole tiles of one block and of pairs, partial sums; with and without a mask
GIVE_UP = [(1, 256, 128, 0.0), (5, 300, 700, 0.0), (5, 300, 700, 0.3), (64, 4096, 4096, 0.0), (2600, 2700, 700, 0.0), (2600, 2700, 700, 0.3),
           (129, 9000, 4200, 0.0), (1300, 1301, 3000, 0.0), (3000, 40, 40, 0.0)]


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K,p", GIVE_UP)
def test_a_product_that_gives_up_says_so(dev, M, N, K, p, out):
    """Blocks that take no look at their barriers leave NaN and an error that the next product raises; the one after it is whole."""
    import ctypes
    from approxtorch_b200.backend import _C, ops
    g = torch.Generator(dev).manual_seed(M + N)
    a, b = ops.fp8_quantize_rows(_x(g, M, K)), ops.fp8_quantize_blocks(_x(g, N, K) / 64, transposed=False)
    bias, state = torch.randn(N, device=dev), torch.tensor([1, 2], dtype=torch.int64, device=dev)
    call = lambda: ops.fp8_gemm(*a, *b, bias=bias, out_dtype=out, drop_p=p, rng=state if p else None)   # noqa: E731
    want = call()
    kept = torch.ones_like(want, dtype=torch.bool) if not p else ops.dropout(torch.ones(M, N, device=dev), p, state) != 0
    status = ctypes.c_int(-1)
    assert torch.isfinite(want).all() and _C.lib.atb_fp8_status(ctypes.byref(status)) == 0 and status.value == 0
    _C.lib.atb_fp8_patience(0)
    try:
        y = call()
        torch.cuda.synchronize()
    finally:
        _C.lib.atb_fp8_patience(-1)
    assert torch.isnan(y[kept]).all()
    with pytest.raises(RuntimeError, match="gave up waiting"):
        call()
    assert torch.equal(call(), want)
    _C.lib.atb_fp8_patience(0)
    try:
        call()
    finally:
        _C.lib.atb_fp8_patience(-1)
    for value in (1, 0):
        assert _C.lib.atb_fp8_status(ctypes.byref(status)) == 0 and status.value == value
    assert torch.equal(call(), want)


def test_a_state_that_moved_on_is_refused_in_the_backward_pass(dev):
    """The mask of the backward pass is drawn from the state that the forward pass was given: one that changed since raises, as
    every saved tensor that was changed in place does; a state handed out by dropout_advance stays as it is."""
    import approxtorch_b200 as at
    from approxtorch_b200.backend import ops
    x, w = torch.randn(40, 96, device=dev, requires_grad=True), torch.randn(50, 96, device=dev, requires_grad=True)
    for run in (lambda r: at.nn.dropout.counter_dropout(x, 0.5, r), lambda r: at.nn.gemm_fp8.linear_fp8(x, w, None, 0.5, r)):
        state = torch.tensor([3, 0], dtype=torch.int64, device=dev)
        want, = torch.autograd.grad(run(state).sum(), x)
        y = run(state)
        taken = ops.dropout_advance(state)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y.sum(), x)
        y = run(taken)
        ops.dropout_advance(state)
        assert torch.equal(torch.autograd.grad(y.sum(), x)[0], want)
    with torch.inference_mode():
        state = torch.tensor([3, 0], dtype=torch.int64, device=dev)
        assert ops.dropout_advance(state).tolist() == [3, 0]
    assert ops.dropout_advance(state).tolist() == [3, 1] and state.tolist() == [3, 2]     # an inference tensor has no version


def test_streams_that_share_a_state_take_offsets_of_their_own(dev):
    from approxtorch_b200.backend import ops
    state = torch.tensor([3, 100], dtype=torch.int64, device=dev)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(8)]
    taken = []
    for _ in range(100):
        for s in streams:
            with torch.cuda.stream(s):
                taken.append(ops.dropout_advance(state))
    torch.cuda.synchronize()
    assert state.tolist() == [3, 900]
    got = torch.stack(taken)
    assert (got[:, 0] == 3).all() and sorted(got[:, 1].tolist()) == list(range(100, 900))


def test_negative_views_are_resolved(dev):
    """Views that only note that they are negative (the imaginary part of a conjugate) count as the values they stand for, as
    inputs, weights, biases and incoming gradients; as operands and states they are refused."""
    import approxtorch_b200 as at
    from approxtorch_b200.backend import ops
    g = torch.Generator(dev).manual_seed(6)
    state = torch.tensor([3, 0], dtype=torch.int64, device=dev)
    base = torch.randn(40, 96, generator=g, device=dev)
    imag = torch.randn(40, 96, dtype=torch.complex64, generator=g, device=dev).conj().imag
    for x in (torch._neg_view(base), torch._neg_view(base.t()), imag, torch._neg_view(base.bfloat16())):
        assert x.is_neg()
        ref = torch.empty(x.shape, dtype=x.dtype, device=dev).copy_(x)
        assert not ref.is_neg() and (ref != 0).any()
        for f in (ops.fp8_quantize_rows, ops.fp8_quantize_both, ops.fp8_quantize_blocks, lambda t: (ops.dropout(t, 0.5, state),),
                  lambda t: (ops.dropout(t, 0.0, None),)):
            for got, want in zip(f(x), f(ref)):
                assert torch.equal(got.contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))
    w, b, go = (torch.randn(s, generator=g, device=dev) for s in ((50, 96), (50,), (40, 50)))
    neg = torch._neg_view
    leaves = [t.clone().requires_grad_(True) for t in (-base, -w, -b)]
    want = at.nn.gemm_fp8.linear_fp8(*leaves, 0.25, state)
    views = [t.clone().requires_grad_(True) for t in (base, w, b)]
    got = at.nn.gemm_fp8.linear_fp8(*(neg(t) for t in views), 0.25, state)
    assert torch.equal(got, want)
    for p, q in zip(torch.autograd.grad(got, views, neg(go)), torch.autograd.grad(want, leaves, go)):
        assert torch.equal(p, q)                             # two signs: of the view and of the incoming gradient
    a = ops.fp8_quantize_rows(base)
    assert torch.equal(ops.fp8_gemm(*a, *a, bias=neg(b[:40])), ops.fp8_gemm(*a, *a, bias=-b[:40]))
    assert torch.equal(ops.fp8_gemm(*a, *a, bias=neg(b[:40].half())), ops.fp8_gemm(*a, *a, bias=-b[:40].half()))
    for bad in (lambda: ops.dropout(base, 0.5, neg(state)), lambda: ops.dropout_advance(neg(state)), lambda: ops.fp8_gemm(neg(a[0]), a[1], *a),
                lambda: ops.fp8_gemm(a[0], neg(a[1].view(torch.uint8)), *a)):
        with pytest.raises(RuntimeError):
            bad()
    assert state.tolist() == [3, 0]


def test_saved_operands_that_come_back_changed_are_refused(dev):
    """Hooks for saved tensors may hand back anything: what is not the memory that was saved is refused before a launch."""
    import approxtorch_b200 as at
    state = torch.tensor([3, 0], dtype=torch.int64, device=dev)
    x, w, go = torch.randn(40, 96, device=dev, requires_grad=True), torch.randn(50, 96, device=dev, requires_grad=True), torch.randn(40, 50, device=dev)
    lin = lambda p: at.nn.gemm_fp8.linear_fp8(x, w, None, p, state)          # noqa: E731
    want = torch.autograd.grad(lin(0.3), (x, w), go)
    only = lambda size, f: lambda t: f(t) if (t.numel() == 2) == size else t                                   # noqa: E731
    for change in (only(False, lambda t: t.cpu()), only(False, lambda t: t[:-1]), only(False, lambda t: t[::2]), only(False, lambda t: t.short()),
                   only(True, lambda t: t.cpu()), only(True, lambda t: t.float()), only(True, lambda t: t[:1])):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            y = lin(0.3)
            z = at.nn.dropout.counter_dropout(x, 0.3, state)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, (x, w), go)
        if change(state) is not state:
            with pytest.raises(RuntimeError):
                torch.autograd.grad(z.sum(), x)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(dev)):
        y = lin(0.3)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, (x, w), go), want))


def _exact(a, b):
    """A B^T and |A| |B|^T in 64 bits, from the bytes of values and scales, a stretch of the reduction at a time."""
    (qa, sa), (qb, sb) = a, b
    out = [torch.zeros(qa.shape[0], qb.shape[0], dtype=torch.float64, device=qa.device) for _ in range(2)]
    part = lambda q, s, i: q[:, 128 * i:128 * (i + 512)].float().double() * torch.exp2(                        # noqa: E731
        s[:, i:i + 512].contiguous().view(torch.uint8).double() - 127).repeat_interleave(128, 1)[:, :q.shape[1] - 128 * i]
    for i in range(0, sa.shape[1], 512):
        da, db = part(qa, sa, i), part(qb, sb, i)
        out[0] += da @ db.t()
        out[1] += da.abs() @ db.abs().t()
    return out


@pytest.mark.parametrize("out,M,N,K", [(torch.float16, 8, 300, 2 ** 18), (torch.float16, 8, 300, 2 ** 20 - 77), (torch.bfloat16, 8, 300, 2 ** 20),
                                       (torch.float16, 2, 3, 2 ** 22 + 130), (torch.bfloat16, 2, 3, 2 ** 22), (torch.float16, 700, 500, 2 ** 18),
                                       (torch.bfloat16, 300, 290, 2 ** 19 + 5), (torch.float32, 8, 300, 2 ** 20)])
def test_long_sums_of_one_sign_keep_their_size(dev, out, M, N, K):
    """The accumulator cuts: an MMA adds 32 products to it, and each of the 33 may lose a unit, 2^-23 of the running sum at most.  Over
    the 32 MMAs of a partial sum that grows evenly this is 33 (1 + ... + 32) / 32 2^-23 = 545 2^-23 of it; the K / 1024 partial sums
    are added in fp32, half a unit of the running sum each; the epilogue rounds twice in fp32 and once to the result's type."""
    from approxtorch_b200.backend import ops
    g = torch.Generator(dev).manual_seed(K)
    a, b = (ops.fp8_quantize_rows(torch.randn(n, K, generator=g, device=dev).abs()) for n in (M, N))
    ref, _ = _exact(a, b)
    alpha = 2.0 ** -18
    bias = torch.rand(N, generator=g, device=dev)
    for p in (0.0, 0.5):
        state = torch.tensor([4, 2], dtype=torch.int64, device=dev)
        want = alpha * ref + bias.double()
        if p:
            want = torch.where(ops.dropout(torch.ones(M, N, device=dev), p, state) != 0, want, 0.0)
        y = ops.fp8_gemm(*a, *b, bias=bias, alpha=alpha, out_dtype=out, drop_p=p, rng=state).double()
        # evenly: quantised magnitudes of normal numbers, whose sums over 1024 steps are within a tenth of one another
        tol = 1.1 * 545 * 2.0 ** -23 + (-(-K // 1024) + 2) * 2.0 ** -24 + torch.finfo(out).eps / 2
        assert ((y - want).abs() <= tol * want.abs()).all(), ((y - want).abs() / want.abs().clamp(min=1e-30)).max().item()


def _whole_numbers(g, R, K):
    """An operand of the numbers -2 .. 2 with a scale of 1, 2, 4 or 8 for each row and slice."""
    q = torch.randint(-2, 3, (R, K), generator=g, device=g.device, dtype=torch.int8).half().to(E4)
    return q, torch.randint(127, 131, (R, -(-K // 128)), generator=g, device=g.device, dtype=torch.uint8)


# one and several blocks to a tile, pairs, partial sums of every result's type
WHOLE = [(1, 1000, 2048), (17, 700, 33000), (1, 300, 100000), (3, 200, 200000), (700, 64, 65536), (300, 500, 2049), (300, 500, 20000),
         (2600, 1500, 5000), (256, 1000, 2048), (40, 60, 300001), (520, 300, 270000)]


@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", WHOLE)
def test_every_slice_counts_once(dev, M, N, K, out):
    """Whole numbers whose magnitudes add up to less than 2^24: every order of additions is exact, so a result equals the exact one
    rounded once.  A slice left out, taken twice or scaled by the next power of two would change most of them."""
    from approxtorch_b200.backend import ops
    g = torch.Generator(dev).manual_seed(M + N + K)
    a, b = _whole_numbers(g, M, K), _whole_numbers(g, N, K)
    b[1].clamp_(max=128)
    ref, mag = _exact(a, b)
    assert mag.max() < 2 ** 24
    alpha = 2.0 ** -6 if out == torch.float16 else 1.0
    round_ = lambda v: (v * alpha).float().to(out)           # noqa: E731  (v fits fp32)
    assert torch.equal(ops.fp8_gemm(*a, *b, alpha=alpha, out_dtype=out), round_(ref))
    # what a fault of one slice would do, on the reference
    for i in (0, a[1].shape[1] // 3, a[1].shape[1] - 1):
        part = [(q[:, 128 * i:128 * (i + 1)].contiguous(), s[:, i:i + 1].contiguous()) for q, s in (a, b)]
        one = _exact(*part)[0]
        for fault in (ref - one, ref + one):                 # left out; taken twice, or twice the scale
            assert (round_(fault) != round_(ref)).float().mean() > 0.3


@pytest.mark.parametrize("M,N", [(8, 300), (512, 512)])
@pytest.mark.parametrize("K", [128, 256, 512, 1000, 1024, 1500, 2048, 4096, 8192])
def test_sums_to_fp32_lose_little(dev, M, N, K):
    """Sums of one sign.  An MMA's result is cut to 24 bits: half a unit on average, a unit being 2^-23 of the running sum at most;
    over the n = K / 32 MMAs of a sum that grows evenly n / 4 units, n 2^-25 of the result (n = 64 at most, then partial sums
    are added in fp32), and the last rounding.  The root mean square of the errors stays within that."""
    from approxtorch_b200.backend import ops
    g = torch.Generator(dev).manual_seed(K)
    a, b = (ops.fp8_quantize_rows(torch.randn(n, K, generator=g, device=dev).abs()) for n in (M, N))
    ref, _ = _exact(a, b)
    err = (ops.fp8_gemm(*a, *b, out_dtype=torch.float32).double() - ref) / ref
    n = min(-(-K // 32), 64)
    assert err.square().mean().sqrt() <= n * 2.0 ** -25 + (1 + -(-K // 1024)) * 2.0 ** -24


def test_transforms_are_refused(dev):
    """No batching rule and no forward derivative: torch refuses both instead of computing something else."""
    import approxtorch_b200 as at
    from approxtorch_b200.backend import ops
    state = torch.tensor([3, 0], dtype=torch.int64, device=dev)
    x, w = torch.randn(4, 40, 96, device=dev), torch.randn(50, 96, device=dev)
    lin, drop = at.nn.gemm_fp8.linear_fp8, at.nn.dropout.counter_dropout
    for f in (lambda t: lin(t, w), lambda t: drop(t, 0.5, state), lambda t: ops.fp8_quantize_rows(t), lambda t: ops.dropout(t, 0.5, state)):
        with pytest.raises(RuntimeError):
            torch.vmap(f)(x)
    for f in (lambda t: lin(t, w), lambda t: drop(t, 0.5, state)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x[0],), (x[1],))
        with pytest.raises(RuntimeError):
            with torch.autograd.forward_ad.dual_level():
                f(torch.autograd.forward_ad.make_dual(x[0], x[1]))


def test_tensors_without_data_are_refused(dev):
    """What a tracer hands in (shapes without memory) reaches no kernel."""
    import approxtorch_b200 as at
    from approxtorch_b200.backend import ops
    from torch._subclasses.fake_tensor import FakeTensorMode
    x, w, b = torch.randn(40, 96, device=dev), torch.randn(50, 96, device=dev), torch.randn(50, device=dev)
    state = torch.tensor([3, 0], dtype=torch.int64, device=dev)
    a, aw = ops.fp8_quantize_rows(x), ops.fp8_quantize_rows(w)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        fake = mode.from_tensor
        for call in (lambda: ops.dropout(fake(x), 0.5, state), lambda: ops.dropout(x, 0.5, fake(state)), lambda: ops.dropout_advance(fake(state)),
                     lambda: ops.fp8_quantize_rows(fake(x)), lambda: ops.fp8_quantize_both(fake(x.t())), lambda: ops.fp8_quantize_rows(x, drop_p=0.5, rng=fake(state)),
                     lambda: at.nn.gemm_fp8.linear_fp8(fake(x), w, b), lambda: at.nn.gemm_fp8.linear_fp8(x, fake(w), b),
                     lambda: at.nn.gemm_fp8.linear_fp8(x, w, fake(b)), lambda: ops.fp8_gemm(fake(a[0]), a[1], *aw), lambda: ops.fp8_gemm(a[0], fake(a[1]), *aw),
                     lambda: ops.fp8_gemm(*a, fake(aw[0]), aw[1]), lambda: ops.fp8_gemm(*a, *aw, bias=fake(b))):
            with pytest.raises(RuntimeError):
                call()


FIRST = """
import threading, torch
from approxtorch_b200.backend import ops
dev = torch.device("cuda:0")
x, w = torch.randn(130, 700, device=dev), torch.randn(300, 700, device=dev)
a, b = ops.fp8_quantize_rows(x), ops.fp8_quantize_blocks(w, transposed=False)
torch.cuda.synchronize()
{first}
torch.cuda.synchronize()
want = ops.fp8_gemm(*a, *b)
assert torch.isfinite(want).all() and len(got) > 0 and all(torch.equal(y, want) for y in got)
print("whole")
"""
CAPTURED = """
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = [ops.fp8_gemm(*a, *b)]
graph.replay()
"""
THREADS = """
got, start = [], threading.Barrier(8)
def work():
    with torch.cuda.stream(torch.cuda.Stream()):
        start.wait()
        for _ in range(20):
            got.append(ops.fp8_gemm(*a, *b))
        torch.cuda.current_stream().synchronize()
threads = [threading.Thread(target=work) for _ in range(8)]
for t in threads: t.start()
for t in threads: t.join()
assert len(got) == 160
"""


@pytest.mark.parametrize("first", [CAPTURED, THREADS], ids=["captured", "threads"])
def test_first_product_of_a_process(dev, first):
    """The first product sets up what later ones find (allowed shared memory, the error word): inside a capture, or by several host
    threads at once."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST.format(first=first)], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "whole" in done.stdout, done.stderr[-2000:]

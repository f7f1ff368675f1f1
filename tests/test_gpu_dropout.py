"""GPU parity of counter-based dropout and of the fully connected layer that folds it in."""

import numpy as np
import pytest
import torch

from oracle import fp8_oracle as fo

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _d(t):
    return t.detach().double().cpu().numpy()


def _state(dev, seed, offset):
    return torch.tensor([seed, offset], dtype=torch.int64, device=dev)


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n,p", [(1, 0.5), (7, 0.3), (8, 0.1), (1000, 0.1), (4099, 0.75), (1 << 18, 0.5), (333, 0.0), (100, 1.0), (64, 1e-9)])
def test_dropout_draws_the_defined_mask(dev, n, p, dt):
    """x f in fp32 (f = 1/(1 - rate) rounded: 2^-24, the product: 2^-24) and half a step of the type."""
    from approxtorch_b200.backend import ops
    seed, offset = 0x7EDCBA9876543210 - n, (5 << 32) + n
    x = torch.randn(n, device=dev).to(DT[dt])
    y = ops.dropout(x, p, _state(dev, seed, offset))
    keep = fo.keep_mask((n,), p, seed, offset)
    ref = np.where(keep, _d(x), 0.0) * ops.drop_factor(p)
    assert y.dtype == x.dtype
    assert ((_d(y) != 0) <= keep).all()
    half = torch.finfo(DT[dt]).eps / 2
    assert (np.abs(_d(y) - ref) <= (half + 2 * 2.0 ** -24) * (1 + 2.0 ** -20) * np.abs(ref) + float(torch.finfo(DT[dt]).tiny) * half).all()


def test_dropout_offsets_strides_and_contents(dev):
    from approxtorch_b200.backend import ops
    st = _state(dev, 9, 1)
    base = torch.randn(2, 515, 6, device=dev)
    for x in (base[:, 1:], base.transpose(0, 2), base[..., ::2], base.flatten()[1:]):
        assert torch.equal(ops.dropout(x, 0.4, st), ops.dropout(x.contiguous().clone(), 0.4, st))
    keep = torch.from_numpy(fo.keep_mask((4096,), 0.4, 9, 1)).to(dev)
    x = torch.where(keep, 1.0, float("nan"))
    assert torch.equal(ops.dropout(x, 0.4, st), torch.where(keep, ops.drop_factor(0.4), 0.0))
    x = torch.where(keep, 1.0, float("-inf"))
    assert torch.equal(ops.dropout(x, 0.4, st), torch.where(keep, ops.drop_factor(0.4), 0.0))
    assert ops.dropout(torch.zeros(0, 3, device=dev), 0.4, st).shape == (0, 3)
    for bad in (lambda: ops.dropout(base, 0.4, None), lambda: ops.dropout(base, 0.4, st.cpu()), lambda: ops.dropout(base, 0.4, st.int()),
                lambda: ops.dropout(base.double(), 0.4, st), lambda: ops.dropout(base, -0.4, st), lambda: ops.dropout_advance(st[:1])):
        with pytest.raises(RuntimeError):
            bad()


def test_dropout_beyond_32_bit_element_numbers(dev):
    """Elements past 2^32 draw from their own counters (9 GB of bf16 in and out)."""
    from approxtorch_b200.backend import ops
    n = (1 << 32) + 4100
    x = torch.ones(n, dtype=torch.bfloat16, device=dev)
    y = ops.dropout(x, 0.5, _state(dev, 5, 6))
    for first in (0, (1 << 32) - 2048, (1 << 32) + 1):
        el = np.arange(first, first + 4000, dtype=np.uint64)
        np.testing.assert_array_equal(_d(y[first:first + 4000]), np.where(fo.kept(el, 0.5, 5, 6), 2.0, 0.0))


def test_dropout_rate(dev):
    """Kept elements of n draws lie within five standard deviations of n (1 - p) (a chance of 6e-7 each)."""
    from approxtorch_b200.backend import ops
    n = 1 << 22
    for p in (0.01, 0.3, 0.5, 0.95):
        kept = int((ops.dropout(torch.ones(n, device=dev), p, _state(dev, 123, 0)) != 0).sum())
        assert abs(kept - n * (1 - p)) <= 5 * (n * p * (1 - p)) ** 0.5 + n * 2.0 ** -17


def test_dropout_layer_gradient_and_state(dev):
    import approxtorch_b200 as at
    layer = at.nn.CounterDropout(0.3, seed=21).to(dev)
    x = torch.randn(50, 33, device=dev, requires_grad=True)
    for step in range(3):
        y = layer(x)
        keep = torch.from_numpy(fo.keep_mask((50, 33), 0.3, 21, step)).to(dev)
        f = 65536 / (65536 - round(0.3 * 65536))
        assert torch.equal(y != 0, keep)
        go = torch.randn_like(x)
        gx, = torch.autograd.grad(y, x, go)
        torch.testing.assert_close(gx, torch.where(keep, go * f, 0.0), rtol=2 ** -22, atol=0)
    assert layer.rng.tolist() == [21, 3]
    saved = layer.state_dict()
    other = at.nn.CounterDropout(0.3, seed=0).to(dev)
    other.load_state_dict(saved)
    assert torch.equal(other(x), layer(x))
    # an expanded gradient
    y = layer(x)
    gx, = torch.autograd.grad(y.sum(), x)
    assert torch.equal(gx != 0, y != 0)


def test_captured_dropout_draws_anew_in_every_replay(dev):
    import approxtorch_b200 as at
    layer = at.nn.CounterDropout(0.5, seed=4).to(dev)
    x = torch.ones(4096, device=dev)
    layer(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x)
    for step in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(_d(y), np.where(fo.keep_mask((4096,), 0.5, 4, step), 2.0, 0.0))


# ---------------------------------------------------------------------------------------------------- linear_fp8
def _linear64(x, w, b, dy, keep, f):
    """(y, dx, dW, db) and for each the magnitudes that its fp32 sums run over, from the definition."""
    def held(v, rows=1):
        return fo.dequantise(*fo.quantise(v, "e4m3", rows))
    xm = np.where(keep, x, 0.0)
    xq, xt, wq, gq, gt = held(xm), held(xm.T), held(w, 128), held(dy), held(dy.T)
    y, my = f * (xq @ wq.T) + b, f * (np.abs(xq) @ np.abs(wq).T) + np.abs(b)
    dx, mx = np.where(keep, f * (gq @ wq), 0.0), f * (np.abs(gq) @ np.abs(wq))
    dw, mw = f * (gt @ xt.T), f * (np.abs(gt) @ np.abs(xt).T)
    return (y, my), (dx, mx), (dw, mw), (dy.sum(0), np.abs(dy).sum(0))


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("M,N,K", [(1, 40, 72), (3, 130, 200), (130, 260, 130), (256, 1000, 512)])
def test_linear_fp8_forward_and_gradients(dev, M, N, K, p, dt):
    """Each fp32 sum of L terms is off by at most L 2^-23 of its magnitudes, then rounded to the result's type."""
    import approxtorch_b200 as at
    torch.manual_seed(M + N + K)
    x = (torch.randn(M, K, device=dev) * torch.exp2(torch.randint(-4, 4, (M, 1), device=dev))).to(DT[dt]).requires_grad_(True)
    w = torch.randn(N, K, device=dev, requires_grad=True)
    b = torch.randn(N, device=dev, requires_grad=True)
    dy = torch.randn(M, N, device=dev).to(DT[dt])
    y = at.nn.gemm_fp8.linear_fp8(x, w, b, drop_p=p, rng=_state(dev, 1, 2))
    got = (y, *torch.autograd.grad(y, (x, w, b), dy))
    f = at.backend.ops.drop_factor(p)
    want = _linear64(_d(x), _d(w), _d(b), _d(dy), fo.keep_mask((M, K), p, 1, 2), f)
    for g, (ref, mag), terms in zip(got, want, (K, N, M, M)):
        half = torch.finfo(g.dtype).eps / 2
        tol = (terms * 2.0 ** -23 + 3 * 2.0 ** -24) * mag
        tol = tol + half * (np.abs(ref) + tol)
        assert tuple(g.shape) == ref.shape
        assert (np.abs(_d(g) - ref) <= tol).all(), (np.abs(_d(g) - ref) / np.maximum(tol, 1e-300)).max()
    assert got[0].dtype == got[1].dtype == DT[dt] and got[2].dtype == torch.float32


def test_linear_fp8_gradient_against_differences(dev):
    """Operands on a grid that e4m3 holds exactly (small integers) make the layer an ordinary product, whose gradient is
    checked against central differences of the layer itself (steps of 1 stay on the grid; every sum is an exact integer)."""
    import approxtorch_b200 as at
    rng = np.random.default_rng(0)
    t = lambda *s: torch.from_numpy(rng.integers(-3, 4, s).astype(np.float32)).to(dev)     # noqa: E731
    x, w, c = t(6, 40), t(9, 40), t(6, 9)
    st = _state(dev, 3, 3)
    loss = lambda x, w: (at.nn.gemm_fp8.linear_fp8(x, w, None, 0.5, st) * c).sum()        # noqa: E731
    x.requires_grad_(True), w.requires_grad_(True)
    gx, gw = torch.autograd.grad(loss(x, w), (x, w))
    with torch.no_grad():
        for i, j in ((0, 0), (3, 17), (5, 39), (2, 8)):
            d = torch.zeros_like(x)
            d[i, j] = 1
            assert (loss(x + d, w) - loss(x - d, w)).item() / 2 == gx[i, j].item()
            d = torch.zeros_like(w)
            d[i, j] = 1
            assert (loss(x, w + d) - loss(x, w - d)).item() / 2 == gw[i, j].item()


def test_linear_fp8_layer(dev):
    import approxtorch_b200 as at
    torch.manual_seed(0)
    layer = at.nn.Linear_fp8(96, 50, dropout=0.2, seed=8).to(dev)
    x = torch.randn(4, 7, 96, device=dev, requires_grad=True)
    y = layer(x)
    assert y.shape == (4, 7, 50) and layer.rng.tolist() == [8, 1]
    y.square().sum().backward()
    assert x.grad.shape == x.shape and layer.weight.grad.shape == (50, 96) and layer.bias.grad.shape == (50,)
    keep = torch.from_numpy(fo.keep_mask((28, 96), 0.2, 8, 0)).to(dev).view(4, 7, 96)
    assert (x.grad[~keep] == 0).all() and (x.grad[keep] != 0).any()
    layer.eval()
    with torch.no_grad():
        want = layer(x)
        layer.freeze_weight()
        assert torch.equal(layer(x), want)
        layer.weight.mul_(2)
        assert torch.equal(layer(x), want)                   # frozen: the change is not seen
        layer.load_state_dict(layer.state_dict())
        assert not torch.equal(layer(x), want)               # loading unfreezes
        layer.freeze_weight()
        layer.to(dev).unfreeze_weight()
        assert layer(x[:0].reshape(0, 96)).shape == (0, 50)
    # partial gradients and an empty batch
    layer.train().weight.requires_grad_(False)
    y = layer(x)
    y.sum().backward()
    e = torch.zeros(0, 96, device=dev, requires_grad=True)
    layer.weight.requires_grad_(True)
    layer.zero_grad()
    layer(e).sum().backward()
    assert e.grad.shape == (0, 96) and (layer.weight.grad == 0).all() and (layer.bias.grad == 0).all()


def test_linear_fp8_training_step_captured(dev):
    """Forward and backward of a two-layer head captured once and replayed: the same gradients as the eager step with the
    same state, new masks in every replay."""
    import approxtorch_b200 as at
    torch.manual_seed(1)
    net = torch.nn.Sequential(at.nn.Linear_fp8(200, 130, dropout=0.1, seed=1), torch.nn.ReLU(), at.nn.CounterDropout(0.3, seed=2),
                              at.nn.Linear_fp8(130, 40)).to(dev)
    x, go = torch.randn(150, 200, device=dev), torch.randn(150, 40, device=dev)
    params = list(net.parameters())

    def step():
        y = net(x)
        return (y, *torch.autograd.grad(y, params, go))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    before = {k: v.clone() for k, v in net.state_dict().items()}
    graph.replay()
    torch.cuda.synchronize()
    first = [t.clone() for t in out]
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(out[0], first[0])
    net.load_state_dict(before)
    for a, b in zip(step(), first):
        assert torch.equal(a.detach(), b)

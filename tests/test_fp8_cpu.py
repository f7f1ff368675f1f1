"""CPU-side checks of the 8-bit floating point operators and of counter-based dropout: the oracle against published
answers and torch's own casts, argument refusals, layer surface."""

import numpy as np
import pytest
import torch

import approxtorch_b200 as at
from approxtorch_b200.backend import _C, ops
from oracle import fp8_oracle as fo


def test_philox_oracle_gives_the_published_answers():
    """Known answers of Philox4x32-10 published with the method's reference implementation."""
    assert fo.philox4x32_10([0] * 4, [0] * 2) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert fo.philox4x32_10([0xffffffff] * 4, [0xffffffff] * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert fo.philox4x32_10([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0]) == \
        [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


def test_vectorised_draws_follow_the_scalar_ones():
    seed, offset = 0x123456789ABCDEF0, (1 << 40) + 7
    for first in (0, 5, (1 << 35) - 3):
        el = np.arange(first, first + 20, dtype=np.uint64)
        got = fo.kept(el, 0.3, seed, offset)
        for e, g in zip(el.tolist(), got.tolist()):
            w = fo.philox4x32_10([(e >> 3) & 0xFFFFFFFF, e >> 35, offset & 0xFFFFFFFF, offset >> 32], [seed & 0xFFFFFFFF, seed >> 32])
            assert g == ((w[(e & 7) >> 1] >> (16 * (e & 1))) & 0xFFFF >= round(0.3 * 65536))


@pytest.mark.parametrize("fmt,dtype", [("e4m3", torch.float8_e4m3fn), ("e5m2", torch.float8_e5m2)])
def test_oracle_rounding_agrees_with_torch_casts(fmt, dtype):
    rng = np.random.default_rng(0)
    v = (rng.standard_normal(20000) * np.exp2(rng.integers(-20, 6, 20000))).astype(np.float32)
    v = np.clip(v, -fo.FORMATS[fmt][0], fo.FORMATS[fmt][0])
    np.testing.assert_array_equal(fo.round_to_format(v.astype(np.float64), fmt), torch.from_numpy(v).to(dtype).double().numpy())


def test_refusals_before_any_launch():
    x = torch.zeros(4, 4)
    for call in (lambda: ops.fp8_quantize_rows(x), lambda: ops.fp8_quantize_both(x), lambda: ops.fp8_quantize_blocks(x),
                 lambda: ops.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64)),
                 lambda: ops.dropout_advance(torch.zeros(2, dtype=torch.int64)),
                 lambda: ops.fp8_gemm(x.to(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8),
                                      x.to(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    for bad in (-0.1, 1.1, float("nan")):
        with pytest.raises(RuntimeError, match="drop rate"):
            ops.drop_threshold(bad)
        with pytest.raises(ValueError):
            at.nn.CounterDropout(bad)
        with pytest.raises(ValueError):
            at.nn.Linear_fp8(4, 4, dropout=bad)
    assert ops.drop_factor(0.5) == 2.0 and ops.drop_factor(1.0) == 0.0 and ops.drop_threshold(1e-7) == 0
    with pytest.raises(RuntimeError):
        at.nn.Linear_fp8(4, 3)(torch.zeros(2, 5))
    with pytest.raises(RuntimeError):
        at.nn.gemm_fp8.linear_fp8(torch.zeros(2, 5), torch.zeros(3, 4))


def test_c_entries_refuse_bad_arguments():
    """Refused on the host before anything is launched (addresses are never touched)."""
    lib, p = _C.lib, 1 << 20
    q = lambda **k: lib.atb_fp8_quantize(*{**dict(x=p, dt=0, R=4, C=200, ldx=200, f8=5, br=1, q=p, ldq=208, s=p, lds=2, qt=None,   # noqa: E731
                                                  ldqt=0, st=None, ldst=0, sums=None, t=0, rng=None, stream=None), **k}.values())
    for bad in (dict(f8=3), dict(br=2), dict(R=-1), dict(ldx=100), dict(ldq=200), dict(q=p + 8), dict(lds=1), dict(x=None), dict(dt=1),
                dict(qt=p), dict(qt=p, st=p, ldqt=4, ldst=1), dict(qt=p, st=p, ldqt=16, ldst=0), dict(t=5), dict(t=70000, rng=p),
                dict(t=5, rng=p, br=128), dict(t=5, rng=p + 4), dict(sums=p), dict(sums=p, qt=p, st=p, ldqt=16, ldst=1, br=128),
                dict(sums=p, qt=p, st=p, ldqt=16, ldst=1, t=5, rng=p)):
        assert q(**bad) == 1, bad
        assert _C.last_error()
    g = lambda **k: lib.atb_fp8_gemm(*{**dict(a=p, af=5, lda=208, sa=p, ldsa=4, ar=1, b=p, bf=5, ldb=208, sb=p, ldsb=4, br=128, bias=None,   # noqa: E731
                                              alpha=1.0, y=p, yd=0, ldy=64, M=4, N=64, K=200, t=0, rng=None, stream=None), **k}.values())
    for bad in (dict(a=None), dict(af=0), dict(bf=4), dict(lda=200), dict(ldb=192), dict(a=p + 1), dict(ldsa=2), dict(ldsa=0), dict(sa=p + 2),
                dict(ar=64), dict(yd=1), dict(ldy=63), dict(M=-1), dict(y=None), dict(bias=p + 2), dict(t=9), dict(t=65537, rng=p)):
        assert g(**bad) == 1, bad
    assert lib.atb_sum_rows(p, -1, 4, p, None) == 1 and lib.atb_sum_rows(None, 1, 4, p, None) == 1 and lib.atb_sum_rows(None, 0, 0, None, None) == 0
    assert g(M=0) == 0 and g(N=0, ldy=0) == 0 and q(R=0) == 0
    d = lambda **k: lib.atb_dropout(*{**dict(x=p, y=p, dt=0, n=4, t=9, rng=p, stream=None), **k}.values())   # noqa: E731
    for bad in (dict(x=None), dict(y=None), dict(dt=2), dict(n=-1), dict(t=-1), dict(t=65537), dict(rng=None), dict(rng=p + 4)):
        assert d(**bad) == 1, bad
    assert d(n=0) == 0
    assert lib.atb_dropout_advance(None, p, None) == 1 and lib.atb_dropout_advance(p, p + 4, None) == 1


def test_c_entries_refuse_misaligned_elements():
    lib, p = _C.lib, 1 << 20
    quant = lambda x, dt: lib.atb_fp8_quantize(x, dt, 4, 200, 200, 5, 1, p, 208, p, 2, None, 0, None, 0, None, 0, None, None)   # noqa: E731
    gemm = lambda y, yd, K=200, bias=None, t=0: lib.atb_fp8_gemm(p, 5, 208, p, 4, 1, p, 5, 208, p, 4, 128, bias, 1.0, y, yd, 64, 4, 64, K, t, p, None)   # noqa: E731
    drop = lambda x, y, dt: lib.atb_dropout(x, y, dt, 4, 9, p, None)         # noqa: E731
    for code, size in ((0, 4), (3, 2), (4, 2)):
        assert quant(p + size // 2, code) == 1 and gemm(p + size // 2, code) == 1
        assert drop(p + size // 2, p, code) == 1 and drop(p, p + size // 2, code) == 1
    assert gemm(p, 0, 0, p + 2) == 1 and gemm(p, 0, 0, p, 9) == 1            # without a reduction too; a masked bias alone is refused
    for q, s, qt, st in ((None, p, p, p), (p, None, p, p), (None, None, None, None), (None, None, p, None), (None, None, None, p)):
        assert lib.atb_fp8_quantize(p, 0, 4, 200, 200, 5, 1, q, 208, s, 2, qt, 16, st, 1, None, 0, None, None) == 1
    assert lib.atb_fp8_quantize(p, 0, 4, 200, 200, 5, 128, None, 0, None, 0, p, 16, p, 1, None, 0, None, None) == 1
    assert lib.atb_sum_rows(p + 2, 2, 4, p, None) == 1 and lib.atb_sum_rows(p, 2, 4, p + 2, None) == 1


def test_layer_surface():
    layer = at.nn.Linear_fp8(12, 5, dropout=0.25, seed=3)
    assert set(layer.state_dict()) == {"weight", "bias", "rng"} and layer.rng.tolist() == [3, 0]
    ref = torch.nn.Linear(12, 5)
    plain = at.nn.Linear_fp8(12, 5)
    plain.load_state_dict(ref.state_dict())
    assert torch.equal(plain.weight, ref.weight) and torch.equal(plain.bias, ref.bias)
    assert at.nn.Linear_fp8(12, 5, bias=False).bias is None
    torch.manual_seed(0)
    a = at.nn.CounterDropout(0.5)
    torch.manual_seed(0)
    assert torch.equal(a.rng, at.nn.CounterDropout(0.5).rng)
    x = torch.randn(3)
    assert a.eval()(x) is x and at.nn.CounterDropout(0.0)(x) is x

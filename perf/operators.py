"""Cases of the 8-bit floating point operators: the block quantiser, the block-scaled matrix product with its two gradient
products, counter-based dropout, and the fully connected layer that runs them together.

Numbers are held in blocks of 128 along the reduction (or 128 x 128 for weights): a block with largest magnitude a has the
scale s = 2^e, the smallest power of two with a <= F s (F = 448 for e4m3, 57344 for e5m2; e at least -126), and holds
x / s rounded to nearest even.  Division by a power of two is exact, so quantised values are equal bit for bit however
they are computed.  Dropout draws 16 bits per element from Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011): key = seed,
counter = (element / 8, offset); an element is kept when its 16 bits are >= round(p 65536)."""

import math

import numpy as np
import torch

own = False

_OUT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_LARGEST = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}


def listed():
    return [
        # one token through a 4096 x 4096 projection, 128 x 128 weight blocks: the latency of serving
        {"name": "product_1_token", "op": "product", "m": 1, "n": 4096, "k": 4096, "b": "blocks", "out": "bf16", "bias": True, "f8": "e4m3"},
        # an odd batch of tokens through a wide projection
        {"name": "product_37_tokens", "op": "product", "m": 37, "n": 16384, "k": 4096, "b": "blocks", "out": "bf16", "bias": False, "f8": "e4m3"},
        # ragged sizes, no multiple of anything, half-precision result
        {"name": "product_ragged", "op": "product", "m": 1003, "n": 1777, "k": 2345, "b": "blocks", "out": "fp16", "bias": True, "f8": "e4m3"},
        # prefill or the forward product of a training step
        {"name": "product_8192", "op": "product", "m": 8192, "n": 8192, "k": 8192, "b": "blocks", "out": "bf16", "bias": False, "f8": "e4m3"},
        # weight gradient: both operands carry a scale per row and 128 steps, the sum over tokens stays in fp32
        {"name": "product_weight_grad", "op": "product", "m": 4096, "n": 4096, "k": 8192, "b": "rows", "out": "fp32", "bias": False, "f8": "e4m3"},
        # activations of a forward pass that keeps no transposed copy
        {"name": "quantise_rows", "op": "quantise", "rows": 8192, "cols": 8192, "form": "rows", "x": "bf16", "f8": "e4m3", "p": 0.0},
        # activations of a training step: operand and transposed operand of the weight gradient, dropout on the way
        {"name": "quantise_both_drop", "op": "quantise", "rows": 8192, "cols": 4096, "form": "both", "x": "bf16", "f8": "e4m3", "p": 0.1},
        # fp32 master weights, 128 x 128 blocks, both layouts
        {"name": "quantise_weight", "op": "quantise", "rows": 4096, "cols": 4096, "form": "blocks", "x": "fp32", "f8": "e4m3", "p": 0.0},
        # hidden activations of a training step
        {"name": "dropout_bf16", "op": "dropout", "rows": 8192, "cols": 8192, "x": "bf16", "p": 0.1},
        # odd sizes in fp32 (no row starts on a draw of eight)
        {"name": "dropout_odd", "op": "dropout", "rows": 1001, "cols": 4097, "x": "fp32", "p": 0.5},
        # the classifier of a ResNet-50 at batch 256, dropout before it: forward and all gradients
        {"name": "linear_head", "op": "linear", "m": 256, "n": 1000, "k": 2048, "x": "fp32", "p": 0.2},
        # a hidden layer of an MLP on 8192 tokens: forward and all gradients
        {"name": "linear_mlp", "op": "linear", "m": 8192, "n": 8192, "k": 2048, "x": "bf16", "p": 0.1},
    ]


def _size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["product", "product", "quantise", "dropout", "linear"])
    if op == "product":
        m, n, k = _size(rng, 1, 8192), _size(rng, 64, 16384), _size(rng, 64, 8192)
        return {"op": op, "m": m, "n": n if m * n * k <= 2 ** 39 else 8192, "k": k, "b": rng.choice(["blocks", "rows"]),
                "out": rng.choice(["bf16", "fp16", "fp32"]), "bias": rng.random() < 0.5, "f8": rng.choice(["e4m3", "e4m3", "e5m2"])}
    if op == "quantise":
        form = rng.choice(["rows", "both", "blocks"])
        return {"op": op, "rows": _size(rng, 1, 8192), "cols": _size(rng, 64, 8192), "form": form,
                "x": rng.choice(["bf16", "fp16", "fp32"]), "f8": rng.choice(["e4m3", "e4m3", "e5m2"]),
                "p": 0.0 if form == "blocks" else rng.choice([0.0, round(rng.uniform(0.05, 0.6), 3)])}
    if op == "dropout":
        return {"op": op, "rows": _size(rng, 1, 8192), "cols": _size(rng, 64, 8192), "x": rng.choice(["bf16", "fp16", "fp32"]),
                "p": round(rng.uniform(0.05, 0.6), 3)}
    return {"op": op, "m": _size(rng, 16, 8192), "n": _size(rng, 64, 8192), "k": _size(rng, 64, 2048),
            "x": rng.choice(["bf16", "fp32"]), "p": rng.choice([0.0, round(rng.uniform(0.05, 0.6), 3)])}


# ---------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, rows, cols, dtype):
    """Activations or gradients: normal, with rows of different size as they leave a network without normalisation."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    return (x * torch.exp(torch.randn(rows, 1, device="cuda", generator=g))).to(dtype)


def _held(x, block_rows, f8):
    """x as a program holds a quantised operand: values with the row pitch padded to 16 bytes, scales to 4 bytes."""
    q, s = _quantise(x, block_rows, 128, f8)
    r, c = q.shape
    data = torch.zeros(r, -(-c // 16) * 16, dtype=torch.uint8, device="cuda")
    data[:, :c] = q.view(torch.uint8)
    sr, sc = s.shape
    byte = torch.zeros(sr, -(-sc // 4) * 4, dtype=torch.uint8, device="cuda")
    byte[:, :sc] = s
    return data.view(f8)[:, :c], byte.view(torch.float8_e8m0fnu)[:, :sc]


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    rng_state = torch.tensor([seed * 7919 + 5, seed % 1000], dtype=torch.int64, device="cuda")
    if op == "product":
        f8 = _F8[case["f8"]]
        a = _held(_normal(g, case["m"], case["k"], torch.float32), 1, f8)
        w = _normal(g, case["n"], case["k"], torch.float32) / math.sqrt(case["k"])
        b = _held(w, 128 if case["b"] == "blocks" else 1, torch.float8_e4m3fn)
        bias = torch.randn(case["n"], device="cuda", generator=g) if case["bias"] else None
        return {"op": op, "a": a, "b": b, "bias": bias, "out": _OUT[case["out"]]}
    if op == "quantise":
        return {"op": op, "x": _normal(g, case["rows"], case["cols"], _OUT[case["x"]]), "form": case["form"], "f8": _F8[case["f8"]],
                "p": case["p"], "rng": rng_state}
    if op == "dropout":
        x = _normal(g, case["rows"], case["cols"], _OUT[case["x"]]).requires_grad_(True)
        return {"op": op, "x": x, "dy": _normal(g, case["rows"], case["cols"], _OUT[case["x"]]), "p": case["p"], "rng": rng_state}
    dt = _OUT[case["x"]]
    x = _normal(g, case["m"], case["k"], dt).requires_grad_(True)
    w = (torch.randn(case["n"], case["k"], device="cuda", generator=g) / math.sqrt(case["k"])).requires_grad_(True)
    bias = torch.randn(case["n"], device="cuda", generator=g).requires_grad_(True)
    dy = (_normal(g, case["m"], case["n"], torch.float32) / case["m"]).to(dt)
    return {"op": op, "x": x, "w": w, "bias": bias, "dy": dy, "p": case["p"], "rng": rng_state}


# ---------------------------------------------------------------------------------------------------- the plain form
def _quantise(x, block_rows, block_cols, f8):
    """(values [R, C] in f8, scale bytes [ceil(R / block_rows), ceil(C / block_cols)]), in 32 bits."""
    r, c = x.shape
    nr, nc = -(-r // block_rows), -(-c // block_cols)
    v = torch.nn.functional.pad(x.float(), (0, nc * block_cols - c, 0, nr * block_rows - r)).view(nr, block_rows, nc, block_cols)
    mant, exp = torch.frexp(v.abs().amax(dim=(1, 3)))                   # a = mant 2^exp, mant in [0.5, 1)
    top_mant, top_exp = math.frexp(_LARGEST[f8])
    e = (exp - top_exp + (mant > top_mant)).clamp(min=-126)
    e = torch.where(mant == 0, torch.full_like(e, -126), e).int()
    inverse = ((127 - e) << 23).view(torch.float32)                     # 2^-e, exactly
    q = (v * inverse[:, None, :, None]).view(nr * block_rows, nc * block_cols)[:r, :c]
    return q.to(f8), (e + 127).to(torch.uint8)


def _dequantise(q, s):
    block_rows = 1 if s.shape[0] == q.shape[0] else 128
    s = s.float().repeat_interleave(block_rows, 0)[:q.shape[0]].repeat_interleave(128, 1)[:, :q.shape[1]]
    return q.float() * s


def _kept(shape, p, state):
    """Truth values of the kept elements, from Philox4x32-10 on the element numbers."""
    n = math.prod(shape)
    mask32 = 0xFFFFFFFF
    group = torch.arange(-(-n // 8), dtype=torch.int64, device=state.device)
    k0, k1 = state[0] & mask32, (state[0] >> 32) & mask32
    c0, c1 = group & mask32, group >> 32
    c2, c3 = (state[1] & mask32).expand_as(group), ((state[1] >> 32) & mask32).expand_as(group)
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57                         # modulo 2^64: both halves are right
        c0, c1, c2, c3 = ((b >> 32) & mask32) ^ c1 ^ k0, b & mask32, ((a >> 32) & mask32) ^ c3 ^ k1, a & mask32
        k0, k1 = (k0 + 0x9E3779B9) & mask32, (k1 + 0xBB67AE85) & mask32
    words = torch.stack((c0, c1, c2, c3), 1)
    halves = torch.stack((words & 0xFFFF, words >> 16), 2).view(-1)[:n]
    return (halves >= round(p * 65536)).view(shape)


def _dropped(x, p, state):
    t = round(p * 65536)
    return torch.where(_kept(x.shape, p, state), x.float() * (65536.0 / (65536 - t)), 0.0).to(x.dtype)


def _plain(s):
    if s["op"] == "product":
        y = _dequantise(*s["a"]) @ _dequantise(*s["b"]).t()
        return (y if s["bias"] is None else y + s["bias"]).to(s["out"])
    if s["op"] == "quantise":
        x = s["x"] if s["p"] == 0.0 else torch.where(_kept(s["x"].shape, s["p"], s["rng"]), s["x"], 0.0)
        rows = 128 if s["form"] == "blocks" else 1
        q, e = _quantise(x, rows, 128, s["f8"])
        if s["form"] == "rows":
            return q, e.view(torch.float8_e8m0fnu)
        qt, et = _quantise(x.t().contiguous(), rows, 128, s["f8"])
        return q, e.view(torch.float8_e8m0fnu), qt, et.view(torch.float8_e8m0fnu)
    if s["op"] == "dropout":
        return _dropped(s["x"].detach(), s["p"], s["rng"]), _dropped(s["dy"], s["p"], s["rng"])
    x, w, dy, p = s["x"].detach(), s["w"].detach(), s["dy"], s["p"]
    f8, alpha = torch.float8_e4m3fn, 65536.0 / (65536 - round(p * 65536))
    kept = _kept(x.shape, p, s["rng"])
    xm = torch.where(kept, x, 0.0)

    def held(v, rows):
        q, e = _quantise(v, rows, 128, f8)
        return _dequantise(q, e.view(torch.float8_e8m0fnu))

    wq = held(w, 128)
    y = alpha * (held(xm, 1) @ wq.t()) + s["bias"].detach()
    dx = torch.where(kept, alpha * (held(dy, 1) @ wq), 0.0)
    dw = alpha * (held(dy.t().contiguous(), 1) @ held(xm.t().contiguous(), 1).t())
    return y.to(x.dtype), dx.to(x.dtype), dw, dy.float().sum(0)


# ---------------------------------------------------------------------------------------------------- the framework's calls
def _calls(s):
    import approxtorch_b200 as at
    ops = at.backend.ops
    if s["op"] == "product":
        return ops.fp8_gemm(*s["a"], *s["b"], bias=s["bias"], out_dtype=s["out"])
    if s["op"] == "quantise":
        if s["form"] == "rows":
            return ops.fp8_quantize_rows(s["x"], s["f8"], drop_p=s["p"], rng=s["rng"])
        if s["form"] == "blocks":
            return ops.fp8_quantize_blocks(s["x"], s["f8"])
        return ops.fp8_quantize_both(s["x"], s["f8"], drop_p=s["p"], rng=s["rng"])
    if s["op"] == "dropout":
        y = at.nn.dropout.counter_dropout(s["x"], s["p"], s["rng"])
        return y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]
    y = at.nn.gemm_fp8.linear_fp8(s["x"], s["w"], s["bias"], drop_p=s["p"], rng=s["rng"])
    return (y.detach(), *torch.autograd.grad(y, (s["x"], s["w"], s["bias"]), s["dy"]))


def run(state):
    return _calls(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        scales = (m + (n if case["b"] == "rows" else -(-n // 128))) * -(-k // 128)
        return {"bytes": m * k + n * k + scales + m * n * size[case["out"]] + (4 * n if case["bias"] else 0), "flops": 2.0 * m * n * k}
    if case["op"] == "quantise":
        r, c = case["rows"], case["cols"]
        br, bc = -(-r // 128), -(-c // 128)
        scales = {"rows": r * bc, "both": r * bc + c * br, "blocks": 2 * br * bc}[case["form"]]
        return {"bytes": r * c * (size[case["x"]] + (1 if case["form"] == "rows" else 2)) + scales, "flops": 0.0}
    if case["op"] == "dropout":
        return {"bytes": 4.0 * case["rows"] * case["cols"] * size[case["x"]], "flops": 0.0}
    m, n, k, e = case["m"], case["n"], case["k"], size[case["x"]]
    return {"bytes": 2.0 * e * (m * k + m * n) + 8.0 * n * k + 8.0 * n, "flops": 6.0 * m * n * k}


# ---------------------------------------------------------------------------------------------------- the definition in 64 bits
def _values(data):
    """The numbers that bytes of e4m3 or e5m2 stand for, from their bits."""
    mbits = 3 if data.dtype == torch.float8_e4m3fn else 2
    bias = 7 if mbits == 3 else 15
    b = data.view(torch.uint8).to(torch.int64)
    e, f = (b >> mbits) & (15 if mbits == 3 else 31), (b & ((1 << mbits) - 1)).double()
    mag = torch.where(e == 0, torch.ldexp(f, torch.tensor(1 - bias - mbits, device=b.device)),
                      torch.ldexp(f + (1 << mbits), e - bias - mbits))
    return torch.where(b >= 128, -mag, mag)


def _operand64(held):
    data, scale = held
    r, c = data.shape
    s = torch.ldexp(torch.ones(scale.shape, dtype=torch.float64, device=data.device), scale.view(torch.uint8).to(torch.int64) - 127)
    row = torch.arange(r, device=data.device) // (1 if scale.shape[0] == r else 128)
    return _values(data) * s[row][:, torch.arange(c, device=data.device) // 128]


def _rounded64(x, by_rows, f8):
    """(x / s rounded to the type's grid, s for each block), both in 64 bits; blocks of by_rows x 128."""
    r, c = x.shape
    br, bc = -(-r // by_rows), -(-c // 128)
    full = torch.zeros(br * by_rows, bc * 128, dtype=torch.float64, device=x.device)
    full[:r, :c] = x
    a = full.abs().reshape(br, by_rows, bc * 128).amax(1).reshape(br, bc, 128).amax(2)
    largest = _LARGEST[f8]
    e = torch.ceil(torch.log2(torch.clamp(a, min=1e-300) / largest))
    e = torch.where(a > largest * torch.exp2(e), e + 1, torch.where(a <= largest * torch.exp2(e - 1), e - 1, e)).clamp(min=-126)
    s = torch.exp2(e)
    v = full / s.repeat_interleave(by_rows, 0).repeat_interleave(128, 1)
    mbits, least = (3, -6) if f8 == torch.float8_e4m3fn else (2, -14)
    place = torch.floor(torch.log2(torch.clamp(v.abs(), min=2.0 ** least))).clamp(min=least)
    unit = torch.exp2(place - mbits)
    return (torch.round(v / unit) * unit)[:r, :c], s


def _times(q, s, by_rows):
    r, c = q.shape
    return q * s.repeat_interleave(by_rows, 0).repeat_interleave(128, 1)[:r, :c]


def _kept64(shape, p, state):
    seed, offset = (int(v) & (2 ** 64 - 1) for v in state.tolist())
    n = int(np.prod(shape))
    low = np.uint64(0xFFFFFFFF)
    i = np.arange((n + 7) // 8, dtype=np.uint64)
    x = [i & low, i >> np.uint64(32), np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p0, p1 = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(p1 >> np.uint64(32)) ^ x[1] ^ np.uint64(key[0]), p1 & low, (p0 >> np.uint64(32)) ^ x[3] ^ np.uint64(key[1]), p0 & low]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    bits = np.stack(x, axis=1).astype("<u4").reshape(-1).view("<u2")[:n]
    return torch.from_numpy(bits.astype(np.int32) >= int(np.floor(p * 65536 + 0.5))).reshape(shape).cuda()


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "product":
        y = _operand64(s["a"]) @ _operand64(s["b"]).t()
        return y if s["bias"] is None else y + s["bias"].double()
    if s["op"] == "quantise":
        x = s["x"].double()
        if s["p"]:
            x = x * _kept64(x.shape, s["p"], s["rng"]).double()
        rows = 128 if s["form"] == "blocks" else 1
        out = _rounded64(x, rows, s["f8"])
        return out if s["form"] == "rows" else (*out, *_rounded64(x.t(), rows, s["f8"]))
    keep = _kept64(s["x"].shape, s["p"], s["rng"]).double()
    factor = 1.0 / (1.0 - math.floor(s["p"] * 65536 + 0.5) / 65536)
    x, dy = s["x"].detach().double(), s["dy"].double()
    if s["op"] == "dropout":
        return x * keep * factor, dy * keep * factor
    f8 = torch.float8_e4m3fn
    w = _times(*_rounded64(s["w"].detach().double(), 128, f8), 128)
    xm, xt = (_times(*_rounded64(v, 1, f8), 1) for v in (x * keep, (x * keep).t()))
    g, gt = (_times(*_rounded64(v, 1, f8), 1) for v in (dy, dy.t()))
    return factor * (xm @ w.t()) + s["bias"].detach().double(), factor * keep * (g @ w), factor * (gt @ xt.t()), dy.sum(0)

// Python binding of the 8-bit floating point operators and of counter-based dropout: argument checks, outputs, the current
// stream, and the autograd functions, around the same C ABI that ctypes binds elsewhere.  Native because these operators
// are called where latency counts: checking and calling one from Python took 17 to 26 us, several times what the kernels
// take for one token or a small head, and a layer's forward and backward 300 us.
#include <ATen/cuda/CUDAContextLight.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>
#include <tuple>

#include "../../../include/approxtorch_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

constexpr auto kScale = at::kFloat8_e8m0fnu;

int float_code(at::ScalarType t)
{
    return t == at::kFloat ? ATB_F32 : t == at::kBFloat16 ? ATB_BF16 : t == at::kHalf ? ATB_F16 : -1;
}
int f8_code(at::ScalarType t) { return t == at::kFloat8_e4m3fn ? ATB_E4M3 : t == at::kFloat8_e5m2 ? ATB_E5M2 : -1; }

void check_status(int status, const char* what)
{
    TORCH_CHECK(status == ATB_OK, what, ": ", atb_last_error(), " (status ", status, ")");
}

// the device of the operands made current, and its current stream
struct On {
    c10::cuda::OptionalCUDAGuard guard;
    void* stream;
    explicit On(const Tensor& t)
    {
        if (t.device().index() != c10::cuda::current_device()) guard.set_device(t.device());
        stream = c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
    }
};

// an uninitialised contiguous tensor on the device of `like` (without the dispatcher: half the time of at::empty)
Tensor fresh(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor& like)
{
    return Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt));
}

// A tensor whose memory holds its values: a view that only notes that it is negative (the imaginary part of a conjugate) is what
// the dispatcher resolves on the way to a kernel, and these operators are called beside it.
Tensor in_memory(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// The gradient node of a leaf belongs to the stream on which an operator first asked for it, for as long as a result of that
// operator lives.  Where that is the default stream and a backward pass is being captured, the engine would make the default
// stream wait for the captured one, which CUDA refuses at a point where an exception ends the process: refused here, before.
void check_captured_backward()
{
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
    const auto node = torch::autograd::get_current_node();
    for (size_t i = 0; node && i < node->num_outputs(); ++i) {
        const auto& next = node->next_edge(i).function;
        if (!next || !node->task_should_compute_output(i)) continue;
        const auto stream = next->stream();
        TORCH_CHECK(!stream || *stream != c10::cuda::getDefaultCUDAStream(stream->device_index()).unwrap(),
                    "a captured backward pass reaches a gradient node of the default stream: let go of all results that were computed from "
                    "the same tensors outside the capture (or compute them on a side stream)");
    }
}

// ---- dropout -------------------------------------------------------------------------------------------------------
int drop_threshold(double p)
{
    TORCH_CHECK(p >= 0.0 && p <= 1.0, "the drop rate must lie in [0, 1], got ", p);
    return static_cast<int>(std::nearbyint(p * 65536));
}

double drop_factor(double p)
{
    const int t = drop_threshold(p);
    return t == 65536 ? 0.0 : 65536.0 / (65536 - t);
}

const void* drop_state(int threshold, const std::optional<Tensor>& rng, const c10::Device& device)
{
    if (threshold == 0) return nullptr;
    TORCH_CHECK(rng.has_value() && rng->scalar_type() == at::kLong && rng->numel() == 2 && rng->is_contiguous() && !rng->is_neg() && rng->device() == device,
                "rng must be a contiguous int64 tensor {seed, offset} on the input's device");
    return rng->const_data_ptr();
}

Tensor dropout(const Tensor& x, double p, const std::optional<Tensor>& rng)
{
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    const int code = float_code(x.scalar_type()), threshold = drop_threshold(p);
    TORCH_CHECK(code >= 0, "x must be float32, bfloat16 or float16");
    const void* state = drop_state(threshold, rng, x.device());
    const Tensor xc = in_memory(x).contiguous();
    if (threshold == 0) return xc.clone();
    Tensor y = fresh(xc.sizes(), xc.scalar_type(), xc);
    if (y.numel()) {
        const On on(x);
        check_status(atb_dropout(xc.const_data_ptr(), y.mutable_data_ptr(), code, xc.numel(), threshold, state, on.stream), "atb_dropout");
    }
    return y;
}

Tensor dropout_advance(const Tensor& rng)
{
    TORCH_CHECK(rng.is_cuda(), "rng must be a CUDA tensor");
    TORCH_CHECK(rng.scalar_type() == at::kLong && rng.numel() == 2 && rng.is_contiguous() && !rng.is_neg(), "rng must be a contiguous int64 tensor {seed, offset}");
    Tensor taken = fresh({2}, at::kLong, rng);
    const On on(rng);
    check_status(atb_dropout_advance(rng.mutable_data_ptr(), taken.mutable_data_ptr(), on.stream), "atb_dropout_advance");
    // a change in place: a graph that saved `rng` itself refuses its backward pass instead of drawing another mask
    if (!rng.is_inference()) rng.unsafeGetTensorImpl()->bump_version();
    return taken;
}

// y = dropout(x): linear in x, so its gradient is the same function of the incoming gradient (any number of times)
struct CounterDropout : torch::autograd::Function<CounterDropout> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, const std::optional<Tensor>& rng)
    {
        ctx->saved_data["p"] = p;
        ctx->save_for_backward({rng.value_or(Tensor())});
        return dropout(x, p, rng);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        check_captured_backward();
        const Tensor rng = ctx->get_saved_variables()[0];
        const double p = ctx->saved_data["p"].toDouble();
        return {CounterDropout::apply(grads[0], p, rng.defined() ? std::optional<Tensor>(rng) : std::nullopt), Tensor(), Tensor()};
    }
};

Tensor counter_dropout(const Tensor& x, double p, const std::optional<Tensor>& rng) { return CounterDropout::apply(x, p, rng); }

// ---- quantiser -----------------------------------------------------------------------------------------------------
// Where a quantised matrix lies: values [R, C] with a pitch of whole 16 bytes, scales likewise.
struct Held {
    uint8_t* q = nullptr;
    uint8_t* s = nullptr;
    int64_t R = 0, C = 0, ldq = 0, lds = 0;
    int block_rows = 1;
    Held() = default;
    Held(int64_t R_, int64_t C_, int rows) : R(R_), C(C_), ldq(up(C_, 16)), lds(up((C_ + 127) / 128, 16)), block_rows(rows) {}
    int64_t scale_rows() const { return block_rows == 1 ? R : (R + 127) / 128; }
    int64_t bytes() const { return up(R * ldq, 256) + up(scale_rows() * lds, 256); }
    uint8_t* place(uint8_t* at)
    {
        q = at;
        s = at + up(R * ldq, 256);
        return at + bytes();
    }
};

// rows that the kernel can read as they lie, or a copy
Tensor quantiser_input(const Tensor& given, const char* name = "x")
{
    const Tensor x = in_memory(given);
    TORCH_CHECK(x.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(float_code(x.scalar_type()) >= 0, name, " must be float32, bfloat16 or float16");
    TORCH_CHECK(x.dim() == 2, name, " must have shape [R, C]");
    const int64_t R = x.size(0), C = x.size(1);
    return (C == 1 || x.stride(1) == 1) && (R == 1 || x.stride(0) >= C) ? x : x.contiguous();
}

void quantise(const Tensor& x, int f8, const Held& h, const Held* t, float* sums, int threshold, const void* state, void* stream)
{
    const int64_t R = x.size(0), C = x.size(1);
    if (R == 0 || C == 0) return;
    check_status(atb_fp8_quantize(x.const_data_ptr(), float_code(x.scalar_type()), R, C, R > 1 ? x.stride(0) : C, f8, h.block_rows, h.q, h.ldq,
                                  h.s, h.lds, t ? t->q : nullptr, t ? t->ldq : 0, t ? t->s : nullptr, t ? t->lds : 0, sums, threshold, state, stream),
                 "atb_fp8_quantize");
}

// [rows, cols] of a 1-byte type with a pitch of whole 16 bytes
Tensor padded(int64_t rows, int64_t cols, at::ScalarType dtype, const Tensor& like)
{
    Tensor t = fresh({rows, up(cols, 16)}, dtype, like);
    if (cols % 16) t.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef({rows, cols}), at::IntArrayRef({up(cols, 16), 1}));
    return t;
}

std::vector<Tensor> fp8_quantize(const Tensor& x_in, at::ScalarType dtype, int block_rows, bool transposed, double drop_p,
                                 const std::optional<Tensor>& rng)
{
    const Tensor x = quantiser_input(x_in);
    const int f8 = f8_code(dtype), threshold = drop_threshold(drop_p);
    TORCH_CHECK(f8 >= 0, "dtype must be torch.float8_e4m3fn or torch.float8_e5m2");
    const void* state = drop_state(threshold, rng, x.device());
    const int64_t R = x.size(0), C = x.size(1);
    auto make = [&](Held& h) -> std::pair<Tensor, Tensor> {
        Tensor q = padded(h.R, h.C, dtype, x), s = padded(h.scale_rows(), (h.C + 127) / 128, kScale, x);
        h.q = static_cast<uint8_t*>(q.mutable_data_ptr());
        h.s = static_cast<uint8_t*>(s.mutable_data_ptr());
        return {q, s};
    };
    Held h(R, C, block_rows), t(C, R, block_rows);
    auto [q, s] = make(h);
    std::vector<Tensor> out{q, s};
    if (transposed) {
        auto [qt, st] = make(t);
        out.push_back(qt);
        out.push_back(st);
    }
    const On on(x);
    quantise(x, f8, h, transposed ? &t : nullptr, nullptr, threshold, state, on.stream);
    return out;
}

// ---- product -------------------------------------------------------------------------------------------------------
struct Operand {
    Tensor values, scales;      // what keeps the memory
    Held at;
    int f8;
};

// whether every row of t can be read up to `width` bytes
bool room(const Tensor& t, int64_t pitch, int64_t width)
{
    return static_cast<int64_t>(t.storage().nbytes()) >= t.storage_offset() + (t.size(0) - 1) * pitch + width;
}

Tensor repacked(const Tensor& t)
{
    Tensor out = padded(t.size(0), t.size(1), t.scalar_type(), t);
    out.view(at::kByte).copy_(t.view(at::kByte));
    return out;
}

// an operand as the kernels read it; copies only what lies otherwise
Operand operand(const Tensor& t, const Tensor& scale, const char* name)
{
    TORCH_CHECK(t.is_cuda() && scale.is_cuda(), name, " and ", name, "_scale must be CUDA tensors");
    Operand o{t, scale, Held(), f8_code(t.scalar_type())};
    TORCH_CHECK(o.f8 >= 0, name, " must be torch.float8_e4m3fn or torch.float8_e5m2");
    TORCH_CHECK(scale.scalar_type() == kScale || scale.scalar_type() == at::kByte, name, "_scale must be torch.float8_e8m0fnu (or its bytes)");
    TORCH_CHECK(t.dim() == 2 && scale.dim() == 2, name, " and ", name, "_scale must have two dimensions");
    TORCH_CHECK(scale.device() == t.device(), name, " and ", name, "_scale must be on one device");
    TORCH_CHECK(!t.is_neg() && !scale.is_neg(), name, " and ", name, "_scale must not be negative views");
    Held& h = o.at;
    h.R = t.size(0);
    h.C = t.size(1);
    const int64_t nb = (h.C + 127) / 128, rows = scale.size(0);
    TORCH_CHECK(scale.size(1) == nb && (rows == h.R || rows == (h.R + 127) / 128), name, "_scale must have shape [", h.R, " or ",
                (h.R + 127) / 128, ", ", nb, "], got ", scale.sizes());
    h.block_rows = rows == h.R ? 1 : 128;
    if (h.R == 0 || h.C == 0) return o;
    TORCH_CHECK(t.const_data_ptr() != nullptr && scale.const_data_ptr() != nullptr, name, " and ", name, "_scale must hold data");
    h.ldq = h.R > 1 ? t.stride(0) : up(h.C, 16);
    if ((h.C > 1 && t.stride(1) != 1) || h.ldq % 16 || h.ldq < h.C || reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16) {
        o.values = repacked(t);
        h.ldq = up(h.C, 16);
    }
    // the kernels read words of the scales, or 16 bytes at a time where base and pitch allow it
    const uintptr_t base = reinterpret_cast<uintptr_t>(scale.const_data_ptr());
    h.lds = rows > 1 ? scale.stride(0) : up(nb, 4);
    const int64_t width = up(nb, h.lds % 16 == 0 && base % 16 == 0 ? 16 : 4);
    if ((nb > 1 && scale.stride(1) != 1) || h.lds % 4 || h.lds < nb || base % 4 || (width > nb && !room(scale, h.lds, width))) {
        o.scales = repacked(scale);
        h.lds = up(nb, 16);
    }
    h.q = static_cast<uint8_t*>(const_cast<void*>(o.values.const_data_ptr()));
    h.s = static_cast<uint8_t*>(const_cast<void*>(o.scales.const_data_ptr()));
    return o;
}

void product(const Held& a, int a_f8, const Held& b, int b_f8, const float* bias, double alpha, Tensor& y, int threshold, const void* state,
             void* stream)
{
    const int64_t M = a.R, N = b.R, K = a.C;
    if (M == 0 || N == 0) return;
    check_status(atb_fp8_gemm(a.q, a_f8, a.ldq, a.s, a.lds, a.block_rows, b.q, b_f8, b.ldq, b.s, b.lds, b.block_rows, bias,
                              static_cast<float>(alpha), y.mutable_data_ptr(), float_code(y.scalar_type()), N, static_cast<int>(M),
                              static_cast<int>(N), static_cast<int>(K), threshold, state, stream),
                 "atb_fp8_gemm");
}

// fp32, contiguous, on the device; undefined without one
Tensor bias_vector(const std::optional<Tensor>& bias, int64_t N, const c10::Device& device)
{
    if (!bias.has_value() || !bias->defined()) return Tensor();
    TORCH_CHECK(bias->device() == device && bias->dim() == 1 && bias->size(0) == N && float_code(bias->scalar_type()) >= 0,
                "bias must be a float tensor of ", N, " elements on the operands' device");
    Tensor b = in_memory(bias->detach().to(at::kFloat)).contiguous();
    TORCH_CHECK(N == 0 || b.const_data_ptr() != nullptr, "bias holds no data");          // (a null pointer means none)
    return b;
}
const float* bias_pointer(const Tensor& bias) { return bias.defined() ? bias.const_data_ptr<float>() : nullptr; }

Tensor fp8_gemm(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale, const std::optional<Tensor>& bias, double alpha,
                at::ScalarType out_dtype, double drop_p, const std::optional<Tensor>& rng)
{
    TORCH_CHECK(float_code(out_dtype) >= 0, "out_dtype must be float32, bfloat16 or float16");
    TORCH_CHECK(a.is_cuda() && b.is_cuda(), "a and b must be CUDA tensors");
    TORCH_CHECK(a.device() == b.device(), "a and b must be on one device");
    const On on(a);                                          // before the operands: a repacking copy runs on this stream
    const Operand l = operand(a, a_scale, "a"), r = operand(b, b_scale, "b");
    TORCH_CHECK(l.at.C == r.at.C, "a.size(1) must equal b.size(1), got ", l.at.C, " vs ", r.at.C);
    TORCH_CHECK(std::max({l.at.R, r.at.R, l.at.C}) <= 0x7FFFF000, "dimension too large");
    const Tensor bias32 = bias_vector(bias, r.at.R, a.device());
    const int threshold = drop_threshold(drop_p);
    const void* state = drop_state(threshold, rng, a.device());
    Tensor y = fresh({l.at.R, r.at.R}, out_dtype, a);
    product(l.at, l.f8, r.at, r.f8, bias_pointer(bias32), alpha, y, threshold, state, on.stream);
    return y;
}

// ---- fully connected layer -----------------------------------------------------------------------------------------
//   y = f q(m x) q(W)^T + b,  dx = m f q(dy) q(W),  dW = f q(dy^T) q((m x)^T)^T,  db = sum of dy
// m, f: dropout's mask and factor; the mask goes into the quantiser and the store of dx, the factor is the products' alpha.
struct LinearFp8 : torch::autograd::Function<LinearFp8> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias, double p,
                          const std::optional<Tensor>& rng, bool need_x, bool need_w)
    {
        const Tensor x2 = quantiser_input(x.reshape({-1, x.size(-1)})), w = quantiser_input(weight, "weight");
        TORCH_CHECK(w.device() == x2.device(), "x and weight must be on one device");
        const int64_t M = x2.size(0), N = w.size(0), K = w.size(1);
        TORCH_CHECK(std::max({M, N, K}) <= 0x7FFFF000, "dimension too large");
        const Tensor bias32 = bias_vector(bias, N, x2.device());
        const int threshold = drop_threshold(p);
        const void* state = drop_state(threshold, rng, x2.device());
        const On on(x2);
        // operands in one allocation, what the backward pass reads in another
        Held xq(M, K, 1), wq(N, K, 128), xt(K, M, 1), wt(K, N, 128);
        Tensor scratch = fresh({xq.bytes() + wq.bytes()}, at::kByte, x2), kept;
        wq.place(xq.place(scratch.mutable_data_ptr<uint8_t>()));
        if (need_x || need_w) {
            kept = fresh({(need_w ? xt.bytes() : 0) + (need_x ? wt.bytes() : 0)}, at::kByte, x2);
            uint8_t* at = kept.mutable_data_ptr<uint8_t>();
            if (need_w) at = xt.place(at);
            if (need_x) wt.place(at);
        }
        quantise(x2, ATB_E4M3, xq, need_w ? &xt : nullptr, nullptr, threshold, state, on.stream);
        quantise(w, ATB_E4M3, wq, need_x ? &wt : nullptr, nullptr, 0, nullptr, on.stream);
        std::vector<int64_t> shape = x.sizes().vec();
        shape.back() = N;
        Tensor y = fresh(shape, x2.scalar_type(), x2);
        product(xq, ATB_E4M3, wq, ATB_E4M3, bias_pointer(bias32), drop_factor(p), y, 0, nullptr, on.stream);
        if (need_x || need_w || (bias.has_value() && bias->defined())) {
            ctx->save_for_backward({kept, threshold ? *rng : Tensor()});
            ctx->saved_data["p"] = p;
            ctx->saved_data["need"] = static_cast<int64_t>(need_x) | static_cast<int64_t>(need_w) << 1;
            ctx->saved_data["x_shape"] = x.sizes().vec();
            ctx->saved_data["N"] = N;
            ctx->saved_data["w_type"] = static_cast<int64_t>(weight.scalar_type());
            ctx->saved_data["b_type"] = bias.has_value() && bias->defined() ? static_cast<int64_t>(bias->scalar_type()) : int64_t(-1);
        }
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        TORCH_CHECK(!at::GradMode::is_enabled(), "linear_fp8 has no second derivative (create_graph=True)");
        check_captured_backward();
        const auto saved = ctx->get_saved_variables();
        const Tensor kept = saved[0], rng = saved[1];
        const double p = ctx->saved_data["p"].toDouble();
        const std::vector<int64_t> x_shape = ctx->saved_data["x_shape"].toIntVector();
        const int64_t N = ctx->saved_data["N"].toInt(), K = x_shape.back(), need = ctx->saved_data["need"].toInt();
        // laid out: what the forward pass kept; wanted: of that, what this backward pass asks for
        const bool laid_x = need & 1, laid_w = need & 2, need_x = laid_x && ctx->needs_input_grad(0), need_w = laid_w && ctx->needs_input_grad(1);
        const Tensor go = quantiser_input(grads[0].reshape({-1, N}), "the gradient");
        const int64_t M = go.size(0);
        const int threshold = drop_threshold(p);
        const double alpha = drop_factor(p);
        const On on(go);
        Held gq(M, N, 1), gt(N, M, 1), xt(K, M, 1), wt(K, N, 128);
        const int64_t b_type = ctx->saved_data["b_type"].toInt();
        const bool need_b = b_type >= 0 && ctx->needs_input_grad(2);
        // the bias gradient comes out of the quantiser's pass over the gradient where that makes both layouts
        const int64_t sum_rows = (M + 127) / 128, sum_bytes = need_b && need_w && M ? up(sum_rows * N * 4, 256) : 0;
        Tensor scratch, dx, dw, db;
        // hooks for saved tensors may hand back anything, and the kernels would read it as device memory
        TORCH_CHECK(!threshold || (rng.defined() && drop_state(threshold, rng, go.device())), "the saved state of the dropout is missing");
        if (need_x || need_w) {
            TORCH_CHECK(kept.defined() && kept.device() == go.device() && kept.scalar_type() == at::kByte && kept.is_contiguous() &&
                            kept.numel() == (laid_w ? xt.bytes() : 0) + (laid_x ? wt.bytes() : 0),
                        "the saved operands of linear_fp8 came back on another device or in another form");
            uint8_t* at = kept.mutable_data_ptr<uint8_t>();
            if (laid_w) at = xt.place(at);
            if (laid_x) wt.place(at);
            scratch = fresh({(need_x ? gq.bytes() : 0) + (need_w ? gt.bytes() : 0) + sum_bytes}, at::kByte, go);
            at = scratch.mutable_data_ptr<uint8_t>();
            if (need_x) at = gq.place(at);
            if (need_w) at = gt.place(at);
            float* sums = sum_bytes ? reinterpret_cast<float*>(at) : nullptr;
            if (sums) {
                db = fresh({N}, at::kFloat, go);
                if (sum_rows == 1) sums = db.mutable_data_ptr<float>();      // one tile of rows: nothing to add up
            }
            quantise(go, ATB_E4M3, gq, need_w ? &gt : nullptr, sums, 0, nullptr, on.stream);
            if (sums && sum_rows > 1) check_status(atb_sum_rows(sums, static_cast<int>(sum_rows), N, db.mutable_data_ptr<float>(), on.stream), "atb_sum_rows");
        }
        if (need_x) {
            dx = fresh(x_shape, go.scalar_type(), go);
            product(gq, ATB_E4M3, wt, ATB_E4M3, nullptr, alpha, dx, threshold, threshold ? rng.const_data_ptr() : nullptr, on.stream);
        }
        if (need_w) {
            dw = fresh({N, K}, static_cast<at::ScalarType>(ctx->saved_data["w_type"].toInt()), go);
            product(gt, ATB_E4M3, xt, ATB_E4M3, nullptr, alpha, dw, 0, nullptr, on.stream);
        }
        if (need_b) {
            if (!db.defined()) db = go.sum(at::IntArrayRef{0}, false, at::kFloat);
            db = db.to(static_cast<at::ScalarType>(b_type));
        }
        return {dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor linear_fp8(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias, double p, const std::optional<Tensor>& rng)
{
    TORCH_CHECK(x.dim() >= 1 && weight.dim() == 2 && x.size(-1) == weight.size(1), "expected x [..., in] and weight [out, in], got ", x.sizes(),
                " and ", weight.sizes());
    TORCH_CHECK(weight.size(0) > 0 && weight.size(1) > 0, "weight must not be empty, got ", weight.sizes());
    const bool grad = at::GradMode::is_enabled();
    return LinearFp8::apply(x, weight, bias, p, rng, grad && x.requires_grad(), grad && weight.requires_grad());
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.def("drop_threshold", torch::wrap_pybind_function(drop_threshold));
    m.def("drop_factor", torch::wrap_pybind_function(drop_factor));
    m.def("dropout", torch::wrap_pybind_function(dropout));
    m.def("dropout_advance", torch::wrap_pybind_function(dropout_advance));
    m.def("counter_dropout", torch::wrap_pybind_function(counter_dropout));
    m.def("fp8_quantize", torch::wrap_pybind_function(fp8_quantize));
    m.def("fp8_gemm", torch::wrap_pybind_function(fp8_gemm));
    m.def("linear_fp8", torch::wrap_pybind_function(linear_fp8));
}

// Dropout whose mask is drawn from a counter and never stored.
//
//   y[i] = kept(i) ? x[i] * f : 0,   f = 65536 / (65536 - t),   t = round(p * 65536)
//
// kept(i) depends on (seed, offset, i) alone, so the gradient is the same call on the incoming gradient: nothing but
// the 16-byte state is saved for the backward pass.  What is dropped is written as zero without being looked at (a NaN
// or an infinity there leaves no trace).  One read and one write of the tensor, the floor of the operation.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "philox.cuh"

namespace atb {

template <class T> __device__ __forceinline__ float drop_load(T v);
template <> __device__ __forceinline__ float drop_load<float>(float v) { return v; }
template <> __device__ __forceinline__ float drop_load<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float drop_load<__half>(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T drop_store(float v);
template <> __device__ __forceinline__ float drop_store<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 drop_store<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half drop_store<__half>(float v) { return __float2half_rn(v); }

template <class T> struct alignas(16) Eight { T v[8]; };

// ALIGNED: 16 bytes at a time; else 2-byte types as the words that hold them (the first may begin, the last end, with an element
// that is not theirs), shifted into place.  2^26 bf16 elements from an odd one on: 54 us (aligned 46), 201 element by element.
template <class T, bool ALIGNED>
__device__ __forceinline__ Eight<T> eight_load(const T* p)
{
    Eight<T> e;
    if constexpr (!ALIGNED) {
        unsigned* const w = reinterpret_cast<unsigned*>(&e);
        if constexpr (sizeof(T) == 2) {
            const unsigned odd = static_cast<unsigned>(reinterpret_cast<uintptr_t>(p)) & 2u;
            const unsigned* const q = reinterpret_cast<const unsigned*>(reinterpret_cast<uintptr_t>(p) - odd);
            unsigned v[5] = {read4(q), read4(q + 1), read4(q + 2), read4(q + 3), 0u};
            if (odd) v[4] = read4(q + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(v[i], v[i + 1], 8u * odd);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = read4(p + i);
        }
        return e;
    }
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(e) / 16); ++i) reinterpret_cast<uint4*>(&e)[i] = read16_once(p + 16 / sizeof(T) * i);
    return e;
}

// One thread takes whole groups of 8 elements (one draw each), kAhead of them at a time, requested together.  VEC: y is 16-byte
// aligned; ALIGNED: x too.  2^26 bf16 elements: 45.9 us (a copy: 42.5 us, floor 41.0 us); 2^24 fp32: 22.4 us (a copy: 22.4 us).  Measured
// against it, 1, 2 or 4 groups ahead and 2, 3 or 4 blocks to an SM: 47 to 74 us.
template <class T, bool VEC, bool ALIGNED>
__global__ void __launch_bounds__(256, 4) dropout_kernel(const T* x, T* y, long long numel, DropState d, float factor)
{
    constexpr int kAhead = sizeof(T) == 2 ? 4 : 1;
    after_previous();
    PhiloxKey key(d.rng);
    key.settle();
    const long long whole = VEC ? numel >> 3 : 0, groups = (numel + 7) >> 3;
    const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
    long long g = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    auto finish = [&](long long at, Eight<T>& e) {
        const uint4 r = philox4x32_10(key, at);
        const uint32_t v[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned h = j & 1 ? v[j >> 1] >> 16 : v[j >> 1] & 0xFFFFu;
            e.v[j] = drop_store<T>(h >= d.threshold ? drop_load(e.v[j]) * factor : 0.0f);
        }
        uint4* dst = reinterpret_cast<uint4*>(y + (at << 3));
#pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof(e) / 16); ++j) __stcs(dst + j, reinterpret_cast<const uint4*>(&e)[j]);
    };
    for (; g + (kAhead - 1) * stride < whole; g += kAhead * stride) {
        Eight<T> e[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) e[i] = eight_load<T, ALIGNED>(x + ((g + i * stride) << 3));
#pragma unroll
        for (int i = 0; i < kAhead; ++i) finish(g + i * stride, e[i]);
    }
    for (; g < whole; g += stride) {
        Eight<T> e = eight_load<T, ALIGNED>(x + (g << 3));
        finish(g, e);
    }
    for (; g < groups; g += stride) {                        // an unaligned result, and what a last group is short of 8
        const unsigned m = philox_keep8(key, g, d.threshold);
        for (int j = 0; j < 8 && (g << 3) + j < numel; ++j)
            y[(g << 3) + j] = drop_store<T>((m >> j) & 1u ? drop_load(x[(g << 3) + j]) * factor : 0.0f);
    }
}

// state = {seed, offset}: `taken` gets the state that this call draws from, the offset moves on by one.  On the device, so that
// every replay of a captured graph draws anew; in one step, so that calls of several streams get offsets of their own.
__global__ void drop_advance_kernel(unsigned long long* state, unsigned long long* taken)
{
    after_previous();
    taken[0] = state[0];
    taken[1] = atomicAdd(state + 1, 1ull);
}

template <class T>
static void launch_dropout(const void* x, void* y, long long numel, const DropState& d, float factor, cudaStream_t s)
{
    const int grid = grid_for((numel + 7) / 8, 256, 8 * sm_count());
    const auto go = [&](void (*kernel)(const T*, T*, long long, DropState, float)) {
        launch_after(kernel, dim3(grid), dim3(256), 0, s, 0, static_cast<const T*>(x), static_cast<T*>(y), numel, d, factor);
    };
    if (!aligned_to(y, 16)) go(dropout_kernel<T, false, false>);
    else if (aligned_to(x, 16)) go(dropout_kernel<T, true, true>);
    else go(dropout_kernel<T, true, false>);
}

}  // namespace atb

using namespace atb;

extern "C" int atb_dropout(const void* x, void* y, int dtype, long long numel, int threshold, const void* rng, void* stream)
{
    ATB_REQUIRE(numel >= 0, "negative numel");
    ATB_REQUIRE(threshold >= 0 && threshold <= 65536, "threshold must lie in [0, 65536]");
    if (numel == 0) return ATB_OK;
    ATB_REQUIRE(x && y && rng, "null pointer");
    ATB_REQUIRE(aligned_to(rng, 8) && aligned_to(x, dtype == ATB_F32 ? 4 : 2) && aligned_to(y, dtype == ATB_F32 ? 4 : 2),
                "rng must be 8-byte aligned, x and y aligned to their elements");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const DropState d{static_cast<const unsigned long long*>(rng), static_cast<unsigned>(threshold)};
    const float factor = threshold == 65536 ? 0.0f : static_cast<float>(65536.0 / (65536 - threshold));
    if (dtype == ATB_F32) launch_dropout<float>(x, y, numel, d, factor, s);
    else if (dtype == ATB_BF16) launch_dropout<__nv_bfloat16>(x, y, numel, d, factor, s);
    else if (dtype == ATB_F16) launch_dropout<__half>(x, y, numel, d, factor, s);
    else return fail_invalid("dtype must be fp32, bf16 or fp16");
    return check_launch("dropout_kernel");
}

extern "C" int atb_dropout_advance(void* state, void* taken, void* stream)
{
    ATB_REQUIRE(state && taken && aligned_to(state, 8) && aligned_to(taken, 8), "state and taken must be 8-byte aligned device pointers");
    launch_after(drop_advance_kernel, dim3(1), dim3(1), 0, static_cast<cudaStream_t>(stream), 0, static_cast<unsigned long long*>(state),
                 static_cast<unsigned long long*>(taken));
    return check_launch("drop_advance_kernel");
}

// Block quantisation to 8-bit floating point with power-of-two scales.
//
// A block (128 consecutive elements of a row, or 128 x 128 for weights) with largest magnitude a gets the scale
// s = 2^e, the smallest power of two with a <= F s (F = 448 for e4m3, 57344 for e5m2; e >= -126), and holds x / s
// rounded to nearest even.  Why powers of two: a floating-point grid is the same at every power of two, so a scale with
// more digits buys at most one binade of range; dividing by one is exact (the stored value is the correctly rounded one,
// whatever computes it), and the tensor core applies it inside the product (kind::mxf8f6f4).  The scale is stored as its
// exponent byte e + 127.  A block that holds a NaN or an infinity gets the scale NaN (byte 255) and NaN in every place:
// it cannot pass unseen.
//
// The reduction over magnitudes works on the bit patterns as unsigned integers: |x| orders like its bits, infinities come
// out above every number and NaNs above them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "philox.cuh"

namespace atb {

struct QuantArgs {
    const void* x;
    long long R, C, ldx;
    uint8_t* q;       // [R, ldq]
    long long ldq;
    uint8_t* s;       // [R or ceil(R/128), lds]
    long long lds;
    uint8_t* qt;      // [C, ldqt]
    long long ldqt;
    uint8_t* st;      // [C or ceil(C/128), ldst]
    long long ldst;
    DropState drop;
};

template <class T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

// 8 consecutive elements of a row from column c on (beyond the row's end: zeros)
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ row, long long c, long long C, float (&v)[8])
{
    if (VEC && c + 8 <= C) {
        T raw[8];
        const uint4* src = reinterpret_cast<const uint4*>(row + c);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(raw) / 16); ++i) reinterpret_cast<uint4*>(raw)[i] = __ldcs(src + i);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_float(raw[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < C ? to_float(row[c + i]) : 0.0f;
    }
}

__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// scale byte of a block from its largest magnitude's bits; 448 = 1.75 * 2^8, 57344 = 1.75 * 2^15
template <bool E5>
__device__ __forceinline__ unsigned scale_byte(unsigned amax)
{
    if (amax >= 0x7F800000u) return 255u;
    const int e = static_cast<int>(amax >> 23) - (E5 ? 15 : 8) + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return static_cast<unsigned>(max(e, 1));
}
// 1 / s (exact); NaN for a block that is not finite
__device__ __forceinline__ float inverse_scale(unsigned byte)
{
    return byte == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float((254u - byte) << 23);
}

template <bool E5>
__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d)
{
    constexpr __nv_fp8_interpretation_t kind = E5 ? __NV_E5M2 : __NV_E4M3;
    const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, kind);
    const unsigned hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, kind);
    return lo | (hi << 16);
}

__device__ __forceinline__ unsigned max16(unsigned v)      // over the 16 lanes that share a block of 128
{
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}

// ---- 1 x 128 blocks along the rows, one layout ---------------------------------------------------------------------
// 16 lanes x 8 elements = one block; a block of threads takes 16 at a time.
template <class T, bool E5, bool VEC, bool DROP>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantArgs a)
{
    const long long nb = (a.C + 127) >> 7, total = a.R * nb;
    const int sub = threadIdx.x >> 4, l16 = threadIdx.x & 15;
    for (long long base = static_cast<long long>(blockIdx.x) * 16; base < total; base += static_cast<long long>(gridDim.x) * 16) {
        const long long id = base + sub;
        const bool live = id < total;
        const long long r = live ? id / nb : 0, b = live ? id - r * nb : 0, c = (b << 7) + l16 * 8;
        float v[8];
        load8<T, VEC>(static_cast<const T*>(a.x) + r * a.ldx, live ? c : a.C, a.C, v);
        if (DROP) {
            const PhiloxKey key(a.drop.rng);
            const unsigned m = philox_keep8_at(key, static_cast<unsigned long long>(r * a.C + c), a.drop.threshold);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (m >> i) & 1u ? v[i] : 0.0f;
        }
        unsigned amax = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = max(amax, magnitude(v[i]));
        amax = max16(amax);
        const unsigned byte = scale_byte<E5>(amax);
        const float inv = inverse_scale(byte);
        if (live) {
            if (c < a.ldq)
                *reinterpret_cast<uint2*>(a.q + r * a.ldq + c) =
                    make_uint2(pack4<E5>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                               pack4<E5>(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
            if (l16 == 0) a.s[r * a.lds + b] = static_cast<uint8_t>(byte);
        }
    }
}

// ---- both layouts in one pass over x ---------------------------------------------------------------------------------
// One block of threads = a 128 x 128 tile, each thread an 8 x 8 piece in registers: row maxima over 16 lanes, column
// maxima over the thread's rows and then over the tile, both images from the same registers.  SQUARE: one scale for the
// whole tile (weights) instead of one for each row and for each column.  The transposed image turns through shared
// memory so that both leave in 128-byte rows.
//
// The turned tile is 128 rows of 128 bytes; the 16-byte piece p of row c sits at place p ^ ((c >> 3) & 7), so that the
// 16 lanes that write one column piece each (rows 8 apart) spread over all banks.  (A padded pitch cannot: eight rows
// of any 16-byte multiple are a multiple of the 128-byte bank cycle.)
__device__ __forceinline__ int turn_at(int c, int byte) { return c * 128 + (byte ^ (((c >> 3) & 7) << 4)); }

template <class T, bool E5, bool VEC, bool DROP, bool SQUARE>
__global__ void __launch_bounds__(256, 2) quantize_tile_kernel(const QuantArgs a)
{
    __shared__ unsigned s_col[8][128];
    __shared__ __align__(16) uint8_t s_turn[128 * 128];
    const int warp = threadIdx.x >> 5, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const long long r0 = static_cast<long long>(blockIdx.y) * 128, c0 = static_cast<long long>(blockIdx.x) * 128;
    const long long c = c0 + tx * 8;
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long r = r0 + ty * 8 + i;
        load8<T, VEC>(static_cast<const T*>(a.x) + (r < a.R ? r : 0) * a.ldx, r < a.R ? c : a.C, a.C, v[i]);
    }
    if (DROP) {
        const PhiloxKey key(a.drop.rng);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned m = philox_keep8_at(key, static_cast<unsigned long long>((r0 + ty * 8 + i) * a.C + c), a.drop.threshold);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = (m >> j) & 1u ? v[i][j] : 0.0f;
        }
    }
    // maxima
    unsigned rowmax[8], colmax[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) colmax[j] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        rowmax[i] = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned m = magnitude(v[i][j]);
            rowmax[i] = max(rowmax[i], m);
            colmax[j] = max(colmax[j], m);
        }
    }
    unsigned rbyte[8], cbyte[8];
    if (SQUARE) {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, rowmax[i]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        if ((threadIdx.x & 31) == 0) s_col[warp][0] = m;
        __syncthreads();
        m = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) m = max(m, s_col[w][0]);
        const unsigned b = scale_byte<E5>(m);
#pragma unroll
        for (int i = 0; i < 8; ++i) { rbyte[i] = b; cbyte[i] = b; }
        if (threadIdx.x == 0) {
            a.s[blockIdx.y * a.lds + blockIdx.x] = static_cast<uint8_t>(b);
            if (a.st) a.st[blockIdx.x * a.ldst + blockIdx.y] = static_cast<uint8_t>(b);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            rbyte[i] = scale_byte<E5>(max16(rowmax[i]));
            const long long r = r0 + ty * 8 + i;
            if (tx == 0 && r < a.R) a.s[r * a.lds + blockIdx.x] = static_cast<uint8_t>(rbyte[i]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) colmax[j] = max(colmax[j], __shfl_xor_sync(0xFFFFFFFFu, colmax[j], 16));
        if ((threadIdx.x & 31) < 16) {
#pragma unroll
            for (int j = 0; j < 8; ++j) s_col[warp][tx * 8 + j] = colmax[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            unsigned m = 0;
#pragma unroll
            for (int w = 0; w < 8; ++w) m = max(m, s_col[w][tx * 8 + j]);
            cbyte[j] = scale_byte<E5>(m);
            if (ty == 0 && c + j < a.C) a.st[(c + j) * a.ldst + blockIdx.y] = static_cast<uint8_t>(cbyte[j]);
        }
    }
    // the image as it lies
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long r = r0 + ty * 8 + i;
        const float inv = inverse_scale(rbyte[i]);
        if (r < a.R && c < a.ldq)
            *reinterpret_cast<uint2*>(a.q + r * a.ldq + c) =
                make_uint2(pack4<E5>(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv),
                           pack4<E5>(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv));
    }
    if (a.qt == nullptr) return;
    // the transposed image: 8 rows of one column are 8 consecutive bytes of it
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float inv = inverse_scale(cbyte[j]);
        *reinterpret_cast<uint2*>(s_turn + turn_at(tx * 8 + j, ty * 8)) =
            make_uint2(pack4<E5>(v[0][j] * inv, v[1][j] * inv, v[2][j] * inv, v[3][j] * inv),
                       pack4<E5>(v[4][j] * inv, v[5][j] * inv, v[6][j] * inv, v[7][j] * inv));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int cc = (threadIdx.x >> 3) + 32 * i, k = (threadIdx.x & 7) * 16;
        if (c0 + cc < a.C && r0 + k < a.ldqt)
            *reinterpret_cast<uint4*>(a.qt + (c0 + cc) * a.ldqt + r0 + k) = *reinterpret_cast<const uint4*>(s_turn + turn_at(cc, k));
    }
}

template <class T, bool E5, bool VEC, bool DROP>
static int launch_quantize2(const QuantArgs& a, bool square, cudaStream_t s)
{
    if (a.qt == nullptr && !square) {
        const long long total = a.R * ((a.C + 127) >> 7);
        quantize_rows_kernel<T, E5, VEC, DROP><<<grid_for(total, 16, 16 * sm_count()), 256, 0, s>>>(a);
        return check_launch("quantize_rows_kernel");
    }
    const dim3 grid(static_cast<unsigned>((a.C + 127) >> 7), static_cast<unsigned>((a.R + 127) >> 7));
    ATB_REQUIRE((a.R + 127) >> 7 <= 65535, "too many rows");
    if (square) quantize_tile_kernel<T, E5, VEC, false, true><<<grid, 256, 0, s>>>(a);
    else quantize_tile_kernel<T, E5, VEC, DROP, false><<<grid, 256, 0, s>>>(a);
    return check_launch("quantize_tile_kernel");
}

template <class T>
static int launch_quantize(const QuantArgs& a, bool e5, bool square, cudaStream_t s)
{
    const bool vec = aligned_to(a.x, 16) && (a.ldx * static_cast<long long>(sizeof(T))) % 16 == 0;
    const bool drop = a.drop.rng != nullptr;
    if (e5) {
        if (vec) return drop ? launch_quantize2<T, true, true, true>(a, square, s) : launch_quantize2<T, true, true, false>(a, square, s);
        return drop ? launch_quantize2<T, true, false, true>(a, square, s) : launch_quantize2<T, true, false, false>(a, square, s);
    }
    if (vec) return drop ? launch_quantize2<T, false, true, true>(a, square, s) : launch_quantize2<T, false, true, false>(a, square, s);
    return drop ? launch_quantize2<T, false, false, true>(a, square, s) : launch_quantize2<T, false, false, false>(a, square, s);
}

}  // namespace atb

using namespace atb;

extern "C" int atb_fp8_quantize(const void* x, int x_dtype, long long R, long long C, long long ldx, int f8, int block_rows,
                                void* q, long long ldq, uint8_t* s, long long lds, void* qt, long long ldqt, uint8_t* st,
                                long long ldst, int drop_threshold, const void* rng, void* stream)
{
    ATB_REQUIRE(R >= 0 && C >= 0, "negative dimension");
    ATB_REQUIRE(f8 == ATB_E4M3 || f8 == ATB_E5M2, "the result must be e4m3 or e5m2");
    ATB_REQUIRE(block_rows == 1 || block_rows == 128, "block_rows must be 1 or 128");
    ATB_REQUIRE(drop_threshold >= 0 && drop_threshold <= 65536, "threshold must lie in [0, 65536]");
    if (R == 0 || C == 0) return ATB_OK;
    ATB_REQUIRE(x && q && s, "null pointer");
    ATB_REQUIRE((qt == nullptr) == (st == nullptr), "the transposed image and its scales come together");
    ATB_REQUIRE(ldx >= C || R == 1, "row pitch of x below its width");
    const long long nb = (C + 127) / 128, nbt = (R + 127) / 128;
    ATB_REQUIRE(ldq >= C && ldq % 16 == 0 && aligned_to(q, 16) && lds >= nb, "q needs 16-byte aligned rows, s a column for every block");
    if (qt) ATB_REQUIRE(ldqt >= R && ldqt % 16 == 0 && aligned_to(qt, 16) && ldst >= nbt, "qt needs 16-byte aligned rows, st a column for every block");
    ATB_REQUIRE(rng == nullptr || block_rows == 1, "dropout goes with blocks of one row");
    ATB_REQUIRE(drop_threshold == 0 || (rng != nullptr && aligned_to(rng, 8)), "dropout needs an 8-byte aligned state");
    QuantArgs a{x, R, C, ldx, static_cast<uint8_t*>(q), ldq, s, lds, static_cast<uint8_t*>(qt), ldqt, st, ldst,
                DropState{drop_threshold ? static_cast<const unsigned long long*>(rng) : nullptr, static_cast<unsigned>(drop_threshold)}};
    cudaStream_t stm = static_cast<cudaStream_t>(stream);
    const bool e5 = f8 == ATB_E5M2, square = block_rows == 128;
    if (x_dtype == ATB_F32) return launch_quantize<float>(a, e5, square, stm);
    if (x_dtype == ATB_BF16) return launch_quantize<__nv_bfloat16>(a, e5, square, stm);
    if (x_dtype == ATB_F16) return launch_quantize<__half>(a, e5, square, stm);
    return fail_invalid("x must be fp32, bf16 or fp16");
}

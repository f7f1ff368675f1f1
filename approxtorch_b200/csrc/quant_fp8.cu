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
// The reduction over magnitudes takes the maximum of absolute values as one instruction (max.xorsign.abs: the result's sign is
// the exclusive or of the operands' and is cleared at the end), a NaN winning over everything; scales are made from the bits.
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
    float* sums;      // [ceil(R/128), C]
    DropState drop;
    long long wq, wqt;       // what may be written of a row of q, qt: its width up to 16 bytes
    unsigned ct, tiles;      // tiles of 128 columns; of the matrix
};

// What a lane holds of a row: 16 bytes in the input's own type (8 bf16 or fp16, 4 fp32).  Magnitudes are compared in that
// type, two halves at a time where it has 16 bits.  Element order: word by word, low half first.
template <class T> struct Piece;
template <> struct Piece<float> {
    static constexpr int kElems = 4;
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b)
    {
        float m;
        asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(m) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
        return __float_as_uint(m);
    }
    static __device__ __forceinline__ unsigned fp32_bits(unsigned m) { return m & 0x7FFFFFFFu; }               // of a whole word's maximum
    template <int J> static __device__ __forceinline__ float get(const unsigned (&w)[4]) { return __uint_as_float(w[J]); }
};
template <> struct Piece<__nv_bfloat16> {
    static constexpr int kElems = 8;
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b)
    {
        unsigned m;
        asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
        return m;
    }
    static __device__ __forceinline__ unsigned fp32_bits(unsigned m) { return max(m << 16 & 0x7FFFFFFFu, m & 0x7FFF0000u); }   // of both halves
    template <int J> static __device__ __forceinline__ float get(const unsigned (&w)[4])
    {
        return __uint_as_float(J & 1 ? w[J / 2] & 0xFFFF0000u : w[J / 2] << 16);
    }
};
template <> struct Piece<__half> {
    static constexpr int kElems = 8;
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b)
    {
        unsigned m;
        asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
        return m;
    }
    static __device__ __forceinline__ unsigned fp32_bits(unsigned m)
    {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
        return max(__float_as_uint(f.x) & 0x7FFFFFFFu, __float_as_uint(f.y) & 0x7FFFFFFFu);
    }
    template <int J> static __device__ __forceinline__ float get(const unsigned (&w)[4])
    {
        const __half2 h = *reinterpret_cast<const __half2*>(&w[J / 2]);
        return J & 1 ? __high2float(h) : __low2float(h);
    }
};

// the 16 bytes from byte `by` (even, 0 .. 14) of lo, hi on
__device__ __forceinline__ void shifted(const uint4& lo, const uint4& hi, unsigned by, unsigned (&out)[4])
{
    unsigned w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 7; ++i) w[i] = by & 4u ? w[i + 1] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = by & 8u ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = __funnelshift_r(w[i], w[i + 1], 8u * (by & 3u));
}
__device__ __forceinline__ uint4 from_next_lane(const uint4& v)
{
    return make_uint4(__shfl_down_sync(0xFFFFFFFFu, v.x, 1), __shfl_down_sync(0xFFFFFFFFu, v.y, 1), __shfl_down_sync(0xFFFFFFFFu, v.z, 1),
                      __shfl_down_sync(0xFFFFFFFFu, v.w, 1));
}

// `left` elements from p on (zeros beyond), wherever p lies; WHOLE: there are enough.  Whole pieces of 2-byte types come as the
// words that hold them (the first may begin, the last end, with an element that is not theirs), shifted into place: 8191 x 4095
// bf16, rows 21.9 us, both layouts 31.8 us, where element by element took 28.1 and 39.1, aligned 16-byte words with any shift
// 52.6 (both), 8-byte words 20.8 and 30.9 but with draws 40.3 instead of 39.4 (rows).
template <class T, bool WHOLE>
__device__ __forceinline__ void load_piece(const T* p, long long left, unsigned (&w)[4])
{
    if constexpr (WHOLE && sizeof(T) == 2) {
        const unsigned odd = static_cast<unsigned>(reinterpret_cast<uintptr_t>(p)) & 2u;
        const unsigned* const q = reinterpret_cast<const unsigned*>(reinterpret_cast<uintptr_t>(p) - odd);
        unsigned v[5] = {q[0], q[1], q[2], q[3], 0u};        // each holds an element of the piece
        if (odd) v[4] = q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(v[i], v[i + 1], 8u * odd);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = 0;
#pragma unroll
        for (int i = 0; i < Piece<T>::kElems; ++i) {
            if (!WHOLE && i >= left) continue;
            if constexpr (Piece<T>::kElems == 4) w[i] = __float_as_uint(p[i]);
            else w[i / 2] |= static_cast<unsigned>(reinterpret_cast<const unsigned short*>(p)[i]) << (16 * (i & 1));
        }
    }
}

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

// clears what is dropped: word i of d holds the 16 bits of elements 2 i and 2 i + 1 of a group of 8
__device__ __forceinline__ void drop_draws8(unsigned (&w)[4], const uint4& d, unsigned high)      // high = threshold << 16
{
    const unsigned v[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (v[i] < high) w[i] &= 0x0000FFFFu;
        if ((v[i] << 16) < high) w[i] &= 0xFFFF0000u;
    }
}
__device__ __forceinline__ void drop_draws4(unsigned (&w)[4], unsigned d0, unsigned d1, unsigned high)
{
    if ((d0 << 16) < high) w[0] = 0;
    if (d0 < high) w[1] = 0;
    if ((d1 << 16) < high) w[2] = 0;
    if (d1 < high) w[3] = 0;
}

// ---- the quantiser ------------------------------------------------------------------------------------------------------
// A block of threads takes a tile of 128 rows x 128 columns; a lane holds 8 rows x 16 bytes of it in registers, in the
// input's own type, so that enough threads are resident for their loads to cover the memory's latency.
//   kRows     one layout, a scale for each row's 128 elements; warps do not meet
//   kBoth     and the transposed layout, a scale for each column's 128 elements, from the same registers
//   kSquare   one scale for the tile (weights), one or both layouts
// A row's block is 16 (fp32: 32) lanes.  The maxima of a lane's 8 rows go through an exchange that halves the rows a lane
// deals with in every step, so that a lane ends with one row, makes its scale once and hands 1 / scale around: instructions
// are what bounds this kernel besides memory, and a scale made by every lane for every row was a third of them.
// The transposed image turns through shared memory so that it leaves in 128-byte rows: column c is row c of s_turn, its
// 8-byte pieces (8 rows of one lane) permuted by the column so that the lanes of a write spread over all banks.
//
// Measured, bf16 8192 x 8192: kRows 32.5 us (floor 30.7), kBoth 47.8 us (41.0), with dropout 49 and 64 us (the draws take 22 us of
// the multiply pipe); fp32 4096 x 4096 kSquare, both layouts, 19.0 us (15.4).  Rows that start anywhere (8191 x 4095): kRows
// 21.9 us (15.4), kBoth 31.8 us (20.5).
enum QuantMode { kRows = 0, kBoth = 1, kSquare = 2 };
template <class T> constexpr int kQuantThreads = 16 * 128 / Piece<T>::kElems;      // 256, fp32: 512

// SUM: the columns' sums over the tile's rows besides (a bias gradient reads the same matrix).  ALIGNED: rows start on
// 16-byte boundaries and have a multiple of 8 elements, so that a lane's 16 bytes are one load and one draw.
//
// AHEAD: two blocks to an SM that go from tile to tile and ask for the next one (cp.async into the lane's own places) while
// they work on this one.  For both layouts of 2-byte types without draws, where more tiles than that are waiting: bf16
// 8192 x 8192 47.7 us instead of 51.4, 8192 x 4096 25.0 instead of 27.0.  Elsewhere it costs more than it hides (same size:
// rows 34.1 instead of 32.6 us, squares 45.7 and 45.0, both layouts with draws 73 instead of 64, bound by instructions; fp32
// 4096 x 4096 both layouts 20.3 and 20.2).
template <class T, bool E5, bool ALIGNED, bool DROP, int MODE, bool SUM = false, bool AHEAD = false>
__global__ void __launch_bounds__(kQuantThreads<T>, sizeof(T) == 2 && !AHEAD ? 3 : 2) quantize_kernel(const QuantArgs a)
{
    static_assert(!AHEAD || (ALIGNED && MODE == kBoth), "the next tile is asked for 16 aligned bytes at a time");
    using P = Piece<T>;
    constexpr int kElems = P::kElems, kLanes = 128 / kElems;                       // of a row
    constexpr int kWarps = kQuantThreads<T> / 32, kWords = 128 * static_cast<int>(sizeof(T)) / 4;   // words of a row
    extern __shared__ __align__(16) uint4 s_ahead[];         // AHEAD: [8][kQuantThreads], a lane's rows
    __shared__ __align__(16) unsigned s_max[MODE == kRows ? 1 : kWarps][MODE == kRows ? 4 : kWords];
    __shared__ __align__(16) float s_inv[MODE == kBoth ? 128 : 4];
    __shared__ float s_sum[SUM ? kWarps : 1][SUM ? 128 : 1];
    __shared__ __align__(16) uint8_t s_turn[MODE == kRows ? 16 : 128 * 128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, in_row = lane % kLanes;
    const int strip = threadIdx.x / kLanes;                                        // of 8 rows, 0 .. 15
    auto ask = [&](unsigned tile) {                          // zeros for what lies outside the matrix
        const unsigned tile_r = tile / a.ct, tile_c = tile - tile_r * a.ct;
        const long long r0 = static_cast<long long>(tile_r) * 128 + strip * 8, c = static_cast<long long>(tile_c) * 128 + in_row * kElems;
        const T* const x = static_cast<const T*>(a.x) + r0 * a.ldx + c;
        const long long rows = c < a.C ? a.R - r0 : 0;
        const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(s_ahead + threadIdx.x));
#pragma unroll
        for (int i = 0; i < 8; ++i)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + i * kQuantThreads<T> * 16),
                         "l"(i < rows ? x + i * a.ldx : static_cast<const T*>(a.x)), "r"(i < rows ? 16 : 0) : "memory");
    };
    unsigned tile = blockIdx.x;
    if (AHEAD) {
        after_previous();
        ask(tile);
    }
    do {
        const unsigned tile_r = tile / a.ct, tile_c = tile - tile_r * a.ct;
        const long long r0 = static_cast<long long>(tile_r) * 128 + strip * 8, c0 = static_cast<long long>(tile_c) * 128;
        const long long c = c0 + in_row * kElems;
        const int rows = static_cast<int>(max(0ll, min(8ll, a.R - r0)));
        if (MODE == kRows && a.R <= r0 - (strip * 8) % (32 / kLanes * 8)) return;      // nothing for this warp
        const T* const x = static_cast<const T*>(a.x) + r0 * a.ldx + c;
        if (!AHEAD) after_previous();

        unsigned v[8][4];
        const bool whole = rows == 8 && c0 + 128 <= a.C;         // the same for the block's warps but in the last tiles
        if (AHEAD) {
            asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint4 q = s_ahead[i * kQuantThreads<T> + threadIdx.x];
                v[i][0] = q.x; v[i][1] = q.y; v[i][2] = q.z; v[i][3] = q.w;
            }
        } else if (ALIGNED && whole) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint4 q = read16_once(x + i * a.ldx);
                v[i][0] = q.x; v[i][1] = q.y; v[i][2] = q.z; v[i][3] = q.w;
            }
        } else if (ALIGNED) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint4 q = i < rows && c < a.C ? read16_once(x + i * a.ldx) : make_uint4(0, 0, 0, 0);
                v[i][0] = q.x; v[i][1] = q.y; v[i][2] = q.z; v[i][3] = q.w;
            }
        } else if (whole) {
#pragma unroll
            for (int i = 0; i < 8; ++i) load_piece<T, true>(x + i * a.ldx, kElems, v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) load_piece<T, false>(x + i * a.ldx, i < rows ? a.C - c : 0, v[i]);
        }
        if (DROP) {
            PhiloxKey key(a.drop.rng);
            key.settle();
            const unsigned high = a.drop.threshold << 16;
            if (a.drop.threshold >= 65536u) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[i][j] = 0;
            } else if (ALIGNED) {
                const unsigned long long g = static_cast<unsigned long long>(r0 * a.C + c) >> 3, row = static_cast<unsigned long long>(a.C) >> 3;
                if (kElems == 8) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) drop_draws8(v[i], philox4x32_10(key, g + i * row), high);
                } else {
                    // a group of 8 elements is two lanes' share of a row: each draws for four rows and they exchange halves
                    const bool odd = lane & 1;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 d = philox4x32_10(key, g + (odd ? i + 4 : i) * row);
                        const unsigned e0 = __shfl_xor_sync(0xFFFFFFFFu, odd ? d.x : d.z, 1), e1 = __shfl_xor_sync(0xFFFFFFFFu, odd ? d.y : d.w, 1);
                        drop_draws4(v[i], odd ? e0 : d.x, odd ? e1 : d.y, high);
                        drop_draws4(v[i + 4], odd ? d.z : e0, odd ? d.w : e1, high);
                    }
                }
            } else {
                // Pieces straddle groups of 8 draws: a lane draws the group of its first element and takes the next group from the
                // next lane.  What the last lanes of the 8 (16) rows are short of, a lane each draws for one row, in one call.
                const int extra_row = lane % 8, extra_strip = strip - lane / kLanes + lane / 8 % (32 / kLanes);
                const unsigned long long e_extra = static_cast<unsigned long long>((static_cast<long long>(tile_r) * 128 + extra_strip * 8 + extra_row) * a.C + c0 + 128 - kElems);
                const uint4 extra = philox4x32_10(key, (e_extra >> 3) + 1);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const unsigned long long e = static_cast<unsigned long long>((r0 + i) * a.C + c);
                    const uint4 own = philox4x32_10(key, e >> 3);
                    uint4 next = from_next_lane(own);
                    const int from = lane / kLanes * 8 + i;      // of the lane that drew for this row
                    const uint4 x = make_uint4(__shfl_sync(0xFFFFFFFFu, extra.x, from), __shfl_sync(0xFFFFFFFFu, extra.y, from),
                                               __shfl_sync(0xFFFFFFFFu, extra.z, from), __shfl_sync(0xFFFFFFFFu, extra.w, from));
                    if (in_row == kLanes - 1) next = x;
                    unsigned d[4];
                    shifted(own, next, 2u * static_cast<unsigned>(e & 7u), d);
                    if (kElems == 8) drop_draws8(v[i], make_uint4(d[0], d[1], d[2], d[3]), high);
                    else drop_draws4(v[i], d[0], d[1], high);
                }
            }
        }

        // maxima of the rows, and of the columns over this lane's rows
        unsigned top[8], col[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            top[i] = P::larger(P::larger(v[i][0], v[i][1]), P::larger(v[i][2], v[i][3]));
            if (MODE == kBoth) {
#pragma unroll
                for (int j = 0; j < 4; ++j) col[j] = i ? P::larger(col[j], v[i][j]) : v[i][j];
            }
        }
        float inv[8];                                            // 1 / scale of this lane's rows
        if (MODE == kSquare) {
            unsigned m = top[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) m = P::larger(m, top[i]);
            m = __reduce_max_sync(0xFFFFFFFFu, P::fp32_bits(m));
            if (lane == 0) s_max[warp][0] = m;
            __syncthreads();
            m = __reduce_max_sync(0xFFFFFFFFu, lane < kWarps ? s_max[lane][0] : 0u);
            const unsigned byte = scale_byte<E5>(m);
            inv[0] = inverse_scale(byte);
#pragma unroll
            for (int i = 1; i < 8; ++i) inv[i] = inv[0];
            if (threadIdx.x == 0) {
                a.s[tile_r * a.lds + tile_c] = static_cast<uint8_t>(byte);
                if (a.st) a.st[tile_c * a.ldst + tile_r] = static_cast<uint8_t>(byte);
            }
        } else {
            if (MODE == kBoth) {
                if (kLanes == 16) {                              // the warp's two strips
#pragma unroll
                    for (int j = 0; j < 4; ++j) col[j] = P::larger(col[j], __shfl_xor_sync(0xFFFFFFFFu, col[j], 16));
                }
                if (lane < kLanes) *reinterpret_cast<uint4*>(&s_max[warp][in_row * 4]) = make_uint4(col[0], col[1], col[2], col[3]);
                if constexpr (SUM) {
                    auto add = [&](int j, float f) {
                        if (kLanes == 16) f += __shfl_xor_sync(0xFFFFFFFFu, f, 16);
                        if (lane < kLanes) s_sum[warp][in_row * kElems + j] = f;
                    };
#define ATB_COLUMN(J) (((P::template get<J>(v[0]) + P::template get<J>(v[1])) + (P::template get<J>(v[2]) + P::template get<J>(v[3]))) + \
                           ((P::template get<J>(v[4]) + P::template get<J>(v[5])) + (P::template get<J>(v[6]) + P::template get<J>(v[7]))))
                    add(0, ATB_COLUMN(0)); add(1, ATB_COLUMN(1)); add(2, ATB_COLUMN(2)); add(3, ATB_COLUMN(3));
                    if constexpr (kElems == 8) { add(4, ATB_COLUMN(4)); add(5, ATB_COLUMN(5)); add(6, ATB_COLUMN(6)); add(7, ATB_COLUMN(7)); }
#undef ATB_COLUMN
                }
            }
            // 8 rows x kLanes lanes: with every step a lane keeps half of its rows, the upper half if its bit is set
#pragma unroll
            for (int half = 4, bit = kLanes / 2; half >= 1; half >>= 1, bit >>= 1) {
                const bool upper = lane & bit;
#pragma unroll
                for (int i = 0; i < half; ++i) {
                    const unsigned keep = upper ? top[i + half] : top[i], give = upper ? top[i] : top[i + half];
                    top[i] = P::larger(keep, __shfl_xor_sync(0xFFFFFFFFu, give, bit));
                }
            }
#pragma unroll
            for (int bit = kLanes / 16; bit >= 1; bit >>= 1) top[0] = P::larger(top[0], __shfl_xor_sync(0xFFFFFFFFu, top[0], bit));
            if (AHEAD && tile + gridDim.x < a.tiles) ask(tile + gridDim.x);          // the maxima have used every value: all are in registers
            const int row = in_row / (kLanes / 8);               // the one this lane is left with
            const unsigned byte = scale_byte<E5>(P::fp32_bits(top[0]));
            const float mine = inverse_scale(byte);
            if (in_row % (kLanes / 8) == 0 && row < rows && (MODE != kBoth || a.q != nullptr)) a.s[(r0 + row) * a.lds + tile_c] = static_cast<uint8_t>(byte);
#pragma unroll
            for (int i = 0; i < 8; ++i) inv[i] = __shfl_sync(0xFFFFFFFFu, mine, i * (kLanes / 8), kLanes);
        }
        // the image as it lies, unless only the transposed one is asked for (bf16 8192 x 8192 36.7 us)
        if (MODE != kBoth || a.q != nullptr) {
            uint8_t* const q = a.q + r0 * a.ldq + c;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned lo = pack4<E5>(P::template get<0>(v[i]) * inv[i], P::template get<1>(v[i]) * inv[i],
                                              P::template get<2>(v[i]) * inv[i], P::template get<3>(v[i]) * inv[i]);
                if constexpr (kElems == 8) {
                    const unsigned hi = pack4<E5>(P::template get<4>(v[i]) * inv[i], P::template get<5>(v[i]) * inv[i],
                                                  P::template get<6>(v[i]) * inv[i], P::template get<7>(v[i]) * inv[i]);
                    if (i < rows && c < a.wq) *reinterpret_cast<uint2*>(q + i * a.ldq) = make_uint2(lo, hi);
                } else {
                    if (i < rows && c < a.wq) *reinterpret_cast<unsigned*>(q + i * a.ldq) = lo;
                }
            }
        }
        if (MODE == kRows || a.qt == nullptr) return;

        if (MODE == kBoth) {
            __syncthreads();
            if (SUM && threadIdx.x >= kQuantThreads<T> - 128) {  // (not the warps that make the scales)
                const int cc = threadIdx.x - (kQuantThreads<T> - 128);
                float f = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) f += s_sum[w][cc];
                if (c0 + cc < a.C) a.sums[tile_r * a.C + c0 + cc] = f;
            }
            if (threadIdx.x < kWords) {                          // a word's columns (one, or two halves)
                unsigned m = s_max[0][threadIdx.x];
#pragma unroll
                for (int w = 1; w < kWarps; ++w) m = P::larger(m, s_max[w][threadIdx.x]);
                constexpr int kPer = 128 / kWords;
#pragma unroll
                for (int h = 0; h < kPer; ++h) {
                    const int cc = threadIdx.x * kPer + h;
                    const unsigned one = kPer == 1 ? m : h ? m >> 16 : m & 0xFFFFu;
                    const unsigned byte = scale_byte<E5>(P::fp32_bits(one));
                    s_inv[cc] = inverse_scale(byte);
                    if (c0 + cc < a.C) a.st[(c0 + cc) * a.ldst + tile_r] = static_cast<uint8_t>(byte);
                }
            }
            __syncthreads();
        }
        auto turn = [&](int j, float f0, float f1, float f2, float f3, float f4, float f5, float f6, float f7) {
            const float by = MODE == kBoth ? s_inv[in_row * kElems + j] : inv[0];
            const int cc = in_row * kElems + j;
            *reinterpret_cast<uint2*>(s_turn + cc * 128 + ((strip ^ in_row % 16) << 3)) =
                make_uint2(pack4<E5>(f0 * by, f1 * by, f2 * by, f3 * by), pack4<E5>(f4 * by, f5 * by, f6 * by, f7 * by));
        };
#define ATB_TURN(J) turn(J, P::template get<J>(v[0]), P::template get<J>(v[1]), P::template get<J>(v[2]), P::template get<J>(v[3]), \
                             P::template get<J>(v[4]), P::template get<J>(v[5]), P::template get<J>(v[6]), P::template get<J>(v[7]))
        ATB_TURN(0); ATB_TURN(1); ATB_TURN(2); ATB_TURN(3);
        if constexpr (kElems == 8) { ATB_TURN(4); ATB_TURN(5); ATB_TURN(6); ATB_TURN(7); }
#undef ATB_TURN
        __syncthreads();
        const long long rt = static_cast<long long>(tile_r) * 128;
#pragma unroll
        for (int i = 0; i < 1024 / kQuantThreads<T>; ++i) {
            const int cc = (threadIdx.x >> 3) + kQuantThreads<T> / 8 * i, piece = threadIdx.x & 7, by = cc / kElems % 16;
            uint4 o = *reinterpret_cast<const uint4*>(s_turn + cc * 128 + ((piece ^ (by >> 1)) << 4));
            if (by & 1) o = make_uint4(o.z, o.w, o.x, o.y);
            if (c0 + cc < a.C && rt + piece * 16 < a.wqt) *reinterpret_cast<uint4*>(a.qt + (c0 + cc) * a.ldqt + rt + piece * 16) = o;
        }
        // (what the next tile writes to shared memory is written one barrier at least after this tile's last read of it)
    } while (AHEAD && (tile += gridDim.x) < a.tiles);
}

// out[c] = the sum of column c of p [rows, C], in the order of the rows
__global__ void __launch_bounds__(256) sum_rows_kernel(const float* p, int rows, long long C, float* out)
{
    after_previous();
    const long long c = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (c >= C) return;
    float f = 0.0f;
#pragma unroll 8
    for (int r = 0; r < rows; ++r) f += p[r * C + c];
    out[c] = f;
}

// both layouts of an aligned matrix of a 2-byte type, more tiles than two blocks an SM
template <class T, bool E5, bool SUM>
static int launch_quantize_ahead(const QuantArgs& a, cudaStream_t s)
{
    const int smem = 8 * 16 * kQuantThreads<T>;              // with what is declared in the kernel, above the default limit
    static bool done[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= 64 || !done[dev]))
        e = cudaFuncSetAttribute(quantize_kernel<T, E5, true, false, kBoth, SUM, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail_invalid(cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) done[dev] = true;
    launch_after(quantize_kernel<T, E5, true, false, kBoth, SUM, true>, dim3(2 * sm_count()), dim3(kQuantThreads<T>), smem, s, 0, a);
    return check_launch("quantize_kernel");
}

template <class T, bool E5, bool ALIGNED>
static int launch_quantize_as(const QuantArgs& a, bool square, cudaStream_t s)
{
    const dim3 grid(a.tiles), block(kQuantThreads<T>);
    const bool drop = a.drop.rng != nullptr;
    if constexpr (ALIGNED && sizeof(T) == 2) {
        if (!square && a.qt != nullptr && !drop && a.tiles > 2u * sm_count())
            return a.sums ? launch_quantize_ahead<T, E5, true>(a, s) : launch_quantize_ahead<T, E5, false>(a, s);
    }
    if (square) launch_after(quantize_kernel<T, E5, ALIGNED, false, kSquare>, grid, block, 0, s, 0, a);
    else if (a.qt == nullptr) {
        if (drop) launch_after(quantize_kernel<T, E5, ALIGNED, true, kRows>, grid, block, 0, s, 0, a);
        else launch_after(quantize_kernel<T, E5, ALIGNED, false, kRows>, grid, block, 0, s, 0, a);
    } else if (a.sums) launch_after(quantize_kernel<T, E5, ALIGNED, false, kBoth, true>, grid, block, 0, s, 0, a);
    else if (drop) launch_after(quantize_kernel<T, E5, ALIGNED, true, kBoth>, grid, block, 0, s, 0, a);
    else launch_after(quantize_kernel<T, E5, ALIGNED, false, kBoth>, grid, block, 0, s, 0, a);
    return check_launch("quantize_kernel");
}

template <class T, bool E5>
static int launch_quantize(QuantArgs a, bool square, cudaStream_t s)
{
    const long long ct = (a.C + 127) >> 7, tiles = ((a.R + 127) >> 7) * ct;
    ATB_REQUIRE(tiles < (1ll << 31), "matrix too large");
    a.ct = static_cast<unsigned>(ct);
    a.tiles = static_cast<unsigned>(tiles);
    const bool aligned = aligned_to(a.x, 16) && (a.ldx * static_cast<long long>(sizeof(T))) % 16 == 0 && a.C % 8 == 0;
    return aligned ? launch_quantize_as<T, E5, true>(a, square, s)
                   : launch_quantize_as<T, E5, false>(a, square, s);
}

}  // namespace atb

using namespace atb;

extern "C" int atb_fp8_quantize(const void* x, int x_dtype, long long R, long long C, long long ldx, int f8, int block_rows,
                                void* q, long long ldq, uint8_t* s, long long lds, void* qt, long long ldqt, uint8_t* st,
                                long long ldst, float* column_sums, int drop_threshold, const void* rng, void* stream)
{
    ATB_REQUIRE(R >= 0 && C >= 0, "negative dimension");
    ATB_REQUIRE(f8 == ATB_E4M3 || f8 == ATB_E5M2, "the result must be e4m3 or e5m2");
    ATB_REQUIRE(block_rows == 1 || block_rows == 128, "block_rows must be 1 or 128");
    ATB_REQUIRE(drop_threshold >= 0 && drop_threshold <= 65536, "threshold must lie in [0, 65536]");
    if (R == 0 || C == 0) return ATB_OK;
    ATB_REQUIRE(x && (q || (qt && block_rows == 1)), "null pointer");
    ATB_REQUIRE(aligned_to(x, x_dtype == ATB_F32 ? 4 : 2), "x must be aligned to its elements");
    ATB_REQUIRE((q == nullptr) == (s == nullptr) && (qt == nullptr) == (st == nullptr), "an image and its scales come together");
    ATB_REQUIRE(ldx >= C || R == 1, "row pitch of x below its width");
    const long long nb = (C + 127) / 128, nbt = (R + 127) / 128;
    if (q) ATB_REQUIRE(ldq >= C && ldq % 16 == 0 && aligned_to(q, 16) && lds >= nb, "q needs 16-byte aligned rows, s a column for every block");
    if (qt) ATB_REQUIRE(ldqt >= R && ldqt % 16 == 0 && aligned_to(qt, 16) && ldst >= nbt, "qt needs 16-byte aligned rows, st a column for every block");
    ATB_REQUIRE(rng == nullptr || block_rows == 1, "dropout goes with blocks of one row");
    ATB_REQUIRE(column_sums == nullptr || (qt && block_rows == 1 && drop_threshold == 0 && aligned_to(column_sums, 4)),
                "column sums go with both layouts, blocks of one row and no dropout");
    ATB_REQUIRE(drop_threshold == 0 || (rng != nullptr && aligned_to(rng, 8)), "dropout needs an 8-byte aligned state");
    QuantArgs a{x, R, C, ldx, static_cast<uint8_t*>(q), ldq, s, lds, static_cast<uint8_t*>(qt), ldqt, st, ldst, column_sums,
                DropState{drop_threshold ? static_cast<const unsigned long long*>(rng) : nullptr, static_cast<unsigned>(drop_threshold)},
                (C + 15) / 16 * 16, (R + 15) / 16 * 16, 0, 0};
    cudaStream_t stm = static_cast<cudaStream_t>(stream);
    const bool e5 = f8 == ATB_E5M2, square = block_rows == 128;
    if (x_dtype == ATB_F32) return e5 ? launch_quantize<float, true>(a, square, stm) : launch_quantize<float, false>(a, square, stm);
    if (x_dtype == ATB_BF16) return e5 ? launch_quantize<__nv_bfloat16, true>(a, square, stm) : launch_quantize<__nv_bfloat16, false>(a, square, stm);
    if (x_dtype == ATB_F16) return e5 ? launch_quantize<__half, true>(a, square, stm) : launch_quantize<__half, false>(a, square, stm);
    return fail_invalid("x must be fp32, bf16 or fp16");
}

extern "C" int atb_sum_rows(const float* p, int rows, long long C, float* out, void* stream)
{
    ATB_REQUIRE(rows >= 0 && C >= 0, "negative dimension");
    if (C == 0) return ATB_OK;
    ATB_REQUIRE(out && (p || rows == 0) && aligned_to(p, 4) && aligned_to(out, 4), "p and out must be 4-byte aligned pointers");
    ATB_REQUIRE((C + 255) / 256 < (1ll << 31), "too many columns");
    launch_after(sum_rows_kernel, dim3(static_cast<unsigned>((C + 255) / 256)), dim3(256), 0, static_cast<cudaStream_t>(stream), 0, p, rows, C, out);
    return check_launch("sum_rows_kernel");
}

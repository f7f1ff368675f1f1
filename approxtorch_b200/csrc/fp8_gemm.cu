// Matrix product of 8-bit floating point operands with a power-of-two scale for each block of 128.
//
//   y[m, n] = alpha * sum_k  A[m, k] 2^(sa[m', k/128] - 127)  B[n, k] 2^(sb[n', k/128] - 127)  + bias[n]
//
// with m' = m or m / 128 (one scale for a row's block, or for a 128 x 128 block), n' likewise; the sum in the tensor core's 24-bit
// accumulator, which cuts instead of rounding (what that costs, and what is done about it: SUMS below), one rounding at the end.
// The scales are applied by the tensor core itself: tcgen05.mma kind::mxf8f6f4.block_scale takes one exponent byte per row and
// 32 steps of the reduction from tensor memory, and four consecutive instructions read the same byte.  So the product runs at the
// rate of an unscaled 8-bit product; promoting every 128-step partial sum through registers instead would cost a read of the
// accumulator per 128 steps.
//
// fp8_gemm_kernel, for products of many tiles: one block of threads per SM (CG = 1), or two blocks on two SMs that work on
// one tile of 256 rows (CG = 2), walk over the output tiles:
//   warp 0      one thread requests the operand tiles by TMA (128-byte swizzle, one 128-step slice = one 128-byte row);
//   warp 1      one thread moves the scales to tensor memory (tcgen05.cp) and issues the MMAs (of the pair: the first
//               block's thread, for both);
//   warps 2-3   gather the scale bytes, 16 slices at a time (one load per row), and hand them over four slices (a quad) at a
//               time in the order in which tcgen05.cp wants them: 32 rows of 16 bytes, word j of row i = operand row
//               i + 32 j (warp 3 also owns the tensor-memory allocation);
//   warps 4-11  read finished accumulators, scale, add the bias, mask and store, 32 x 32 elements at a time through shared
//               memory so that a row's bytes leave together (four warps instead of eight: 4096 x 8192 x 128 24.0 instead of
//               19.5 us, 4096 x 8192 x 1024 with a mask 58 instead of 46 us).
// Two accumulators let the epilogue of a tile run under the MMAs of the next; where two of 256 columns and the scales do
// not fit the 512 columns of tensor memory, they share 24 columns, which the epilogue reads first.  Why pairs: each block of
// a pair holds its own 128 rows of A and half the rows of B and the tensor core reads both halves, so a slice of a 256 x 256
// tile costs each SM 32 KB from L2 instead of the 48 KB of a 128 x 256 tile.
//
// What bounds it: the tensor core, at the clock that the power limit leaves.  8192^3: 541 clocks for a slice of a 256 x 256 tile,
// first loads and last results included, where the tensor core's nominal rate is 512.  One call by itself 353 us (3.1 PFLOP/s) at
// 1.39 GHz, the fifth in a row 400 at 1.30, four seconds of them 450 at 1.13 GHz (990 W, the power limit the only reason; a library
// product of the same operands with a scale for each 32: 404).  What it took to get there, and what a change should not lose: the issuing warp
// runs converged and walks uniform values (a branch on the lane number cost 40 %), the scales arrive a quad ahead, and only
// hand-overs of memory between the blocks pay for cluster scope.
//
// fp8_split_kernel, for products of few tiles (serving, small heads): see there.
//
// Operand rows beyond M or N and steps beyond K are zeros that TMA fills in; scale bytes beyond the last block are
// never selected, and rows beyond the last take its scales: a row's products go to its own row of the result alone.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <atomic>

#include "common.cuh"
#include "philox.cuh"

namespace atb {

constexpr int kF8Threads = 384, kF8EpiWarp = 4, kF8EpiWarps = 8, kF8SplitThreads = 256;
constexpr int kF8SumTileN = 192, kF8SumQuads = 2;            // with fp32 sums of partial products
constexpr int kF8TileM = 128, kF8MaxTileN = 256;          // of one block; a pair's tile has twice the rows
constexpr int kF8SfSlots = 8, kF8SfSlotBytes = 3 * 512;   // a run of quads for each gathering warp; 128 rows of A, up to 256 of B
constexpr int kF8SfCol = 488, kF8SfCols = 12;             // tensor-memory columns of the two scale buffers
constexpr int kF8Smem = 226 * 1024, kF8MaxStages = 8;
constexpr int kF8SplitSmem = kF8Smem - kF8TileM * 16;    // fp8_split_kernel: its mask besides
constexpr int kF8SumsFrom = 16;                          // slices beyond which an fp32 result is added up from partial sums,
constexpr int kF8SumsFromFp16 = 256, kF8SumsFromBf16 = 2048;     // a 16-bit one
constexpr int kF8MaxQuads = 40;                           // of one block of fp8_split_kernel
constexpr int kF8Group = 8;                               // row tiles that are walked together (their operands meet in L2)

struct Fp8Params {
    const uint8_t* sa;
    const uint8_t* sb;
    long long ldsa, ldsb;
    int a_shift, b_shift;                // 0: a scale per row, 7: per 128 rows
    bool sf_vec;                         // scale rows of both operands start on 16-byte boundaries
    const float* bias;
    float alpha;
    void* y;
    long long ldy;
    int M, N, kblocks;
    int tile_n, mt, nt, stages;
    uint32_t idesc;
    bool vec;                            // rows of y start on 16-byte boundaries
    DropState drop;
    int patience;                        // see f8_wait
    int* error;                          // pinned host memory
};

__device__ __forceinline__ uint32_t f8_smem(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void f8_bar_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void f8_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void f8_expect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Bounded wait (`patience` looks at the barrier) that also gives up when another role of the block has.  CLUSTER: the arrivals it
// waits for order another block's writes (an acquire over the cluster costs far more than one over the block; only the
// hand-overs that need it pay for it).
//
// A block that gave up fills what it has not written with NaN, waits for its copies and MMAs in flight, says so in a word of
// pinned host memory that the next call looks at, and returns.
constexpr int kF8Patience = 1 << 18;                      // about a second
template <bool CLUSTER = false>
__device__ __forceinline__ bool f8_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int patience)
{
    for (int i = 0; i < patience; ++i) {
        uint32_t ok;
        if (CLUSTER)
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                         : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        else
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                         : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if ((i & 63) == 63 && *abort_flag) return false;
    }
    *abort_flag = 1;
    return false;
}
// the wait for what is in flight when a block ends, whoever has given up before
__device__ __forceinline__ bool f8_settle(uint32_t bar, uint32_t parity)
{
    int never = 0;
    return f8_wait(bar, parity, &never, kF8Patience);
}
__device__ __forceinline__ void f8_report(int* error)
{
    *static_cast<volatile int*>(error) = 1;
    __threadfence_system();
}
// one look at a barrier
__device__ __forceinline__ bool f8_test(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// one lane of a converged warp.  (The roles below run as whole warps and issue under this predicate: a branch on the lane
// number instead makes the compiler rebuild every descriptor operand lane by lane, and the MMA issue became the bound.)
__device__ __forceinline__ bool f8_elect()
{
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
// the same shared address in the first block of the pair
__device__ __forceinline__ uint32_t f8_leader(uint32_t addr)
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
// An arrival at a barrier of the pair's first block.  It orders no memory by itself: it says that tensor memory has been
// read (the tcgen05 fences on both sides order that), or follows an f8_release_cluster.
__device__ __forceinline__ void f8_arrive_leader(uint32_t local_bar)
{
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(f8_leader(local_bar)) : "memory");
}
__device__ __forceinline__ void f8_release_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }
__device__ __forceinline__ void f8_cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// CG = 2: the bytes land here, the barrier may be the other block's
template <int CG>
__device__ __forceinline__ void f8_tma(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar)
{
    if (CG == 1)
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
// K-major operand with 128-byte swizzle: 8-row atoms 1024 bytes apart
__device__ __forceinline__ uint64_t f8_desc(uint32_t saddr)
{
    return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(1) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
// 32 rows of 16 bytes without swizzle: 8-row groups 128 bytes apart
__device__ __forceinline__ uint64_t f8_sf_desc(uint32_t saddr)
{
    return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(1) << 16) |
           (static_cast<uint64_t>(128 >> 4) << 32) | (static_cast<uint64_t>(1) << 46);
}
template <int CG>
__device__ __forceinline__ void f8_copy_scales(uint32_t tmem, uint64_t desc)
{
    if (CG == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// one 32-step MMA; a_lo, b_lo: the low words of the operands' descriptors (f8_desc)
template <int CG>
__device__ __forceinline__ void f8_mma(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t sfa, uint32_t sfb, bool accumulate)
{
    const uint32_t acc = accumulate ? 1u : 0u, hi = static_cast<uint32_t>(f8_desc(0) >> 32);
    if (CG == 1)
        asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %6, 0;\n\tmov.b64 da, {%1, %7};\n\tmov.b64 db, {%2, %7};\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc), "r"(hi) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %6, 0;\n\tmov.b64 da, {%1, %7};\n\tmov.b64 db, {%2, %7};\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc), "r"(hi) : "memory");
}
// arrives at the barrier when the MMAs issued so far are done; CG = 2: at the same barrier of both blocks
template <int CG>
__device__ __forceinline__ void f8_commit(uint32_t bar)
{
    if (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}
// the same, at this block's barrier alone
template <int CG>
__device__ __forceinline__ void f8_commit_here(uint32_t bar)
{
    if (CG == 1) asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    else asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void f8_tmem_ld32(uint32_t (&v)[32], uint32_t addr)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                   "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
                   "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
                   "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void f8_tmem_ld16(uint32_t (&v)[16], uint32_t addr)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                   "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

template <class T> __device__ __forceinline__ T f8_out(float v);
template <> __device__ __forceinline__ float f8_out<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 f8_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half f8_out<__half>(float v) { return __float2half_rn(v); }
template <class T> __device__ __forceinline__ uint32_t f8_pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t f8_pack2<__nv_bfloat16>(float a, float b)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t f8_pack2<__half>(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// 16 bytes of results to shared memory and back
template <class T>
__device__ __forceinline__ void f8_put16(uint32_t addr, const float* f)
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
        else w[i] = f8_pack2<T>(f[2 * i], f[2 * i + 1]);
    }
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}
__device__ __forceinline__ uint4 f8_get16(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
template <class T>
__device__ __forceinline__ T f8_get(uint32_t addr)
{
    T r;
    if constexpr (sizeof(T) == 4) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(addr) : "memory");
    else {
        uint16_t h;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(addr) : "memory");
        r = *reinterpret_cast<T*>(&h);
    }
    return r;
}
// bit j set: element + j is kept (j < 32).  Out of line: long enough to push the loop out of the instruction cache, and not
// every product has a mask.  The four (five) draws are independent of one another, so that they fill each other's latency.
__device__ __noinline__ unsigned f8_keep32(PhiloxKey key, unsigned threshold, unsigned long long element)
{
    const unsigned long long group = element >> 3;
    const unsigned shift = static_cast<unsigned>(element & 7u);
    unsigned keep[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) keep[g] = philox_keep8(key, group + g, threshold);
    const unsigned m = keep[0] | keep[1] << 8 | keep[2] << 16 | keep[3] << 24;
    return shift ? __funnelshift_r(m, philox_keep8(key, group + 4, threshold), shift) : m;
}

__device__ __forceinline__ uint32_t f8_word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// row and column tile of the t-th output tile: kF8Group row tiles at a time, column by column
__device__ __forceinline__ void f8_tile(int t, int mt, int nt, int& tm, int& tn)
{
    const int per = kF8Group * nt, g = t / per, rows = min(kF8Group, mt - g * kF8Group), in = t - g * per;
    tn = in / rows;
    tm = g * kF8Group + (in - tn * rows);
}

// NaN for what an epilogue warp still had to write when it gave up: its part of the tiles t, t + step, ...  Out of line: the
// loop need not carry it.
template <class T, bool SUMS>
__device__ __noinline__ void f8_blank(const Fp8Params& p, int t, int step, int cg, int rank)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = (warp - kF8EpiWarp) >> 2;
    const int c0 = SUMS ? p.tile_n / 2 * group : 32 * group, c1 = SUMS ? c0 + p.tile_n / 2 : p.tile_n, by = SUMS ? 32 : 64;
    for (; t < p.mt * p.nt; t += step) {
        int tm, tn;
        f8_tile(t, p.mt, p.nt, tm, tn);
        const int m0 = (tm * cg + rank) * kF8TileM + (warp & 3) * 32, m1 = min(m0 + 32, p.M);
        for (int c = c0; c < c1; c += by) {
            const int n = tn * p.tile_n + c + lane;
            if (n < p.N)
                for (int m = m0; m < m1; ++m) static_cast<T*>(p.y)[m * p.ldy + n] = f8_out<T>(__uint_as_float(0x7FC00000u));
        }
    }
}

// SUMS: the tensor core's accumulator has the 24 bits of fp32, but cuts what does not fit instead of rounding it, at several
// places of an MMA, which leaves a bias towards zero that grows with the number of additions.  Measured with magnitudes of normal
// numbers, which is a sum without cancellation: 1.8e-7 of the result over 1024 steps, 5e-7 over 2048, 4e-4 over 2^18, 3e-3 over
// 2^20, 8e-2 over 2^24 (of numbers of both signs the magnitudes' 1e-8 and less).  So a long reduction reads the accumulators
// every 1024 steps (kF8SumQuads quads) and adds them up, rounded, in the registers of the epilogue warps, the two accumulators
// taking turns: beyond 2048 steps to fp32 (8192 steps 117 us, every 2048 steps 114, never 111; 2e-7 to 5e-7), and where the bias
// would near a quarter of a step of a 16-bit result, n 2^-23 for n = steps / 32 additions as an estimate: 2^15 steps to fp16, 2^18
// to bf16.
template <class T, int CG, bool SUMS>
__global__ void __launch_bounds__(kF8Threads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ Fp8Params p)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    __shared__ __align__(8) uint64_t s_full[kF8MaxStages], s_empty[kF8MaxStages], s_sf_full[kF8SfSlots], s_sf_empty[kF8SfSlots], s_acc_full[2], s_acc_empty[2], s_acc_part, s_mma_done;
    constexpr int kPitch = 32 * sizeof(T) + 16;              // of a staged row: 16-byte accesses without bank conflicts
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);  // the same for a warp, and the compiler knows it
    const int rank = CG == 2 ? static_cast<int>(blockIdx.x & 1u) : 0;
    const int first = blockIdx.x / CG, step = gridDim.x / CG;
    const uint32_t smem0 = (f8_smem(smem_raw) + 1023u) & ~1023u;
    const int b_rows = p.tile_n / CG;                        // rows of B that this block holds
    const uint32_t stage_bytes = kF8TileM * 128 + b_rows * 128;
    const uint32_t sf0 = smem0 + p.stages * stage_bytes, stage0 = sf0 + kF8SfSlots * kF8SfSlotBytes;
    const uint32_t full0 = f8_smem(s_full), empty0 = f8_smem(s_empty), sff0 = f8_smem(s_sf_full), sfe0 = f8_smem(s_sf_empty);
    const uint32_t accf0 = f8_smem(s_acc_full), acce0 = f8_smem(s_acc_empty), accp = f8_smem(&s_acc_part), done0 = f8_smem(&s_mma_done);
    const int ntiles = p.mt * p.nt, kb_n = p.kblocks, quads = (kb_n + 3) >> 2, runs = (kb_n + 15) >> 4;
    volatile int* abort_flag = &s_abort;

    // 16 bytes (a run of up to four quads) of the scale rows of a tile: lane i gets operand rows i, i + 32, ...  Rows beyond
    // the last repeat it: their products are never stored.
    uint4 w[12];
    auto fetch = [&](int turn, int run) {
        int tm, tn;
        f8_tile(first + turn * step, p.mt, p.nt, tm, tn);
        const int m0 = (tm * CG + rank) * kF8TileM + lane, n0 = tn * p.tile_n + lane;
        const uint8_t* a = p.sa + 16 * run;
        const uint8_t* b = p.sb + 16 * run;
        if (p.sf_vec) {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = read16(a + static_cast<long long>(min(m0 + 32 * j, p.M - 1) >> p.a_shift) * p.ldsa);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (32 * j < p.tile_n) w[4 + j] = read16(b + static_cast<long long>(min(n0 + 32 * j, p.N - 1) >> p.b_shift) * p.ldsb);
        } else {
            const int words = quads - 4 * run;               // that this run has left
            const uint8_t* src[12];
#pragma unroll
            for (int j = 0; j < 12; ++j) {
                src[j] = j < 4 ? a + static_cast<long long>(min(m0 + 32 * j, p.M - 1) >> p.a_shift) * p.ldsa
                               : b + static_cast<long long>(min(n0 + 32 * (j - 4), p.N - 1) >> p.b_shift) * p.ldsb;
                if (j < 4 || 32 * (j - 4) < p.tile_n) w[j].x = read4(src[j]);
            }
#pragma unroll
            for (int i = 1; i < 4; ++i) {
                if (i >= words) break;
#pragma unroll
                for (int j = 0; j < 12; ++j) {
                    if (j >= 4 && 32 * (j - 4) >= p.tile_n) continue;
                    const uint32_t v = read4(src[j] + 4 * i);
                    if (i == 1) w[j].y = v; else if (i == 2) w[j].z = v; else w[j].w = v;
                }
            }
        }
    };
    const int my_turns = first < ntiles ? (ntiles - 1 - first) / step + 1 : 0;
    int sf_turn = 0, sf_run = warp - 2;                      // of the scale warps' next run: tile of this block, run of the tile
    auto sf_settle = [&] { while (sf_run >= runs) { sf_run -= runs; ++sf_turn; } };

    if (warp == 0) {
        if (lane == 0) s_abort = 0;
        for (int i = lane; i < kF8MaxStages; i += 32) { f8_bar_init(full0 + 8 * i, 1); f8_bar_init(empty0 + 8 * i, 1); }
        if (lane < kF8SfSlots) { f8_bar_init(sff0 + 8 * lane, CG); f8_bar_init(sfe0 + 8 * lane, 1); }
        if (lane < 2) { f8_bar_init(accf0 + 8 * lane, 1); f8_bar_init(acce0 + 8 * lane, kF8EpiWarps * CG); }
        if (lane == 0) { f8_bar_init(accp, kF8EpiWarps / 2 * CG); f8_bar_init(done0, 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    } else if (warp == 1) {
        if (f8_elect()) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
        }
    } else if (warp == 3) {
        if (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(f8_smem(&s_tmem)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(f8_smem(&s_tmem)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    if (warp == 2 || (CG == 1 && warp == 3)) {
        // the first scales are what the first MMA waits for: asked for before the blocks meet, and without waiting for
        // them there (this warp has written nothing that others read)
        after_previous();
        sf_settle();
        if (sf_turn < my_turns) fetch(sf_turn, sf_run);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (CG == 2) {
        if (warp == 2) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
        else asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    after_previous();
    const uint32_t tmem = s_tmem;
    // Two accumulators side by side, or, where they and the scales do not fit, sharing columns: the epilogue then reads the
    // shared ones first and says so, and the next tile's MMAs start.
    const uint32_t d_step = min(p.tile_n, kF8SfCol - p.tile_n);
    const bool overlap = d_step < static_cast<uint32_t>(p.tile_n);

    if (warp == 0) {
        uint32_t s = 0, parity = 1, issued = 0;
        bool ok = true;
        for (int t = first; t < ntiles && ok; t += step) {
            int tm, tn;
            f8_tile(t, p.mt, p.nt, tm, tn);
            const int m0 = (tm * CG + rank) * kF8TileM, n0 = tn * p.tile_n + rank * b_rows;
            for (int kb = 0; kb < kb_n; ++kb, ++issued) {
                if (!(ok = f8_wait(empty0 + 8 * s, parity, abort_flag, p.patience))) break;
                if (f8_elect()) {
                    if (rank == 0) f8_expect(full0 + 8 * s, CG * stage_bytes);
                    const uint32_t bar = CG == 2 ? f8_leader(full0 + 8 * s) : full0 + 8 * s;
                    f8_tma<CG>(smem0 + s * stage_bytes, &map_a, kb * 128, m0, bar);
                    f8_tma<CG>(smem0 + s * stage_bytes + kF8TileM * 128, &map_b, kb * 128, n0, bar);
                }
                __syncwarp();
                if (++s == static_cast<uint32_t>(p.stages)) { s = 0; parity ^= 1u; }
            }
        }
        // nothing may be in flight when the block ends (all of it has landed unless a role gave up); the second block of a pair
        // has no barrier for its own share, which lands in microseconds: it waits a millisecond
        if (rank == 0) {
            for (uint32_t j = issued > static_cast<uint32_t>(p.stages) ? issued - p.stages : 0; j < issued; ++j)
                if (!f8_settle(full0 + 8 * (j % p.stages), (j / p.stages) & 1u)) break;
        } else if (!ok) {
            for (int i = 0; i < 100; ++i) __nanosleep(10000);
        }
    } else if (warp == 1) {
        if (rank == 0) {
            uint32_t parity = 0, quad = 0, tile = 0;         // tile: accumulators used so far
            // Scales of a quad to tensor memory, one quad ahead of the MMAs.  The gathering warps fill four slots each, in turn
            // by runs; a scale buffer is free when the MMAs of two quads before are done.
            uint32_t staged = 0, run = 0, run_left = 0, tile_left = 0, taken[2] = {0, 0};
            uint32_t older_bar = 0, older_parity = 0, last_bar = 0, last_parity = 0;
            const uint32_t total = static_cast<uint32_t>(my_turns) * quads;
            auto stage_scales = [&]() -> bool {
                if (staged >= total) return true;
                if (tile_left == 0) tile_left = quads;
                if (run_left == 0) { run_left = min(tile_left, 4u); ++run; }
                const uint32_t from = (run - 1) & 1u, n = from ? taken[1] : taken[0], slot = 4 * from + (n & 3u), turn_parity = (n >> 2) & 1u;
                if (staged >= 2 && !f8_wait(older_bar, older_parity, abort_flag, p.patience)) return false;
                if (!f8_wait<CG == 2>(sff0 + 8 * slot, turn_parity, abort_flag, p.patience)) return false;
                older_bar = last_bar; older_parity = last_parity;
                last_bar = sfe0 + 8 * slot; last_parity = turn_parity;
                if (from) ++taken[1]; else ++taken[0];
                --run_left; --tile_left;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t src = sf0 + slot * kF8SfSlotBytes, dst = tmem + kF8SfCol + (staged & 1u) * kF8SfCols;
                if (f8_elect()) {
                    f8_copy_scales<CG>(dst, f8_sf_desc(src));
                    f8_copy_scales<CG>(dst + 4, f8_sf_desc(src + 512));
                    if (p.tile_n > 128) f8_copy_scales<CG>(dst + 8, f8_sf_desc(src + 1024));
                }
                __syncwarp();
                ++staged;
                return true;
            };
            // a stage's barrier and the low word of its A descriptor, walked side by side
            const uint32_t a_first = static_cast<uint32_t>(f8_desc(smem0)), a_step = stage_bytes >> 4, a_end = a_first + p.stages * a_step;
            uint32_t a_lo = a_first, full = full0;
            bool ok = stage_scales(), ready = false;
            const int item_quads = SUMS ? kF8SumQuads : quads, items = (quads + item_quads - 1) / item_quads * my_turns;
            for (int it = 0, left = quads; it < items && ok; ++it, ++tile) {
                const uint32_t buf = tile & 1u, d = tmem + buf * d_step;
                const int now = min(left, item_quads), kb_left = min(4 * now, kb_n - 4 * (quads - left));   // of this accumulator
                left = left == now ? quads : left - now;
                if (!(ok = f8_wait(acce0 + 8 * buf, ((tile >> 1) & 1u) ^ 1u, abort_flag, p.patience))) break;
                if (overlap && tile > 0 && !(ok = f8_wait(accp, (tile - 1) & 1u, abort_flag, p.patience))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int q = 0; q < now && ok; ++q, ++quad) {
                    const uint32_t sfa = tmem + kF8SfCol + (quad & 1u) * kF8SfCols, slot = last_bar;
                    const int slices = min(4, kb_left - 4 * q);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (i >= slices) break;
                        if (!ready && !(ok = f8_wait(full, parity, abort_flag, p.patience))) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t at = a_lo, empty = full + (empty0 - full0);
                        a_lo += a_step;
                        full += 8;
                        if (a_lo == a_end) { a_lo = a_first; full = full0; parity ^= 1u; }
                        ready = f8_test(full, parity);           // answered while the MMAs below are issued
                        const uint32_t idesc = p.idesc | (static_cast<uint32_t>(i) << 29) | (static_cast<uint32_t>(i) << 4);
                        if (f8_elect()) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) f8_mma<CG>(d, at + 2 * j, at + (kF8TileM * 128 >> 4) + 2 * j, idesc, sfa, sfa + 4, q > 0 || i > 0 || j > 0);
                            f8_commit<CG>(empty);
                            if (i == slices - 1) f8_commit<CG>(slot);
                        }
                        __syncwarp();
                        if (i == min(1, slices - 1) && !(ok = stage_scales())) break;
                    }
                }
                if (ok && f8_elect()) f8_commit<CG>(accf0 + 8 * buf);
                __syncwarp();
            }
            if (f8_elect()) f8_commit_here<CG>(done0);
            __syncwarp();
            f8_settle(done0, 0);
        }
    } else if (warp < kF8EpiWarp) {
        // Warps 2 and 3 take every other run.  A warp asks for its next run after the hand-over of the one before (the fence of
        // a hand-over would wait for loads in flight).
        if (CG == 2 && warp == 3) {
            sf_settle();
            if (sf_turn < my_turns) fetch(sf_turn, sf_run);
        }
        uint32_t handed = 0;                                 // quads of this warp so far; it fills four slots of its own in turn
        bool ok = true;
        while (ok && sf_turn < my_turns) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (4 * sf_run + q >= quads) break;
                const uint32_t n = handed + q, slot = 4 * (warp - 2) + (n & 3u), dst = sf0 + slot * kF8SfSlotBytes + lane * 16;
                if (!(ok = f8_wait(sfe0 + 8 * slot, ((n >> 2) & 1u) ^ 1u, abort_flag, p.patience))) break;
#pragma unroll
                for (int j = 0; j < 3; ++j)
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + 512 * j), "r"(f8_word(w[4 * j], q)), "r"(f8_word(w[4 * j + 1], q)),
                                 "r"(f8_word(w[4 * j + 2], q)), "r"(f8_word(w[4 * j + 3], q)) : "memory");
                if (CG == 1) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) f8_arrive(sff0 + 8 * slot);
                }
            }
            if (!ok) break;
            const int count = min(4, quads - 4 * sf_run);
            if (CG == 2) {                                   // one hand-over for the run: a release over the cluster takes about 1500 clocks
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    f8_release_cluster();
                    for (int q = 0; q < count; ++q) f8_arrive_leader(sff0 + 8 * (4 * (warp - 2) + ((handed + q) & 3u)));
                }
            }
            handed += count;
            sf_run += 2;
            sf_settle();
            if (ok && sf_turn < my_turns) fetch(sf_turn, sf_run);
        }
    } else if (warp >= kF8EpiWarp) {
        const int row0 = (warp & 3) * 32;
        const uint32_t stage = stage0 + (warp - kF8EpiWarp) * 32 * kPitch;
        const uint32_t lanes = static_cast<uint32_t>(row0) << 16;
        T* const y = static_cast<T*>(p.y);
        PhiloxKey key;
        if (p.drop.rng != nullptr) key = PhiloxKey(p.drop.rng);
        // the bias of column n + lane
        auto bias_of = [&](int n) { return p.bias != nullptr ? __uint_as_float(read4(p.bias + min(n + lane, p.N - 1))) : 0.0f; };
        // 32 x 32 results: f holds this lane's row, columns n ..., bias is bias_of(n), asked for ahead
        auto emit = [&](float (&f)[32], int m0, int n, int rows, float bias) {
            const int cols = min(32, p.N - n);
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] *= p.alpha;
            if (p.bias != nullptr) {                         // one load a lane, handed around (32 loads a lane cost 650 clocks)
#pragma unroll
                for (int j = 0; j < 32; ++j) f[j] += __shfl_sync(0xFFFFFFFFu, bias, j);
            }
            if (p.drop.rng != nullptr) {
                const unsigned m = f8_keep32(key, p.drop.threshold, static_cast<unsigned long long>(m0 + lane) * p.N + n);
#pragma unroll
                for (int j = 0; j < 32; ++j) f[j] = (m >> j) & 1u ? f[j] : 0.0f;
            }
            constexpr int kPer = 16 / sizeof(T), kPieces = 32 / kPer;           // of a 32-element row
            __syncwarp();                                                       // the last chunk's readers are through
#pragma unroll
            for (int j = 0; j < kPieces; ++j) f8_put16<T>(stage + lane * kPitch + 16 * j, f + j * kPer);
            __syncwarp();
            if (p.vec && cols == 32) {
                const int piece = lane % kPieces, r0 = lane / kPieces;
                T* dst = y + static_cast<long long>(m0 + r0) * p.ldy + n + piece * kPer;
                uint4 e[kPieces];
#pragma unroll
                for (int j = 0; j < kPieces; ++j) e[j] = f8_get16(stage + (r0 + j * (32 / kPieces)) * kPitch + 16 * piece);
                if (rows >= 32) {
#pragma unroll
                    for (int j = 0; j < kPieces; ++j) *reinterpret_cast<uint4*>(dst + j * (32 / kPieces) * p.ldy) = e[j];
                } else {
#pragma unroll
                    for (int j = 0; j < kPieces; ++j)
                        if (r0 + j * (32 / kPieces) < rows) *reinterpret_cast<uint4*>(dst + j * (32 / kPieces) * p.ldy) = e[j];
                }
            } else if (lane < cols) {
                T* dst = y + static_cast<long long>(m0) * p.ldy + n + lane;
                const int live_rows = min(rows, 32);
#pragma unroll 8
                for (int r = 0; r < live_rows; ++r) dst[r * p.ldy] = f8_get<T>(stage + r * kPitch + lane * sizeof(T));
            }
        };
        auto release = [&](uint32_t buf) {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) { if (CG == 2) f8_arrive_leader(acce0 + 8 * buf); else f8_arrive(acce0 + 8 * buf); }
        };
        // an accumulator may take long where the reduction is: a second for every 65536 slices, which take 26 ms
        const int patience = p.patience * (1 + (kb_n >> 16));
        uint32_t item = 0;                                   // accumulators read so far
        bool ok = true;
        int t = first;
        for (; t < ntiles; t += step) {
            int tm, tn;
            f8_tile(t, p.mt, p.nt, tm, tn);
            const int m0 = (tm * CG + rank) * kF8TileM + row0, n0 = tn * p.tile_n, rows = p.M - m0;
            if constexpr (SUMS) {
                // the eight warps share the columns in halves of up to 96
                const int half = p.tile_n / 2, c0 = half * ((warp - kF8EpiWarp) >> 2);
                float sums[kF8SumTileN / 64][32];
                for (int q = 0; q < quads; q += kF8SumQuads, ++item) {
                    const uint32_t buf = item & 1u;
                    if (!(ok = f8_wait(accf0 + 8 * buf, (item >> 1) & 1u, abort_flag, patience))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (int i = 0; i < kF8SumTileN / 64; ++i) {
                        if (32 * i >= half) break;
                        uint32_t v[32];
                        f8_tmem_ld32(v, tmem + buf * d_step + lanes + c0 + 32 * i);
#pragma unroll
                        for (int j = 0; j < 32; ++j) sums[i][j] = q == 0 ? __uint_as_float(v[j]) : sums[i][j] + __uint_as_float(v[j]);
                    }
                    release(buf);
                }
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < kF8SumTileN / 64; ++i) {
                    if (32 * i >= half) break;
                    const int n = n0 + c0 + 32 * i;
                    if (n < p.N && rows > 0) emit(sums[i], m0, n, rows, bias_of(n));
                }
            } else {
                const int chunks = p.tile_n / 32;
                const uint32_t buf = item & 1u;
                auto column = [&](int i) { return 32 * (overlap && buf == 0 ? (i == 0 ? chunks - 1 : i - 1) : i); };
                const int half = (warp - kF8EpiWarp) >> 2;   // the chunks' turn: four warps the even ones, four the odd ones
                float bias_next = bias_of(n0 + column(half));
                if (!(ok = f8_wait(accf0 + 8 * buf, (item >> 1) & 1u, abort_flag, patience))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t src = tmem + buf * d_step + lanes;
                for (int i = half; i < chunks; i += 2) {
                    const int c = column(i), n = n0 + c;
                    const float bias = bias_next;
                    if (i + 2 < chunks) bias_next = bias_of(n0 + column(i + 2));
                    const bool live = n < p.N && rows > 0;   // the same for the whole warp
                    uint32_t v[32];
                    if (live) f8_tmem_ld32(v, src + c);
                    if (overlap && i == 0) {
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) { if (CG == 2) f8_arrive_leader(accp); else f8_arrive(accp); }
                    }
                    if (!live) continue;
                    float f[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]);
                    emit(f, m0, n, rows, bias);
                }
                release(buf);
                ++item;
            }
        }
        if (!ok) f8_blank<T, SUMS>(p, t, step, CG, rank);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (CG == 2) f8_cluster_sync(); else __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (tid == 0 && s_abort) f8_report(p.error);
    if (warp == 3) {
        if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// ---- products of few tiles --------------------------------------------------------------------------------------------
// y = alpha A B^T + bias for few rows of A (serving) or small matrices: one tile of 128 rows of B by tile_c rows of A, and
// the reduction cut over the S blocks of a cluster, so that 4096 x 4096 weights and one row of A keep 128 SMs reading
// instead of 32.  B supplies the MMA's 128 rows whatever M is, so no tensor-core row is wasted on a missing token; each
// block requests its whole share of B at once (up to kF8MaxStages slices).  The S partial tiles meet in shared memory: every
// block adds up its share of the columns over the cluster in the order of the blocks (bit for bit repeatable) and stores
// it.  No workspace, no counters, one launch.  Measured back to back, bf16 results, against the best tile of
// fp8_gemm_kernel: 1 x 4096 x 4096 5.6 us (12.3; the weights' 17 MB pass at 3.0 TB/s), 64 x 4096 x 4096 7.2 us (11.5),
// 256 x 1000 x 2048 5.6 us (7.3).
// (128 bytes, with the two maps 384 of a launch: at 400 the same kernel takes 0.2 to 0.6 us longer)
struct Fp8SplitParams {
    const uint8_t* sa;
    const uint8_t* sb;
    long long ldsa, ldsb;
    const float* bias;
    void* y;
    long long ldy;
    DropState drop;
    int* error;
    float alpha;
    int patience;
    int M, N, kblocks;
    int tile_c, ct;                          // rows of A to a tile, column tiles
    uint32_t tmem_cols;
    uint32_t idesc;
    uint8_t a_shift, b_shift, splits, stages;
};
static_assert(sizeof(Fp8SplitParams) <= 128, "see above");

__device__ __forceinline__ float f8_remote(uint32_t addr, uint32_t block)
{
    float v;
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.f32 %0, [r];\n\t}"
                 : "=f"(v) : "r"(addr), "r"(block) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t f8_cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// CUT: more than one block to a tile.  A form for each (and the rare path marked as such): what follows the product is short
// enough for fetching its instructions to show, 256 x 1000 x 2048 5.6 instead of 6.1 us, 128 x 2048 x 1000 4.4 instead of 4.7.
template <class T, bool CUT>
__global__ void __launch_bounds__(kF8SplitThreads)
fp8_split_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a, const Fp8SplitParams p)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    __shared__ __align__(8) uint64_t s_full[kF8MaxStages], s_empty[kF8MaxStages], s_sf[kF8MaxQuads], s_acc, s_mma_done;
    __shared__ unsigned s_keep[kF8TileM][4];                 // [row of A]: a bit for each row of B
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
    const uint32_t rank = CUT ? f8_cluster_rank() : 0u;
    const int tile = blockIdx.x / (CUT ? p.splits : 1), n0 = (tile / p.ct) * kF8TileM, m0 = (tile % p.ct) * p.tile_c;
    const int kb0 = CUT ? static_cast<int>(static_cast<long long>(p.kblocks) * rank / p.splits) : 0;
    const int kb1 = CUT ? static_cast<int>(static_cast<long long>(p.kblocks) * (rank + 1) / p.splits) : p.kblocks;
    const uint32_t smem0 = (f8_smem(smem_raw) + 1023u) & ~1023u;
    const uint32_t stage_bytes = (kF8TileM + p.tile_c) * 128, sf0 = smem0 + p.stages * stage_bytes;
    const uint32_t full0 = f8_smem(s_full), empty0 = f8_smem(s_empty), sff0 = f8_smem(s_sf), acc0 = f8_smem(&s_acc), done0 = f8_smem(&s_mma_done);
    volatile int* abort_flag = &s_abort;
    if (warp == 0) {
        if (lane == 0) { s_abort = 0; f8_bar_init(acc0, 1); f8_bar_init(done0, 1); }
        if (lane < kF8MaxStages) { f8_bar_init(full0 + 8 * lane, 1); f8_bar_init(empty0 + 8 * lane, 1); }
        for (int i = lane; i < kF8MaxQuads; i += 32) f8_bar_init(sff0 + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    } else if (warp == 1) {
        if (f8_elect()) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
        }
    } else if (warp == 3) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(f8_smem(&s_tmem)), "r"(p.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    after_previous();
    const uint32_t tmem = s_tmem;
    const int q0 = kb0 >> 2, quads = ((kb1 + 3) >> 2) - q0;      // of this block, by place in a scale row
    uint32_t issued = 0;                                     // slices asked for (warp 0)
    bool ok = true;

    if (warp == 0) {
        uint32_t s = 0, parity = 1;
        for (int kb = kb0; kb < kb1; ++kb, ++issued) {
            if (!f8_wait(empty0 + 8 * s, parity, abort_flag, p.patience)) break;
            if (f8_elect()) {
                f8_expect(full0 + 8 * s, stage_bytes);
                f8_tma<1>(smem0 + s * stage_bytes, &map_b, kb * 128, n0, full0 + 8 * s);
                f8_tma<1>(smem0 + s * stage_bytes + kF8TileM * 128, &map_a, kb * 128, m0, full0 + 8 * s);
            }
            __syncwarp();
            if (++s == static_cast<uint32_t>(p.stages)) { s = 0; parity ^= 1u; }
        }
    } else if (warp == 1) {
        const uint32_t a_first = static_cast<uint32_t>(f8_desc(smem0)), a_step = stage_bytes >> 4, a_end = a_first + p.stages * a_step;
        uint32_t a_lo = a_first, full = full0, parity = 0, sfa = tmem + p.tile_c - 8;
        bool ready = false;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (kb == kb0 || (kb & 3) == 0) {
                const int q = (kb >> 2) - q0;
                sfa += 8;
                if (!(ok = f8_wait(sff0 + 8 * q, 0, abort_flag, p.patience))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (f8_elect()) {
                    f8_copy_scales<1>(sfa, f8_sf_desc(sf0 + q * 1024));
                    f8_copy_scales<1>(sfa + 4, f8_sf_desc(sf0 + q * 1024 + 512));
                }
                __syncwarp();
            }
            if (!ready && !(ok = f8_wait(full, parity, abort_flag, p.patience))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t at = a_lo, empty = full + (empty0 - full0);
            a_lo += a_step;
            full += 8;
            if (a_lo == a_end) { a_lo = a_first; full = full0; parity ^= 1u; }
            ready = f8_test(full, parity);
            const uint32_t idesc = p.idesc | (static_cast<uint32_t>(kb & 3) << 29) | (static_cast<uint32_t>(kb & 3) << 4);
            if (f8_elect()) {
#pragma unroll
                for (int j = 0; j < 4; ++j) f8_mma<1>(tmem, at + 2 * j, at + (kF8TileM * 128 >> 4) + 2 * j, idesc, sfa, sfa + 4, kb > kb0 || j > 0);
                f8_commit<1>(empty);
            }
            __syncwarp();
        }
        if (f8_elect()) f8_commit<1>(ok ? acc0 : done0);
        __syncwarp();
    } else if (warp < kF8EpiWarp) {
        // scale words of a quad: lane i takes rows i, i + 32, ... of both operands
        for (int q = warp - 2; q < quads; q += 2) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint8_t* src = j < 4 ? p.sb + static_cast<long long>(min(n0 + lane + 32 * j, p.N - 1) >> p.b_shift) * p.ldsb
                                           : p.sa + static_cast<long long>(min(m0 + lane + 32 * (j - 4), p.M - 1) >> p.a_shift) * p.ldsa;
                w[j] = j < 4 || 32 * (j - 4) < p.tile_c ? read4(src + 4 * (q0 + q)) : 0x7F7F7F7Fu;
            }
            const uint32_t dst = sf0 + q * 1024 + lane * 16;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + 512 * j), "r"(w[4 * j]), "r"(w[4 * j + 1]),
                             "r"(w[4 * j + 2]), "r"(w[4 * j + 3]) : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) f8_arrive(sff0 + 8 * q);
        }
    }
    const int cols = min(p.tile_c, p.M - m0);
    T* const y = static_cast<T*>(p.y) + static_cast<long long>(m0) * p.ldy;
    auto store = [&](int n, int c, float v, float bias) {
        float f = p.alpha * v + bias;
        if (p.drop.rng != nullptr && !((s_keep[c][(n - n0) >> 5] >> ((n - n0) & 31)) & 1u)) f = 0.0f;
        y[c * p.ldy + n] = f8_out<T>(f);
    };
    if (warp >= kF8EpiWarp) {
        if (p.drop.rng != nullptr) {                         // the mask of this block's share, while the product is made
            const PhiloxKey key(p.drop.rng);
            for (int i = tid - 32 * kF8EpiWarp; i < 4 * ((cols - static_cast<int>(rank) + p.splits - 1) / p.splits); i += 128) {
                const int c = static_cast<int>(rank) + p.splits * (i >> 2), n = n0 + 32 * (i & 3);
                if (n < p.N) s_keep[c][i & 3] = f8_keep32(key, p.drop.threshold, static_cast<unsigned long long>(m0 + c) * p.N + n);
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
        }
        if (f8_wait(acc0, 0, abort_flag, p.patience)) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int row = (warp & 3) * 32 + lane, n = n0 + row;
            const float bias = !CUT && p.bias != nullptr && n < p.N ? __uint_as_float(read4(p.bias + n)) : 0.0f;
            for (int c = 0; c < cols; c += 16) {
                uint32_t v[16];
                f8_tmem_ld16(v, tmem + c + (static_cast<uint32_t>((warp & 3) * 32) << 16));
                if constexpr (!CUT) {                        // nothing to meet: straight to y, a warp's lanes side by side
                    if (n < p.N) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) if (c + j < cols) store(n, c + j, __uint_as_float(v[j]), bias);
                    }
                } else {                                     // over the stages: all MMAs are done
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(smem0 + ((c + j) * kF8TileM + row) * 4), "r"(v[j]) : "memory");
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        }
    }
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (__builtin_expect(s_abort, 0)) {                      // once nothing is in flight, NaN for this block's part or its results
        if (warp == 0)
            for (uint32_t j = issued > static_cast<uint32_t>(p.stages) ? issued - p.stages : 0; j < issued; ++j)
                if (!f8_settle(full0 + 8 * (j % p.stages), (j / p.stages) & 1u)) break;
        if (warp == 1) f8_settle(ok ? acc0 : done0, 0);
        __syncthreads();
        const float nan = __uint_as_float(0x7FC00000u);
        if (tid == 0) f8_report(p.error);
        for (int i = tid; i < cols * kF8TileM; i += kF8SplitThreads) {
            const int c = i / kF8TileM, n = n0 + i % kF8TileM;
            if (CUT) asm volatile("st.shared.f32 [%0], %1;" ::"r"(smem0 + 4 * i), "f"(nan) : "memory");
            else if (n < p.N) y[c * p.ldy + n] = f8_out<T>(nan);
        }
        __syncwarp();
    }
    // Tensor memory goes back before this block waits for the others of its cluster: tcgen05.alloc waits without a limit, so a
    // block that kept its columns while it waited for one that still waits for columns could close a circle through a tensor-core
    // kernel of another stream that shares their SMs.
    if (warp == 3) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
    if (!CUT) return;
    f8_cluster_sync();                                       // the parts are in place
    // ---- every block finishes its share of the columns, four at a time so that the reads overlap
    const int row = tid & (kF8TileM - 1), n = n0 + row;
    if (n < p.N) {
        const float bias = p.bias != nullptr ? __uint_as_float(read4(p.bias + n)) : 0.0f;
        const int step = 2 * p.splits;
        for (int c = static_cast<int>(rank) + p.splits * (tid >> 7); c < cols; c += 4 * step) {
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int j = 0; j < p.splits; ++j) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c + i * step < cols) sum[i] += f8_remote(smem0 + ((c + i * step) * kF8TileM + row) * 4, j);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) if (c + i * step < cols) store(n, c + i * step, sum[i], bias);
        }
    }
    f8_cluster_sync();                                       // no block leaves while another reads its part
}

// y = bias (a product over nothing)
template <class T>
__global__ void fp8_bias_kernel(T* y, long long ldy, const float* bias, int M, int N)
{
    after_previous();
    const long long total = static_cast<long long>(M) * N, stride = static_cast<long long>(gridDim.x) * blockDim.x;
    for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += stride) {
        const long long m = i / N, n = i - m * N;
        y[m * ldy + n] = f8_out<T>(bias ? bias[n] : 0.0f);
    }
}

// ---- host side -----------------------------------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled()
{
    static const EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return fn;
}

// rows x 128-byte slices of a byte matrix [R, C] with row pitch ld
static int operand_map(CUtensorMap* map, const void* base, long long R, long long C, long long ld, int box_rows)
{
    const EncodeTiled fn = encode_tiled();
    if (fn == nullptr) { set_error("cuTensorMapEncodeTiled is not available"); return ATB_ERR_CUDA; }
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(C), static_cast<cuuint64_t>(R)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
    const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)}, step[2] = {1, 1};
    const CUresult rc = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, step,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) { set_error("cuTensorMapEncodeTiled: error %d", static_cast<int>(rc)); return ATB_ERR_CUDA; }
    return ATB_OK;
}

// the kernels' shared memory is above the default limit: allowed once per device
template <class K>
static cudaError_t allow_smem(K kernel, int bytes, bool (&done)[64])
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev >= 0 && dev < 64 && done[dev])) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
    return e;
}

// blocks of clusters of `size` that the device runs at a time, one to an SM (148 SMs hold 132 blocks of clusters of 4)
static int fp8_cluster_blocks(int size)
{
    static int known[64][9];
    static bool done[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sm_count() / size * size;
    if (known[dev][size] == 0) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(size);
        cfg.blockDim = dim3(kF8SplitThreads);
        cfg.dynamicSmemBytes = kF8SplitSmem;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = size;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (allow_smem(fp8_split_kernel<float, true>, kF8SplitSmem, done) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, fp8_split_kernel<float, true>, &cfg) != cudaSuccess || n <= 0) {
            cudaGetLastError();                              // an estimate does; the launch reports what is wrong
            n = sm_count() / size;
        }
        known[dev][size] = n * size;
    }
    return known[dev][size];
}

// How a product is cut: the kernel, tile and number of blocks to a tile with the least estimated time.  Microseconds as
// measured on B200 (8-bit operands of random numbers): a slice (128 steps) of a tile costs 0.06 + 0.0013 per column to a
// pair of blocks (the MMAs; 0.22 at least, the issue), 0.165 + 0.00106 per column to a single block; a tile besides, 0.4 +
// 0.003 per column; a launch with a first load, 3.5 (pairs: 4.6).  The split kernel: 0.14 + 0.0016 per row of A for a slice,
// 0.8 + 0.025 per row of A and 0.06 per block of the cluster for a tile, 2.0 for the launch, 2.8 with clusters (blocks that
// share an SM take nearly as long as one after the other, so they count as further rounds).  Over 600 products drawn at
// random (rows 1 to 4000, columns and reduction 64 to 8192, bf16 and fp32 results) the choice took 1.02 of the time of the
// best choice on average and 1.37 at worst.
struct Fp8Plan {
    int cg, tile;            // fp8_gemm_kernel: blocks to a tile, columns
    int splits;              // fp8_split_kernel where not 0: blocks to a tile; tile = rows of A
};

// A reduction over more than sums_from slices is added up from partial sums (SUMS): tiles of 64, 128 or 192 columns, and no block
// of the split kernel gets more slices than that.
static Fp8Plan fp8_plan(int M, int N, int kblocks, int sums_from)
{
    const bool sums = kblocks > sums_from;
    Fp8Plan best{1, sums ? 64 : 32, 0};
    double least = 1e300;
    const int sms = sm_count();
    for (int cg = 1; cg <= 2; ++cg) {
        const double mt = (M + cg * kF8TileM - 1) / (cg * kF8TileM);
        const int unit = sums ? 64 : 32;
        for (int tile = unit; tile <= (sums ? kF8SumTileN : kF8MaxTileN); tile += unit) {
            if (tile > unit && tile - unit >= N) break;
            const double nt = (N + tile - 1) / tile, waves = ceil(mt * nt / (sms / cg));
            const double slice = cg == 2 ? fmax(0.22, 0.06 + 0.0013 * tile) : 0.165 + 0.00106 * tile;
            const double t = waves * (kblocks * slice + 0.4 + 0.003 * tile) + (cg == 2 ? 4.6 : 3.5);
            if (t < least) { least = t; best = Fp8Plan{cg, tile, 0}; }
        }
    }
    const double nt = (N + kF8TileM - 1) / kF8TileM;
    for (int tile = 16; tile <= kF8TileM; tile += 16) {
        if (tile > 16 && tile - 16 >= M) break;
        const double mt = (M + tile - 1) / tile;
        if (mt * nt > 16.0 * sms) continue;                  // many tiles: never the better kernel
        for (int splits = 1; splits <= 8 && splits <= kblocks; ++splits) {
            const int slices = (kblocks + splits - 1) / splits;
            if (slices / 4 + 2 > kF8MaxQuads || slices > sums_from) continue;
            const double waves = ceil(mt * nt * splits / fp8_cluster_blocks(splits));
            const double t = waves * (slices * (0.14 + 0.0016 * tile) + 0.8 + 0.025 * tile + 0.06 * splits) + (splits > 1 ? 2.8 : 2.0);
            if (t < least) { least = t; best = Fp8Plan{1, tile, splits}; }
        }
    }
    return best;
}

template <class T, int CG, bool SUMS>
static int launch_fp8(const CUtensorMap& ma, const CUtensorMap& mb, const Fp8Params& p, cudaStream_t s)
{
    static bool done[64];
    cudaError_t e = allow_smem(fp8_gemm_kernel<T, CG, SUMS>, kF8Smem, done);
    const int tiles = p.mt * p.nt, fit = sm_count() / CG;
    if (e == cudaSuccess)
        e = launch_after(fp8_gemm_kernel<T, CG, SUMS>, dim3(CG * (tiles < fit ? tiles : fit)), dim3(kF8Threads), kF8Smem, s,
                         CG == 2 ? 2 : 0, ma, mb, p);
    if (e != cudaSuccess) { set_error("fp8_gemm_kernel: %s", cudaGetErrorString(e)); return ATB_ERR_CUDA; }
    return check_launch("fp8_gemm_kernel");
}

template <class T>
static int launch_fp8_cg(const CUtensorMap& ma, const CUtensorMap& mb, const Fp8Params& p, int cg, bool sums, cudaStream_t s)
{
    if (sums) return cg == 2 ? launch_fp8<T, 2, true>(ma, mb, p, s) : launch_fp8<T, 1, true>(ma, mb, p, s);
    return cg == 2 ? launch_fp8<T, 2, false>(ma, mb, p, s) : launch_fp8<T, 1, false>(ma, mb, p, s);
}

template <class T, bool CUT>
static int launch_split(const CUtensorMap& mb, const CUtensorMap& ma, const Fp8SplitParams& p, int tiles, size_t smem, cudaStream_t s)
{
    static bool done[64];
    cudaError_t e = allow_smem(fp8_split_kernel<T, CUT>, kF8SplitSmem, done);
    if (e == cudaSuccess) e = launch_after(fp8_split_kernel<T, CUT>, dim3(tiles * p.splits), dim3(kF8SplitThreads), smem, s, p.splits, mb, ma, p);
    if (e != cudaSuccess) { set_error("fp8_split_kernel: %s", cudaGetErrorString(e)); return ATB_ERR_CUDA; }
    return check_launch("fp8_split_kernel");
}

template <class T>
static int launch_split_cut(const CUtensorMap& mb, const CUtensorMap& ma, const Fp8SplitParams& p, int tiles, size_t smem, cudaStream_t s)
{
    return p.splits > 1 ? launch_split<T, true>(mb, ma, p, tiles, smem, s) : launch_split<T, false>(mb, ma, p, tiles, smem, s);
}

template <class T>
static int launch_bias(void* y, long long ldy, const float* bias, int M, int N, cudaStream_t s)
{
    launch_after(fp8_bias_kernel<T>, dim3(grid_for(static_cast<long long>(M) * N, 256, 16 * sm_count())), dim3(256), 0, s, 0, static_cast<T*>(y), ldy, bias, M, N);
    return check_launch("fp8_bias_kernel");
}

// A word that the kernels of every device set when a block gave up, in pinned host memory so that the host sees it without
// waiting for a device: 4 bytes, allocated by the first product and kept.
static std::atomic<int*> g_error_word{nullptr};
static std::atomic<int> g_patience{kF8Patience};

static int* error_word()
{
    int* word = g_error_word.load(std::memory_order_acquire);
    if (word != nullptr) return word;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;      // the first product may come inside a capture
    cudaThreadExchangeStreamCaptureMode(&mode);
    int* fresh = nullptr;
    if (cudaHostAlloc(reinterpret_cast<void**>(&fresh), sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped) == cudaSuccess) {
        *fresh = 0;
        if (g_error_word.compare_exchange_strong(word, fresh)) word = fresh;
        else cudaFreeHost(fresh);                            // another thread was first: `word` is its
    } else {
        cudaGetLastError();
    }
    cudaThreadExchangeStreamCaptureMode(&mode);
    return word;
}

}  // namespace atb

using namespace atb;

extern "C" int atb_fp8_gemm(const void* a, int a_f8, long long lda, const uint8_t* sa, long long ldsa, int a_block_rows,
                            const void* b, int b_f8, long long ldb, const uint8_t* sb, long long ldsb, int b_block_rows,
                            const float* bias, float alpha, void* y, int y_dtype, long long ldy, int M, int N, int K,
                            int drop_threshold, const void* rng, void* stream)
{
    ATB_REQUIRE(M >= 0 && N >= 0 && K >= 0, "negative dimension");
    ATB_REQUIRE(M <= 0x7FFFF000 && N <= 0x7FFFF000 && K <= 0x7FFFF000, "dimension too large");   // tile coordinates are 32-bit
    ATB_REQUIRE((a_f8 == ATB_E4M3 || a_f8 == ATB_E5M2) && (b_f8 == ATB_E4M3 || b_f8 == ATB_E5M2), "operands must be e4m3 or e5m2");
    ATB_REQUIRE((a_block_rows == 1 || a_block_rows == 128) && (b_block_rows == 1 || b_block_rows == 128), "block rows must be 1 or 128");
    ATB_REQUIRE(y_dtype == ATB_F32 || y_dtype == ATB_BF16 || y_dtype == ATB_F16, "y must be fp32, bf16 or fp16");
    ATB_REQUIRE(drop_threshold >= 0 && drop_threshold <= 65536, "threshold must lie in [0, 65536]");
    ATB_REQUIRE(drop_threshold == 0 || (rng != nullptr && aligned_to(rng, 8)), "dropout needs an 8-byte aligned state");
    if (M == 0 || N == 0) return ATB_OK;
    ATB_REQUIRE(y != nullptr && ldy >= N, "null y, or its row pitch below N");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int size = y_dtype == ATB_F32 ? 4 : 2;
    ATB_REQUIRE(aligned_to(y, size) && aligned_to(bias, 4), "y and bias must be aligned to their elements");
    if (K == 0) {
        ATB_REQUIRE(drop_threshold == 0 || bias == nullptr, "dropout needs a product");
        if (y_dtype == ATB_F32) return launch_bias<float>(y, ldy, bias, M, N, s);
        if (y_dtype == ATB_BF16) return launch_bias<__nv_bfloat16>(y, ldy, bias, M, N, s);
        return launch_bias<__half>(y, ldy, bias, M, N, s);
    }
    ATB_REQUIRE(a && b && sa && sb, "null pointer");
    ATB_REQUIRE(aligned_to(a, 16) && aligned_to(b, 16) && lda >= K && ldb >= K && lda % 16 == 0 && ldb % 16 == 0,
                "operand rows must start on 16-byte boundaries");
    const int kblocks = (K + 127) / 128;
    ATB_REQUIRE(aligned_to(sa, 4) && aligned_to(sb, 4) && ldsa >= kblocks && ldsb >= kblocks && ldsa % 4 == 0 && ldsb % 4 == 0,
                "scale rows must start on 4-byte boundaries");

    int* const error = error_word();
    if (error == nullptr) { set_error("no pinned memory for the product's error word"); return ATB_ERR_CUDA; }
    if (__atomic_load_n(error, __ATOMIC_RELAXED) != 0 && __atomic_exchange_n(error, 0, __ATOMIC_ACQ_REL) != 0) {
        set_error("an earlier product gave up waiting for its operands: the results that it left out are NaN (this call has done nothing)");
        return ATB_ERR_CUDA;
    }
    const int patience = g_patience.load(std::memory_order_relaxed);

    Fp8Params p{};
    p.patience = patience; p.error = error;
    p.sa = sa; p.sb = sb; p.ldsa = ldsa; p.ldsb = ldsb;
    p.a_shift = a_block_rows == 128 ? 7 : 0; p.b_shift = b_block_rows == 128 ? 7 : 0;
    p.sf_vec = aligned_to(sa, 16) && ldsa % 16 == 0 && aligned_to(sb, 16) && ldsb % 16 == 0;
    p.bias = bias; p.alpha = alpha; p.y = y; p.ldy = ldy; p.M = M; p.N = N; p.kblocks = kblocks;
    const int sums_from = y_dtype == ATB_F32 ? kF8SumsFrom : y_dtype == ATB_F16 ? kF8SumsFromFp16 : kF8SumsFromBf16;
    const Fp8Plan plan = fp8_plan(M, N, kblocks, sums_from);
    const bool sums = kblocks > sums_from && !plan.splits;
    const DropState drop{drop_threshold ? static_cast<const unsigned long long*>(rng) : nullptr, static_cast<unsigned>(drop_threshold)};
    const uint32_t formats = (1u << 23);                     // scales are powers of two (ue8m0)
    CUtensorMap ma, mb;
    if (plan.splits) {
        Fp8SplitParams q{sa, sb, ldsa, ldsb, bias, y, ldy, drop, error, alpha, patience, M, N, kblocks};
        q.a_shift = static_cast<uint8_t>(p.a_shift);
        q.b_shift = static_cast<uint8_t>(p.b_shift);
        q.tile_c = plan.tile;
        q.ct = (M + plan.tile - 1) / plan.tile;
        q.splits = static_cast<uint8_t>(plan.splits);
        const int kbs = (kblocks + plan.splits - 1) / plan.splits, quads = kbs / 4 + 2, stage = (kF8TileM + plan.tile) * 128;
        const int sums = plan.tile * kF8TileM * 4;           // the partial tile takes the stages' place
        int stages = (kF8SplitSmem - 1024 - quads * 1024) / stage;
        stages = stages < kbs ? stages : kbs;
        stages = stages < kF8MaxStages ? stages : kF8MaxStages;
        stages = stages * stage >= sums ? stages : (sums + stage - 1) / stage;
        q.stages = static_cast<uint8_t>(stages);
        q.tmem_cols = 32;
        while (q.tmem_cols < static_cast<uint32_t>(plan.tile + 8 * quads)) q.tmem_cols *= 2;
        q.idesc = formats | (b_f8 == ATB_E5M2 ? 1u << 7 : 0u) | (a_f8 == ATB_E5M2 ? 1u << 10 : 0u) | (static_cast<uint32_t>(plan.tile >> 3) << 17) | (1u << 27);
        // At least the tensor memory's share of an SM's 228 KB: blocks that fit an SM together then find their columns at once
        // instead of waiting for a neighbour's.
        const size_t share = 456 * static_cast<size_t>(q.tmem_cols) - 1024;
        size_t smem = 1024 + static_cast<size_t>(stages) * stage + static_cast<size_t>(quads) * 1024;
        smem = smem < share ? share : smem;
        smem = smem < kF8SplitSmem ? smem : kF8SplitSmem;    // (which leaves no room for a second block either)
        const int tiles = ((N + kF8TileM - 1) / kF8TileM) * q.ct;
        int rc = operand_map(&mb, b, N, K, ldb, kF8TileM);
        if (rc == ATB_OK) rc = operand_map(&ma, a, M, K, lda, plan.tile);
        if (rc != ATB_OK) return rc;
        if (y_dtype == ATB_F32) return launch_split_cut<float>(mb, ma, q, tiles, smem, s);
        if (y_dtype == ATB_BF16) return launch_split_cut<__nv_bfloat16>(mb, ma, q, tiles, smem, s);
        return launch_split_cut<__half>(mb, ma, q, tiles, smem, s);
    }
    const int cg = plan.cg;
    p.tile_n = plan.tile;
    p.mt = (M + cg * kF8TileM - 1) / (cg * kF8TileM);
    p.nt = (N + p.tile_n - 1) / p.tile_n;
    ATB_REQUIRE(static_cast<long long>(p.mt) * p.nt < (1LL << 30), "too many tiles");
    const int stage = kF8TileM * 128 + p.tile_n / cg * 128;
    p.stages = (kF8Smem - 1024 - kF8SfSlots * kF8SfSlotBytes - kF8EpiWarps * 32 * (32 * size + 16)) / stage;
    if (p.stages > kF8MaxStages) p.stages = kF8MaxStages;
    p.idesc = formats | (a_f8 == ATB_E5M2 ? 1u << 7 : 0u) | (b_f8 == ATB_E5M2 ? 1u << 10 : 0u) |
              (static_cast<uint32_t>(p.tile_n >> 3) << 17) | (static_cast<uint32_t>(cg) << 27);
    p.vec = aligned_to(y, 16) && (ldy * size) % 16 == 0;
    p.drop = drop;
    int rc = operand_map(&ma, a, M, K, lda, kF8TileM);
    if (rc == ATB_OK) rc = operand_map(&mb, b, N, K, ldb, p.tile_n / cg);
    if (rc != ATB_OK) return rc;
    if (y_dtype == ATB_F32) return launch_fp8_cg<float>(ma, mb, p, cg, sums, s);
    if (y_dtype == ATB_BF16) return launch_fp8_cg<__nv_bfloat16>(ma, mb, p, cg, sums, s);
    return launch_fp8_cg<__half>(ma, mb, p, cg, sums, s);
}

extern "C" int atb_fp8_status(int* status)
{
    ATB_REQUIRE(status != nullptr, "null pointer");
    const cudaError_t e = cudaDeviceSynchronize();
    if (e != cudaSuccess) { set_error("cudaDeviceSynchronize: %s", cudaGetErrorString(e)); return ATB_ERR_CUDA; }
    int* const error = g_error_word.load(std::memory_order_acquire);
    *status = error != nullptr ? __atomic_exchange_n(error, 0, __ATOMIC_ACQ_REL) : 0;
    return ATB_OK;
}

extern "C" int atb_fp8_patience(int looks)
{
    return g_patience.exchange(looks < 0 ? kF8Patience : looks < kF8Patience ? looks : kF8Patience);
}

// Matrix product of 8-bit floating point operands with a power-of-two scale for each block of 128.
//
//   y[m, n] = alpha * sum_k  A[m, k] 2^(sa[m', k/128] - 127)  B[n, k] 2^(sb[n', k/128] - 127)  + bias[n]
//
// with m' = m or m / 128 (one scale for a row's block, or for a 128 x 128 block), n' likewise; the sum in fp32 in the
// tensor core, one rounding at the end.  The scales are applied by the tensor core itself: tcgen05.mma
// kind::mxf8f6f4.block_scale takes one exponent byte per row and 32 steps of the reduction from tensor memory, and four
// consecutive instructions read the same byte.  So the product runs at the rate of an unscaled 8-bit product; promoting
// every 128-step partial sum through registers instead would cost a read of the accumulator per 128 steps.
//
// fp8_gemm_kernel, for products of many tiles: one block of threads per SM (CG = 1), or two blocks on two SMs that work on
// one tile of 256 rows (CG = 2), walk over the output tiles:
//   warp 0      one thread requests the operand tiles by TMA (128-byte swizzle, one 128-step slice = one 128-byte row);
//   warp 1      one thread moves the scales to tensor memory (tcgen05.cp) and issues the MMAs (of the pair: the first
//               block's thread, for both);
//   warp 2      gathers the scale bytes of four slices at a time (one 32-bit word per row) into the order in which
//               tcgen05.cp wants them: 32 rows of 16 bytes, word j of row i = operand row i + 32 j;
//   warp 3      owns the tensor-memory allocation;
//   warps 4-7   read finished accumulators, scale, add the bias and store, 32 x 32 elements at a time through shared
//               memory so that a row's bytes leave together.
// Two accumulators let the epilogue of a tile run under the MMAs of the next.  Why pairs: each block of a pair holds its
// own 128 rows of A and half the rows of B and the tensor core reads both halves, so a slice of a 256 x 224 tile costs
// each SM 30 KB instead of the 44 KB of a 128 x 224 tile, and what bounds the product is the path from L2 to the SMs.
//
// fp8_split_kernel, for products of few tiles (serving, small heads): see there.
//
// Operand rows beyond M or N and steps beyond K are zeros that TMA fills in; scale bytes beyond the last block are
// never selected, and rows beyond the last get 1.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "philox.cuh"

namespace atb {

__device__ int g_fp8_status = 0;                      // 1: a block gave up waiting

constexpr int kF8Threads = 256, kF8EpiWarp = 4;
constexpr int kF8TileM = 128, kF8MaxTileN = 224;          // of one block; a pair's tile has twice the rows
constexpr int kF8SfSlots = 4, kF8SfSlotBytes = 3 * 512;   // 128 rows of A, up to 256 rows of B
constexpr int kF8SfCol = 488, kF8SfCols = 12;             // tensor-memory columns of the two scale buffers
constexpr int kF8Smem = 224 * 1024, kF8MaxStages = 8;
constexpr int kF8Group = 8;                               // row tiles that are walked together (their operands meet in L2)

struct Fp8Params {
    const uint8_t* sa;
    const uint8_t* sb;
    long long ldsa, ldsb;
    int a_shift, b_shift;                // 0: a scale per row, 7: per 128 rows
    const float* bias;
    float alpha;
    void* y;
    long long ldy;
    int M, N, kblocks;
    int tile_n, mt, nt, stages;
    uint32_t idesc;
    bool vec;                            // rows of y start on 16-byte boundaries
    DropState drop;
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
// bounded wait that also gives up when another role of the block has
__device__ __forceinline__ bool f8_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag)
{
    for (int i = 0; i < (1 << 21); ++i) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if ((i & 63) == 63 && *abort_flag) return false;
    }
    *abort_flag = 1;
    return false;
}
// the same shared address in the first block of the pair
__device__ __forceinline__ uint32_t f8_leader(uint32_t addr)
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void f8_arrive_cluster(uint32_t bar)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
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
template <int CG>
__device__ __forceinline__ void f8_mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb, bool accumulate)
{
    const uint32_t acc = accumulate ? 1u : 0u;
    if (CG == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc) : "memory");
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

template <class T> __device__ __forceinline__ T f8_out(float v);
template <> __device__ __forceinline__ float f8_out<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 f8_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half f8_out<__half>(float v) { return __float2half_rn(v); }

// row and column tile of the t-th output tile: kF8Group row tiles at a time, column by column
__device__ __forceinline__ void f8_tile(int t, int mt, int nt, int& tm, int& tn)
{
    const int per = kF8Group * nt, g = t / per, rows = min(kF8Group, mt - g * kF8Group), in = t - g * per;
    tn = in / rows;
    tm = g * kF8Group + (in - tn * rows);
}

template <class T, int CG>
__global__ void __launch_bounds__(kF8Threads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Fp8Params p)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    __shared__ __align__(8) uint64_t s_full[kF8MaxStages], s_empty[kF8MaxStages], s_sf_full[kF8SfSlots], s_sf_empty[kF8SfSlots], s_acc_full[2], s_acc_empty[2];
    constexpr int kPitch = 32 * sizeof(T) + 16;              // of a staged row: 16-byte accesses without bank conflicts
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = CG == 2 ? static_cast<int>(blockIdx.x & 1u) : 0;
    const int first = blockIdx.x / CG, step = gridDim.x / CG;
    const uint32_t smem0 = (f8_smem(smem_raw) + 1023u) & ~1023u;
    const int b_rows = p.tile_n / CG;                        // rows of B that this block holds
    const uint32_t stage_bytes = kF8TileM * 128 + b_rows * 128;
    const uint32_t sf0 = smem0 + p.stages * stage_bytes, stage0 = sf0 + kF8SfSlots * kF8SfSlotBytes;
    const uint32_t full0 = f8_smem(s_full), empty0 = f8_smem(s_empty), sff0 = f8_smem(s_sf_full), sfe0 = f8_smem(s_sf_empty);
    const uint32_t accf0 = f8_smem(s_acc_full), acce0 = f8_smem(s_acc_empty);
    volatile int* abort_flag = &s_abort;
    if (tid == 0) {
        s_abort = 0;
        for (int s = 0; s < kF8MaxStages; ++s) { f8_bar_init(full0 + 8 * s, 1); f8_bar_init(empty0 + 8 * s, 1); }
        for (int s = 0; s < kF8SfSlots; ++s) { f8_bar_init(sff0 + 8 * s, CG); f8_bar_init(sfe0 + 8 * s, 1); }
        for (int s = 0; s < 2; ++s) { f8_bar_init(accf0 + 8 * s, 1); f8_bar_init(acce0 + 8 * s, 4 * CG); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (CG == 2) f8_cluster_sync();
    if (warp == 3) {
        if (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(f8_smem(&s_tmem)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(f8_smem(&s_tmem)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (CG == 2) f8_cluster_sync(); else __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;
    const int ntiles = p.mt * p.nt, kb_n = p.kblocks, quads = (kb_n + 3) >> 2;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, parity = 1, issued = 0;
            bool ok = true;
            for (int t = first; t < ntiles && ok; t += step) {
                int tm, tn;
                f8_tile(t, p.mt, p.nt, tm, tn);
                const int m0 = (tm * CG + rank) * kF8TileM, n0 = tn * p.tile_n + rank * b_rows;
                for (int kb = 0; kb < kb_n; ++kb, ++issued) {
                    if (!(ok = f8_wait(empty0 + 8 * s, parity, abort_flag))) break;
                    if (rank == 0) f8_expect(full0 + 8 * s, CG * stage_bytes);
                    const uint32_t bar = CG == 2 ? f8_leader(full0 + 8 * s) : full0 + 8 * s;
                    f8_tma<CG>(smem0 + s * stage_bytes, &map_a, kb * 128, m0, bar);
                    f8_tma<CG>(smem0 + s * stage_bytes + kF8TileM * 128, &map_b, kb * 128, n0, bar);
                    if (++s == static_cast<uint32_t>(p.stages)) { s = 0; parity ^= 1u; }
                }
            }
            // nothing may be in flight when the block ends (all of it has landed unless a role gave up)
            if (rank == 0)
                for (uint32_t j = issued > static_cast<uint32_t>(p.stages) ? issued - p.stages : 0; j < issued; ++j) {
                    int never = 0;
                    f8_wait(full0 + 8 * (j % p.stages), (j / p.stages) & 1u, &never);
                }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            uint32_t s = 0, parity = 0, quad = 0, tile = 0;
            bool ok = true;
            for (int t = first; t < ntiles && ok; t += step, ++tile) {
                const uint32_t buf = tile & 1u, d = tmem + buf * p.tile_n;
                if (!(ok = f8_wait(acce0 + 8 * buf, ((tile >> 1) & 1u) ^ 1u, abort_flag))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int kb = 0; kb < kb_n; ++kb) {
                    const uint32_t sfa = tmem + kF8SfCol + (quad & 1u) * kF8SfCols, sfb = sfa + 4;
                    if ((kb & 3) == 0) {
                        const uint32_t slot = quad % kF8SfSlots;
                        // the buffer's last readers, the MMAs of two quads ago, have to be done
                        if (quad >= 2 && !(ok = f8_wait(sfe0 + 8 * ((quad - 2) % kF8SfSlots), ((quad - 2) / kF8SfSlots) & 1u, abort_flag))) break;
                        if (!(ok = f8_wait(sff0 + 8 * slot, (quad / kF8SfSlots) & 1u, abort_flag))) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t src = sf0 + slot * kF8SfSlotBytes;
                        f8_copy_scales<CG>(sfa, f8_sf_desc(src));
                        f8_copy_scales<CG>(sfb, f8_sf_desc(src + 512));
                        if (p.tile_n > 128) f8_copy_scales<CG>(sfb + 4, f8_sf_desc(src + 1024));
                    }
                    if (!(ok = f8_wait(full0 + 8 * s, parity, abort_flag))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t da = f8_desc(smem0 + s * stage_bytes), db = f8_desc(smem0 + s * stage_bytes + kF8TileM * 128);
                    const uint32_t idesc = p.idesc | (static_cast<uint32_t>(kb & 3) << 29) | (static_cast<uint32_t>(kb & 3) << 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) f8_mma<CG>(d, da + 2 * j, db + 2 * j, idesc, sfa, sfb, kb > 0 || j > 0);
                    f8_commit<CG>(empty0 + 8 * s);
                    if ((kb & 3) == 3 || kb == kb_n - 1) { f8_commit<CG>(sfe0 + 8 * (quad % kF8SfSlots)); ++quad; }
                    if (++s == static_cast<uint32_t>(p.stages)) { s = 0; parity ^= 1u; }
                }
                if (ok) f8_commit<CG>(accf0 + 8 * buf);
            }
        }
    } else if (warp == 2) {
        uint32_t quad = 0;
        bool ok = true;
        for (int t = first; t < ntiles && ok; t += step) {
            int tm, tn;
            f8_tile(t, p.mt, p.nt, tm, tn);
            const int m0 = (tm * CG + rank) * kF8TileM, n0 = tn * p.tile_n;
            for (int q = 0; q < quads; ++q, ++quad) {
                const uint32_t slot = quad % kF8SfSlots, dst = sf0 + slot * kF8SfSlotBytes + lane * 16;
                uint32_t w[12];
#pragma unroll
                for (int j = 0; j < 12; ++j) {
                    const bool is_a = j < 4;
                    const int r = is_a ? m0 + lane + 32 * j : n0 + lane + 32 * (j - 4);
                    const bool in = is_a ? r < p.M : (r < p.N && 32 * (j - 4) < p.tile_n);
                    const uint8_t* src = is_a ? p.sa + static_cast<long long>(r >> p.a_shift) * p.ldsa
                                              : p.sb + static_cast<long long>(r >> p.b_shift) * p.ldsb;
                    w[j] = in ? __ldg(reinterpret_cast<const uint32_t*>(src) + q) : 0x7F7F7F7Fu;
                }
                if (!(ok = f8_wait(sfe0 + 8 * slot, ((quad / kF8SfSlots) & 1u) ^ 1u, abort_flag))) break;
#pragma unroll
                for (int j = 0; j < 3; ++j)
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + 512 * j), "r"(w[4 * j]), "r"(w[4 * j + 1]),
                                 "r"(w[4 * j + 2]), "r"(w[4 * j + 3]) : "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    if (CG == 2) f8_arrive_cluster(f8_leader(sff0 + 8 * slot)); else f8_arrive(sff0 + 8 * slot);
                }
            }
        }
    } else if (warp >= kF8EpiWarp) {
        const int row0 = (warp & 3) * 32;
        uint8_t* const stage = smem_raw + (stage0 - f8_smem(smem_raw)) + (warp & 3) * 32 * kPitch;
        uint32_t tile = 0;
        T* const y = static_cast<T*>(p.y);
        for (int t = first; t < ntiles; t += step, ++tile) {
            int tm, tn;
            f8_tile(t, p.mt, p.nt, tm, tn);
            const int m0 = (tm * CG + rank) * kF8TileM + row0, n0 = tn * p.tile_n;
            const uint32_t buf = tile & 1u;
            if (!f8_wait(accf0 + 8 * buf, (tile >> 1) & 1u, abort_flag)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t src = tmem + buf * p.tile_n + (static_cast<uint32_t>(row0) << 16);
            const int rows = min(32, p.M - m0);
            for (int c = 0; c < p.tile_n; c += 32) {
                const int n = n0 + c;
                if (n >= p.N || rows <= 0) break;            // the same for the whole warp
                uint32_t v[32];
                f8_tmem_ld32(v, src + c);
                const int cols = min(32, p.N - n);
                T out[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    float f = p.alpha * __uint_as_float(v[j]);
                    if (p.bias != nullptr && j < cols) f += __ldg(p.bias + n + j);
                    out[j] = f8_out<T>(f);
                }
                if (p.drop.rng != nullptr) {
                    const PhiloxKey key(p.drop.rng);
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const unsigned keep = philox_keep8_at(key, static_cast<unsigned long long>(m0 + lane) * p.N + n + 8 * g, p.drop.threshold);
#pragma unroll
                        for (int j = 0; j < 8; ++j) if (!((keep >> j) & 1u)) out[8 * g + j] = f8_out<T>(0.0f);
                    }
                }
                constexpr int kPer = 16 / sizeof(T), kPieces = 32 / kPer;       // of a 32-element row
                __syncwarp();                                                   // the last chunk's readers are through
#pragma unroll
                for (int j = 0; j < kPieces; ++j) {
                    uint4 pack;
                    T* e = reinterpret_cast<T*>(&pack);
#pragma unroll
                    for (int i = 0; i < kPer; ++i) e[i] = out[j * kPer + i];
                    *reinterpret_cast<uint4*>(stage + lane * kPitch + 16 * j) = pack;
                }
                __syncwarp();
                if (p.vec && cols == 32) {
                    const int piece = lane % kPieces;
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) {
                        const int r = lane / kPieces + i * (32 / kPieces);
                        if (r < rows)
                            *reinterpret_cast<uint4*>(y + static_cast<long long>(m0 + r) * p.ldy + n + piece * kPer) =
                                *reinterpret_cast<const uint4*>(stage + r * kPitch + 16 * piece);
                    }
                } else if (lane < cols) {
                    for (int r = 0; r < rows; ++r)
                        y[static_cast<long long>(m0 + r) * p.ldy + n + lane] = *reinterpret_cast<const T*>(stage + r * kPitch + lane * sizeof(T));
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (CG == 2) f8_arrive_cluster(f8_leader(acce0 + 8 * buf)); else f8_arrive(acce0 + 8 * buf);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (CG == 2) f8_cluster_sync(); else __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (tid == 0 && s_abort) g_fp8_status = 1;
    if (warp == 3) {
        if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// y = bias (a product over nothing)
template <class T>
__global__ void fp8_bias_kernel(T* __restrict__ y, long long ldy, const float* __restrict__ bias, int M, int N)
{
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

template <class T, int CG>
static int launch_fp8(const CUtensorMap& ma, const CUtensorMap& mb, const Fp8Params& p, cudaStream_t s)
{
    cudaError_t e = cudaFuncSetAttribute(fp8_gemm_kernel<T, CG>, cudaFuncAttributeMaxDynamicSharedMemorySize, kF8Smem);
    const int tiles = p.mt * p.nt, fit = sm_count() / CG;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(CG * (tiles < fit ? tiles : fit));
    cfg.blockDim = dim3(kF8Threads);
    cfg.dynamicSmemBytes = kF8Smem;
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = CG;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = CG == 2 ? 1 : 0;
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, fp8_gemm_kernel<T, CG>, ma, mb, p);
    if (e != cudaSuccess) { set_error("fp8_gemm_kernel: %s", cudaGetErrorString(e)); return ATB_ERR_CUDA; }
    return check_launch("fp8_gemm_kernel");
}

template <class T>
static int launch_fp8_cg(const CUtensorMap& ma, const CUtensorMap& mb, const Fp8Params& p, int cg, cudaStream_t s)
{
    return cg == 2 ? launch_fp8<T, 2>(ma, mb, p, s) : launch_fp8<T, 1>(ma, mb, p, s);
}

template <class T>
static int launch_bias(void* y, long long ldy, const float* bias, int M, int N, cudaStream_t s)
{
    fp8_bias_kernel<T><<<grid_for(static_cast<long long>(M) * N, 256, 16 * sm_count()), 256, 0, s>>>(static_cast<T*>(y), ldy, bias, M, N);
    return check_launch("fp8_bias_kernel");
}

}  // namespace atb

using namespace atb;

extern "C" int atb_fp8_gemm(const void* a, int a_f8, long long lda, const uint8_t* sa, long long ldsa, int a_block_rows,
                            const void* b, int b_f8, long long ldb, const uint8_t* sb, long long ldsb, int b_block_rows,
                            const float* bias, float alpha, void* y, int y_dtype, long long ldy, int M, int N, int K,
                            int drop_threshold, const void* rng, void* stream)
{
    ATB_REQUIRE(M >= 0 && N >= 0 && K >= 0, "negative dimension");
    ATB_REQUIRE((a_f8 == ATB_E4M3 || a_f8 == ATB_E5M2) && (b_f8 == ATB_E4M3 || b_f8 == ATB_E5M2), "operands must be e4m3 or e5m2");
    ATB_REQUIRE((a_block_rows == 1 || a_block_rows == 128) && (b_block_rows == 1 || b_block_rows == 128), "block rows must be 1 or 128");
    ATB_REQUIRE(y_dtype == ATB_F32 || y_dtype == ATB_BF16 || y_dtype == ATB_F16, "y must be fp32, bf16 or fp16");
    ATB_REQUIRE(drop_threshold >= 0 && drop_threshold <= 65536, "threshold must lie in [0, 65536]");
    ATB_REQUIRE(drop_threshold == 0 || (rng != nullptr && aligned_to(rng, 8)), "dropout needs an 8-byte aligned state");
    if (M == 0 || N == 0) return ATB_OK;
    ATB_REQUIRE(y != nullptr && ldy >= N, "null y, or its row pitch below N");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int size = y_dtype == ATB_F32 ? 4 : 2;
    if (K == 0) {
        ATB_REQUIRE(drop_threshold == 0, "dropout needs a product");
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
    ATB_REQUIRE(bias == nullptr || aligned_to(bias, 4), "bias must be 4-byte aligned");

    Fp8Params p{};
    p.sa = sa; p.sb = sb; p.ldsa = ldsa; p.ldsb = ldsb;
    p.a_shift = a_block_rows == 128 ? 7 : 0; p.b_shift = b_block_rows == 128 ? 7 : 0;
    p.bias = bias; p.alpha = alpha; p.y = y; p.ldy = ldy; p.M = M; p.N = N; p.kblocks = kblocks;
    const int cg = M > kF8TileM ? 2 : 1;
    p.tile_n = N >= kF8MaxTileN ? kF8MaxTileN : ((N + 31) / 32) * 32;
    p.mt = (M + cg * kF8TileM - 1) / (cg * kF8TileM);
    p.nt = (N + p.tile_n - 1) / p.tile_n;
    ATB_REQUIRE(static_cast<long long>(p.mt) * p.nt < (1LL << 30), "too many tiles");
    const int stage = kF8TileM * 128 + p.tile_n / cg * 128;
    p.stages = (kF8Smem - 1024 - kF8SfSlots * kF8SfSlotBytes - 4 * 32 * (32 * size + 16)) / stage;
    if (p.stages > kF8MaxStages) p.stages = kF8MaxStages;
    p.idesc = (a_f8 == ATB_E5M2 ? 1u << 7 : 0u) | (b_f8 == ATB_E5M2 ? 1u << 10 : 0u) |
              (static_cast<uint32_t>(p.tile_n >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(cg) << 27);
    p.vec = aligned_to(y, 16) && (ldy * size) % 16 == 0;
    p.drop = DropState{drop_threshold ? static_cast<const unsigned long long*>(rng) : nullptr, static_cast<unsigned>(drop_threshold)};

    CUtensorMap ma, mb;
    int rc = operand_map(&ma, a, M, K, lda, kF8TileM);
    if (rc == ATB_OK) rc = operand_map(&mb, b, N, K, ldb, p.tile_n / cg);
    if (rc != ATB_OK) return rc;
    if (y_dtype == ATB_F32) return launch_fp8_cg<float>(ma, mb, p, cg, s);
    if (y_dtype == ATB_BF16) return launch_fp8_cg<__nv_bfloat16>(ma, mb, p, cg, s);
    return launch_fp8_cg<__half>(ma, mb, p, cg, s);
}

extern "C" int atb_fp8_status(int* status)
{
    ATB_REQUIRE(status != nullptr, "null pointer");
    const cudaError_t e = cudaMemcpyFromSymbol(status, g_fp8_status, sizeof(int));
    if (e != cudaSuccess) { set_error("cudaMemcpyFromSymbol: %s", cudaGetErrorString(e)); return ATB_ERR_CUDA; }
    return ATB_OK;
}

// Counter-based random bits for dropout: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", 2011).  key = the 64-bit seed, counter = (group, offset), both 64 bits; one call serves the 8 elements of
// a group with 16 bits each.  An element is kept when its 16 bits are >= threshold = round(p * 65536), so the rate is
// exact to 2^-17 and no mask has to be stored: whoever knows (seed, offset) has it back.
//
// Why 16 bits an element: a call takes 11.2 us / 2^22 of a B200, half the time in which its memory reads and writes 8 bf16
// elements; with 32 bits each (4 elements a call) the arithmetic would be the bound.
#pragma once

#include <stdint.h>

namespace atb {

struct DropState {                // what a kernel needs to know of a dropout call
    const unsigned long long* rng;    // device: {seed, offset}; null: nothing is dropped
    unsigned threshold;               // 0 .. 65536
};

struct PhiloxKey {
    uint32_t k0, k1, o0, o1;
    PhiloxKey() = default;
    __device__ __forceinline__ explicit PhiloxKey(const unsigned long long* rng)
    {
        const unsigned long long seed = rng[0], off = rng[1];
        k0 = static_cast<uint32_t>(seed); k1 = static_cast<uint32_t>(seed >> 32);
        o0 = static_cast<uint32_t>(off); o1 = static_cast<uint32_t>(off >> 32);
    }
    // by a converged warp: the key in uniform registers, where the ten round keys are made once for all of a thread's calls
    __device__ __forceinline__ void settle()
    {
        k0 = __reduce_max_sync(0xFFFFFFFFu, k0);
        k1 = __reduce_max_sync(0xFFFFFFFFu, k1);
    }
};

// both halves of a product by one instruction (a 64-bit product in C costs 14.6 us instead of 11.2 us for 2^25 elements)
__device__ __forceinline__ void philox_product(uint32_t a, uint32_t b, uint32_t& hi, uint32_t& lo)
{
    asm("{\n\t.reg .b64 t;\n\tmul.wide.u32 t, %2, %3;\n\tmov.b64 {%0, %1}, t;\n\t}" : "=r"(lo), "=r"(hi) : "r"(a), "r"(b));
}

__device__ __forceinline__ uint4 philox4x32_10(const PhiloxKey& key, unsigned long long group)
{
    uint32_t c0 = static_cast<uint32_t>(group), c1 = static_cast<uint32_t>(group >> 32), c2 = key.o0, c3 = key.o1;
    uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        uint32_t ah, al, bh, bl;
        philox_product(c0, 0xD2511F53u, ah, al);
        philox_product(c2, 0xCD9E8D57u, bh, bl);
        c0 = bh ^ c1 ^ k0;
        c1 = bl;
        c2 = ah ^ c3 ^ k1;
        c3 = al;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// bit e set: element e of the group is kept
__device__ __forceinline__ unsigned philox_keep8(const PhiloxKey& key, unsigned long long group, unsigned threshold)
{
    const uint4 w = philox4x32_10(key, group);
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((v[i] & 0xFFFFu) >= threshold) m |= 1u << (2 * i);
        if ((v[i] >> 16) >= threshold) m |= 2u << (2 * i);
    }
    return m;
}

}  // namespace atb

// The dropout mask.  It is never stored: element i of the features is kept if word i % 4 of Philox4x32-10 (J. Salmon,
// M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with the counter
// (i / 4, offset) and the key `seed` is at least floor(p 2^32).  The forward and the backward pass, of any kernel and
// any number of ranks, make the same words from the same numbers.
#pragma once
#include <stdint.h>

namespace agcn {

// What a kernel needs to make its part of a mask again.
struct DropoutMask {
    int on;                       // 0: everything is kept, unscaled
    uint32_t key0, key1;          // seed
    uint32_t threshold;           // floor(p 2^32)
    float scale;                  // 1 / (1 - p)
    int64_t offset;
    const int64_t *step;          // added to offset, read when the kernel runs (null: 0)
    int64_t first;                // number of the first element: row0 * cols
};

// Four words: two 32 x 32 -> 64 bit products, four exclusive ors and two key additions per round, ten rounds.
__device__ __forceinline__ uint4 philox4x32(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1)
{
#pragma unroll
    for (int round = 0; round < 10; round++) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

// Bit e: whether word e of block `block` keeps its element.
__device__ __forceinline__ uint32_t keep_block(const DropoutMask &m, int64_t offset, int64_t block)
{
    const uint4 w = philox4x32((uint32_t)block, (uint32_t)(block >> 32), (uint32_t)offset, (uint32_t)(offset >> 32), m.key0, m.key1);
    return (w.x >= m.threshold ? 1u : 0u) | (w.y >= m.threshold ? 2u : 0u) | (w.z >= m.threshold ? 4u : 0u) | (w.w >= m.threshold ? 8u : 0u);
}

// Bits 0 .. E - 1: whether elements i, i + 1, ... are kept (E a multiple of 4; elements before the first one, i < 0, may
// be asked for and mean nothing).
template <int E>
__device__ __forceinline__ uint32_t keep_bits(const DropoutMask &m, int64_t offset, int64_t i)
{
    const int64_t block = i >> 2;
    const int skip = (int)(i & 3);
    uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < E / 4; k++) bits |= keep_block(m, offset, block + k) << (4 * k);
    if (skip != 0) bits = (bits | keep_block(m, offset, block + E / 4) << E) >> skip;
    return bits;
}

__device__ __forceinline__ int64_t mask_offset(const DropoutMask &m) { return m.on && m.step != nullptr ? m.offset + *m.step : m.offset; }

}  // namespace agcn

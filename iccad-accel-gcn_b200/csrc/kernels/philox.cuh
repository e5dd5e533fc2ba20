// The dropout mask.  It is never stored: element i of the features is kept if word i % 4 of Philox4x32-10 (J. Salmon,
// M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with the counter
// (i / 4, offset) and the key `seed` is at least floor(p 2^32).  The forward and the backward pass, of any kernel and
// any number of ranks, make the same words from the same numbers.
#pragma once
#include <stdint.h>

namespace agcn {

// What a kernel needs to make its part of a mask again.
struct DropoutMask {
    int on;                                // 0: everything is kept, unscaled
    uint32_t key0, key1;                   // seed
    uint32_t threshold;                    // floor(p 2^32)
    float scale;                           // 1 / (1 - p)
    int64_t offset;
    const int64_t *step;                   // added to offset, read when the kernel runs (null: 0)
    int64_t first;                         // number of the first element: row0 * cols
};

// The words of N blocks side by side: two 32 x 32 -> 64 bit products and two three-way exclusive ors a round and block; the
// two additions that make a round's keys serve all N.
template <int N>
__device__ __forceinline__ void philox4x32(const DropoutMask &m, int64_t offset, const int64_t (&block)[N], uint32_t (&w)[N][4])
{
    uint32_t k0 = m.key0, k1 = m.key1;
#pragma unroll
    for (int n = 0; n < N; n++) {
        w[n][0] = (uint32_t)block[n]; w[n][1] = (uint32_t)((uint64_t)block[n] >> 32);
        w[n][2] = (uint32_t)offset; w[n][3] = (uint32_t)((uint64_t)offset >> 32);
    }
#pragma unroll
    for (int round = 0; round < 10; round++) {
#pragma unroll
        for (int n = 0; n < N; n++) {
            const uint64_t a = (uint64_t)w[n][0] * 0xD2511F53u, b = (uint64_t)w[n][2] * 0xCD9E8D57u;
            w[n][0] = (uint32_t)(b >> 32) ^ w[n][1] ^ k0;
            w[n][1] = (uint32_t)b;
            w[n][2] = (uint32_t)(a >> 32) ^ w[n][3] ^ k1;
            w[n][3] = (uint32_t)a;
        }
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
}

// Words of CH chunks of E elements; chunk j begins with word `skip` (0 to 3, alike for all) of block `block[j]`.  Element e
// is kept if its word is at least m.threshold.  (Where the chunks do not begin with a block, a word stands for the answer:
// 0, or all ones.)
template <int CH, int E>
__device__ __forceinline__ void draw_words(const DropoutMask &m, int64_t offset, const int64_t (&block)[CH], int skip, uint32_t (&word)[CH][E])
{
    constexpr int B = E / 4;
    int64_t blocks[CH * B];
    uint32_t w[CH * B][4];
#pragma unroll
    for (int n = 0; n < CH * B; n++) blocks[n] = block[n / B] + n % B;
    philox4x32<CH * B>(m, offset, blocks, w);
#pragma unroll
    for (int j = 0; j < CH; j++)
#pragma unroll
        for (int e = 0; e < E; e++) word[j][e] = w[j * B + e / 4][e % 4];
    if (skip != 0) {
        int64_t more[CH];
        uint32_t v[CH][4];
#pragma unroll
        for (int j = 0; j < CH; j++) more[j] = block[j] + B;
        philox4x32<CH>(m, offset, more, v);
#pragma unroll
        for (int j = 0; j < CH; j++) {
            uint32_t bits = 0;
#pragma unroll
            for (int e = 0; e < E + 4; e++) bits |= ((e < E ? word[j][e < E ? e : 0] : v[j][e < E ? 0 : e - E]) >= m.threshold ? 1u : 0u) << e;
            bits >>= skip;
#pragma unroll
            for (int e = 0; e < E; e++) word[j][e] = bits >> e & 1u ? ~0u : 0u;       // threshold > 0 wherever an element may be dropped
        }
    }
}

// The same where the chunks of consecutive lanes are consecutive and do not begin with a block: bit e of bits[j] says whether element e of
// chunk j is kept.  A chunk's last words are the first ones of the next lane's block, so a lane makes CH chunks' blocks and one more, not
// twice as many.  L: the lanes that share a row, whose first lane has chunk j + 1 behind the last one's chunk j; 0: all 32 and what is
// behind the last one is another warp's.  `lane`: its number among the L (32).  All lanes of the warp call.
// (1 200 000 rows of 116 of 167 columns: 316 us forward, 421 back; with twice the blocks 386 and 478.)
template <int L, int CH, int E>
__device__ __forceinline__ void draw_bits(const DropoutMask &m, int64_t offset, int64_t block, int64_t stride, int skip, int lane, uint32_t (&bits)[CH])
{
    constexpr int B = E / 4, W = L > 0 ? L : 32, AT_ONCE = CH * B > 2 && CH % 2 == 0 ? CH / 2 : CH;
#pragma unroll
    for (int i = 0; i < CH; i += AT_ONCE) {
        int64_t blocks[AT_ONCE];
        uint32_t word[AT_ONCE][E];
#pragma unroll
        for (int j = 0; j < AT_ONCE; j++) blocks[j] = block + (i + j) * stride;
        draw_words<AT_ONCE, E>(m, offset, blocks, 0, word);
#pragma unroll
        for (int j = 0; j < AT_ONCE; j++) {
            bits[i + j] = 0;
#pragma unroll
            for (int e = 0; e < E; e++) bits[i + j] |= (word[j][e] >= m.threshold ? 1u : 0u) << e;
        }
    }
    // the blocks behind the last lane: behind its last chunk, which it makes itself, or (L = 0) behind each, which lane j makes
    const int64_t last = L > 0 ? block + (CH - 1) * stride + B : block + (W - 1 - lane) * B + lane * stride + B;
    const int64_t more[1] = {last};
    uint32_t w[1][4];
    philox4x32<1>(m, offset, more, w);
    const uint32_t behind = (w[0][0] >= m.threshold ? 1u : 0u) | (w[0][1] >= m.threshold ? 2u : 0u) | (w[0][2] >= m.threshold ? 4u : 0u);
    uint32_t next[CH];
#pragma unroll
    for (int j = 0; j < CH; j++) {
        next[j] = __shfl_sync(0xffffffffu, bits[j], lane + 1, W);
        uint32_t wrapped;
        if (L == 0) wrapped = __shfl_sync(0xffffffffu, behind, j, W);
        else wrapped = j + 1 < CH ? __shfl_sync(0xffffffffu, bits[j + 1 < CH ? j + 1 : j], 0, W) : behind;
        if (lane == W - 1) next[j] = wrapped;
    }
#pragma unroll
    for (int j = 0; j < CH; j++) bits[j] = (bits[j] | next[j] << E) >> skip;
}

__device__ __forceinline__ int64_t mask_offset(const DropoutMask &m) { return m.on && m.step != nullptr ? m.offset + *m.step : m.offset; }

}  // namespace agcn

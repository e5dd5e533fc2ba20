// Dropout of features, with the ReLU before it, and their gradient:
//     y = keep relu(v) / (1 - p)            dx = keep [x > 0] dy / (1 - p)
// v is x or dy, gate the x of the second.  One pass over the tensors, a thread with 4 chunks of 16 bytes at a time so that
// enough is under way.  The mask (philox.cuh) costs some 13 instructions per element: bound by HBM in 32 bits; in
// 16 by the mask at 16 warps per SM (57 to 62 % of the issue slots in use, DRAM at 3.8 TB/s forward and 5.2 back).
#pragma once
#include "philox.cuh"
#include "ptx.cuh"
#include "rows.cuh"

namespace agcn {

constexpr int DROPOUT_THREADS = 256;
constexpr int DROPOUT_CHUNKS = 4;          // of one array, at a time
constexpr int DROPOUT_ROWS = 2;            // of a group, at a time
constexpr int DROPOUT_STAGES = 3;
constexpr int DROPOUT_LANES = 1024;        // threads per row, at most

struct DropoutParams {
    const void *v, *gate;                  // gate: of the backward pass with a ReLU, else null
    void *out;
    int64_t rows, cols;
    int relu;                              // of the forward pass
    DropoutMask mask;
    // rows that are not one array: they go round-robin over `groups` groups of `lanes` threads, `turns` each, the first `rest` one more
    int64_t ldv, ldgate, ldout, groups, rest;
    int lanes, turns;
};

// What becomes of U chunks that are in registers: elements lo .. hi - 1 of each (WHOLE: all E of them) are stored, at to[u] on.  Their
// words begin with word `skip` of block[u].  WARP: all lanes of the warp call, with consecutive chunks and the same skip.
template <typename T, bool VEC, bool GATE, bool WHOLE, bool WARP, int U>
__device__ __forceinline__ void dropout_finish(const DropoutParams &p, int64_t offset, T *const (&to)[U], const int64_t (&block)[U], int skip, int lo, int hi,
                                               const uint4 (&v)[U], const uint4 (&gate)[GATE ? U : 1])
{
    constexpr int E = Elem<T>::E;
    constexpr int AT_ONCE = E == 8 && U > 2 ? U / 2 : U;         // chunks whose words are made side by side
    uint32_t bits[U];
    const bool by_bits = WARP && p.mask.on && skip != 0;
    if (by_bits) draw_bits<0, U, E>(p.mask, offset, block[0], block[U - 1 > 0 ? 1 : 0] - block[0], skip, (int)threadIdx.x & 31, bits);
#pragma unroll
    for (int i = 0; i < U; i += AT_ONCE) {
        uint32_t word[AT_ONCE][E];
        if (by_bits) {
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++)
#pragma unroll
                for (int e = 0; e < E; e++) word[u][e] = bits[i + u] >> e & 1u ? ~0u : 0u;
        } else if (p.mask.on) {
            int64_t these[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) these[u] = block[i + u];
            draw_words<AT_ONCE, E>(p.mask, offset, these, WARP ? 0 : skip, word);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            float x[E], g[E];
            Elem<T>::unpack(v[i + u], x);
            if (GATE) Elem<T>::unpack(gate[GATE ? i + u : 0], g);
            if (p.relu) {
#pragma unroll
                for (int e = 0; e < E; e++) x[e] = relu_of(x[e]);
            }
            if (p.mask.on) {
#pragma unroll
                for (int e = 0; e < E; e += 2) unpair(mul2(pair(&x[e]), both(p.mask.scale)), &x[e]);
#pragma unroll
                for (int e = 0; e < E; e++) x[e] = word[u][e] >= p.mask.threshold ? x[e] : 0.f;
            }
            if (GATE) {
#pragma unroll
                for (int e = 0; e < E; e++) x[e] = relu_passes(g[e]) ? x[e] : 0.f;
            }
            if (WHOLE) *reinterpret_cast<uint4 *>(to[i + u]) = Elem<T>::pack(x);
            else store_chunk<T, VEC, false>(to[i + u], ((1u << hi) - 1) & ~((1u << lo) - 1), x);
        }
    }
}

// One chunk of an array of n elements, from element `at` on, which may be in front of it.
template <typename T, bool GATE>
__device__ __forceinline__ void dropout_alone(const DropoutParams &p, int64_t offset, const T *v_base, const T *gate_base, T *out, int64_t at, int64_t n, int skip)
{
    constexpr int E = Elem<T>::E;
    const int lo = at < 0 ? (int)-at : 0, hi = n - at < E ? (int)(n - at) : E;
    float f[E];
    uint4 v[1], gate[1];
    load_chunk<T, true>(v_base + at + lo, -lo, hi - lo, f);
    v[0] = Elem<T>::pack(f);
    if (GATE) {
        load_chunk<T, true>(gate_base + at + lo, -lo, hi - lo, f);
        gate[0] = Elem<T>::pack(f);
    }
    T *to[1] = {out + at};
    const int64_t block[1] = {(p.mask.first + at) >> 2};
    dropout_finish<T, true, GATE, false, false, 1>(p, offset, to, block, skip, lo, hi, v, gate);
}

// Tensors that are one array of n elements each, and sit alike: chunks one behind the other, whatever the width.
template <typename T, bool GATE>
__global__ void __launch_bounds__(DROPOUT_THREADS, 2)
dropout_array_kernel(const __grid_constant__ DropoutParams p)
{
    constexpr int E = Elem<T>::E, U = DROPOUT_CHUNKS;
    wait_for_predecessor();
    const int64_t offset = mask_offset(p.mask), n = p.rows * p.cols;
    const T *const v_base = static_cast<const T *>(p.v), *const gate_base = static_cast<const T *>(p.gate);
    T *const out = static_cast<T *>(p.out);
    const int shift = (int)((reinterpret_cast<uintptr_t>(p.v) / sizeof(T)) & (E - 1));
    const int64_t step = (int64_t)gridDim.x * DROPOUT_THREADS * E;
    int64_t at = ((int64_t)blockIdx.x * DROPOUT_THREADS + threadIdx.x) * E - shift;
    const int skip = (int)((p.mask.first + at) & 3);
    // A warp stays together, so that its chunks are consecutive: where its first one begins in front of the array, ...
    if (__any_sync(0xffffffffu, at < 0)) {
        if (at < n) dropout_alone<T, GATE>(p, offset, v_base, gate_base, out, at, n, skip);
        at += step;
    }
    // U chunks at a time; the next ones are under way while these are worked on
    uint4 v[U], gate[GATE ? U : 1];
    const auto load = [&](int64_t a) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            v[u] = *reinterpret_cast<const uint4 *>(v_base + a + u * step);
            if (GATE) gate[GATE ? u : 0] = *reinterpret_cast<const uint4 *>(gate_base + a + u * step);
        }
    };
    // ... and where its last one is not all there any more
    const int64_t span = (U - 1) * step + E + (31 - ((int)threadIdx.x & 31)) * E;
    if (at + span <= n) load(at);
    for (; at + span <= n; at += U * step) {
        uint4 these[U], its_gate[GATE ? U : 1];
        T *to[U];
        int64_t block[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            these[u] = v[u];
            if (GATE) its_gate[GATE ? u : 0] = gate[GATE ? u : 0];
            to[u] = out + at + u * step;
            block[u] = ((p.mask.first + at) >> 2) + u * (step / 4);
        }
        if (at + U * step + span <= n) load(at + U * step);
        dropout_finish<T, true, GATE, true, true, U>(p, offset, to, block, skip, 0, E, these, its_gate);
    }
    for (; at < n; at += step) dropout_alone<T, GATE>(p, offset, v_base, gate_base, out, at, n, skip);
}

// Rows anywhere.  The number of groups is a multiple of 8, so a group's rows all sit at one offset from a 16-byte boundary and from a
// block of the mask's, and the next ones are under way in a ring in shared memory: a copy of some of a chunk's bytes, where a row
// ends, needs no branch.  (Loads of single elements in a branch are waited for inside it: 1 021 us for 1 000 000 rows of 100 of 128
// columns, two tensors in and one out in 16 bits.)
template <typename T, int LAYOUT, bool GATE>
__global__ void __launch_bounds__(DROPOUT_THREADS)
dropout_rows_kernel(const __grid_constant__ DropoutParams p)
{
    constexpr bool VEC = LAYOUT != ROWS_LOOSE, WHOLE = LAYOUT == ROWS_WHOLE;
    constexpr int E = Elem<T>::E, U = VEC ? DROPOUT_ROWS : 1, STAGES = DROPOUT_STAGES, TENSORS = GATE ? 2 : 1;
    __shared__ uint4 s_ring[VEC ? STAGES * TENSORS * U * DROPOUT_THREADS : 1];
    const int64_t thread = (int64_t)blockIdx.x * DROPOUT_THREADS + threadIdx.x, group = thread / p.lanes;
    if (group >= p.groups) return;
    wait_for_predecessor();
    const int64_t offset = mask_offset(p.mask);
    const int turns = p.turns + (group < p.rest);
    const int64_t v_step = p.groups * p.ldv, gate_step = p.groups * p.ldgate, out_step = p.groups * p.ldout, words = p.groups * p.cols / 4;
    const T *const v_first = static_cast<const T *>(p.v), *const gate_first = static_cast<const T *>(p.gate);
    const int shift = LAYOUT == ROWS_EDGES ? (int)(((int64_t)(reinterpret_cast<uintptr_t>(p.v) / sizeof(T)) + group * p.ldv) & (E - 1)) : 0;
    for (int64_t at = (thread - group * p.lanes) * E - shift; at < p.cols; at += (int64_t)p.lanes * E) {
        const int lo = !WHOLE && at < 0 ? (int)-at : 0, hi = !WHOLE && p.cols - at < E ? (int)(p.cols - at) : E;
        const int64_t number = p.mask.first + group * p.cols + at;
        const T *v_from = v_first + group * p.ldv + at, *gate_from = GATE ? gate_first + group * p.ldgate + at : nullptr;
        T *to[U];
        int64_t block[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            to[u] = static_cast<T *>(p.out) + group * p.ldout + at + u * out_step;
            block[u] = (number >> 2) + u * words;
        }
        RowRing<T, TENSORS, U, STAGES> ring(s_ring);
        const auto fetch = [&](int k, bool near_first) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (k + u < turns) {
                    if (WHOLE) {
                        ring.fetch(0, u, v_from);
                        if (GATE) ring.fetch(TENSORS - 1, u, gate_from);
                    } else if (near_first) {
                        ring.fetch_edge(0, u, v_from, v_first, -lo, hi - lo, hi * (int)sizeof(T));
                        if (GATE) ring.fetch_edge(TENSORS - 1, u, gate_from, gate_first, -lo, hi - lo, hi * (int)sizeof(T));
                    } else {
                        ring.fetch(0, u, v_from, hi * (int)sizeof(T));
                        if (GATE) ring.fetch(TENSORS - 1, u, gate_from, hi * (int)sizeof(T));
                    }
                }
                v_from += v_step;
                if (GATE) gate_from += gate_step;
            }
            commit_copies();
        };
        if (VEC) {
#pragma unroll
            for (int k = 0; k < STAGES; k++) { fetch(k * U, true); ring.next(); }
        }
        for (int k = 0; k < turns; k += U) {
            uint4 v[U], gate[GATE ? U : 1];
            if (VEC) {
                wait_copies<STAGES - 1>();
#pragma unroll
                for (int u = 0; u < U; u++) {
                    v[u] = ring.get(0, u);
                    if (GATE) gate[GATE ? u : 0] = ring.get(TENSORS - 1, u);
                }
                fetch(k + STAGES * U, false);
                ring.next();
            } else {
                float f[E];
                load_chunk<T, false>(v_from + lo, -lo, hi - lo, f);
                v[0] = Elem<T>::pack(f);
                if (GATE) {
                    load_chunk<T, false>(gate_from + lo, -lo, hi - lo, f);
                    gate[0] = Elem<T>::pack(f);
                }
                v_from += v_step;
                if (GATE) gate_from += gate_step;
            }
            if (k + U <= turns) {
                dropout_finish<T, VEC, GATE, WHOLE, false, U>(p, offset, to, block, (int)(number & 3), lo, hi, v, gate);
            } else {
                // the last rows, fewer than U
#pragma unroll
                for (int u = 0; u < U - 1; u++) {
                    if (k + u >= turns) break;
                    T *last[1] = {to[u]};
                    const int64_t its[1] = {block[u]};
                    const uint4 x[1] = {v[u]}, g[1] = {gate[GATE ? u : 0]};
                    dropout_finish<T, VEC, GATE, WHOLE, false, 1>(p, offset, last, its, (int)(number & 3), lo, hi, x, g);
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) { to[u] += U * out_step; block[u] += U * words; }
        }
        wait_copies<0>();                      // the ring is filled anew for the next columns
    }
}

}  // namespace agcn

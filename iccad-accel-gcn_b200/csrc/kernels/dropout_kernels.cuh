// Dropout of features, with the ReLU before it, and their gradient:
//     y = keep relu(v) / (1 - p)            dx = keep [x > 0] dy / (1 - p)
// v is x or dy, gate the x of the second.  One pass over the tensors, a thread with 4 chunks of 16 bytes at a time so that
// enough is under way.  The mask (philox.cuh) costs some 13 instructions per element: bound by HBM in 32 bits, by both
// in 16.
#pragma once
#include "philox.cuh"
#include "ptx.cuh"
#include "rows.cuh"

namespace agcn {

constexpr int DROPOUT_THREADS = 256;
constexpr int DROPOUT_CHUNKS = 4;          // of one array, at a time
__device__ constexpr int DROPOUT_ROW_CHUNKS[3] = {4, 2, 1};       // of rows, by their layout
constexpr int DROPOUT_STAGES = 3;

struct DropoutParams {
    const void *v, *gate;                  // gate: of the backward pass with a ReLU, else null
    void *out;
    int64_t ldv, ldgate, ldout, rows, cols;
    int relu;                              // of the forward pass
    int lanes;                             // threads per row, a power of two (rows that are not one array)
    DropoutMask mask;
};

// A thread's chunks, U of them: where each begins in the three tensors, and the number of its first element.
template <int U>
struct DropoutChunks {
    int64_t v[U], gate[U], out[U], number[U];
};

// What becomes of chunks that are in registers; elements lo .. hi - 1 of each (WHOLE: all E of them) are stored.
template <typename T, bool VEC, bool GATE, bool WHOLE, int U>
__device__ __forceinline__ void dropout_finish(const DropoutParams &p, int64_t offset, const DropoutChunks<U> &c, int lo, int hi,
                                               float (&v)[U][Elem<T>::E], const float (&gate)[GATE ? U : 1][Elem<T>::E])
{
    constexpr int E = Elem<T>::E;
    constexpr int AT_ONCE = E == 8 && U > 1 ? U / 2 : U;         // chunks whose words are made side by side
#pragma unroll
    for (int i = 0; i < U; i += AT_ONCE) {
        uint32_t word[AT_ONCE][E];
        if (p.mask.on) {
            int64_t block[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) block[u] = c.number[i + u] >> 2;
            draw_words<AT_ONCE, E>(p.mask, offset, block, (int)(c.number[i] & 3), word);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            float (&x)[E] = v[i + u];
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
                for (int e = 0; e < E; e++) x[e] = relu_passes(gate[GATE ? i + u : 0][e]) ? x[e] : 0.f;
            }
            T *to = static_cast<T *>(p.out) + c.out[i + u];
            if (WHOLE) *reinterpret_cast<uint4 *>(to) = Elem<T>::pack(x);
            else store_chunk<T, VEC, false>(to, -lo, hi - lo, x);
        }
    }
}

// The same from memory on.
template <typename T, bool VEC, bool GATE, bool WHOLE, int U>
__device__ __forceinline__ void dropout_chunks(const DropoutParams &p, int64_t offset, const DropoutChunks<U> &c, int lo, int hi)
{
    constexpr int E = Elem<T>::E;
    const T *v_base = static_cast<const T *>(p.v), *gate_base = static_cast<const T *>(p.gate);
    float v[U][E], gate[GATE ? U : 1][E];
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (WHOLE) Elem<T>::unpack(*reinterpret_cast<const uint4 *>(v_base + c.v[u]), v[u]);
        else load_chunk<T, VEC>(v_base + c.v[u] + lo, -lo, hi - lo, v[u]);
    }
    if (GATE) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (WHOLE) Elem<T>::unpack(*reinterpret_cast<const uint4 *>(gate_base + c.gate[u]), gate[u]);
            else load_chunk<T, VEC>(gate_base + c.gate[u] + lo, -lo, hi - lo, gate[u]);
        }
    }
    dropout_finish<T, VEC, GATE, WHOLE, U>(p, offset, c, lo, hi, v, gate);
}

// Tensors that are one array of n elements each, and sit alike: chunks one behind the other, whatever the width.
template <typename T, bool GATE>
__global__ void __launch_bounds__(DROPOUT_THREADS)
dropout_array_kernel(const __grid_constant__ DropoutParams p)
{
    constexpr int E = Elem<T>::E, U = DROPOUT_CHUNKS;
    wait_for_predecessor();
    const int64_t offset = mask_offset(p.mask), n = p.rows * p.cols;
    const int shift = (int)((reinterpret_cast<uintptr_t>(p.v) / sizeof(T)) & (E - 1));
    const int64_t step = (int64_t)gridDim.x * DROPOUT_THREADS * E;
    for (int64_t at = ((int64_t)blockIdx.x * DROPOUT_THREADS + threadIdx.x) * E - shift; at < n; at += U * step) {
        if (at >= 0 && at + (U - 1) * step + E <= n) {
            DropoutChunks<U> c;
#pragma unroll
            for (int u = 0; u < U; u++) {
                c.v[u] = c.gate[u] = c.out[u] = at + u * step;
                c.number[u] = p.mask.first + at + u * step;
            }
            dropout_chunks<T, true, GATE, true, U>(p, offset, c, 0, E);
        } else {
#pragma unroll 1
            for (int u = 0; u < U; u++) {
                const int64_t a = at + u * step;
                if (a >= n) break;
                const DropoutChunks<1> c = {{a}, {a}, {a}, {p.mask.first + a}};
                dropout_chunks<T, true, GATE, false, 1>(p, offset, c, a < 0 ? (int)-a : 0, n - a < E ? (int)(n - a) : E);
            }
        }
    }
}

// Rows anywhere: they go round-robin over groups of `lanes` threads, a row's chunks over the group's threads.  The number of groups
// is a multiple of 8, so a group's rows all sit at one offset from a 16-byte boundary and from a block of the mask's.
// Where rows have chunks at their ends that are not the row's alone, the next rows are under way in a ring in shared memory:
// a copy of some of a chunk's bytes needs no branch.  (Loads of single elements in a branch are waited for inside it: 1 021 us in
// place of 299 for 1 000 000 rows of 100 of 128 columns, two tensors in and one out in 16 bits.)
template <typename T, int LAYOUT, bool GATE>
__global__ void __launch_bounds__(DROPOUT_THREADS)
dropout_rows_kernel(const __grid_constant__ DropoutParams p)
{
    constexpr bool WHOLE = LAYOUT == ROWS_WHOLE;
    constexpr int E = Elem<T>::E, U = DROPOUT_ROW_CHUNKS[LAYOUT], STAGES = DROPOUT_STAGES, TENSORS = GATE ? 2 : 1;
    wait_for_predecessor();
    const int64_t offset = mask_offset(p.mask);
    const int64_t thread = (int64_t)blockIdx.x * DROPOUT_THREADS + threadIdx.x;
    const int64_t group = thread / p.lanes, groups = (int64_t)gridDim.x * (DROPOUT_THREADS / p.lanes);
    const T *const v_first = static_cast<const T *>(p.v), *const gate_first = static_cast<const T *>(p.gate);
    const int shift = LAYOUT == ROWS_EDGES ? (int)(((int64_t)(reinterpret_cast<uintptr_t>(p.v) / sizeof(T)) + group * p.ldv) & (E - 1)) : 0;
    __shared__ uint4 s_ring[LAYOUT == ROWS_EDGES ? STAGES * TENSORS * U * DROPOUT_THREADS : 1];
    for (int64_t at = (int64_t)(threadIdx.x & (p.lanes - 1)) * E - shift; at < p.cols; at += (int64_t)p.lanes * E) {
        const int lo = !WHOLE && at < 0 ? (int)-at : 0, hi = !WHOLE && p.cols - at < E ? (int)(p.cols - at) : E;
        int64_t row = group;
        const auto places = [&](int64_t r) {
            DropoutChunks<U> c;
#pragma unroll
            for (int u = 0; u < U; u++, r += groups) {
                c.v[u] = r * p.ldv + at; c.gate[u] = r * p.ldgate + at; c.out[u] = r * p.ldout + at;
                c.number[u] = p.mask.first + r * p.cols + at;
            }
            return c;
        };
        if constexpr (LAYOUT == ROWS_EDGES) {
            RowRing<T, TENSORS, U, STAGES> ring(s_ring);
            int64_t ahead = group;
            const auto fetch = [&]() {
#pragma unroll
                for (int u = 0; u < U; u++, ahead += groups) {
                    if (ahead >= p.rows) continue;
                    ring.fetch_edge(0, u, v_first + ahead * p.ldv + at, v_first, -lo, hi - lo, hi * (int)sizeof(T));
                    if (GATE) ring.fetch_edge(TENSORS - 1, u, gate_first + ahead * p.ldgate + at, gate_first, -lo, hi - lo, hi * (int)sizeof(T));
                }
                commit_copies();
            };
#pragma unroll
            for (int k = 0; k < STAGES; k++) { fetch(); ring.next(); }
            for (; row < p.rows; row += U * groups) {
                float v[U][E], gate[GATE ? U : 1][E];
                wait_copies<STAGES - 1>();
#pragma unroll
                for (int u = 0; u < U; u++) {
                    ring.get(0, u, v[u]);
                    if (GATE) ring.get(TENSORS - 1, u, gate[u]);
                }
                fetch();
                ring.next();
                if (row + (U - 1) * groups < p.rows) {
                    dropout_finish<T, true, GATE, false, U>(p, offset, places(row), lo, hi, v, gate);
                } else {
                    // the last rows: at most U - 1 of them
#pragma unroll
                    for (int u = 0; u < U - 1; u++) {
                        const int64_t r = row + u * groups;
                        if (r >= p.rows) break;
                        const DropoutChunks<1> c = {{0}, {0}, {r * p.ldout + at}, {p.mask.first + r * p.cols + at}};
                        float one[1][E], its[1][E];
#pragma unroll
                        for (int e = 0; e < E; e++) { one[0][e] = v[u][e]; its[0][e] = GATE ? gate[GATE ? u : 0][e] : 0.f; }
                        dropout_finish<T, true, GATE, false, 1>(p, offset, c, lo, hi, one, its);
                    }
                }
            }
            wait_copies<0>();                  // the ring is filled anew for the next columns
        } else {
            for (; row + (U - 1) * groups < p.rows; row += U * groups) dropout_chunks<T, WHOLE, GATE, WHOLE, U>(p, offset, places(row), lo, hi);
#pragma unroll 1
            for (; row < p.rows; row += groups) {
                const DropoutChunks<1> c = {{row * p.ldv + at}, {row * p.ldgate + at}, {row * p.ldout + at}, {p.mask.first + row * p.cols + at}};
                dropout_chunks<T, WHOLE, GATE, WHOLE, 1>(p, offset, c, lo, hi);
            }
        }
    }
}

}  // namespace agcn

// Dropout of features, with the ReLU before it, and their gradient:
//     y = keep relu(v) / (1 - p)            dx = keep [x > 0] dy / (1 - p)
// v is x or dy, gate the x of the second.  One pass over the tensors, bound by HBM in 32 bits; the mask (philox.cuh)
// costs 20 wide multiplies per 4 elements.
#pragma once
#include "philox.cuh"
#include "rows.cuh"

namespace agcn {

constexpr int DROPOUT_THREADS = 256;

struct DropoutParams {
    const void *v, *gate;                  // gate: of the backward pass with a ReLU, else null
    void *out;
    int64_t ldv, ldgate, ldout, rows, cols;
    int relu;                              // of the forward pass
    int lanes;                             // threads per row, a power of two
    DropoutMask mask;
};

// Rows go round-robin over groups of `lanes` threads, the chunks of a row over the group's threads.
template <typename T, bool VEC>
__global__ void __launch_bounds__(DROPOUT_THREADS)
dropout_kernel(const __grid_constant__ DropoutParams p)
{
    constexpr int E = Elem<T>::E;
    const int64_t offset = mask_offset(p.mask);
    const int64_t thread = (int64_t)blockIdx.x * DROPOUT_THREADS + threadIdx.x, threads = (int64_t)gridDim.x * DROPOUT_THREADS;
    for (int64_t row = thread / p.lanes; row < p.rows; row += threads / p.lanes) {
        const T *v_row = static_cast<const T *>(p.v) + row * p.ldv, *gate_row = static_cast<const T *>(p.gate) + (p.gate != nullptr ? row * p.ldgate : 0);
        T *out_row = static_cast<T *>(p.out) + row * p.ldout;
        const int shift = VEC ? (int)((reinterpret_cast<uintptr_t>(v_row) / sizeof(T)) & (E - 1)) : (int)((p.mask.first + row * p.cols) & 3);
        const int64_t first = p.mask.first + row * p.cols;
        for (int64_t c0 = (thread & (p.lanes - 1)) * E - shift; c0 < p.cols; c0 += (int64_t)p.lanes * E) {
            // chunks count from c0: what load_chunk sees fits an int
            const int lo = c0 < 0 ? (int)c0 : 0, left = (int)(p.cols - (c0 < 0 ? 0 : c0) < E ? p.cols - (c0 < 0 ? 0 : c0) : E);
            const int64_t at = c0 < 0 ? 0 : c0;
            float v[E], gate[E];
            load_chunk<T, VEC>(v_row + at, lo, left, v);
            if (p.gate != nullptr) load_chunk<T, VEC>(gate_row + at, lo, left, gate);
            uint32_t word[1][E];
            if (p.mask.on) draw_words<1, E>(p.mask, offset, (first + c0) >> 2, 0, (int)((first + c0) & 3), word);
#pragma unroll
            for (int e = 0; e < E; e++) {
                float x = v[e];
                if (p.relu) x = relu_of(x);
                if (p.mask.on) x *= p.mask.scale;
                v[e] = (!p.mask.on || word[0][e] >= p.mask.threshold) && (p.gate == nullptr || relu_passes(gate[e])) ? x : 0.f;
            }
            store_chunk<T, VEC, false>(out_row + at + lo, lo, left, v);
        }
    }
}

}  // namespace agcn

// Layer norm over the rows of the features, its gradients, and with them in the same pass the ReLU and the dropout that
// follow it in a GCN layer:
//
//   m = mean_c x,  s = 1 / sqrt(mean_c (x - m)^2 + eps),  h = (x - m) s,  z = h w + b,  y = keep relu(z) / (1 - p)
//
//   dz = keep [z > 0] dy / (1 - p),  g = dz w,  dx = s (g - mean_c g - h mean_c (g h)),  dw = sum_r dz h,  db = sum_r dz
//
// Bound by HBM: two (three) passes over the features.  A group of L lanes (L = 0: a thread block) has a row at a time in
// registers, CH chunks of 16 bytes per lane, so every element is read once; rows go round-robin over the groups.  The
// number of groups is a multiple of 8, so a group's rows all sit at one offset from a 16-byte boundary and a lane has the
// same columns in all of them: weights and the sums over the rows stay in registers, and rows of any width are read 16
// bytes at a time (VEC; rows of tensors that do not sit alike are read element by element).
#pragma once
#include "philox.cuh"
#include "rows.cuh"

namespace agcn {

constexpr int NORM_THREADS = 256;          // of the forms with several rows per thread block
constexpr int NORM_MAX_THREADS = 544;      // of the form with one: 8192 columns, 16 per thread, from any offset on
static_assert(NORM_MAX_THREADS <= 32 * ROW_WARPS, "group_sum holds the sums of that many warps");

struct NormForward {
    const void *x;
    void *y;
    int64_t ldx, ldy, rows;
    const float *weight, *bias;            // null: 1, 0
    float2 *stats;                         // [rows] (m, s); null: not wanted
    int cols, relu;
    float eps, inv_cols;
    DropoutMask mask;
};

struct NormBackward {
    const void *dy, *x;
    void *dx;
    int64_t lddy, ldx, lddx, rows;
    const float *weight, *bias;
    const float2 *stats;
    float *dweight, *dbias;                // [gridDim.x][cols] each, one row per thread block; null: not wanted
    int64_t part_stride;                   // floats between two thread blocks' rows
    int cols, relu;
    float inv_cols;
    DropoutMask mask;
};

// Elements that the first of a group's columns stands behind a 16-byte boundary (VEC), or behind a whole block of the
// mask's words; the same for all rows of the group.
template <typename T, bool VEC>
__device__ __forceinline__ int row_shift(const void *x, int64_t ldx, const DropoutMask &mask, int cols, int64_t row)
{
    constexpr int E = Elem<T>::E;
    if (VEC) return (int)(((int64_t)(reinterpret_cast<uintptr_t>(x) / sizeof(T)) + row * ldx) & (E - 1));
    return mask.on ? (int)((mask.first + row * cols) & 3) : 0;
}

template <typename T, int L, int CH, bool VEC>
__global__ void __launch_bounds__(L > 0 ? NORM_THREADS : NORM_MAX_THREADS)
layer_norm_kernel(const __grid_constant__ NormForward p)
{
    constexpr int E = Elem<T>::E;
    __shared__ GroupSums<1> s_one;
    __shared__ GroupSums<2> s_two;
    int turn_one = 0, turn_two = 0;
    if (L == 0) {
        clear_sums(s_one);
        clear_sums(s_two);
        __syncthreads();
    }
    const int lanes = L > 0 ? L : (int)blockDim.x, t = L > 0 ? (int)threadIdx.x % (L > 0 ? L : 1) : (int)threadIdx.x;
    const int sub = L > 0 ? ((int)threadIdx.x & 31) / (L > 0 ? L : 1) : 0;           // group within the warp
    const int64_t groups = (int64_t)gridDim.x * (L > 0 ? NORM_THREADS / (L > 0 ? L : 1) : 1);
    const int64_t group = L > 0 ? ((int64_t)blockIdx.x * NORM_THREADS + threadIdx.x) / (L > 0 ? L : 1) : (int64_t)blockIdx.x;
    const int cols = p.cols, shift = row_shift<T, VEC>(p.x, p.ldx, p.mask, cols, group);
    const int64_t offset = mask_offset(p.mask);

    float w[CH][E], b[CH][E];
    uint32_t ok = 0;                                     // which of the thread's columns there are
#pragma unroll
    for (int j = 0; j < CH; j++) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int c = (j * lanes + t) * E - shift + e;
            const bool in = c >= 0 && c < cols;
            if (in) ok |= 1u << (j * E + e);
            w[j][e] = in && p.weight != nullptr ? p.weight[c] : 1.f;
            b[j][e] = in && p.bias != nullptr ? p.bias[c] : 0.f;
        }
    }

    for (int64_t base = group - sub; base < p.rows; base += groups) {
        const int64_t row = base + sub;
        const bool live = row < p.rows;
        float d[CH][E];
        float one[1] = {0.f}, two[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < CH; j++) {
            const int c0 = (j * lanes + t) * E - shift;
            if (live && c0 < cols) load_chunk<T, VEC>(static_cast<const T *>(p.x) + row * p.ldx, c0, cols, d[j]);
            else {
#pragma unroll
                for (int e = 0; e < E; e++) d[j][e] = 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < E; e++) one[0] += d[j][e];
        group_sum<L, 1>(one, s_one, turn_one);
        // The first mean is off by its own rounding; the second sum says by how much, and the squares are taken around
        // the first: nothing cancels, however far the mean is from zero.
        const float m = one[0] * p.inv_cols;
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < E; e++) {
                d[j][e] = ok >> (j * E + e) & 1u ? d[j][e] - m : 0.f;
                two[0] += d[j][e];
                two[1] = fmaf(d[j][e], d[j][e], two[1]);
            }
        group_sum<L, 2>(two, s_two, turn_two);
        const float off = two[0] * p.inv_cols;
        const float var = fmaf(-off, off, two[1] * p.inv_cols);
        const float s = __frsqrt_rn((var < 0.f ? 0.f : var) + p.eps);
        if (!live) continue;
        if (p.stats != nullptr && t == 0) p.stats[row] = make_float2(m + off, s);
#pragma unroll
        for (int j = 0; j < CH; j++) {
            const int c0 = (j * lanes + t) * E - shift;
            if (c0 >= cols) continue;
            float v[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                v[e] = fmaf((d[j][e] - off) * s, w[j][e], b[j][e]);
                if (p.relu) v[e] = relu_of(v[e]);
            }
            if (p.mask.on) {
                const uint32_t keep = keep_bits<E>(p.mask, offset, p.mask.first + row * cols + c0);
#pragma unroll
                for (int e = 0; e < E; e++) v[e] = keep >> e & 1u ? v[e] * p.mask.scale : 0.f;
            }
            store_chunk<T, VEC>(static_cast<T *>(p.y) + row * p.ldy, c0, cols, v);
        }
    }
}

template <typename T, int L, int CH, bool VEC>
__global__ void __launch_bounds__(L > 0 ? NORM_THREADS : NORM_MAX_THREADS)
layer_norm_backward_kernel(const __grid_constant__ NormBackward p)
{
    constexpr int E = Elem<T>::E;
    __shared__ GroupSums<2> s_two;
    __shared__ float s_cols[L > 0 ? NORM_THREADS * CH * E : 1];
    int turn = 0;
    if (L == 0) {
        clear_sums(s_two);
        __syncthreads();
    }
    const int lanes = L > 0 ? L : (int)blockDim.x, t = L > 0 ? (int)threadIdx.x % (L > 0 ? L : 1) : (int)threadIdx.x;
    const int sub = L > 0 ? ((int)threadIdx.x & 31) / (L > 0 ? L : 1) : 0;
    const int64_t groups = (int64_t)gridDim.x * (L > 0 ? NORM_THREADS / (L > 0 ? L : 1) : 1);
    const int64_t group = L > 0 ? ((int64_t)blockIdx.x * NORM_THREADS + threadIdx.x) / (L > 0 ? L : 1) : (int64_t)blockIdx.x;
    const int cols = p.cols, shift = row_shift<T, VEC>(p.x, p.ldx, p.mask, cols, group);
    const int64_t offset = mask_offset(p.mask);

    float w[CH][E], b[CH][E], sum_w[CH][E], sum_b[CH][E];
    uint32_t ok = 0;
#pragma unroll
    for (int j = 0; j < CH; j++) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int c = (j * lanes + t) * E - shift + e;
            const bool in = c >= 0 && c < cols;
            if (in) ok |= 1u << (j * E + e);
            w[j][e] = in && p.weight != nullptr ? p.weight[c] : 1.f;
            b[j][e] = in && p.bias != nullptr ? p.bias[c] : 0.f;
            sum_w[j][e] = sum_b[j][e] = 0.f;
        }
    }

    for (int64_t base = group - sub; base < p.rows; base += groups) {
        const int64_t row = base + sub;
        const bool live = row < p.rows;
        float h[CH][E], g[CH][E];
        float two[2] = {0.f, 0.f};
        const float2 stats = live ? p.stats[row] : make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < CH; j++) {
            const int c0 = (j * lanes + t) * E - shift;
            if (live && c0 < cols) {
                load_chunk<T, VEC>(static_cast<const T *>(p.x) + row * p.ldx, c0, cols, h[j]);
                load_chunk<T, VEC>(static_cast<const T *>(p.dy) + row * p.lddy, c0, cols, g[j]);
            } else {
#pragma unroll
                for (int e = 0; e < E; e++) h[j][e] = g[j][e] = 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < CH; j++) {
            const int c0 = (j * lanes + t) * E - shift;
            const uint32_t keep = p.mask.on && live && c0 < cols ? keep_bits<E>(p.mask, offset, p.mask.first + row * cols + c0) : ~0u;
            bool near = false;
            uint32_t pass = ~0u;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float x = h[j][e];
                h[j][e] = ok >> (j * E + e) & 1u ? (x - stats.x) * stats.y : 0.f;
                if (p.relu) {
                    const float z = fmaf(h[j][e], w[j][e], b[j][e]);
                    if (!relu_passes(z)) pass &= ~(1u << e);
                    // |z| off by less than 2^-22 |b| where the two terms cancel: the sign is not certain below that
                    near = near || fabsf(z) < 4.76837158e-7f * fabsf(b[j][e]);
                }
            }
            if (near) {
                // One element in millions: in 64 bits, so that a gradient passes where the formula lets it pass.
                float x[E];
                load_chunk<T, VEC>(static_cast<const T *>(p.x) + row * p.ldx, c0, cols, x);
                pass = ~0u;
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (((double)x[e] - (double)stats.x) * (double)stats.y * (double)w[j][e] + (double)b[j][e] <= 0.0) pass &= ~(1u << e);
            }
#pragma unroll
            for (int e = 0; e < E; e++) {
                float dz = g[j][e];
                if (p.mask.on) dz *= p.mask.scale;
                dz = (keep & pass) >> e & 1u ? dz : 0.f;
                sum_w[j][e] = fmaf(dz, h[j][e], sum_w[j][e]);
                sum_b[j][e] += dz;
                g[j][e] = dz * w[j][e];
                two[0] += g[j][e];
                two[1] = fmaf(g[j][e], h[j][e], two[1]);
            }
        }
        group_sum<L, 2>(two, s_two, turn);
        if (!live) continue;
        const float m1 = two[0] * p.inv_cols, m2 = two[1] * p.inv_cols;
#pragma unroll
        for (int j = 0; j < CH; j++) {
            const int c0 = (j * lanes + t) * E - shift;
            if (c0 >= cols) continue;
            float v[E];
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = stats.y * (g[j][e] - m1 - h[j][e] * m2);
            store_chunk<T, VEC>(static_cast<T *>(p.dx) + row * p.lddx, c0, cols, v);
        }
    }

    // The groups' sums, then the thread blocks': always in the same order.
#pragma unroll
    for (int pass = 0; pass < 2; pass++) {
        float *part = pass == 0 ? p.dweight : p.dbias;
        if (part == nullptr) continue;
        part += (int64_t)blockIdx.x * p.part_stride;
        if (L > 0) __syncthreads();
        float *mine = L > 0 ? s_cols + (threadIdx.x / (L > 0 ? L : 1)) * cols : part;
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < E; e++)
                if (ok >> (j * E + e) & 1u) mine[(j * lanes + t) * E - shift + e] = pass == 0 ? sum_w[j][e] : sum_b[j][e];
        if (L > 0) {
            __syncthreads();
            for (int c = threadIdx.x; c < cols; c += NORM_THREADS) {
                float s = 0.f;
                for (int k = 0; k < NORM_THREADS / (L > 0 ? L : 1); k++) s += s_cols[k * cols + c];
                part[c] = s;
            }
        }
    }
}

// Column sums of the thread blocks' rows: 32 columns per thread block, its 8 warps over the rows in turn.
static __global__ void __launch_bounds__(256)
norm_columns_kernel(const float *__restrict__ parts, int64_t part_stride, int n_parts, float *__restrict__ dweight, float *__restrict__ dbias, int cols)
{
    __shared__ float s_sum[8][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float *out = blockIdx.y == 0 ? dweight : dbias;
    if (out == nullptr) return;
    float s = 0.f;
    if (c < cols)
        for (int k = warp; k < n_parts; k += 8) s += parts[k * part_stride + (int64_t)blockIdx.y * cols + c];
    s_sum[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < cols) {
        s = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) s += s_sum[k][lane];
        out[c] = s;
    }
}

}  // namespace agcn

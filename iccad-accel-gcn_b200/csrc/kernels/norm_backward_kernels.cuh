// The backward pass of layer norm, ReLU and dropout (norm_kernels.cuh has the mathematics and the layout): dx row by row, the columns' sums
// in each thread's registers over all of its rows, then over the groups of a thread block, then over the thread blocks, in one order.
#pragma once
#include <cooperative_groups.h>

#include "norm_kernels.cuh"

namespace agcn {

// Bit j * E + e: whether z <= 0 in column c0 + j * stride + e.  Out of line, so that it takes no registers where it is not called.
template <typename T>
__device__ __noinline__ uint32_t closed_in_64_bits(const T *row, const float *weight, const float *bias, float2 stats, int c0, int stride, int chunks, int cols)
{
    constexpr int E = Elem<T>::E;
    uint32_t bits = 0;
    for (int j = 0; j < chunks; j++)
        for (int e = 0; e < E; e++) {
            const int c = c0 + j * stride + e;
            if (c < 0 || c >= cols) continue;
            const double h = ((double)Elem<T>::get(row[c]) - (double)stats.x) * (double)stats.y;
            if (h * (weight != nullptr ? (double)weight[c] : 1.0) + (bias != nullptr ? (double)bias[c] : 0.0) <= 0.0) bits |= 1u << (j * E + e);
        }
    return bits;
}

// Sums over groups and thread blocks are made as eight chains that are added as a tree: with 2 048 rows of 16 a term has at most 22 roundings
// behind it, 135 in one chain.  dbias is off by 0.7e-7 of its norm there (one chain: 1.9e-7), in 5.9 us (6.0); joined in 64 bits it were
// 0.5e-7, in 7.1 us.  A thread's own rows are one chain in fp32, and most of what is left in long calls (2 400 000 x 128: 2.0e-7).
__device__ __forceinline__ float sum8(const float (&v)[8]) { return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])); }

template <typename T, int L, int CH, int LAYOUT>
__global__ void __launch_bounds__(L > 0 ? NORM_THREADS : NORM_MAX_THREADS, L > 0 && CH * Elem<T>::E <= (LAYOUT == ROWS_WHOLE ? 12 : 8) ? 2 : 1)
layer_norm_backward_kernel(const __grid_constant__ NormBackward p)
{
    constexpr int E = Elem<T>::E;
    constexpr bool VEC = LAYOUT != ROWS_LOOSE;
    __shared__ GroupSums<2> s_two;
    int turn = 0;
    if (L == 0) {
        clear_sums(s_two);
        __syncthreads();
    }
    const int cols = p.cols;
    const NormPlace<T, L, CH, LAYOUT> at(p.part, p.x, p.ldx, cols);

    extern __shared__ uint4 s_ring[];
    constexpr int STAGES = norm_backward_stages(L);
    RowRing<T, 2, CH, STAGES> ring(s_ring);
    wait_for_predecessor();
    const T *const x_first = static_cast<const T *>(p.x), *const dy_first = static_cast<const T *>(p.dy);
    const T *x = x_first + at.group * p.ldx + at.column(0), *dy = dy_first + at.group * p.lddy + at.column(0);
    if (VEC) {
#pragma unroll
        for (int k = 0; k < STAGES; k++) {
            ring.clear();
            if (k < at.turns) {
                at.fetch(ring, 0, x, x_first, cols, true);
                at.fetch(ring, 1, dy, dy_first, cols, true);
            }
            commit_copies();
            ring.next();
            x += p.x_step;
            dy += p.dy_step;
        }
    }

    uint4 *s_columns = s_ring + STAGES * 2 * CH * blockDim.x;
    NormColumns<L == 0, CH, E> w(s_columns), b(s_columns + CH * (E / 4) * blockDim.x);
    float sum_w[CH][E], sum_b[CH][E];
    uint32_t own[CH][E];
    float uncertain = 0.f;
#pragma unroll
    for (int j = 0; j < CH; j++) {
        float wj[E], bj[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int c = at.column(j) + e;
            const bool in = c >= 0 && c < cols;
            wj[e] = in && p.weight != nullptr ? p.weight[c] : 1.f;
            bj[e] = !in ? INFINITY : p.bias != nullptr ? p.bias[c] : 0.f;         // a column that is not there is never near zero
            // z = h w + b is off by less than 2^-22 |b| where the two terms cancel: its sign is not certain below that
            if (in) uncertain = fmaxf(uncertain, fabsf(bj[e]) * 4.76837158e-7f);
            sum_w[j][e] = sum_b[j][e] = 0.f;
            own[j][e] = at.mine(j, e);
        }
        w.put(j, wj);
        b.put(j, bj);
    }
    const float scale = p.mask.on ? p.mask.scale : 1.f;       // of all gradients: once per row and at the end
    const float dx_scale = cols > 1 ? scale : 0.f;            // (a row of one column is its own mean: its gradient is zero, not a rounding)
    const int64_t offset = mask_offset(p.mask);
    const int64_t number = p.mask.first + at.group * cols - at.shift;
    const int skip = (int)(number & 3);
    int64_t block = (number >> 2) + at.t * (E / 4);
    T *dx = static_cast<T *>(p.dx) + at.group * p.lddx + at.column(0);
    const float2 *stats_at = p.stats + at.group;
    float2 next_stats = at.turns > 0 ? *stats_at : make_float2(0.f, 0.f);

    for (int k = 0; k < at.warp_turns; k++) {
        const bool live = k < at.turns;
        float h[CH][E], g[CH][E];
        float2 part[2][2] = {};
        const float2 stats = next_stats;
        stats_at += at.groups;
        if (k + 1 < at.turns) next_stats = *stats_at;
        if (VEC) {
            wait_copies<STAGES - 1>();
#pragma unroll
            for (int j = 0; j < CH; j++) {
                ring.get(0, j, h[j]);
                ring.get(1, j, g[j]);
            }
            if (k + STAGES < at.turns) {
                at.fetch(ring, 0, x, x_first, cols, false);
                at.fetch(ring, 1, dy, dy_first, cols, false);
            }
            commit_copies();
            ring.next();
        } else {
#pragma unroll
            for (int j = 0; j < CH; j++) {
                load_chunk<T, false>(x - at.column(0), live ? at.column(j) : cols, cols, h[j]);
                load_chunk<T, false>(dy - at.column(0), live ? at.column(j) : cols, cols, g[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                unpair(mul2(add2(pair(&h[j][e]), both(LAYOUT == ROWS_WHOLE ? masked(-stats.x, own[j][0]) : -stats.x)), both(stats.y)), &h[j][e]);
                if (LAYOUT != ROWS_WHOLE) {
                    // what else a slot holds does not count
#pragma unroll
                    for (int i = e; i < e + 2; i++) {
                        h[j][i] = masked(h[j][i], own[j][i]);
                        if (LAYOUT == ROWS_EDGES && j == 0) g[j][i] = masked(g[j][i], own[j][i]);      // what is behind a row is 0
                    }
                }
            }
        if (p.relu) {
            bool near = false;
#pragma unroll
            for (int j = 0; j < CH; j++) {
                float wj[E], bj[E];
                w.get(j, wj);
                b.get(j, bj);
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const float2 z = fma2(pair(&h[j][e]), pair(&wj[e]), pair(&bj[e]));
                    near = near || fabsf(z.x) < uncertain || fabsf(z.y) < uncertain;
                    g[j][e] = relu_passes(z.x) ? g[j][e] : 0.f;
                    g[j][e + 1] = relu_passes(z.y) ? g[j][e + 1] : 0.f;
                }
            }
            if (near && live) {
                // One element in millions: in 64 bits, so that a gradient passes where the formula lets it pass.
                const int ahead = VEC ? STAGES : 0;
                const uint32_t closed = closed_in_64_bits(x - ahead * p.x_step - at.column(0), p.weight, p.bias, stats, at.column(0), at.lanes * E, CH, cols);
#pragma unroll
                for (int j = 0; j < CH; j++) {
                    load_chunk<T, false>(dy - ahead * p.dy_step - at.column(0), at.column(j), cols, g[j]);
#pragma unroll
                    for (int e = 0; e < E; e++) g[j][e] = closed >> (j * E + e) & 1u ? 0.f : g[j][e];
                }
            }
        }
        x += p.x_step;
        dy += p.dy_step;
        if (p.mask.on) {
            drop<L, CH, E>(p.mask, offset, block, at.lanes * (E / 4), skip, g);
        }
        if (live) {
#pragma unroll
            for (int j = 0; j < CH; j++) {
                float wj[E];
                w.get(j, wj);
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    float2 v = pair(&g[j][e]);
                    unpair(fma2(v, pair(&h[j][e]), pair(&sum_w[j][e])), &sum_w[j][e]);
                    unpair(add2(v, pair(&sum_b[j][e])), &sum_b[j][e]);
                    v = mul2(v, pair(&wj[e]));
                    part[0][e / 2 % 2] = add2(part[0][e / 2 % 2], v);
                    part[1][e / 2 % 2] = fma2(v, pair(&h[j][e]), part[1][e / 2 % 2]);
                    unpair(v, &g[j][e]);
                }
            }
        }
        float two[2] = {sum4(part[0]), sum4(part[1])};
        group_sum<L, 2>(two, s_two, turn);
        if (live) {
            const float s = stats.y * dx_scale, m1 = two[0] * p.inv_cols * s, m2 = two[1] * p.inv_cols * s;
#pragma unroll
            for (int j = 0; j < CH; j++)
#pragma unroll
                for (int e = 0; e < E; e += 2) unpair(fma2(pair(&h[j][e]), both(-m2), fma2(pair(&g[j][e]), both(s), both(-m1))), &g[j][e]);
            at.template store<VEC>(dx, g);
        }
        dx += p.dx_step;
        block += p.part.words;
    }

    if (VEC) wait_copies<0>();
    // The groups' sums, then the thread blocks': always in the same order.  The ring is empty by now and has room for them.
    float *s_cols = reinterpret_cast<float *>(s_ring), *s_parts = s_cols + (L > 0 ? NORM_THREADS * CH * E : 0);
#pragma unroll
    for (int pass = 0; pass < 2; pass++) {
        float *part = pass == 0 ? p.dweight : p.dbias;
        if (part == nullptr) continue;
        part = p.cluster ? s_parts + pass * cols : part + (int64_t)blockIdx.x * p.part_stride;
        if (L > 0 || p.cluster) __syncthreads();               // whoever still has rows, or clears its slots
        float *mine = L > 0 ? s_cols + (threadIdx.x / (L > 0 ? L : 1)) * cols : part;
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < E; e++)
                if (at.ok >> (j * E + e) & 1u) mine[at.column(j) + e] = (pass == 0 ? sum_w[j][e] : sum_b[j][e]) * scale;
        if (L > 0) {
            __syncthreads();
            for (int c = threadIdx.x; c < cols; c += NORM_THREADS) {
                float s[8] = {};                      // of the groups k, k + 8, ...: there are 8 to 128
                for (int k = 0; k < NORM_THREADS / (L > 0 ? L : 1); k += 8)
#pragma unroll
                    for (int u = 0; u < 8; u++) s[u] += s_cols[(k + u) * cols + c];
                part[c] = sum8(s);
            }
        }
    }
    if (p.cluster) {
        // few rows: the thread blocks read each other's sums, in place of a second kernel and a workspace
        cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
        cluster.sync();
        for (int c = blockIdx.x * blockDim.x + threadIdx.x; c < 2 * cols; c += gridDim.x * blockDim.x) {
            float *out = c < cols ? p.dweight : p.dbias;
            if (out == nullptr) continue;
            float v[NORM_CLUSTER];
#pragma unroll
            for (int k = 0; k < NORM_CLUSTER; k++) v[k] = k < (int)gridDim.x ? *cluster.map_shared_rank(s_parts + c, k) : 0.f;
            out[c < cols ? c : c - cols] = sum8(v);
        }
        cluster.sync();                        // nobody leaves while its sums are read
    }
}

// Column sums of the thread blocks' rows: 32 columns per thread block, its 32 warps over the rows in turn, 8 of them under way (one of each chain).
static __global__ void __launch_bounds__(1024)
norm_columns_kernel(const float *parts, int64_t part_stride, int n_parts, float *__restrict__ dweight, float *__restrict__ dbias, int cols)
{
    __shared__ float s_sum[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float *out = blockIdx.y == 0 ? dweight : dbias;
    if (out == nullptr) return;
    wait_for_predecessor();
    float s = 0.f, sums[8] = {};
    if (c < cols) {
        const float *from = parts + (int64_t)blockIdx.y * cols + c;
        int k = warp;
        for (; k + 7 * 32 < n_parts; k += 8 * 32) {
#pragma unroll
            for (int u = 0; u < 8; u++) sums[u] += from[(k + u * 32) * part_stride];
        }
#pragma unroll
        for (int u = 0; u < 7; u++) if (k + u * 32 < n_parts) sums[u] += from[(k + u * 32) * part_stride];
        s = sum8(sums);
    }
    s_sum[warp][lane] = s;
    __syncthreads();
    s = s_sum[lane][warp];                     // lane: the warp that made it; warp: the column
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (lane == 0 && blockIdx.x * 32 + warp < cols) out[blockIdx.x * 32 + warp] = s;
}

}  // namespace agcn

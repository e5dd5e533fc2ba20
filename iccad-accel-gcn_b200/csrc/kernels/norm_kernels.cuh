// Layer norm over the rows of the features, its gradients, and with them in the same pass the ReLU and the dropout that
// follow it in a GCN layer:
//
//   m = mean_c x,  s = 1 / sqrt(mean_c (x - m)^2 + eps),  h = (x - m) s,  z = h w + b,  y = keep relu(z) / (1 - p)
//
//   dz = keep [z > 0] dy / (1 - p),  g = dz w,  dx = s (g - mean_c g - h mean_c (g h)),  dw = sum_r dz h,  db = sum_r dz
//
// Bound by HBM: two (three) passes over the features, 2 400 000 rows of 128 in fp32 with ReLU and dropout in 400-435 us forward (5.7-6.2 TB/s)
// and 615-655 us backward (5.6-6.0 TB/s) where a copy makes 6.56 TB/s; without dropout 545 us backward.  A group of L lanes (L = 0: a
// thread block) has a row at a time in registers, CH chunks of 16 bytes per lane, so every element is read once; rows go round-robin over
// the groups.  The number of groups is a multiple of 8, so a group's rows all sit at one offset from a 16-byte boundary and a lane has the
// same columns in all of them: weights and the sums over the rows stay in registers, and rows of any width are read 16 bytes at a time
// (500 000 rows of 61: 58 us forward, 74-84 backward).  Rows of tensors that do not sit alike are read element by element, with none ahead:
// 1 000 000 x 128 into a slice that begins one column later 271 us in place of 168 forward, 366 of 243 back; bf16 445 of 155, 359 of 227.
// The next rows are under way in a ring in shared memory meanwhile (RowRing): with loads into registers the forward pass took 750 us and
// the backward 2 057.  What bounds it next is how fast 16 warps per SM get through their instructions: a layer's mask costs 14 to 16 per element, the
// rest 11 forward and 25 backward, and a warp waits for the results of its own ones and for the half-rate units that the mask's multiplies and
// exclusive ors need; 54 to 64 % of the issue slots are in use.  In 16 bits, where a row is half the bytes, that is the bound, and nothing
// waits for memory (2 400 000 x 128 bf16: 358-365 and 531 us, 0.53 of the copy).
#pragma once
#include "philox.cuh"
#include "ptx.cuh"
#include "rows.cuh"

namespace agcn {

constexpr int NORM_STAGES = 3;             // rows ahead in the ring
// of the backward pass: with one row per thread block, two tensors of 8192 columns in 32 bits and the weights are 192 KB
__host__ __device__ constexpr int norm_backward_stages(int lanes) { return lanes == 0 ? 2 : NORM_STAGES; }
constexpr int NORM_CLUSTER = 8;            // thread blocks of a backward pass that are one cluster, at most
constexpr int NORM_THREADS = 256;          // of the forms with several rows per thread block
constexpr int NORM_MAX_THREADS = 512;      // of the form with one: 8192 columns, 16 per thread
static_assert(NORM_MAX_THREADS <= 32 * ROW_WARPS, "group_sum holds the sums of that many warps");

// The rows of a call over the groups: every group has `turns` of them, the first `rest` groups one more.
struct NormRows {
    int turns;
    int64_t rest;
    int64_t words;                         // of the mask, in blocks, from one row of a group to its next
};

struct NormForward {
    NormRows part;
    int64_t x_step, y_step;                // elements from one row of a group to its next
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
    NormRows part;
    int64_t dy_step, x_step, dx_step;
    const void *dy, *x;
    void *dx;
    int64_t lddy, ldx, lddx, rows;
    const float *weight, *bias;
    const float2 *stats;
    float *dweight, *dbias;                // [gridDim.x][cols] each, one row per thread block; [cols] where all are one cluster; null: not wanted
    int64_t part_stride;                   // floats between two thread blocks' rows
    int cluster;                           // whether the thread blocks are one cluster
    int cols, relu;
    float inv_cols;
    DropoutMask mask;
};

// Where a thread of a layer norm kernel stands.
template <typename T, int L, int CH, int LAYOUT>
struct NormPlace {
    static constexpr int E = Elem<T>::E;
    int lanes, t;                        // threads of the group, this one's number
    int64_t group, groups;
    int turns, warp_turns;               // rows of the group; the most that a group of this warp has
    int shift;                           // elements that the group's rows begin behind a 16-byte boundary (LOOSE: taken as 0)
    uint32_t ok;                         // which of the thread's CH * E columns there are
    int bytes[CH];                       // of its chunks in a ring, with what is in front of the row
    __device__ __forceinline__ NormPlace(const NormRows &part, const void *x, int64_t ldx, int cols)
    {
        lanes = L > 0 ? L : (int)blockDim.x;
        t = L > 0 ? (int)threadIdx.x & (L - 1) : (int)threadIdx.x;
        groups = (int64_t)gridDim.x * (L > 0 ? NORM_THREADS / (L > 0 ? L : 1) : 1);
        group = L > 0 ? ((int64_t)blockIdx.x * NORM_THREADS + threadIdx.x) / (L > 0 ? L : 1) : (int64_t)blockIdx.x;
        turns = part.turns + (group < part.rest);
        warp_turns = L > 0 ? part.turns + (group - ((int)threadIdx.x & 31) / (L > 0 ? L : 1) < part.rest) : turns;
        shift = 0;
        if (LAYOUT == ROWS_EDGES) shift = (int)(((int64_t)(reinterpret_cast<uintptr_t>(x) / sizeof(T)) + group * ldx) & (E - 1));
        ok = 0;
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < E; e++)
                if (column(j) + e >= 0 && column(j) + e < cols) ok |= 1u << (j * E + e);
#pragma unroll
        for (int j = 0; j < CH; j++) bytes[j] = cols - column(j) >= E ? 16 : (cols - column(j)) * (int)sizeof(T);
    }
    __device__ __forceinline__ int column(int j) const { return (j * lanes + t) * E - shift; }
    // All ones where the thread has the column (WHOLE: a chunk is there or not; a slot of the ring that is never filled is 0)
    __device__ __forceinline__ uint32_t mine(int j, int e) const { return 0u - (ok >> (j * E + (LAYOUT == ROWS_WHOLE ? 0 : e)) & 1u); }
    __device__ __forceinline__ bool has(int j) const { return ok >> (j * E) & ((1u << E) - 1); }
    // The thread's columns of a per-column array (null: `none` in all of them), `missing` where there are none: all loads under way at once.
    __device__ __forceinline__ void load_columns(const float *from, float none, float missing, float (&v)[CH][E]) const
    {
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < E; e++) v[j][e] = ok >> (j * E + e) & 1u ? none : missing;
        if (from == nullptr) return;
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < E; e++) if (ok >> (j * E + e) & 1u) v[j][e] = from[column(j) + e];
    }
    // Starts the copies of a row's chunks, from where this thread's first one is (near_first: the row may be one of the first few).
    template <int N, int STAGES>
    __device__ __forceinline__ void fetch(const RowRing<T, N, CH, STAGES> &ring, int k, const T *from, const T *first, int cols, bool near_first) const
    {
#pragma unroll
        for (int j = 0; j < CH; j++) {
            if (!has(j)) continue;
            if (LAYOUT == ROWS_WHOLE) ring.fetch(k, j, from + j * lanes * E);
            else if (near_first) ring.fetch_edge(k, j, from + j * lanes * E, first, column(j), cols, bytes[j]);
            else ring.fetch(k, j, from + j * lanes * E, bytes[j]);
        }
    }
    // Stores a row's chunks, to where this thread's first one is.
    template <bool VEC>
    __device__ __forceinline__ void store(T *to, const float (&v)[CH][E]) const
    {
#pragma unroll
        for (int j = 0; j < CH; j++)
            if (has(j)) store_chunk<T, VEC, LAYOUT == ROWS_WHOLE>(to + j * lanes * E, ok >> (j * E) & ((1u << E) - 1), v[j]);
    }
};

// One number per column of the thread's: in registers, or (L = 0, where the row's 16 elements per thread take those) in shared
// memory, 16 bytes at a time: quarter q of chunk j at [j][q][thread].
template <bool SHARED, int CH, int E>
struct NormColumns {
    float v[SHARED ? 1 : CH][E];
    float4 *s;
    int threads;
    __device__ __forceinline__ NormColumns(void *memory) : s(static_cast<float4 *>(memory) + threadIdx.x), threads(blockDim.x) {}
    __device__ __forceinline__ void put(int j, const float (&c)[E])
    {
#pragma unroll
        for (int e = 0; e < E; e++) if (!SHARED) v[SHARED ? 0 : j][e] = c[e];
#pragma unroll
        for (int q = 0; q < E / 4; q++) if (SHARED) s[(j * (E / 4) + q) * threads] = make_float4(c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]);
    }
    __device__ __forceinline__ void get(int j, float (&c)[E]) const
    {
#pragma unroll
        for (int e = 0; e < E; e++) if (!SHARED) c[e] = v[SHARED ? 0 : j][e];
#pragma unroll
        for (int q = 0; q < E / 4; q++)
            if (SHARED) {
                const float4 f = s[(j * (E / 4) + q) * threads];
                c[4 * q] = f.x; c[4 * q + 1] = f.y; c[4 * q + 2] = f.z; c[4 * q + 3] = f.w;
            }
    }
};

// 1 / sqrt(v): the approximation and one step of Newton's method, off by 2 roundings at most
__device__ __forceinline__ float inverse_sqrt(float v)
{
    float s;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(v));
    return fmaf(0.5f * s, fmaf(-v * s, s, 1.f), s);
}

// Zeroes what the mask drops of a thread's chunks; the first begins in block `block`, the next `stride` blocks later.
template <int L, int CH, int E>
__device__ __forceinline__ void drop(const DropoutMask &m, int64_t offset, int64_t block, int stride, int skip, float (&v)[CH][E])
{
    // one answer for the warp: its groups may differ
    if (__any_sync(0xffffffffu, skip != 0)) {
        uint32_t bits[CH];
        draw_bits<L, CH, E>(m, offset, block, stride, skip, (int)threadIdx.x & (L > 0 ? L - 1 : 31), bits);
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < E; e++) v[j][e] = bits[j] >> e & 1u ? v[j][e] : 0.f;
        return;
    }
    constexpr int AT_ONCE = CH * E == 16 ? CH / 2 : CH;      // 16 elements in two halves: all at once take the registers of other rows
#pragma unroll
    for (int i = 0; i < CH; i += AT_ONCE) {
        int64_t blocks[AT_ONCE];
        uint32_t word[AT_ONCE][E];
#pragma unroll
        for (int j = 0; j < AT_ONCE; j++) blocks[j] = block + (i + j) * stride;
        draw_words<AT_ONCE, E>(m, offset, blocks, 0, word);
#pragma unroll
        for (int j = 0; j < AT_ONCE; j++)
#pragma unroll
            for (int e = 0; e < E; e++) v[i + j][e] = word[j][e] >= m.threshold ? v[i + j][e] : 0.f;
    }
}

__device__ __forceinline__ float sum4(const float2 (&v)[2])
{
    const float2 s = add2(v[0], v[1]);
    return s.x + s.y;
}

template <typename T, int L, int CH, int LAYOUT>
__global__ void __launch_bounds__(L > 0 ? NORM_THREADS : NORM_MAX_THREADS, L > 0 ? (CH * Elem<T>::E <= 8 ? 3 : 2) : 1)
layer_norm_kernel(const __grid_constant__ NormForward p)
{
    constexpr int E = Elem<T>::E;
    constexpr bool VEC = LAYOUT != ROWS_LOOSE;
    __shared__ GroupSums<1> s_one;
    __shared__ GroupSums<2> s_two;
    int turn_one = 0, turn_two = 0;
    if (L == 0) {
        clear_sums(s_one);
        clear_sums(s_two);
        __syncthreads();
    }
    const int cols = p.cols;
    const NormPlace<T, L, CH, LAYOUT> at(p.part, p.x, p.ldx, cols);

    extern __shared__ uint4 s_ring[];
    constexpr int STAGES = NORM_STAGES;
    RowRing<T, 1, CH, STAGES> ring(s_ring);
    wait_for_predecessor();
    const T *const first = static_cast<const T *>(p.x), *x = first + at.group * p.ldx + at.column(0);
    if (VEC) {
#pragma unroll
        for (int k = 0; k < STAGES; k++) {
            ring.clear();
            if (k < at.turns) at.fetch(ring, 0, x, first, cols, true);
            commit_copies();
            ring.next();
            x += p.x_step;
        }
    }

    float w[CH][E], b[CH][E];
    uint32_t own[CH][E];
    at.load_columns(p.weight, 1.f, 1.f, w);
    at.load_columns(p.bias, 0.f, 0.f, b);
    // the mask's factor is in them: what is kept is multiplied by it, and it is positive
    const float scale = p.mask.on ? p.mask.scale : 1.f;
#pragma unroll
    for (int j = 0; j < CH; j++)
#pragma unroll
        for (int e = 0; e < E; e++) {
            w[j][e] *= scale;
            b[j][e] *= scale;
            own[j][e] = at.mine(j, e);
        }
    const int64_t offset = mask_offset(p.mask);
    const int64_t number = p.mask.first + at.group * cols - at.shift;       // of the row's first element; the same within a block in all rows
    const int skip = (int)(number & 3);
    int64_t block = (number >> 2) + at.t * (E / 4);
    T *y = static_cast<T *>(p.y) + at.group * p.ldy + at.column(0);
    float2 *stats = p.stats + at.group;

    for (int k = 0; k < at.warp_turns; k++) {
        const bool live = k < at.turns;
        float d[CH][E];
        float one[1], two[2];
        float2 part[3][2] = {};
        if (VEC) {
            wait_copies<STAGES - 1>();
#pragma unroll
            for (int j = 0; j < CH; j++) ring.get(0, j, d[j]);
            if (k + STAGES < at.turns) at.fetch(ring, 0, x, first, cols, false);
            commit_copies();
            ring.next();
        } else {
#pragma unroll
            for (int j = 0; j < CH; j++) load_chunk<T, false>(x - at.column(0), live ? at.column(j) : cols, cols, d[j]);
        }
        x += p.x_step;
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                if (LAYOUT == ROWS_EDGES && j == 0) {             // in front of the row; what is behind it is 0
                    d[j][e] = masked(d[j][e], own[j][e]);
                    d[j][e + 1] = masked(d[j][e + 1], own[j][e + 1]);
                }
                part[0][e / 2 % 2] = add2(part[0][e / 2 % 2], pair(&d[j][e]));
            }
        one[0] = sum4(part[0]);
        group_sum<L, 1>(one, s_one, turn_one);
        // The first mean is off by its own rounding; the second sum says by how much, and the squares are taken around
        // the first: nothing cancels, however far the mean is from zero.
        const float m = one[0] * p.inv_cols;
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                float2 v = add2(pair(&d[j][e]), both(LAYOUT == ROWS_WHOLE ? masked(-m, own[j][0]) : -m));
                if (LAYOUT != ROWS_WHOLE) v = make_float2(masked(v.x, own[j][e]), masked(v.y, own[j][e + 1]));
                part[1][e / 2 % 2] = add2(part[1][e / 2 % 2], v);
                part[2][e / 2 % 2] = fma2(v, v, part[2][e / 2 % 2]);
                unpair(v, &d[j][e]);
            }
        two[0] = sum4(part[1]);
        two[1] = sum4(part[2]);
        group_sum<L, 2>(two, s_two, turn_two);
        const float off = two[0] * p.inv_cols;
        const float var = fmaf(-off, off, two[1] * p.inv_cols);
        const float s = inverse_sqrt(relu_of(var) + p.eps);
        const float shifted = -off * s;
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < E; e += 2) unpair(fma2(fma2(pair(&d[j][e]), both(s), both(shifted)), pair(&w[j][e]), pair(&b[j][e])), &d[j][e]);
        if (p.relu) {
#pragma unroll
            for (int j = 0; j < CH; j++)
#pragma unroll
                for (int e = 0; e < E; e++) d[j][e] = relu_of(d[j][e]);
        }
        if (p.mask.on) {
            drop<L, CH, E>(p.mask, offset, block, at.lanes * (E / 4), skip, d);
        }
        if (live) {
            if (p.stats != nullptr && at.t == 0) *stats = make_float2(m + off, s);
            at.template store<VEC>(y, d);
        }
        y += p.y_step;
        stats += at.groups;
        block += p.part.words;
    }
}

}  // namespace agcn

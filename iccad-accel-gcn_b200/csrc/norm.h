// Which form of the layer norm kernels a call takes (norm.cu, norm_backward.cu).
#pragma once
#include "rows.h"
#include "kernels/norm_kernels.cuh"

#include <type_traits>

namespace agcn {

constexpr int64_t NORM_MAX_COLS = AGCN_NORM_MAX_COLS;
constexpr int NORM_ELEMS = 16;              // of a row per thread, at most
// Elements of a row per lane that a group within a warp has at most: 16 forward (with 8, 47 instructions per element in place of 29: 600 us
// for 2 400 000 x 128 in place of 435); 12 backward in 32 bits and 8 in 16, where 16 take over 200 registers (2 000 000 x 96: 496 us with 8,
// 424-442 with 12).  That is what is aimed at with fewer than 32 lanes; 32 go on to 16 elements (backward 385 to 512 columns in 32 bits, 257 to 512 in
// 16) with 216 registers and one thread block per SM, since one warp as a thread block per row is slower with a mask: 200 000 x 512 fp32 194
// us, 210 as that (185, 222 without a mask), 400 000 x 512 bf16 342, 364 (without a mask 241, 221), 400 000 x 384 bf16 347, 363.  Three chunks per lane where that is enough: 2 000 000 x 96 forward 324 -> 279 us, 200 000 x 700 309 -> 252.
constexpr int NORM_FORWARD_ELEMS = 16, NORM_BACKWARD_ELEMS = 12;
// Backward pass: a call whose groups would have up to so many rows in turn runs as one cluster, which adds up the columns itself: 8 where a
// row is a group's within a warp (2 048 rows of 16: 7.9 us a call, 14.8 with a second kernel and a workspace), 2 where it takes a thread
// block (64 rows of 8 192: 29 us as 8 turns of 8, 19 as 64 thread blocks and a second kernel).  Within a warp it goes by the groups that rows on a
// 16-byte boundary have, because the workspace's size is asked for without the addresses: rows off it whose chunk more makes a group twice as wide
// have up to 16 in turn (2 048 x 95: 18.0 us on the GPU; a workspace would make it 6.4).
constexpr int NORM_CLUSTER_TURNS = 8, NORM_CLUSTER_WIDE_TURNS = 2;
constexpr int NORM_MAX_SMEM = 200 * 1024;
static_assert(NORM_MAX_THREADS * NORM_ELEMS * (norm_backward_stages(0) * 2 * 4 + 8) <= NORM_MAX_SMEM, "8192 columns in 32 bits");

struct NormForm {
    int layout;                             // RowLayout
    int lanes;                              // per row; 0: a thread block of `threads`
    int chunks;                             // of 16 bytes per lane
    int threads;
    int64_t rows_per_block;
};

// The form for rows of `cols` elements that begin up to `shift` behind a boundary; `per_lane`: elements of a row per lane of a group
// within a warp that are aimed at.
inline NormForm norm_form_of(int layout, int64_t cols, int dtype, int per_lane, int shift = 0)
{
    const int e = 16 / dtype_bytes(dtype), most_chunks = NORM_ELEMS / e;
    NormForm f = {};
    f.layout = layout;
    // the one thread block that has a row has no room for a chunk more
    if (cols + shift > NORM_MAX_COLS) f.layout = ROWS_LOOSE;
    if (f.layout == ROWS_LOOSE) shift = 0;
    const int chunks = (int)ceil_div(cols + shift, e);
    f.lanes = 2;
    while (f.lanes < 32 && f.lanes * (per_lane / e) < chunks) f.lanes *= 2;
    f.threads = NORM_THREADS;
    f.chunks = (int)ceil_div(chunks, f.lanes);
    if (f.chunks > most_chunks) {
        f.lanes = 0;
        f.threads = 32 * (int)ceil_div(chunks, 32 * most_chunks);
        f.chunks = (int)ceil_div(chunks, f.threads) < 3 ? most_chunks : (int)ceil_div(chunks, f.threads);
    }
    f.rows_per_block = f.lanes > 0 ? NORM_THREADS / f.lanes : 1;
    return f;
}

inline NormForm norm_form(const Rows *t, int n, int64_t cols, int dtype, int per_lane)
{
    int shift = 0;
    const int layout = rows_layout(t, n, cols, dtype, &shift);
    return norm_form_of(layout, cols, dtype, per_lane, shift);
}

// Thread blocks: what the GPU holds at once, a multiple of 8 (every group's rows then sit alike), or fewer.
inline int64_t norm_grid(const NormForm &f, int64_t rows, int64_t resident)
{
    const int64_t needed = ceil_div(rows, f.rows_per_block);
    resident = resident / 8 * 8 > 0 ? resident / 8 * 8 : 8;
    return needed < resident ? needed : resident;
}

// Whether norm_form_of() gives groups of L lanes with CH chunks each, `aim` of them aimed at and `most` the most.
constexpr bool norm_reaches(int L, int CH, int aim, int most)
{
    if (L == 0) return CH == most || CH == 3;
    const int least = L == 2 ? 1 : L / 2 * aim + 1, top = L == 32 ? L * most : L * aim;      // chunks of a row
    return CH >= (least + L - 1) / L && CH <= (top + L - 1) / L;
}

// Calls launch.template operator()<T, L, CH, LAYOUT>() of the form.
template <typename T, int LAYOUT, int L, int CH = 1, typename F> int norm_dispatch_chunks(const NormForm &f, F &&launch)
{
    constexpr int MOST = NORM_ELEMS / Elem<T>::E, AIM = std::decay_t<F>::ELEMS / Elem<T>::E;
    if constexpr (norm_reaches(L, CH, AIM, MOST)) if (f.chunks == CH) return launch.template operator()<T, L, CH, LAYOUT>();
    if constexpr (CH < MOST) return norm_dispatch_chunks<T, LAYOUT, L, CH + 1>(f, launch);
    set_error("no form of %d lanes and %d chunks", f.lanes, f.chunks);
    return AGCN_ERR_INVALID;
}
template <typename T, int LAYOUT, typename F> int norm_dispatch_lanes(const NormForm &f, F &&launch)
{
    switch (f.lanes) {
    case 2: return norm_dispatch_chunks<T, LAYOUT, 2>(f, launch);
    case 4: return norm_dispatch_chunks<T, LAYOUT, 4>(f, launch);
    case 8: return norm_dispatch_chunks<T, LAYOUT, 8>(f, launch);
    case 16: return norm_dispatch_chunks<T, LAYOUT, 16>(f, launch);
    case 32: return norm_dispatch_chunks<T, LAYOUT, 32>(f, launch);
    default: return norm_dispatch_chunks<T, LAYOUT, 0>(f, launch);
    }
}
template <typename T, typename F> int norm_dispatch_layout(const NormForm &f, F &&launch)
{
    if (f.layout == ROWS_WHOLE) return norm_dispatch_lanes<T, ROWS_WHOLE>(f, launch);
    return f.layout == ROWS_EDGES ? norm_dispatch_lanes<T, ROWS_EDGES>(f, launch) : norm_dispatch_lanes<T, ROWS_LOOSE>(f, launch);
}
template <typename F> int norm_dispatch(const NormForm &f, int dtype, F &&launch)
{
    if (dtype == AGCN_F32) return norm_dispatch_layout<float>(f, launch);
    return dtype == AGCN_BF16 ? norm_dispatch_layout<__nv_bfloat16>(f, launch) : norm_dispatch_layout<__half>(f, launch);
}

// Dynamic shared memory: the ring of `tensors` tensors (at the end the groups' column sums) and, where a thread block has one
// row, weight and bias of the backward pass
inline int norm_smem(const NormForm &f, int tensors, int elems)
{
    const int stages = tensors == 2 ? norm_backward_stages(f.lanes) : NORM_STAGES;
    return f.threads * f.chunks * (stages * tensors * 16 + (f.lanes == 0 && tensors == 2 ? 8 * elems : 0));
}

inline NormRows norm_rows(const NormForm &f, int64_t grid, int64_t rows, int64_t cols, int64_t *groups)
{
    *groups = grid * f.rows_per_block;
    NormRows r = {};
    r.turns = (int)(rows / *groups);
    r.rest = rows % *groups;
    r.words = *groups * cols / 4;          // whole wherever a group has a second row: *groups is a multiple of 8 then
    return r;
}

// Thread blocks of a kernel that the current device holds at once, asked for once per device and block size
template <auto KERNEL> int norm_resident(int threads, int smem, int64_t *blocks)
{
    static int per_sm[64][ROW_WARPS + 1] = {};
    int dev = 0, sms = 0;
    const int rc = current_sm_count(&dev, &sms);
    if (rc != AGCN_OK) return rc;
    int &n = per_sm[dev][threads / 32];
    if (n == 0) {
        AGCN_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, NORM_MAX_SMEM));
        AGCN_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, threads, smem));
    }
    *blocks = (int64_t)n * sms;
    return AGCN_OK;
}

}  // namespace agcn

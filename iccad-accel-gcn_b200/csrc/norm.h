// Which form of the layer norm kernels a call takes (norm.cu, norm_backward.cu).
#pragma once
#include "rows.h"
#include "kernels/norm_kernels.cuh"

namespace agcn {

constexpr int64_t NORM_MAX_COLS = AGCN_NORM_MAX_COLS;
constexpr int NORM_ELEMS = 16;              // of a row per thread, at most

struct NormForm {
    bool vec;
    int lanes;                              // per row; 0: a thread block of `threads`
    int chunks;                             // of 16 bytes per lane
    int threads;
    int64_t rows_per_block;
};

inline NormForm norm_form(const Rows *t, int n, int64_t cols, int dtype, bool mask)
{
    const int e = 16 / dtype_bytes(dtype), most_chunks = NORM_ELEMS / e;
    NormForm f = {};
    int shift = 0;
    f.vec = rows_sit_alike(t, n, dtype, &shift);
    if (!f.vec) shift = mask ? 3 : 0;
    const int chunks = (int)ceil_div(cols + shift, e);
    f.lanes = 4;
    while (f.lanes <= 32 && f.lanes * most_chunks < chunks) f.lanes *= 2;
    f.threads = NORM_THREADS;
    if (f.lanes > 32) {
        f.lanes = 0;
        f.threads = 32 * (int)ceil_div(chunks, 32 * most_chunks);
    }
    f.chunks = f.vec && f.lanes > 0 ? (int)ceil_div(chunks, f.lanes) : most_chunks;
    f.rows_per_block = f.lanes > 0 ? NORM_THREADS / f.lanes : 1;
    return f;
}

// Thread blocks: what the GPU holds at once, a multiple of 8 (every group's rows then sit alike), or fewer.
inline int64_t norm_grid(const NormForm &f, int64_t rows, int64_t resident)
{
    const int64_t needed = ceil_div(rows, f.rows_per_block);
    resident = resident / 8 * 8 > 0 ? resident / 8 * 8 : 8;
    return needed < resident ? needed : resident;
}

// Calls launch.template operator()<T, L, CH, VEC>() of the form.
template <typename T, bool VEC, int L, typename F> int norm_dispatch_chunks(const NormForm &f, F &&launch)
{
    constexpr int MOST = NORM_ELEMS / Elem<T>::E;
    if constexpr (VEC && L > 0) {
        if (f.chunks == 1) return launch.template operator()<T, L, 1, VEC>();
        if constexpr (MOST == 4) {
            if (f.chunks == 2) return launch.template operator()<T, L, 2, VEC>();
            if (f.chunks == 3) return launch.template operator()<T, L, 3, VEC>();
        }
    }
    return launch.template operator()<T, L, MOST, VEC>();
}
template <typename T, bool VEC, typename F> int norm_dispatch_lanes(const NormForm &f, F &&launch)
{
    switch (f.lanes) {
    case 4: return norm_dispatch_chunks<T, VEC, 4>(f, launch);
    case 8: return norm_dispatch_chunks<T, VEC, 8>(f, launch);
    case 16: return norm_dispatch_chunks<T, VEC, 16>(f, launch);
    case 32: return norm_dispatch_chunks<T, VEC, 32>(f, launch);
    default: return norm_dispatch_chunks<T, VEC, 0>(f, launch);
    }
}
template <typename F> int norm_dispatch(const NormForm &f, int dtype, F &&launch)
{
    if (dtype == AGCN_F32) return f.vec ? norm_dispatch_lanes<float, true>(f, launch) : norm_dispatch_lanes<float, false>(f, launch);
    if (dtype == AGCN_BF16) return f.vec ? norm_dispatch_lanes<__nv_bfloat16, true>(f, launch) : norm_dispatch_lanes<__nv_bfloat16, false>(f, launch);
    return f.vec ? norm_dispatch_lanes<__half, true>(f, launch) : norm_dispatch_lanes<__half, false>(f, launch);
}

// Thread blocks of a kernel that the current device holds at once, asked for once per device and block size
template <auto KERNEL> int norm_resident(int threads, int64_t *blocks)
{
    static int per_sm[64][ROW_WARPS + 1] = {};
    int dev = 0, sms = 0;
    const int rc = current_sm_count(&dev, &sms);
    if (rc != AGCN_OK) return rc;
    int &n = per_sm[dev][threads / 32];
    if (n == 0) AGCN_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, threads, 0));
    *blocks = (int64_t)n * sms;
    return AGCN_OK;
}

}  // namespace agcn

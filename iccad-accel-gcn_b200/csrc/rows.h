// Host checks shared by the row-wise operators (layer norm, dropout).
#pragma once
#include "host_common.h"
#include "kernels/philox.cuh"
#include "kernels/rows.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace agcn {

constexpr int64_t ROWS_MAX_ELEMENTS = (int64_t)1 << 60;       // numbers of elements, their strides and the mask's counters stay in 64 bits
constexpr int64_t ROWS_MAX_STRIDE = (int64_t)1 << 40;          // times the groups of a launch, too

inline bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
inline int dtype_bytes(int dtype) { return dtype == AGCN_F32 ? 4 : 2; }

// A tensor of features: a device pointer to rows `ld` elements apart.
struct Rows {
    const void *ptr;
    int64_t ld;
    const char *name;
};

inline int check_rows(const char *who, const Rows &t, int64_t rows, int64_t cols, int dtype)
{
    AGCN_REQUIRE(t.ptr != nullptr, "%s: %s is null", who, t.name);
    AGCN_REQUIRE(reinterpret_cast<uintptr_t>(t.ptr) % dtype_bytes(dtype) == 0, "%s: %s is not aligned to its elements", who, t.name);
    AGCN_REQUIRE(t.ld >= cols, "%s: rows of %s are %lld elements apart, fewer than the %lld columns", who, t.name, (long long)t.ld, (long long)cols);
    AGCN_REQUIRE(t.ld <= ROWS_MAX_STRIDE && t.ld <= ROWS_MAX_ELEMENTS / rows, "%s: row stride of %s out of range", who, t.name);
    return AGCN_OK;
}

inline int check_sizes(const char *who, int64_t rows, int64_t cols, int64_t max_cols, int dtype, int activation)
{
    AGCN_REQUIRE(dtype == AGCN_F32 || dtype == AGCN_BF16 || dtype == AGCN_F16, "%s: unknown element type %d", who, dtype);
    AGCN_REQUIRE(activation == AGCN_ACT_NONE || activation == AGCN_ACT_RELU, "%s: unknown activation %d", who, activation);
    AGCN_REQUIRE(cols >= 1 && cols <= max_cols, "%s: %lld columns (1 to %lld are built)", who, (long long)cols, (long long)max_cols);
    AGCN_REQUIRE(rows >= 0 && rows <= ROWS_MAX_ELEMENTS / cols, "%s: row count out of range", who);
    return AGCN_OK;
}

inline int make_mask(const char *who, DropoutMask *m, double p, int64_t seed, int64_t offset, const int64_t *d_step, int64_t row0, int64_t rows, int64_t cols)
{
    AGCN_REQUIRE(p >= 0.0 && p < 1.0, "%s: dropout probability %g (0 <= p < 1)", who, p);
    AGCN_REQUIRE(row0 >= 0 && row0 <= ROWS_MAX_ELEMENTS / cols - rows, "%s: row0 out of range", who);
    AGCN_REQUIRE(reinterpret_cast<uintptr_t>(d_step) % 8 == 0, "%s: step is not aligned to 8 bytes", who);
    *m = DropoutMask{};
    m->on = p > 0.0;
    m->key0 = (uint32_t)(uint64_t)seed;
    m->key1 = (uint32_t)((uint64_t)seed >> 32);
    m->threshold = (uint32_t)(p * 4294967296.0);
    m->scale = (float)(1.0 / (1.0 - p));
    m->offset = offset;
    m->step = d_step;
    m->first = row0 * cols;
    return AGCN_OK;
}

// How the rows of all tensors sit; *most: elements that a row may begin behind a 16-byte boundary.
inline int rows_layout(const Rows *t, int n, int64_t cols, int dtype, int *most)
{
    const int size = dtype_bytes(dtype), e = 16 / size;
    const auto at = [&](const Rows &r) { return (int)(reinterpret_cast<uintptr_t>(r.ptr) / size % e); };
    *most = 0;
    for (int k = 1; k < n; k++)
        if (at(t[k]) != at(t[0]) || t[k].ld % e != t[0].ld % e) return ROWS_LOOSE;
    *most = t[0].ld % e == 0 ? at(t[0]) : e - 1;
    return *most != 0 || cols % e != 0 ? ROWS_EDGES : ROWS_WHOLE;
}

// Streaming multiprocessors of the current device, looked up once
inline int current_sm_count(int *dev, int *count)
{
    static int of[64] = {};
    AGCN_CUDA(cudaGetDevice(dev));
    AGCN_REQUIRE(*dev >= 0 && *dev < 64, "device ordinal %d not supported", *dev);
    if (of[*dev] == 0) AGCN_CUDA(cudaDeviceGetAttribute(&of[*dev], cudaDevAttrMultiProcessorCount, *dev));
    *count = of[*dev];
    return AGCN_OK;
}

}  // namespace agcn

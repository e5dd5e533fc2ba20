// Gradients of layer norm, ReLU and dropout (norm.cu) in one pass over the rows, and the column sums.
#include "norm.h"
#include "kernels/norm_backward_kernels.cuh"

namespace agcn {

// Whether a call's thread blocks are one cluster.  `whole`: the form of rows that fill their chunks; `lanes`: those of the call's own form, which
// is a thread block (0) for the widest rows that a warp has, where they begin behind a boundary (512 x 510 in fp32 as 64 turns of a cluster: 68 us,
// 7.7 as thread blocks and a second kernel).
static bool norm_one_cluster(int64_t rows, const NormForm &whole, int lanes)
{
    return rows <= NORM_CLUSTER * (lanes > 0 ? NORM_CLUSTER_TURNS * whole.rows_per_block : NORM_CLUSTER_WIDE_TURNS);
}

// Thread blocks whose sums the workspace holds: all that are resident, for the forms there are
static int64_t norm_parts(int64_t rows, int64_t cols, int dtype, int lanes, int sms)
{
    const NormForm f = norm_form_of(ROWS_WHOLE, cols, dtype, NORM_BACKWARD_ELEMS);
    if (norm_one_cluster(rows, f, lanes)) return 0;
    // What a thread block writes for its columns (8 bytes each) should be little beside the rows that it reads: 16 of them at
    // least, but two thread blocks per SM where there are few rows.
    const int64_t resident = sms * (2048 / f.threads), few = 2 * sms > rows / 16 ? 2 * sms : rows / 16;
    const int64_t most = few < resident ? few : resident;
    return rows < most ? rows : most;
}

struct NormBackwardLaunch {
    static constexpr int ELEMS = NORM_BACKWARD_ELEMS;
    NormBackward &p;
    const NormForm &f;
    float *work;
    int64_t most_parts;
    cudaStream_t s;
    template <typename T, int L, int CH, int LAYOUT> int operator()() const
    {
        constexpr auto kernel = layer_norm_backward_kernel<T, L, CH, LAYOUT>;
        const size_t smem = norm_smem(f, 2, Elem<T>::E);
        int64_t resident = 0;
        const int rc = norm_resident<layer_norm_backward_kernel<T, L, CH, LAYOUT>>(f.threads, (int)smem, &resident);
        if (rc != AGCN_OK) return rc;
        float *dweight = p.dweight, *dbias = p.dbias;
        const bool wanted = dweight != nullptr || dbias != nullptr;
        int64_t grid = norm_grid(f, p.rows, resident);
        if (wanted && most_parts == 0) {
            const int64_t needed = ceil_div(p.rows, f.rows_per_block);
            for (grid = 1; grid < needed && grid < NORM_CLUSTER; grid *= 2) {}
            p.cluster = grid > 1;              // alone, a thread block's sums are the sums
        } else if (wanted) {
            grid = norm_grid(f, p.rows, resident < most_parts ? resident : most_parts);
            p.part_stride = 2 * p.cols;
            p.dweight = dweight != nullptr ? work : nullptr;
            p.dbias = dbias != nullptr ? work + p.cols : nullptr;
        }
        int64_t groups = 0;
        p.part = norm_rows(f, grid, p.rows, p.cols, &groups);
        p.dy_step = groups * p.lddy;
        p.x_step = groups * p.ldx;
        p.dx_step = groups * p.lddx;
        cudaLaunchAttribute attr[2] = {};
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = (unsigned)grid; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)grid); cfg.blockDim = dim3(f.threads); cfg.dynamicSmemBytes = smem; cfg.stream = s;
        cfg.attrs = attr; cfg.numAttrs = p.cluster ? 2 : 1;
        AGCN_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
        if (wanted && most_parts > 0)
            AGCN_CUDA(launch_early(true, norm_columns_kernel, dim3((unsigned)ceil_div(p.cols, 32), 2), 1024, 0, s, work, p.part_stride, (int)grid, dweight,
                                   dbias, p.cols));
        return AGCN_OK;
    }
};

}  // namespace agcn

extern "C" int agcn_layer_norm_backward_work(int64_t rows, int64_t cols, int dtype, int64_t *bytes)
{
    using namespace agcn;
    clear_error();
    const char *who = "agcn_layer_norm_backward_work";
    AGCN_REQUIRE(bytes != nullptr, "%s: null result pointer", who);
    int dev = 0, sms = 0;
    int rc = check_sizes(who, rows, cols, NORM_MAX_COLS, dtype, AGCN_ACT_NONE);
    if (rc == AGCN_OK) rc = current_sm_count(&dev, &sms);
    if (rc != AGCN_OK) return rc;
    // wherever the rows begin: as far behind a boundary as they can
    const NormForm f = norm_form_of(ROWS_EDGES, cols, dtype, NORM_BACKWARD_ELEMS, 16 / dtype_bytes(dtype) - 1);
    *bytes = norm_parts(rows, cols, dtype, f.lanes, sms) * 2 * cols * (int64_t)sizeof(float);
    return AGCN_OK;
}

extern "C" int agcn_layer_norm_backward(const void *d_dy, int64_t lddy, const void *d_x, int64_t ldx, const float *d_stats, const float *d_weight,
                                        const float *d_bias, void *d_dx, int64_t lddx, float *d_dweight, float *d_dbias, void *d_work,
                                        int64_t work_bytes, int64_t rows, int64_t cols, int dtype, int activation, double p, int64_t seed,
                                        int64_t offset, const int64_t *d_step, int64_t row0, void *stream)
{
    using namespace agcn;
    clear_error();
    const char *who = "agcn_layer_norm_backward";
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    NormBackward a = {};
    int rc = check_sizes(who, rows, cols, NORM_MAX_COLS, dtype, activation);
    if (rc == AGCN_OK) rc = make_mask(who, &a.mask, p, seed, offset, d_step, row0, rows, cols);
    if (rc != AGCN_OK) return rc;
    AGCN_REQUIRE(aligned4(d_weight) && aligned4(d_bias) && aligned4(d_dweight) && aligned4(d_dbias) && aligned4(d_work) &&
                     reinterpret_cast<uintptr_t>(d_stats) % 8 == 0,
                 "%s: weight, bias, their gradients and the workspace must be aligned to 4 bytes, stats to 8", who);
    if (rows == 0) {
        if (d_dweight != nullptr) AGCN_CUDA(cudaMemsetAsync(d_dweight, 0, (size_t)cols * sizeof(float), s));
        if (d_dbias != nullptr) AGCN_CUDA(cudaMemsetAsync(d_dbias, 0, (size_t)cols * sizeof(float), s));
        return AGCN_OK;
    }
    AGCN_REQUIRE(d_stats != nullptr, "%s: stats is null", who);
    const Rows t[3] = {{d_dy, lddy, "dy"}, {d_x, ldx, "x"}, {d_dx, lddx, "dx"}};
    for (const Rows &r : t)
        if ((rc = check_rows(who, r, rows, cols, dtype)) != AGCN_OK) return rc;
    int dev = 0, sms = 0;
    if ((rc = current_sm_count(&dev, &sms)) != AGCN_OK) return rc;
    const NormForm f = norm_form(t, 3, cols, dtype, NORM_BACKWARD_ELEMS);
    const int64_t parts = norm_parts(rows, cols, dtype, f.lanes, sms);
    AGCN_REQUIRE((d_dweight == nullptr && d_dbias == nullptr) || parts == 0 || (d_work != nullptr && work_bytes >= parts * 2 * cols * (int64_t)sizeof(float)),
                 "%s: workspace of %lld bytes, %lld are needed", who, (long long)work_bytes, (long long)(parts * 2 * cols * (int64_t)sizeof(float)));
    a.dy = d_dy; a.lddy = lddy; a.x = d_x; a.ldx = ldx; a.dx = d_dx; a.lddx = lddx; a.rows = rows;
    a.weight = d_weight; a.bias = d_bias;
    a.stats = reinterpret_cast<const float2 *>(d_stats);
    a.dweight = d_dweight; a.dbias = d_dbias;
    a.cols = (int)cols; a.relu = activation == AGCN_ACT_RELU;
    a.inv_cols = 1.f / (float)cols;
    return norm_dispatch(f, dtype, NormBackwardLaunch{a, f, static_cast<float *>(d_work), parts, s});
}

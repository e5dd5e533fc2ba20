// Layer norm of the rows of the features, with the ReLU and the dropout that follow it in a GCN layer: forward pass.
// The reference stops at the sparse product (spmm_accel.cu:104-108); this is what a layer that is trained has behind it.
#include "norm.h"

namespace agcn {

struct NormForwardLaunch {
    static constexpr int ELEMS = NORM_FORWARD_ELEMS;
    NormForward &p;
    const NormForm &f;
    cudaStream_t s;
    template <typename T, int L, int CH, int LAYOUT> int operator()() const
    {
        int64_t resident = 0;
        const int rc = norm_resident<layer_norm_kernel<T, L, CH, LAYOUT>>(f.threads, norm_smem(f, 1, Elem<T>::E), &resident);
        if (rc != AGCN_OK) return rc;
        const int64_t grid = norm_grid(f, p.rows, resident);
        int64_t groups = 0;
        p.part = norm_rows(f, grid, p.rows, p.cols, &groups);
        p.x_step = groups * p.ldx;
        p.y_step = groups * p.ldy;
        AGCN_CUDA(launch_early(true, layer_norm_kernel<T, L, CH, LAYOUT>, (unsigned)grid, f.threads, norm_smem(f, 1, Elem<T>::E), s, p));
        return AGCN_OK;
    }
};

}  // namespace agcn

extern "C" int agcn_layer_norm(const void *d_x, int64_t ldx, const float *d_weight, const float *d_bias, double eps, void *d_y, int64_t ldy,
                               float *d_stats, int64_t rows, int64_t cols, int dtype, int activation, double p, int64_t seed, int64_t offset,
                               const int64_t *d_step, int64_t row0, void *stream)
{
    using namespace agcn;
    clear_error();
    const char *who = "agcn_layer_norm";
    NormForward a = {};
    int rc = check_sizes(who, rows, cols, NORM_MAX_COLS, dtype, activation);
    if (rc == AGCN_OK) rc = make_mask(who, &a.mask, p, seed, offset, d_step, row0, rows, cols);
    if (rc != AGCN_OK) return rc;
    AGCN_REQUIRE(eps >= 1e-30 && eps <= 1e30, "%s: eps %g (1e-30 to 1e30)", who, eps);
    AGCN_REQUIRE(aligned4(d_weight) && aligned4(d_bias) && reinterpret_cast<uintptr_t>(d_stats) % 8 == 0,
                 "%s: weight and bias must be aligned to 4 bytes, stats to 8", who);
    if (rows == 0) return AGCN_OK;
    const Rows t[2] = {{d_x, ldx, "x"}, {d_y, ldy, "y"}};
    for (const Rows &r : t)
        if ((rc = check_rows(who, r, rows, cols, dtype)) != AGCN_OK) return rc;
    a.x = d_x; a.ldx = ldx; a.y = d_y; a.ldy = ldy; a.rows = rows;
    a.weight = d_weight; a.bias = d_bias;
    a.stats = reinterpret_cast<float2 *>(d_stats);
    a.cols = (int)cols; a.relu = activation == AGCN_ACT_RELU;
    a.eps = (float)eps; a.inv_cols = 1.f / (float)cols;
    const NormForm f = norm_form(t, 2, cols, dtype, NORM_FORWARD_ELEMS);
    return norm_dispatch(f, dtype, NormForwardLaunch{a, f, static_cast<cudaStream_t>(stream)});
}

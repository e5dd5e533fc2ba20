// Dropout of features from a counter-based generator, with the ReLU before it, and its gradient.
// The reference stops at the sparse product (spmm_accel.cu:104-108); a layer that is trained has this behind it.
#include "rows.h"
#include "kernels/dropout_kernels.cuh"

namespace agcn {

template <typename T, bool VEC>
static int dropout_launch(DropoutParams &p, cudaStream_t s)
{
    int dev = 0, sms = 0;
    const int rc = current_sm_count(&dev, &sms);
    if (rc != AGCN_OK) return rc;
    const int64_t chunks = ceil_div(p.cols, Elem<T>::E);
    p.lanes = 1;
    while (p.lanes < DROPOUT_THREADS && p.lanes < chunks) p.lanes *= 2;
    const int64_t needed = ceil_div(p.rows * p.lanes, DROPOUT_THREADS), most = (int64_t)sms * 8;
    dropout_kernel<T, VEC><<<(unsigned)(needed < most ? needed : most), DROPOUT_THREADS, 0, s>>>(p);
    AGCN_LAUNCH_CHECK("dropout_kernel");
    return AGCN_OK;
}

static int dropout_run(const char *who, const Rows &v, const Rows &gate, const Rows &out, int64_t rows, int64_t cols, int dtype, int activation,
                       bool backward, double prob, int64_t seed, int64_t offset, const int64_t *d_step, int64_t row0, cudaStream_t s)
{
    DropoutParams a = {};
    int rc = check_sizes(who, rows, cols, ROWS_MAX_ELEMENTS, dtype, activation);
    if (rc == AGCN_OK) rc = make_mask(who, &a.mask, prob, seed, offset, d_step, row0, rows, cols);
    if (rc != AGCN_OK || rows == 0) return rc;
    const bool gated = backward && activation == AGCN_ACT_RELU;
    const Rows t[3] = {v, out, gate};
    const int n = gated ? 3 : 2;
    for (int k = 0; k < n; k++)
        if ((rc = check_rows(who, t[k], rows, cols, dtype)) != AGCN_OK) return rc;
    a.v = v.ptr; a.ldv = v.ld; a.out = const_cast<void *>(out.ptr); a.ldout = out.ld;
    if (gated) { a.gate = gate.ptr; a.ldgate = gate.ld; }
    a.rows = rows; a.cols = cols;
    a.relu = !backward && activation == AGCN_ACT_RELU;
    int shift = 0;
    const bool vec = rows_sit_alike(t, n, dtype, &shift);
    if (dtype == AGCN_F32) return vec ? dropout_launch<float, true>(a, s) : dropout_launch<float, false>(a, s);
    if (dtype == AGCN_BF16) return vec ? dropout_launch<__nv_bfloat16, true>(a, s) : dropout_launch<__nv_bfloat16, false>(a, s);
    return vec ? dropout_launch<__half, true>(a, s) : dropout_launch<__half, false>(a, s);
}

}  // namespace agcn

extern "C" int agcn_dropout(const void *d_x, int64_t ldx, void *d_y, int64_t ldy, int64_t rows, int64_t cols, int dtype, int activation, double p,
                            int64_t seed, int64_t offset, const int64_t *d_step, int64_t row0, void *stream)
{
    agcn::clear_error();
    return agcn::dropout_run("agcn_dropout", {d_x, ldx, "x"}, {nullptr, 0, ""}, {d_y, ldy, "y"}, rows, cols, dtype, activation, false, p, seed, offset,
                             d_step, row0, static_cast<cudaStream_t>(stream));
}

extern "C" int agcn_dropout_backward(const void *d_dy, int64_t lddy, const void *d_x, int64_t ldx, void *d_dx, int64_t lddx, int64_t rows,
                                     int64_t cols, int dtype, int activation, double p, int64_t seed, int64_t offset, const int64_t *d_step,
                                     int64_t row0, void *stream)
{
    agcn::clear_error();
    return agcn::dropout_run("agcn_dropout_backward", {d_dy, lddy, "dy"}, {d_x, ldx, "x"}, {d_dx, lddx, "dx"}, rows, cols, dtype, activation, true, p,
                             seed, offset, d_step, row0, static_cast<cudaStream_t>(stream));
}

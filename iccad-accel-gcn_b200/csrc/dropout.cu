// Dropout of features from a counter-based generator, with the ReLU before it, and its gradient.
// The reference stops at the sparse product (spmm_accel.cu:104-108); a layer that is trained has this behind it.
#include "rows.h"
#include "kernels/dropout_kernels.cuh"

namespace agcn {

// Thread blocks of a kernel that the current device holds at once
template <auto KERNEL> static int dropout_resident(int64_t *blocks)
{
    static int per_sm[64] = {};
    int dev = 0, sms = 0;
    const int rc = current_sm_count(&dev, &sms);
    if (rc != AGCN_OK) return rc;
    if (per_sm[dev] == 0) AGCN_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm[dev], KERNEL, DROPOUT_THREADS, 0));
    *blocks = (int64_t)per_sm[dev] * sms;
    return AGCN_OK;
}

// `rounds` thread blocks for one that the GPU holds: the reader of two tensors gains by it (2 400 000 x 64: 302 us with one, 275 with 4),
// that of one loses (199, 205).
template <auto KERNEL> static int dropout_array(const DropoutParams &p, int64_t chunks, int rounds, cudaStream_t s)
{
    int64_t resident = 0;
    const int rc = dropout_resident<KERNEL>(&resident);
    if (rc != AGCN_OK) return rc;
    const int64_t needed = ceil_div(chunks, DROPOUT_THREADS);
    resident *= rounds;
    AGCN_CUDA(launch_early(true, KERNEL, (unsigned)(needed < resident ? needed : resident), DROPOUT_THREADS, 0, s, p));
    return AGCN_OK;
}

template <auto KERNEL> static int dropout_rows(DropoutParams &p, int64_t chunks, cudaStream_t s)
{
    int64_t resident = 0;
    const int rc = dropout_resident<KERNEL>(&resident);
    if (rc != AGCN_OK) return rc;
    p.lanes = (int)(chunks < DROPOUT_LANES ? chunks : DROPOUT_LANES);
    p.groups = resident * DROPOUT_THREADS / p.lanes / 8 * 8;       // at least 8: an SM holds 256 threads, and there are 32 and more
    if (p.rows < p.groups) p.groups = p.rows;
    AGCN_REQUIRE(p.groups > 0 && p.rows / p.groups < INT32_MAX, "dropout: row count out of range");
    p.turns = (int)(p.rows / p.groups);
    p.rest = p.rows % p.groups;
    AGCN_CUDA(launch_early(true, KERNEL, (unsigned)ceil_div(p.groups * p.lanes, DROPOUT_THREADS), DROPOUT_THREADS, 0, s, p));
    return AGCN_OK;
}

template <typename T, bool GATE>
static int dropout_launch(DropoutParams &p, bool array, int layout, int shift, cudaStream_t s)
{
    if (array) return dropout_array<dropout_array_kernel<T, GATE>>(p, ceil_div(p.rows * p.cols + shift, Elem<T>::E), GATE ? 4 : 1, s);
    const int64_t chunks = ceil_div(p.cols + shift, Elem<T>::E);
    if (layout == ROWS_WHOLE) return dropout_rows<dropout_rows_kernel<T, ROWS_WHOLE, GATE>>(p, chunks, s);
    return layout == ROWS_EDGES ? dropout_rows<dropout_rows_kernel<T, ROWS_EDGES, GATE>>(p, chunks, s)
                                : dropout_rows<dropout_rows_kernel<T, ROWS_LOOSE, GATE>>(p, chunks, s);
}

template <typename T>
static int dropout_typed(DropoutParams &p, bool array, int layout, int shift, cudaStream_t s)
{
    return p.gate != nullptr ? dropout_launch<T, true>(p, array, layout, shift, s) : dropout_launch<T, false>(p, array, layout, shift, s);
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
    const int layout = rows_layout(t, n, cols, dtype, &shift);
    bool array = layout != ROWS_LOOSE;
    for (int k = 0; k < n; k++) array = array && (t[k].ld == cols || rows == 1);
    if (dtype == AGCN_F32) return dropout_typed<float>(a, array, layout, shift, s);
    return dtype == AGCN_BF16 ? dropout_typed<__nv_bfloat16>(a, array, layout, shift, s) : dropout_typed<__half>(a, array, layout, shift, s);
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

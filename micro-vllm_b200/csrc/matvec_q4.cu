// matvec_q4.cu -- host entries of the few-row products with 4-bit weights.
#include "host.hpp"
#include "matvec_q4.cuh"

using namespace mvb;

namespace {

using bf = __nv_bfloat16;

template <typename TX, typename TY>
int matvec_launch(cudaStream_t st, bool grad, int nb, const MatvecArgs &a, const TX *x,
                  int64_t ldx, TY *y, int64_t ldy) {
    if (grad)
        MVB_TRY(launch_serial(matvec_grad_simple_kernel<TX, TY>, dim3((a.I + 255) / 256, nb),
                              dim3(256), 0, st, a, x, ldx, y, ldy));
    else
        MVB_TRY(launch_serial(matvec_simple_kernel<TX, TY>, dim3((a.O + 7) / 8, nb), dim3(256), 0,
                              st, a, x, ldx, y, ldy));
    return MVLLM_OK;
}

int matvec_any(const char *who, void *stream, bool grad, int nb, const MatvecArgs &a,
               const void *x, int x_dtype, int64_t ldx, void *y, int y_dtype, int64_t ldy) {
    const int out = grad ? a.I : a.O;
    if ((a.fmt != MVLLM_FMT_INT4_G64 && a.fmt != MVLLM_FMT_MXFP4) ||
        (a.rows > 0 && (!x || !y)) || a.I < 1 ||
        a.O < 1 || a.rows < 0 || ldx < 0 || ldy < out ||
        (x_dtype != MVLLM_DTYPE_F32 && x_dtype != MVLLM_DTYPE_BF16) ||
        (y_dtype != MVLLM_DTYPE_F32 && y_dtype != MVLLM_DTYPE_BF16))
        return host_fail(MVLLM_ERR_INVALID, "%s: invalid arguments", who);
    DeviceScope dev;
    if (int rc = dev.enter())
        return rc;
    if (a.rows == 0)
        return MVLLM_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool fx = x_dtype == MVLLM_DTYPE_F32, fy = y_dtype == MVLLM_DTYPE_F32;
    if (fx && fy)
        return matvec_launch(st, grad, nb, a, static_cast<const float *>(x), ldx,
                             static_cast<float *>(y), ldy);
    if (fx)
        return matvec_launch(st, grad, nb, a, static_cast<const float *>(x), ldx,
                             static_cast<bf *>(y), ldy);
    if (fy)
        return matvec_launch(st, grad, nb, a, static_cast<const bf *>(x), ldx,
                             static_cast<float *>(y), ldy);
    return matvec_launch(st, grad, nb, a, static_cast<const bf *>(x), ldx, static_cast<bf *>(y),
                         ldy);
}

int matvec_one(const char *who, void *stream, bool grad, int fmt, const void *x, int x_dtype,
               int64_t ldx, const void *w, const void *s, int S, int I, int O, void *y,
               int y_dtype, int64_t ldy) {
    if (!w || !s || (fmt == MVLLM_FMT_INT4_G64 && (reinterpret_cast<uintptr_t>(s) & 3u)))
        return host_fail(MVLLM_ERR_INVALID, "%s: invalid arguments", who);
    MatvecArgs a{};
    a.fmt = fmt, a.I = I, a.O = O, a.w = w, a.s = s, a.rows = S;
    return matvec_any(who, stream, grad, 1, a, x, x_dtype, ldx, y, y_dtype, ldy);
}

int matvec_experts(const char *who, void *stream, bool grad, int fmt, int nb, const void *x,
                   int x_dtype, int64_t ldx, int rows_cap, const int *nr, const int *xoff,
                   const void *const *wt, const void *const *st, int I, int O, void *y,
                   int y_dtype, int64_t ldy) {
    if (!wt || !st || !nr || !xoff || nb < 1 || nb > 1024)
        return host_fail(MVLLM_ERR_INVALID, "%s: invalid arguments", who);
    MatvecArgs a{};
    a.fmt = fmt, a.I = I, a.O = O, a.wt = wt, a.st = st, a.nr = nr, a.xoff = xoff;
    a.rows = rows_cap;
    return matvec_any(who, stream, grad, nb, a, x, x_dtype, ldx, y, y_dtype, ldy);
}

} // namespace

extern "C" {

int mvllm_matvec_q4_dev(void *stream, int fmt, const void *x, int x_dtype, int64_t ldx,
                        const void *w, const void *scales, int S, int I, int O, void *y,
                        int y_dtype, int64_t ldy) {
    return matvec_one("matvec_q4_dev", stream, false, fmt, x, x_dtype, ldx, w, scales, S, I, O, y,
                      y_dtype, ldy);
}

int mvllm_matvec_q4_grad_dev(void *stream, int fmt, const void *dy, int dy_dtype, int64_t lddy,
                             const void *w, const void *scales, int S, int I, int O, void *dx,
                             int dx_dtype, int64_t lddx) {
    return matvec_one("matvec_q4_grad_dev", stream, true, fmt, dy, dy_dtype, lddy, w, scales, S,
                      I, O, dx, dx_dtype, lddx);
}

int mvllm_moe_matvec_q4_dev(void *stream, int fmt, int nb, const void *x, int x_dtype,
                            int64_t ldx, int rows_cap, const int *nr, const int *xoff,
                            const void *const *w, const void *const *scales, int I, int O,
                            void *y, int y_dtype, int64_t ldy) {
    return matvec_experts("moe_matvec_q4_dev", stream, false, fmt, nb, x, x_dtype, ldx, rows_cap,
                          nr, xoff, w, scales, I, O, y, y_dtype, ldy);
}

int mvllm_moe_matvec_q4_grad_dev(void *stream, int fmt, int nb, const void *dy, int dy_dtype,
                                 int64_t lddy, int rows_cap, const int *nr, const int *xoff,
                                 const void *const *w, const void *const *scales, int I, int O,
                                 void *dx, int dx_dtype, int64_t lddx) {
    return matvec_experts("moe_matvec_q4_grad_dev", stream, true, fmt, nb, dy, dy_dtype, lddy,
                          rows_cap, nr, xoff, w, scales, I, O, dx, dx_dtype, lddx);
}

} // extern "C"

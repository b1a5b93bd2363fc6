// matvec_q4.cuh -- products of few rows with 4-bit weights and their
// gradient, for one matrix or for the expert-sorted rows of many.
//
//   forward   y[r, o]  = sum_i W[o, i] x[r, i]
//   gradient  dx[r, i] = sum_o W[o, i] dy[r, o]
// with W[o, i] = q[o, i] s[o, i / G] decoded from the packed formats (int4
// with a f32 scale per G = 64 columns, MXFP4 with a ue8m0 scale per G = 32).
// Sums are f32.
#pragma once

#include "row_kernels.cuh"

namespace mvb {

struct MatvecArgs {
    int fmt, I, O;
    const void *w, *s;               // one matrix, or
    const void *const *wt, *const *st; // device tables of the experts' matrices
    const int *nr, *xoff;            // segments of the rows (tables only)
    int rows;                        // rows of x and y
};

// One weight, from the formats' bit fields.
__device__ __forceinline__ float q4_weight(const void *w, const void *s, int fmt, int o, int i,
                                           int I) {
    const uint32_t b = static_cast<const uint8_t *>(w)[int64_t(o) * ((I + 1) / 2) + (i >> 1)];
    const uint32_t code = (i & 1) ? b >> 4 : b & 15u;
    if (fmt == MVLLM_FMT_INT4_G64)
        return (static_cast<int>(code) - 8) *
               static_cast<const float *>(s)[int64_t(o) * ((I + 63) / 64) + (i >> 6)];
    uint32_t h0, h1, h2, h3;
    e2m1x8_to_f16x8(code, h0, h1, h2, h3);
    return __half2float(__ushort_as_half(static_cast<unsigned short>(h0))) *
           ue8m0_to_f32(static_cast<const uint8_t *>(s)[int64_t(o) * ((I + 31) / 32) + (i >> 5)]);
}

// Matrix and row range of expert e; an expert without weights has w null.
__device__ __forceinline__ bool matvec_expert(const MatvecArgs &a, int e, const void *&w,
                                              const void *&s, int &r0, int &r1) {
    if (!a.wt) {
        w = a.w, s = a.s, r0 = 0, r1 = a.rows;
        return r1 > 0;
    }
    const int64_t off = a.xoff[e], n = a.nr[e];
    if (n <= 0 || off < 0)
        return false;
    r0 = static_cast<int>(min(off, int64_t(a.rows)));
    r1 = static_cast<int>(min(off + n, int64_t(a.rows)));
    w = a.wt[e], s = a.st[e];
    if (!s)
        w = nullptr;
    return r0 < r1;
}

// A warp per output column o, lanes over I.
template <typename TX, typename TY>
__global__ void __launch_bounds__(256)
    matvec_simple_kernel(const MatvecArgs a, const TX *__restrict__ x, int64_t ldx,
                         TY *__restrict__ y, int64_t ldy) {
    pdl_wait();
    const void *w, *s;
    int r0, r1;
    const int lane = threadIdx.x & 31, o = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (!matvec_expert(a, blockIdx.y, w, s, r0, r1) || o >= a.O)
        return;
    for (int r = r0; r < r1; ++r) {
        float acc = 0.f;
        if (w)
            for (int i = lane; i < a.I; i += 32) {
                float v[1];
                load_row<1>(x + r * ldx + i, v);
                acc = fmaf(q4_weight(w, s, a.fmt, o, i, a.I), v[0], acc);
            }
#pragma unroll
        for (int m = 16; m > 0; m >>= 1)
            acc += __shfl_xor_sync(0xffffffffu, acc, m);
        const float out[1] = {acc};
        if (lane == 0)
            store_row<1>(y + r * ldy + o, out);
    }
}

// A thread per input column i.
template <typename TX, typename TY>
__global__ void __launch_bounds__(256)
    matvec_grad_simple_kernel(const MatvecArgs a, const TX *__restrict__ dy, int64_t lddy,
                              TY *__restrict__ dx, int64_t lddx) {
    pdl_wait();
    const void *w, *s;
    int r0, r1;
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (!matvec_expert(a, blockIdx.y, w, s, r0, r1) || i >= a.I)
        return;
    for (int r = r0; r < r1; ++r) {
        float acc = 0.f;
        if (w)
            for (int o = 0; o < a.O; ++o) {
                float v[1];
                load_row<1>(dy + r * lddy + o, v);
                acc = fmaf(q4_weight(w, s, a.fmt, o, i, a.I), v[0], acc);
            }
        const float out[1] = {acc};
        store_row<1>(dx + r * lddx + i, out);
    }
}

} // namespace mvb

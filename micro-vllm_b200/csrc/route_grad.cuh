// route_grad.cuh -- the gradient of the router's weights (route_kernels.cuh).
//
// Forward: z = x . router^T, s = sigmoid(z) or sqrt(softplus(z)), ids by the
// choice s + bias, m_k = max(s[idx_k], 0), M = sum_k m_k and
// wt_k = c m_k / M (c = routed_scale).  The bias only selects.  Backward,
// with g_k = c dwt_k:
//   dm_k = (g_k - sum_j g_j m_j / M) / M          (0 where m_k or M is 0)
//   dz_k = dm_k s'(z_k),  s' = s (1 - s)                     sigmoid
//                         s' = (1 - e^(-s^2)) / (2 s)        sqrt(softplus),
// the second from softplus' = sigmoid(z) = 1 - e^(-softplus) and s^2 =
// softplus: both need the scores alone.  Then
//   dx[t]      = sum_k dz_k router[idx_k]
//   drouter[e] = sum over the tokens routed to e of dz x[t].
// Only K of a token's E logits have a gradient, so the two products are
// gathers over the permutation's order, 4 T K H operations in place of 4 T E H.
#pragma once

#include "row_kernels.cuh"

namespace mvb {

struct RouteGradArgs {
    const int *idx;      // [T, K]
    const float *scores; // [T, E]
    const float *dwt;    // [T, K]
    const int *tok_pos;  // [T, KK]
    const float *router; // [E, H]
    int T, K, KK, E, H, cap, score_fn, accumulate;
    float scale;
    float *dzp; // [cap] dz of each sorted position
};

// dz of lane k's slot (K <= 32, one warp a token); 0 for lanes past K and ids
// outside [0, E).
__device__ __forceinline__ float route_slot_grad(const RouteGradArgs &a, int64_t t, int &e) {
    const int lane = threadIdx.x & 31;
    e = lane < a.K ? a.idx[t * a.K + lane] : -1;
    if (e >= a.E)
        e = -1;
    float m = 0.f, g = 0.f;
    if (e >= 0) {
        m = fmaxf(a.scores[t * a.E + e], 0.f);
        g = a.scale * a.dwt[t * a.K + lane];
    }
    float M = 0.f, G = 0.f;
    for (int k = 0; k < a.K; ++k) { // slot order, the same on every lane
        const float mk = __shfl_sync(0xffffffffu, m, k), gk = __shfl_sync(0xffffffffu, g, k);
        M += mk;
        G = fmaf(gk, mk, G);
    }
    if (e < 0 || !(m > 0.f))
        return 0.f;
    const float dm = (g - G / M) / M;
    const float slope = a.score_fn == MVLLM_SCORE_SQRT_SOFTPLUS ? -expm1f(-m * m) / (2.f * m)
                                                                : m * (1.f - m);
    return dm * slope;
}

// A warp per token: dz, and its value at the sorted position of each slot
// (slots that repeat an id add to the first one's).
__global__ void __launch_bounds__(256) route_dz_kernel(const RouteGradArgs a) {
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t t = blockIdx.x * int64_t(blockDim.x >> 5) + (threadIdx.x >> 5);
    if (t >= a.T)
        return;
    int e;
    const float dz = route_slot_grad(a, t, e);
    float sum = 0.f;
    for (int k = 0; k < a.K; ++k) {
        const float dk = __shfl_sync(0xffffffffu, dz, k);
        if (__shfl_sync(0xffffffffu, e, k) == e)
            sum += dk;
    }
    if (lane < a.K) {
        const int p = a.tok_pos[t * a.KK + lane];
        if (p >= 0 && p < a.cap)
            a.dzp[p] = sum;
    }
}

// dx[t] = sum_k dz_k router[idx_k], a CTA per token.
template <typename TO>
__global__ void __launch_bounds__(256)
    route_dx_kernel(const RouteGradArgs a, TO *__restrict__ dx, int64_t lddx) {
    pdl_wait();
    __shared__ float sdz[32];
    __shared__ int se[32];
    const int64_t t = blockIdx.x;
    if (threadIdx.x < 32) {
        int e;
        sdz[threadIdx.x] = route_slot_grad(a, t, e);
        se[threadIdx.x] = e;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.H; c += blockDim.x) {
        float acc[1] = {0.f};
        if (a.accumulate)
            load_row<1>(dx + t * lddx + c, acc);
        for (int k = 0; k < a.K; ++k)
            if (se[k] >= 0)
                acc[0] = fmaf(sdz[k], a.router[int64_t(se[k]) * a.H + c], acc[0]);
        store_row<1>(dx + t * lddx + c, acc);
    }
}

// drouter[e] = sum over e's sorted rows of dz x[rows], a CTA per (expert,
// columns), rows in ascending order.
template <typename TX>
__global__ void __launch_bounds__(256)
    route_dw_kernel(const RouteGradArgs a, const TX *__restrict__ x, int64_t ldx,
                    const int *__restrict__ nr, const int *__restrict__ xoff,
                    const int *__restrict__ rows, float *__restrict__ drouter) {
    pdl_wait();
    const int e = blockIdx.x, c = blockIdx.y * blockDim.x + threadIdx.x;
    if (c >= a.H)
        return;
    const int n = nr[e], off = xoff[e];
    float acc = a.accumulate ? drouter[int64_t(e) * a.H + c] : 0.f;
    for (int i = 0; i < n; ++i) {
        const int p = off + i;
        if (p < 0 || p >= a.cap)
            break;
        const int t = rows[p];
        if (t < 0 || t >= a.T)
            continue;
        float v[1];
        load_row<1>(x + t * ldx + c, v);
        acc = fmaf(a.dzp[p], v[0], acc);
    }
    drouter[int64_t(e) * a.H + c] = acc;
}

} // namespace mvb

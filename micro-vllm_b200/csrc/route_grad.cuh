// route_grad.cuh -- the gradient of the router's weights (route_kernels.cuh).
//
// Forward: z = x . router^T, s = sigmoid(z) or sqrt(softplus(z)), ids by the
// choice s + bias, m_k = max(s[idx_k], 0), M = sum_k m_k and
// wt_k = c m_k / M (c = routed_scale).  The bias only selects.  Backward,
// with g_k = c dwt_k:
//   dm_k = (g_k - sum_j g_j m_j / M) / M          (0 where m_k is 0, or where
//                         M is 0 or NaN: the forward pass has wt_k = c / K there)
//   dz_k = dm_k s'(z_k),  s' = s (1 - s)                     sigmoid
//                         s' = (1 - e^(-s^2)) / (2 s)        sqrt(softplus),
// the second from softplus' = sigmoid(z) = 1 - e^(-softplus) and s^2 =
// softplus: both need the scores alone.  With w_k = m_k / M the product is
// taken as (g_k - sum_j g_j w_j) w_k (s' / m_k), whose factors stay in range
// where all scores of a token are tiny.  Then
//   dx[t]      = sum_k dz_k router[idx_k]
//   drouter[e] = sum over the tokens routed to e of dz x[t].
// Only K of a token's E logits have a gradient, so the two products are
// gathers over the permutation's order, 4 T K H operations in place of 4 T E H.
#pragma once

#include "row_kernels.cuh"

#include <type_traits>

namespace mvb {

struct RouteGradArgs {
    const int *idx;      // [T, K]
    const float *scores; // [T, E]
    const float *dwt;    // [T, K]
    const int *tok_pos;  // [T, KK]
    const float *router; // [E, H]
    int T, K, KK, E, H, cap, score_fn, accumulate;
    int block;      // sorted rows of a drouter item
    int counters;   // of `arrived`; 0 where drouter is not asked for
    float scale;
    float *dzp;     // [cap] the sorted positions' dz, null likewise
    int *arrived;   // [E, column blocks] partial sums of an expert that are done,
                    // and one more: the drouter items taken
    float *partial; // [row blocks][H]
};

constexpr int kRgCols = 256; // columns of a drouter item
constexpr int kRgRows = 64; // sorted rows of a drouter item, at least
constexpr int kRgThreads = 256; // of a dx CTA

// dz of lane k's slot (K <= 32, one warp a token); 0 for lanes past K and ids
// outside [0, E).
__device__ __forceinline__ float route_slot_grad(const RouteGradArgs &a, int64_t t, int &e) {
    const int lane = threadIdx.x & 31;
    e = lane < a.K ? a.idx[t * a.K + lane] : -1;
    if (e >= a.E)
        e = -1;
    float m = 0.f, g = 0.f;
    if (e >= 0) {
        m = a.scores[t * a.E + e];
        m = m < 0.f ? 0.f : m; // NaN stays, as in the forward pass
        g = a.scale * a.dwt[t * a.K + lane];
    }
    float M = 0.f, G = 0.f; // sums in slot order, the same on every lane
    for (int k = 0; k < a.K; ++k)
        M += __shfl_sync(0xffffffffu, m, k);
    const bool live = e >= 0 && m > 0.f && M > 0.f;
    const float w = live ? m / M : 0.f;
    for (int k = 0; k < a.K; ++k)
        G = fmaf(__shfl_sync(0xffffffffu, g, k), __shfl_sync(0xffffffffu, w, k), G);
    if (!live)
        return 0.f;
    const float mm = m * m;
    const float slope = a.score_fn != MVLLM_SCORE_SQRT_SOFTPLUS ? 1.f - m
                        : mm < 0x1p-24f                         ? 0.5f // 1 - e^-mm = mm
                                                                : -expm1f(-mm) / (2.f * mm);
    return (g - G) * w * slope;
}

// At the sorted position of each id the sum of its slots' dz (slots that
// repeat an id add to the first one's), for drouter.
__device__ __forceinline__ void route_put_grad(const RouteGradArgs &a, int64_t t, int e, float dz) {
    const int lane = threadIdx.x & 31;
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
// Clears the drouter kernel's counters.
__device__ __forceinline__ void route_clear(const RouteGradArgs &a) {
    for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < a.counters;
         i += int64_t(gridDim.x) * blockDim.x)
        a.arrived[i] = 0;
}

// What drouter needs, where dx is not asked for: a warp per token.
__global__ void __launch_bounds__(256) route_dz_kernel(const RouteGradArgs a) {
    pdl_wait();
    pdl_trigger();
    route_clear(a);
    const int64_t t = blockIdx.x * int64_t(blockDim.x >> 5) + (threadIdx.x >> 5);
    if (t >= a.T)
        return;
    int e;
    const float dz = route_slot_grad(a, t, e);
    route_put_grad(a, t, e, dz);
}

// dx[t] = sum_k dz_k router[idx_k], the router's rows gathered: a CTA takes
// (token, segment of the row).  The gathers are 4 T K H bytes, 1.9 GB in 102 us
// for 8192 tokens of 8 out of 384 experts, H 7168; half of the sectors hit L1,
// whose throughput and the issue slots both stand at 78%.  (A form with some
// columns of every expert in shared memory, which the CTA's tokens then read,
// took 25 to 60% longer up to 64 slots per expert and was never more than 7%
// ahead; eight columns a lane split the sectors, 117 us in place of 82 on 6144
// tokens.)
template <typename TO, int N>
__global__ void __launch_bounds__(kRgThreads)
    route_dx_kernel(const RouteGradArgs a, int nseg, int seg, TO *__restrict__ dx, int64_t lddx) {
    pdl_wait();
    pdl_trigger();
    __shared__ float sdz[32];
    __shared__ int se[32];
    const int64_t t = blockIdx.x / nseg;
    const int part = static_cast<int>(blockIdx.x % nseg);
    const int s0 = part * seg, s1 = min(a.H, s0 + seg);
    if (threadIdx.x < 32) {
        int e;
        const float dz = route_slot_grad(a, t, e);
        sdz[threadIdx.x] = dz, se[threadIdx.x] = e;
        if (part == 0 && a.dzp)
            route_put_grad(a, t, e, dz);
    }
    route_clear(a);
    __syncthreads();
    for (int c = s0 + threadIdx.x * N; c < s1; c += kRgThreads * N) {
        float acc[N] = {};
        if (a.accumulate)
            load_row<N>(dx + t * lddx + c, acc);
#pragma unroll 4
        for (int k = 0; k < a.K; ++k) {
            if (se[k] >= 0) {
                float v[N];
                load_row<N>(a.router + int64_t(se[k]) * a.H + c, v);
#pragma unroll
                for (int q = 0; q < N; ++q)
                    acc[q] = fmaf(sdz[k], v[q], acc[q]);
            }
        }
        store_row<N>(dx + t * lddx + c, acc);
    }
}

// drouter[e] = sum over e's sorted rows of dz x[rows].  An item is (a block of
// kRgCols columns, an expert, `block` of its rows); each warp takes the next
// one, and has four rows' loads under way: 32 warps per SM so hide more of the
// gathers' latency than 16 with eight rows each (97 against 103 us on 65536
// slots spread evenly over 384 experts, H 7168, bf16; 112 where they are uneven).
// Items run by groups of eight column blocks, so the columns of x that all
// experts gather from (16 T kRgCols bytes in bf16) stay in L2.  An expert of several items leaves its partial sums in
// the workspace, and the warp that arrives last adds them in order; one without
// rows gets zeros.  Bound by the latency of the gathers, a third of whose
// sectors miss the near L2; issue slots stand at 52%.  (Rows through a ring of
// asynchronous copies, three times as many under way, took 140 us.)
template <typename TX>
__global__ void __launch_bounds__(256, sizeof(TX) == 4 ? 2 : 4)
    route_dw_kernel(const RouteGradArgs a, const TX *__restrict__ x, int64_t ldx, int vec,
                    const int *__restrict__ nr, const int *__restrict__ xoff,
                    const int *__restrict__ rows, float *__restrict__ drouter) {
    constexpr int B = 4;
    __shared__ int first[1025]; // row blocks before each expert
    __shared__ int wsum[8];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // Prefix sums of the experts' row blocks, four experts a thread.
    int n4[4], v = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int e = 4 * int(threadIdx.x) + k;
        n4[k] = e < a.E ? max(1, (min(nr[e], a.cap) + a.block - 1) / a.block) : 0;
        v += n4[k];
    }
    int before = -v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        v += lane >= o ? u : 0;
    }
    if (lane == 31)
        wsum[warp] = v;
    __syncthreads();
    before += v;
    for (int k = 0; k < warp; ++k)
        before += wsum[k];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int e = 4 * int(threadIdx.x) + k;
        if (e < a.E)
            first[e] = before;
        before += n4[k];
        if (e == a.E - 1)
            first[a.E] = before;
    }
    __syncthreads();
    // (No more than the workspace holds, whatever nr says.)
    const int blocks = min(first[a.E], a.cap / a.block + a.E);
    const int ncol = (a.H + kRgCols - 1) / kRgCols, groups = (ncol + 7) / 8;
    const int total = blocks * groups * 8;
    for (;;) { // a warp at a time: items differ in rows by a hundredfold
        int ticket = 0;
        if (lane == 0)
            ticket = atomicAdd(&a.arrived[a.E * ncol], 1);
        ticket = __shfl_sync(0xffffffffu, ticket, 0);
        if (ticket >= total)
            break;
        const int cg = ticket / (blocks * 8), slot = ticket / 8 - cg * blocks;
        const int cb = cg * 8 + (ticket & 7);
        if (cb >= ncol)
            continue;
        int lo = 0, hi = a.E; // the last expert with first[e] <= slot
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first[mid] <= slot)
                lo = mid;
            else
                hi = mid;
        }
        const int e = lo, rb = slot - first[e], nblk = first[e + 1] - first[e];
        const int off = xoff[e], n = min(nr[e], a.cap);
        const int p0 = off + rb * a.block, p1 = min(min(off + n, p0 + a.block), a.cap);
        const int c = cb * kRgCols + lane * 8;
        const bool inside = vec && (cb + 1) * kRgCols <= a.H;
        float acc[8] = {};
        // 32 rows at a time, their tokens and dz by lane; one that does not
        // count loads token 0's and is not added
        auto slots = [&](int pb, int &t, float &dz) {
            const int p = pb + lane;
            t = -1, dz = 0.f;
            if (p >= 0 && p < p1) {
                t = rows[p];
                dz = a.dzp[p];
                if (t < 0 || t >= a.T)
                    t = -1;
            }
        };
        int t_next;
        float dz_next;
        slots(p0, t_next, dz_next);
        for (int pb = p0; pb < p1; pb += 32) {
            const int t = t_next;
            const float dz = dz_next;
            slots(pb + 32, t_next, dz_next);
            const int cnt = min(32, p1 - pb);
            const uint32_t odd = __ballot_sync(0xffffffffu, t < 0);
            const int whole = odd ? __ffs(odd) - 1 : 32; // rows that count, from the first on
            for (int j0 = 0; j0 < cnt; j0 += B) {
                Raw8<TX> xv[B];
                int tj[B];
                float dj[B];
#pragma unroll
                for (int j = 0; j < B; ++j) {
                    tj[j] = __shfl_sync(0xffffffffu, t, j0 + j);
                    dj[j] = __shfl_sync(0xffffffffu, dz, j0 + j);
                }
                if (inside) { // uniform over the warp: loads side by side
#pragma unroll
                    for (int j = 0; j < B; ++j)
                        xv[j].load_whole(x + max(tj[j], 0) * ldx + c);
                } else {
#pragma unroll
                    for (int j = 0; j < B; ++j)
                        xv[j].load(x + max(tj[j], 0) * ldx, min(c, a.H), a.H, vec);
                }
                auto add = [&](auto some) { // `some` of them may not count
#pragma unroll
                    for (int j = 0; j < B; ++j) {
                        if (some.value && tj[j] < 0)
                            continue;
                        float f[8];
                        xv[j].get(f);
#pragma unroll
                        for (int s = 0; s < 8; s += 2)
                            ffma2(acc[s], acc[s + 1], f[s], f[s + 1], dj[j]);
                    }
                };
                if (j0 + B <= whole)
                    add(std::false_type{});
                else
                    add(std::true_type{});
            }
        }
        float *out = drouter + int64_t(e) * a.H + c;
        const bool whole = (a.H & 3) == 0 && (reinterpret_cast<uintptr_t>(drouter) & 15u) == 0;
        auto put = [&](float *to, const float (&f)[8]) {
            if (whole && c + 8 <= a.H) {
                store_row<8>(to, f);
                return;
            }
#pragma unroll
            for (int s = 0; s < 8; ++s)
                if (c + s < a.H)
                    to[s] = f[s];
        };
        float base[8] = {};
        if (nblk > 1) {
            float *mine = a.partial + int64_t(slot) * a.H + c;
            put(mine, acc);
            __threadfence();
            __syncwarp();
            int arrived = 0;
            if (lane == 0)
                arrived = atomicAdd(&a.arrived[e * ncol + cb], 1);
            if (__shfl_sync(0xffffffffu, arrived, 0) != nblk - 1)
                continue;
            __threadfence();
#pragma unroll
            for (int s = 0; s < 8; ++s)
                acc[s] = 0.f;
            const float *from = a.partial + int64_t(first[e]) * a.H + c;
            if (whole && (cb + 1) * kRgCols <= a.H) {
#pragma unroll 4
                for (int k = 0; k < nblk; ++k, from += a.H) {
                    const float4 u = __ldcg(reinterpret_cast<const float4 *>(from));
                    const float4 w = __ldcg(reinterpret_cast<const float4 *>(from) + 1);
                    acc[0] += u.x, acc[1] += u.y, acc[2] += u.z, acc[3] += u.w;
                    acc[4] += w.x, acc[5] += w.y, acc[6] += w.z, acc[7] += w.w;
                }
            } else {
                for (int k = 0; k < nblk; ++k, from += a.H)
#pragma unroll
                    for (int s = 0; s < 8; ++s)
                        if (c + s < a.H)
                            acc[s] += __ldcg(from + s);
            }
        }
        if (a.accumulate) {
#pragma unroll
            for (int s = 0; s < 8; ++s)
                if (c + s < a.H)
                    base[s] = out[s];
        }
#pragma unroll
        for (int s = 0; s < 8; ++s)
            acc[s] += base[s];
        put(out, acc);
    }
}

} // namespace mvb

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
// softplus: both need the scores alone.  With w_k = m_k / M the product is
// taken as (g_k - sum_j g_j w_j) w_k (s' / m_k), whose factors stay in range
// where all scores of a token are tiny.  Then
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
    float *dz;      // [T, K] the slots' dz
    float *dzp;     // [cap] the sorted positions' dz
    int *arrived;   // [E, column blocks] partial sums of an expert that are done,
                    // and one more: the drouter items taken
    float *partial; // [row blocks][H]
};

constexpr int kRgCols = 256; // columns of a drouter item
constexpr int kRgRows = 128; // sorted rows of a drouter item
constexpr int kRgSmem = 200 * 1024;
constexpr int kRgWarps = 32; // of a dx CTA

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
    float M = 0.f, G = 0.f; // sums in slot order, the same on every lane
    for (int k = 0; k < a.K; ++k)
        M += __shfl_sync(0xffffffffu, m, k);
    const bool live = e >= 0 && m > 0.f;
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

// A warp per token: the slots' dz, and at the sorted position of each id their
// sum (slots that repeat an id add to the first one's).  Clears the drouter
// kernel's counters.
__global__ void __launch_bounds__(256) route_dz_kernel(const RouteGradArgs a, int counters) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < counters; i += gridDim.x * blockDim.x)
        a.arrived[i] = 0;
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
        a.dz[t * a.K + lane] = dz;
        const int p = a.tok_pos[t * a.KK + lane];
        if (p >= 0 && p < a.cap)
            a.dzp[p] = sum;
    }
}

// dx[t] = sum_k dz_k router[idx_k], each router row gathered from L2: a CTA
// per token, for calls of fewer slots than experts.
template <typename TO, int N>
__global__ void __launch_bounds__(256)
    route_dx_gather_kernel(const RouteGradArgs a, TO *__restrict__ dx, int64_t lddx) {
    pdl_wait();
    pdl_trigger();
    __shared__ float sdz[32];
    __shared__ int se[32];
    const int64_t t = blockIdx.x;
    if (threadIdx.x < 32) {
        int e = -1;
        if (int(threadIdx.x) < a.K)
            e = a.idx[t * a.K + threadIdx.x];
        sdz[threadIdx.x] = e >= 0 && e < a.E ? a.dz[t * a.K + threadIdx.x] : 0.f;
        se[threadIdx.x] = e >= a.E ? -1 : e;
    }
    __syncthreads();
    for (int c = threadIdx.x * N; c < a.H; c += blockDim.x * N) {
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

// The same with the router's columns in shared memory.  Gathered from L2 the
// rows are 4 T K H bytes (1.9 GB for 8192 tokens of 8 out of 384 experts, H
// 7168), which L2 serves at about half of what shared memory does; so a CTA
// keeps LPT * 4 columns of every expert (and a row of zeros for slots without
// one) and goes through tokens, LPT lanes each.  The (column block, token) plane is cut evenly over the
// CTAs, column blocks outermost.
template <typename TO, int LPT>
__global__ void __launch_bounds__(32 * kRgWarps)
    route_dx_tile_kernel(const RouteGradArgs a, TO *__restrict__ dx, int64_t lddx, int vec) {
    extern __shared__ __align__(16) float rg_tile[];
    __shared__ __align__(16) int2 pairs[kRgWarps][2][32]; // (row of the tile, dz) of a warp's slots
    constexpr int COLS = LPT * 4, TPW = 32 / LPT; // tokens a warp has at a time
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane / LPT, col4 = (lane % LPT) * 4;
    const int blocks = (a.H + COLS - 1) / COLS;
    const int64_t plane = int64_t(blocks) * a.T;
    int64_t at = plane * blockIdx.x / gridDim.x;
    const int64_t end = plane * (blockIdx.x + 1) / gridDim.x;
    while (at < end) {
        const int b = int(at / a.T), c0 = b * COLS;
        const int t0 = int(at - int64_t(b) * a.T);
        const int t1 = int(min(int64_t(a.T), t0 + end - at));
        __syncthreads(); // the last block's readers are done
        for (int i = threadIdx.x; i < (a.E + 1) * LPT; i += blockDim.x) {
            const int e = i / LPT, c = (i - e * LPT) * 4;
            const float *src = a.router + int64_t(e) * a.H + c0 + c;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (e == a.E) {
                // zeros
            } else if (vec && c0 + c + 4 <= a.H) {
                v = *reinterpret_cast<const float4 *>(src);
            } else {
                if (c0 + c < a.H)
                    v.x = src[0];
                if (c0 + c + 1 < a.H)
                    v.y = src[1];
                if (c0 + c + 2 < a.H)
                    v.z = src[2];
                if (c0 + c + 3 < a.H)
                    v.w = src[3];
            }
            *reinterpret_cast<float4 *>(rg_tile + e * COLS + c) = v;
        }
        __syncthreads();
        // A group of LPT lanes takes BT tokens at a time, their slots' ids and dz
        // by lane, the next batch's loaded before this one is worked off.
        const int bt = max(1, LPT / a.K), lk = lane % LPT;
        const int stride = kRgWarps * TPW * bt;
        auto fetch = [&](int t, int k0) { // slots k0.. of tokens t..
            int e = a.E;
            float dz = 0.f;
            const int tt = t + (a.K <= LPT ? lk / a.K : 0), k = a.K <= LPT ? lk % a.K : k0 + lk;
            if (tt < min(t1, t + bt) && k < a.K) {
                e = a.idx[int64_t(tt) * a.K + k];
                dz = a.dz[int64_t(tt) * a.K + k];
                if (e < 0 || e >= a.E)
                    e = a.E, dz = 0.f;
            }
            return make_int2(e * COLS, __float_as_int(dz));
        };
        const int c = c0 + col4;
        const bool whole = vec && c + 4 <= a.H;
        auto old = [&](int64_t t, float (&acc)[4]) {
            if (whole) {
                load_row<4>(dx + t * lddx + c, acc);
                return;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float o[1] = {0.f};
                if (c + q < a.H)
                    load_row<1>(dx + t * lddx + c + q, o);
                acc[q] = o[0];
            }
        };
        int tb = t0 + (warp * TPW + sub) * bt;
        int2 next = fetch(tb, 0);
        const int rounds = (t1 - t0 + stride - 1) / stride; // the same for every lane
        for (int i = 0; i < rounds; ++i, tb += stride) {
            // Two buffers: the last round's readers may still be at theirs.
            const int2 *slots = pairs[warp][i & 1] + sub * LPT;
            pairs[warp][i & 1][lane] = next;
            __syncwarp();
            next = fetch(tb + stride, 0);
            for (int s = 0; s < bt; ++s) {
                const int t = tb + s;
                const bool live = t < t1;
                float acc[4] = {};
                if (live && a.accumulate)
                    old(t, acc);
                for (int k0 = 0; k0 < a.K; k0 += LPT) {
                    if (k0 > 0) { // more slots than lanes: bt is 1
                        __syncwarp();
                        pairs[warp][i & 1][lane] = fetch(tb, k0);
                        __syncwarp();
                    }
                    const int n = min(LPT, a.K - k0);
#pragma unroll 8
                    for (int j = 0; j < n; ++j) {
                        const int2 p = slots[s * a.K + j];
                        const float4 v =
                            *reinterpret_cast<const float4 *>(rg_tile + p.x + col4);
                        const float dj = __int_as_float(p.y);
                        acc[0] = fmaf(dj, v.x, acc[0]), acc[1] = fmaf(dj, v.y, acc[1]);
                        acc[2] = fmaf(dj, v.z, acc[2]), acc[3] = fmaf(dj, v.w, acc[3]);
                    }
                }
                if (live) {
                    if (whole) {
                        store_row<4>(dx + t * lddx + c, acc);
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const float o[1] = {acc[q]};
                            if (c + q < a.H)
                                store_row<1>(dx + t * lddx + c + q, o);
                        }
                    }
                }
            }
        }
        at += t1 - t0;
    }
}

// drouter[e] = sum over e's sorted rows of dz x[rows].  An item is (a block of
// kRgCols columns, an expert, kRgRows of its rows); each warp takes the next
// one, and has eight (f32: four) rows' loads under way.  Items run by groups of
// eight column blocks, so the columns of x that all experts gather from (16 T
// kRgCols bytes in bf16) stay in L2.  An expert of several items leaves its
// partial sums in the workspace, and the warp that arrives last adds them in
// order; one without rows gets zeros.
template <typename TX>
__global__ void __launch_bounds__(256)
    route_dw_kernel(const RouteGradArgs a, const TX *__restrict__ x, int64_t ldx, int vec,
                    const int *__restrict__ nr, const int *__restrict__ xoff,
                    const int *__restrict__ rows, float *__restrict__ drouter) {
    constexpr int B = sizeof(TX) == 4 ? 4 : 8;
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
        n4[k] = e < a.E ? max(1, (min(nr[e], a.cap) + kRgRows - 1) / kRgRows) : 0;
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
    const int blocks = min(first[a.E], a.cap / kRgRows + a.E);
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
        const int p0 = off + rb * kRgRows, p1 = min(min(off + n, p0 + kRgRows), a.cap);
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
#pragma unroll
                for (int j = 0; j < B; ++j) {
                    float f[8];
                    xv[j].get(f);
#pragma unroll
                    for (int s = 0; s < 8; ++s)
                        acc[s] = tj[j] >= 0 ? fmaf(dj[j], f[s], acc[s]) : acc[s];
                }
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

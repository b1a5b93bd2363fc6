// row_kernels.cuh -- token rows to the expert-sorted order and back, each
// with its gradient, as steps of their own (the fused layer does them inside
// its staging and combine kernels).
//
// With p(t, j) = tok_pos[t, j] >= 0 the sorted position of token t's slot j,
// as the permutation writes it:
//   dispatch            xs[p] = x[t]
//   dispatch gradient   dx[t] = sum_j dxs[p]
//   combine             out[t] = sum_j rw[p] y[p]
//   combine gradient    dy[p] = rw[p] dout[t],  drw[p] = <dout[t], y[p]>
// The first and third are each other's adjoint up to the weights, so there
// are three kernels: one copies a token's row to its positions, one adds up
// its positions' rows (weights optional), one does both for the combine's
// gradient.  All are bound by memory: every byte is moved once.
#pragma once

#include "common.cuh"

namespace mvb {

constexpr int kMaxSlots = 64; // slots of a token: two per lane of a warp

// N elements of a row as f32; the address is a multiple of min(16, N * size).
template <int N> __device__ __forceinline__ void load_row(const float *p, float (&v)[N]) {
    if constexpr (N == 1) {
        v[0] = *p;
    } else if constexpr (N == 2) {
        const float2 a = *reinterpret_cast<const float2 *>(p);
        v[0] = a.x, v[1] = a.y;
    } else {
#pragma unroll
        for (int q = 0; q < N; q += 4) {
            const float4 a = *reinterpret_cast<const float4 *>(p + q);
            v[q] = a.x, v[q + 1] = a.y, v[q + 2] = a.z, v[q + 3] = a.w;
        }
    }
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
template <int N> __device__ __forceinline__ void load_row(const __nv_bfloat16 *p, float (&v)[N]) {
    if constexpr (N == 1) {
        v[0] = __bfloat162float(*p);
    } else if constexpr (N == 2) {
        const uint32_t a = *reinterpret_cast<const uint32_t *>(p);
        v[0] = bf16_lo(a), v[1] = bf16_hi(a);
    } else if constexpr (N == 4) {
        const uint2 a = *reinterpret_cast<const uint2 *>(p);
        v[0] = bf16_lo(a.x), v[1] = bf16_hi(a.x), v[2] = bf16_lo(a.y), v[3] = bf16_hi(a.y);
    } else {
        static_assert(N == 8, "row vector");
        const uint4 a = *reinterpret_cast<const uint4 *>(p);
        v[0] = bf16_lo(a.x), v[1] = bf16_hi(a.x), v[2] = bf16_lo(a.y), v[3] = bf16_hi(a.y);
        v[4] = bf16_lo(a.z), v[5] = bf16_hi(a.z), v[6] = bf16_lo(a.w), v[7] = bf16_hi(a.w);
    }
}

// N elements as loaded (32, 16, 8, 4 or 2 bytes), to be converted when used.
template <int BYTES> struct RowWord;
struct alignas(16) Word32 {
    uint4 lo, hi;
};
template <> struct RowWord<32> { using type = Word32; };
template <> struct RowWord<16> { using type = uint4; };
template <> struct RowWord<8> { using type = uint2; };
template <> struct RowWord<4> { using type = uint32_t; };
template <> struct RowWord<2> { using type = uint16_t; };
template <typename T, int N> struct RowVec {
    using Word = typename RowWord<N * sizeof(T)>::type;
    Word w;
    __device__ __forceinline__ void load(const T *p) { w = *reinterpret_cast<const Word *>(p); }
    __device__ __forceinline__ void get(float (&v)[N]) const {
        load_row<N>(reinterpret_cast<const T *>(&w), v);
    }
};

// The same way out; bf16 rounds once, to nearest even.
template <int N> __device__ __forceinline__ void store_row(float *p, const float (&v)[N]) {
    if constexpr (N == 1) {
        *p = v[0];
    } else if constexpr (N == 2) {
        *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
    } else {
#pragma unroll
        for (int q = 0; q < N; q += 4)
            *reinterpret_cast<float4 *>(p + q) =
                make_float4(v[q], v[q + 1], v[q + 2], v[q + 3]);
    }
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <int N> __device__ __forceinline__ void store_row(__nv_bfloat16 *p, const float (&v)[N]) {
    if constexpr (N == 1) {
        *p = __float2bfloat16_rn(v[0]);
    } else if constexpr (N == 2) {
        *reinterpret_cast<uint32_t *>(p) = pack_bf16(v[0], v[1]);
    } else if constexpr (N == 4) {
        *reinterpret_cast<uint2 *>(p) =
            make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
    } else {
        static_assert(N == 8, "row vector");
        *reinterpret_cast<uint4 *>(p) =
            make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                       pack_bf16(v[6], v[7]));
    }
}

// 8 elements of a row, as loaded; 0 past K.
template <typename TX> struct Raw8 {
    uint4 u[sizeof(TX) / 2];
    __device__ __forceinline__ void load_whole(const TX *p) {
#pragma unroll
        for (int q = 0; q < int(sizeof(TX)) / 2; ++q)
            u[q] = reinterpret_cast<const uint4 *>(p)[q];
    }
    __device__ __forceinline__ void load(const TX *row, int c, int K, bool vec) {
        if (vec && c + 8 <= K) {
#pragma unroll
            for (int q = 0; q < int(sizeof(TX)) / 2; ++q) // stays where it is written
                asm volatile("ld.global.v4.b32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(u[q].x), "=r"(u[q].y), "=r"(u[q].z), "=r"(u[q].w)
                             : "l"(reinterpret_cast<const uint4 *>(row + c) + q)
                             : "memory");
        } else {
            uint32_t w[sizeof(TX) * 2];
#pragma unroll
            for (int q = 0; q < int(sizeof(TX)) * 2; ++q) {
                w[q] = 0;
                if constexpr (sizeof(TX) == 4) {
                    if (c + q < K)
                        w[q] = __float_as_uint(row[c + q]);
                } else {
#pragma unroll
                    for (int b = 0; b < 2; ++b)
                        if (c + 2 * q + b < K)
                            w[q] |= uint32_t(__bfloat16_as_ushort(row[c + 2 * q + b])) << (16 * b);
                }
            }
#pragma unroll
            for (int q = 0; q < int(sizeof(TX)) / 2; ++q)
                u[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint4 a = u[0];
        if constexpr (sizeof(TX) == 4) {
            const uint4 b = u[1];
            v[0] = __uint_as_float(a.x), v[1] = __uint_as_float(a.y);
            v[2] = __uint_as_float(a.z), v[3] = __uint_as_float(a.w);
            v[4] = __uint_as_float(b.x), v[5] = __uint_as_float(b.y);
            v[6] = __uint_as_float(b.z), v[7] = __uint_as_float(b.w);
        } else {
            v[0] = bf16_lo(a.x), v[1] = bf16_hi(a.x), v[2] = bf16_lo(a.y), v[3] = bf16_hi(a.y);
            v[4] = bf16_lo(a.z), v[5] = bf16_hi(a.z), v[6] = bf16_lo(a.w), v[7] = bf16_hi(a.w);
        }
    }
};

// A token's slots, KK <= kMaxSlots, held by one warp: lane l keeps slots l
// and l + 32.  A slot counts when its position lies in [0, cap).
struct WarpSlots {
    int p0, p1; // positions, -1 = none
    __device__ __forceinline__ void load(const int *__restrict__ tok_pos, size_t t, int KK,
                                         int cap) {
        const int lane = threadIdx.x & 31;
        const int *row = tok_pos + t * KK;
        p0 = lane < KK ? row[lane] : -1;
        p1 = lane + 32 < KK ? row[lane + 32] : -1;
        if (p0 >= cap)
            p0 = -1;
        if (p1 >= cap)
            p1 = -1;
    }
    // Sorts the positions ascending over (lane, half) and returns their
    // number: each value goes to the place its rank names.  Slots with the same
    // position rank by slot, so that every place gets a value.
    __device__ __forceinline__ int sort(int KK, int *smem) {
        const int lane = threadIdx.x & 31;
        int r0 = 0, r1 = 0;
        for (int u = 0; u < KK; ++u) {
            const int q = __shfl_sync(0xffffffffu, u < 32 ? p0 : p1, u & 31);
            r0 += (q >= 0 && (u < lane ? q <= p0 : q < p0)) ? 1 : 0;
            r1 += (q >= 0 && (u < lane + 32 ? q <= p1 : q < p1)) ? 1 : 0;
        }
        const int n = __popc(__ballot_sync(0xffffffffu, p0 >= 0)) +
                      __popc(__ballot_sync(0xffffffffu, p1 >= 0));
        __syncwarp(); // the readers of the last token are done with smem
        if (p0 >= 0)
            smem[r0] = p0;
        if (p1 >= 0)
            smem[r1] = p1;
        __syncwarp();
        return n;
    }
};

// dispatch: a warp takes (token, piece of the row), loads Q words a lane and
// stores them at each of the token's positions: a copy of the bits, so W is
// only the widest word (16, 4 or 2 bytes) that rows, pitches and addresses are
// multiples of.  ldx, ldxs and D count words.  Bound by memory: 4096 tokens to
// 8 positions each, 7168 bf16, 6.1 TB/s.
template <typename W, int Q>
__global__ void __launch_bounds__(256)
    dispatch_rows_kernel(const W *__restrict__ x, int64_t ldx, const int *__restrict__ tok_pos,
                         int64_t units, int pieces, int KK, int D, W *__restrict__ xs,
                         int64_t ldxs, int cap) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t unit = blockIdx.x * int64_t(blockDim.x >> 5) + (threadIdx.x >> 5);
    if (unit >= units)
        return;
    const int64_t t = unit / pieces;
    const int col = static_cast<int>(unit - t * pieces) * 32 * Q + lane;
    WarpSlots sl;
    sl.load(tok_pos, t, KK, cap);
    const uint32_t m0 = __ballot_sync(0xffffffffu, sl.p0 >= 0);
    const uint32_t m1 = __ballot_sync(0xffffffffu, sl.p1 >= 0);
    if (!(m0 | m1))
        return;
    W v[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q)
        if (col + 32 * q < D)
            v[q] = x[t * ldx + col + 32 * q];
    auto copy = [&](int64_t p) {
        W *to = xs + p * ldxs + col;
#pragma unroll
        for (int q = 0; q < Q; ++q)
            if (col + 32 * q < D)
                to[32 * q] = v[q];
    };
    for (uint32_t m = m0; m; m &= m - 1)
        copy(__shfl_sync(0xffffffffu, sl.p0, __ffs(m) - 1));
    for (uint32_t m = m1; m; m &= m - 1)
        copy(__shfl_sync(0xffffffffu, sl.p1, __ffs(m) - 1));
}

// combine and the dispatch gradient: out[t] = (out[t] +) sum of rw[p] y[p]
// over the token's positions in ascending order (ascending expert id), f32
// fused multiply-adds, one rounding at the end.  rw == nullptr: weight 1.
// A warp takes (token, segment of the row) and has eight positions' loads under
// way at a time.  Bound by memory: 4096 tokens of 8 rows of 7168 bf16 into f32
// move 587 MB in 93 us, 6.3 TB/s.
template <typename TY, typename TO, int N>
__global__ void __launch_bounds__(256)
    combine_rows_kernel(const TY *__restrict__ y, int64_t ldy, int cap,
                        const float *__restrict__ rw, const int *__restrict__ tok_pos,
                        int64_t units, int nseg, int seg, int KK, int D, TO *__restrict__ out,
                        int64_t ldo, int accumulate) {
    pdl_wait();
    pdl_trigger();
    constexpr int B = 8;
    __shared__ int spos[8][kMaxSlots + B];
    __shared__ float sw[8][kMaxSlots + B];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t unit = blockIdx.x * int64_t(blockDim.x >> 5) + warp;
    if (unit >= units)
        return;
    const int64_t t = unit / nseg;
    const int s0 = static_cast<int>(unit - t * nseg) * seg, s1 = min(D, s0 + seg);
    WarpSlots sl;
    sl.load(tok_pos, t, KK, cap);
    const int n = sl.sort(KK, spos[warp]);
    // The last batch is filled up with the last position: loaded again, not added.
    const int fill = n ? spos[warp][n - 1] : 0;
    for (int j = lane; j < n + B; j += 32) {
        if (j >= n)
            spos[warp][j] = fill;
        else
            sw[warp][j] = rw ? rw[spos[warp][j]] : 1.f;
    }
    __syncwarp();
    // Narrow vectors, whose many steps repeat the address arithmetic, keep the
    // first batch's rows and weights in registers; for 16-byte vectors those
    // registers cost more (109 against 91 us on 4096 tokens of 8 rows of 7168
    // bf16 summed into f32).
    constexpr bool HELD = N * sizeof(TY) < 16;
    const TY *row[HELD ? B : 1];
    float w[HELD ? B : 1];
    auto hold = [&](int j0) {
        if constexpr (HELD) {
#pragma unroll
            for (int b = 0; b < B; ++b) {
                row[b] = y + int64_t(spos[warp][j0 + b]) * ldy;
                w[b] = sw[warp][j0 + b];
            }
        }
    };
    hold(0);
    for (int c = s0 + lane * N; c < s1; c += 32 * N) {
        float acc[N];
        if (accumulate)
            load_row<N>(out + t * ldo + c, acc);
        else
#pragma unroll
            for (int q = 0; q < N; ++q)
                acc[q] = 0.f;
        for (int j0 = 0; j0 < n; j0 += B) {
            if (n > B)
                hold(j0);
            RowVec<TY, N> v[B];
#pragma unroll
            for (int b = 0; b < B; ++b) {
                if constexpr (HELD)
                    v[b].load(row[b] + c);
                else
                    v[b].load(y + int64_t(spos[warp][j0 + b]) * ldy + c);
            }
#pragma unroll
            for (int b = 0; b < B; ++b) {
                float f[N];
                v[b].get(f);
                if constexpr (HELD) {
#pragma unroll
                    for (int q = 0; q < N; ++q)
                        acc[q] = j0 + b < n ? fmaf(w[b], f[q], acc[q]) : acc[q];
                } else if (j0 + b < n) {
#pragma unroll
                    for (int q = 0; q < N; ++q)
                        acc[q] = fmaf(sw[warp][j0 + b], f[q], acc[q]);
                }
            }
        }
        store_row<N>(out + t * ldo + c, acc);
    }
}

// The combine's gradient, a CTA per token (4096 of 8 rows of 7168 bf16, 10% of
// them padding: 147 us, 6.1 TB/s): dy[p] = rw[p] dout[t] and
// drw[p] = <dout[t], y[p]> (f32, warps' partial sums added in warp order),
// then dwt[t, k] = drw of the position that token t has for expert idx[t, k]
// (a repeated id shares the position of its first slot), 0 where it has none.
template <typename TD, typename TY, int N>
__global__ void __launch_bounds__(256)
    combine_grad_kernel(const TD *__restrict__ dout, int64_t lddo, const TY *__restrict__ y,
                        int64_t ldy, int cap, const float *__restrict__ rw,
                        const int *__restrict__ tok_pos, const int *__restrict__ idx, int K,
                        int KK, int D, TY *__restrict__ dy, int64_t lddy,
                        float *__restrict__ dwt) {
    pdl_wait();
    pdl_trigger();
    // Vectors of dout a thread keeps while it goes through the positions.
    constexpr int C = 4;
    __shared__ float part[8][kMaxSlots];
    __shared__ int spos[kMaxSlots];
    __shared__ float sw[kMaxSlots];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int64_t t = blockIdx.x;
    for (int j = threadIdx.x; j < KK; j += blockDim.x) {
        int p = tok_pos[t * KK + j];
        if (p >= cap)
            p = -1;
        spos[j] = p;
        sw[j] = p >= 0 ? rw[p] : 0.f;
    }
    for (int j = lane; j < KK; j += 32)
        part[warp][j] = 0.f;
    __syncthreads();
    const int step = blockDim.x * N;
    for (int c0 = threadIdx.x * N; c0 - int(threadIdx.x) * N < D; c0 += C * step) {
        RowVec<TD, N> g[C];
#pragma unroll
        for (int q = 0; q < C; ++q)
            if (c0 + q * step < D)
                g[q].load(dout + t * lddo + c0 + q * step);
#pragma unroll 2
        for (int j = 0; j < KK; ++j) {
            const int64_t p = spos[j];
            if (p < 0)
                continue; // uniform over the CTA
            const float w = sw[j];
            RowVec<TY, N> v[C];
#pragma unroll
            for (int q = 0; q < C; ++q)
                if (c0 + q * step < D)
                    v[q].load(y + p * ldy + c0 + q * step);
            float dot = 0.f;
#pragma unroll
            for (int q = 0; q < C; ++q) {
                if (c0 + q * step < D) {
                    float gf[N], vf[N], o[N];
                    g[q].get(gf);
                    v[q].get(vf);
#pragma unroll
                    for (int s = 0; s < N; ++s) {
                        dot = fmaf(gf[s], vf[s], dot);
                        o[s] = w * gf[s];
                    }
                    store_row<N>(dy + p * lddy + c0 + q * step, o);
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
                dot += __shfl_xor_sync(0xffffffffu, dot, o);
            if (lane == 0)
                part[warp][j] += dot;
        }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < K; k += blockDim.x) {
        const int e = idx[t * K + k];
        float d = 0.f;
        for (int j = 0; j <= k; ++j) {
            if (idx[t * K + j] == e) { // the id's first slot
                if (spos[j] >= 0)
                    for (int w = 0; w < warps; ++w)
                        d += part[w][j];
                break;
            }
        }
        dwt[t * K + k] = d;
    }
}

} // namespace mvb

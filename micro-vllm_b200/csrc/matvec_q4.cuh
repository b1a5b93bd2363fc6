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
    int nb;                          // experts
};

// Matrix and row range of expert e; an expert without weights has w null.
__device__ __forceinline__ bool matvec_expert(const MatvecArgs &a, int e, const uint8_t *&w,
                                              const uint8_t *&s, int &r0, int &r1) {
    if (!a.wt) {
        w = static_cast<const uint8_t *>(a.w), s = static_cast<const uint8_t *>(a.s);
        r0 = 0, r1 = a.rows;
        return r1 > 0;
    }
    const int64_t off = a.xoff[e], n = a.nr[e];
    if (n <= 0 || off < 0)
        return false;
    r0 = static_cast<int>(min(off, int64_t(a.rows)));
    r1 = static_cast<int>(min(off + n, int64_t(a.rows)));
    w = static_cast<const uint8_t *>(a.wt[e]), s = static_cast<const uint8_t *>(a.st[e]);
    if (!s)
        w = nullptr;
    return r0 < r1;
}

constexpr int kMvWarps = 16, kMvThreads = 32 * kMvWarps;
constexpr int kMvRows = 32, kMvCols = 128; // weights of a warp's stage
constexpr int kMvMaxExperts = 1024;
constexpr int kMvSmem = 226 * 1024; // dynamic part of the 227 KB

// How a launch cuts its work, filled by the host (matvec_plan).
struct MatvecPlan {
    int N, K;      // outputs and reduction length: (O, I) forward, (I, O) gradient
    int range;     // outputs of a unit
    int nranges;   // units that cover N
    int wo, wk;    // warps along the outputs and along the reduction
    int slice;     // stages of the reduction per CTA of the cluster
    int chunk;     // stages whose rows are staged in shared memory at a time
    int x_vec;     // rows of x start on 16-byte boundaries
    int y_f32;
    int off_x, off_ex, off_red, off_list; // shared memory (ring at 0)
};

// Per-format geometry of a stage.
template <int FMT> struct MvFormat {
    static constexpr int G = FMT == MVLLM_FMT_INT4_G64 ? 64 : 32; // columns of a scale
    static constexpr int SB = FMT == MVLLM_FMT_INT4_G64 ? 8 : 4;  // scale bytes of a stage row
    static constexpr int STAGE = kMvRows * (kMvCols / 2 + SB);
};

// Parts an x element is split into, and rows that 8 * NT operand columns hold.
template <int FMT, typename TX, bool GRAD> struct MvTerms {
    static constexpr bool F32 = sizeof(TX) == 4;
    // forward: f16 parts, 11 bits each, scaled per group: bf16 fits one, f32
    // takes two (22 bits).  Gradient: bf16 parts, 8 bits each: bf16 rows of
    // an MXFP4 matrix fit one; times an int4 matrix's f32 scale two keep 16 to
    // 17 bits; f32 takes three (24 bits).
    static constexpr int T = GRAD ? (F32 ? 3 : FMT == MVLLM_FMT_INT4_G64 ? 2 : 1) : (F32 ? 2 : 1);
};

__device__ __forceinline__ void cp_async16_part(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void cp_async4_part(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void mv_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void mv_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t mv_prmt(uint32_t a, uint32_t b, uint32_t sel) {
    return __byte_perm(a, b, sel);
}
__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], uint32_t a0, uint32_t a1,
                                               uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ void mv_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\t"
                 "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t mv_cluster_addr(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// A stage in shared memory: 32 weight rows of 64 bytes, 16-byte chunk c of
// row r at chunk c ^ f(r), then the rows' scales.  f gives the 8 rows (4 rows
// by 32 bytes) that the forward (gradient) lanes read together 8 different
// bank groups.
__device__ __forceinline__ uint32_t mv_chunk(int row, int c) {
    const int f = (row & 2) | ((row >> 2) & 1);
    return row * 64 + ((c ^ f) << 4);
}

// Fills a stage with rows row0.. of a matrix [rows, I] and columns
// 128 * cs...  Bytes past the matrix's rows or columns become 0, their scales
// too.  Aligned matrices are copied asynchronously, others through registers
// byte by byte where their addresses ask for it.
template <int FMT>
__device__ __forceinline__ void mv_fill(uint32_t st, const uint8_t *w, const uint8_t *s, int rows,
                                        int I, int row0, int cs, bool w_al, bool s_al) {
    using F = MvFormat<FMT>;
    const int lane = threadIdx.x & 31;
    const int rb = (I + 1) >> 1;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int id = lane + 32 * q, r = id >> 2, c = id & 3;
        const int at = cs * 64 + c * 16;
        const uint8_t *src = w + int64_t(row0 + r) * rb + at;
        const bool in = row0 + r < rows;
        const uint32_t dst = st + mv_chunk(r, c);
        if (w_al) {
            const bool ok = in && at < rb;
            cp_async16_part(dst, ok ? src : w, ok ? 16 : 0);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t v = 0;
                if (in) {
                    const uint8_t *p = src + 4 * k;
                    const int left = rb - at - 4 * k;
                    if (left >= 4 && (reinterpret_cast<uintptr_t>(p) & 3u) == 0)
                        v = *reinterpret_cast<const uint32_t *>(p);
                    else
                        for (int b = 0; b < 4 && b < left; ++b)
                            v |= uint32_t(p[b]) << (8 * b);
                }
                sts32(dst + 4 * k, v);
            }
        }
    }
    // Scales: lane = row.
    const uint32_t sd = st + kMvRows * 64 + lane * F::SB;
    const int ng = (I + F::G - 1) / F::G;
    const bool in = row0 + lane < rows;
    if constexpr (FMT == MVLLM_FMT_INT4_G64) {
        const int g0 = cs * 2;
        const uint8_t *src = s + (int64_t(row0 + lane) * ng + g0) * 4;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const bool ok = in && g0 + k < ng;
            if (s_al) {
                cp_async4_part(sd + 4 * k, ok ? src + 4 * k : s, ok ? 4 : 0);
            } else {
                uint32_t v = 0;
                if (ok)
                    for (int b = 0; b < 4; ++b)
                        v |= uint32_t(src[4 * k + b]) << (8 * b);
                sts32(sd + 4 * k, v);
            }
        }
    } else {
        const int g0 = cs * 4;
        const uint8_t *src = s + int64_t(row0 + lane) * ng + g0;
        if (s_al) {
            const bool ok = in && g0 < ng;
            cp_async4_part(sd, ok ? src : s, ok ? 4 : 0);
        } else {
            uint32_t v = 0;
            for (int b = 0; b < 4; ++b)
                if (in && g0 + b < ng)
                    v |= uint32_t(src[b]) << (8 * b);
            sts32(sd, v);
        }
    }
}

// 8 elements of a row from column c, 0 past K.
template <typename TX>
__device__ __forceinline__ void mv_load8(const TX *row, int c, int K, bool vec, float (&v)[8]) {
    if (vec && c + 8 <= K) {
        if constexpr (sizeof(TX) == 4) {
            load_row<8>(row + c, v);
        } else {
            load_row<8>(row + c, v);
        }
    } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            float e[1] = {0.f};
            if (c + q < K)
                load_row<1>(row + c + q, e);
            v[q] = e[0];
        }
    }
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// f32 with all but the upper 16 bits cleared: a bf16 value, never above v.
__device__ __forceinline__ float trunc_bf16(float v) {
    return __uint_as_float(__float_as_uint(v) & 0xffff0000u);
}
// Part `term` of T of v (rounded to bf16 by the caller): leading 8 bits, the
// next 8, the rest.  Infinities and NaN are all in the first.
template <int T> __device__ __forceinline__ float mv_term(float v, int term) {
    if (T == 1)
        return v;
    const bool fin = fabsf(v) <= 3.402823466e38f;
    const float h = fin ? trunc_bf16(v) : v;
    float r = fin ? v - h : 0.f;
    if (T == 2)
        return term == 0 ? h : r;
    const float m = trunc_bf16(r);
    return term == 0 ? h : term == 1 ? m : r - m;
}

// Stages rows [r0, r0 + n) of x, columns c0 .. c0 + cols, as the B operand.
// Forward: f16 parts of x * 2^e with e per row and scale group such that the
// group's largest finite value lies in [2^14, 2^15): parts [8 NT][cols]
// (8-column chunks; int4 in its nibble pair order) and 2^-e as ex[group][row].
// A value 2^-24 of its group's largest keeps all the bits that matter next to
// it.  Gradient: bf16 parts (MXFP4) or plain f32 (int4), 16 rows of the
// matrix in the order lane t's four rows t, t + 4, t + 8, t + 12.
template <int FMT, typename TX, int NT, bool GRAD>
__device__ __forceinline__ void mv_stage_x(uint8_t *xs, float *ex, int pitch, const TX *x,
                                           int64_t ldx, int r0, int n, int c0, int cols, int K,
                                           bool vec) {
    constexpr int T = MvTerms<FMT, TX, GRAD>::T, RP = 8 * NT / T;
    if constexpr (!GRAD) {
        constexpr int GL = MvFormat<FMT>::G / 8; // lanes of a group
        const int per = cols / 8, tasks = per * RP;
        for (int b = (threadIdx.x & ~31); b < tasks; b += kMvThreads) {
            const int id = b + (threadIdx.x & 31);
            const int r = id / per, q = id - r * per;
            float v[8] = {};
            if (id < tasks && r < n)
                mv_load8(x + int64_t(r0 + r) * ldx, c0 + q * 8, K, vec, v);
            float m = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float a = fabsf(v[k]);
                m = a <= 3.402823466e38f ? fmaxf(m, a) : m;
            }
#pragma unroll
            for (int o = 1; o < GL; o <<= 1)
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            // 2^(14 - floor(log2 m)) and its reciprocal, both normal f32.
            const int e = m > 0.f ? max(14 - (int(__float_as_uint(m) >> 23) - 127), -113) : 0;
            const int sh = min(e, 126);
            const float sc = __uint_as_float(uint32_t(127 + sh) << 23);
            if (id >= tasks)
                continue;
            float h[8], l[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float a = v[k] * sc;
                h[k] = a;
                l[k] = fabsf(a) <= 3.402823466e38f ? a - __half2float(__float2half_rn(a)) : 0.f;
            }
            const bool i4 = FMT == MVLLM_FMT_INT4_G64;
#pragma unroll
            for (int term = 0; term < T; ++term) {
                const float(&p)[8] = term ? l : h;
                const uint4 w = i4 ? make_uint4(pack_f16(p[0], p[4]), pack_f16(p[1], p[5]),
                                                pack_f16(p[2], p[6]), pack_f16(p[3], p[7]))
                                   : make_uint4(pack_f16(p[0], p[1]), pack_f16(p[2], p[3]),
                                                pack_f16(p[4], p[5]), pack_f16(p[6], p[7]));
                *reinterpret_cast<uint4 *>(xs + (r * T + term) * pitch + q * 16) = w;
            }
            if ((q & (GL - 1)) == 0)
                ex[(q / GL) * RP + r] = __uint_as_float(uint32_t(127 - sh) << 23);
        }
    } else {
        constexpr bool I4 = FMT == MVLLM_FMT_INT4_G64;
        constexpr int R = I4 ? RP : (8 * NT + T - 1) / T; // the last may be partial
        for (int id = threadIdx.x; id < cols * R; id += kMvThreads) {
            const int r = id / cols, o = id - r * cols;
            float v[1] = {0.f};
            if (r < n && c0 + o < K)
                load_row<1>(x + int64_t(r0 + r) * ldx + c0 + o, v);
            if (v[0] != v[0])
                v[0] = __uint_as_float(0x7fc00000u);
            const int at = (o & ~15) + (o & 3) * 4 + ((o >> 2) & 3);
            if constexpr (I4) {
                *reinterpret_cast<float *>(xs + r * pitch + at * 4) = v[0];
            } else {
#pragma unroll
                for (int term = 0; term < T; ++term)
                    if (r * T + term < 8 * NT)
                        *reinterpret_cast<__nv_bfloat16 *>(xs + (r * T + term) * pitch + at * 2) =
                            __float2bfloat16_rn(mv_term<T>(v[0], term));
            }
        }
    }
}

// Forward product of one stage: 32 weight rows x 128 columns on the staged
// columns from xc on.  A lane holds rows g and g + 8 of two 16-row tiles and,
// of every 32 columns, its own 8: their order along the MMA's K is the same
// for both operands, so no nibble moves between lanes.  Each scale group's
// sum starts from zero and is scaled into the f32 accumulator.
template <int FMT, typename TX, int NT>
__device__ __forceinline__ void mv_forward(uint32_t st, uint32_t xs, const float *ex, int pitch,
                                           float (&acc)[2][NT][4]) {
    using F = MvFormat<FMT>;
    constexpr int T = MvTerms<FMT, TX, false>::T, RP = 8 * NT / T;
    constexpr int BPG = F::G / 32; // 32-column blocks of a group
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float sc[2][2][kMvCols / F::G];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t at = st + kMvRows * 64 + (mt * 16 + h * 8 + g) * F::SB;
            if constexpr (FMT == MVLLM_FMT_INT4_G64) {
                const uint2 v = lds64(at);
                sc[mt][h][0] = __uint_as_float(v.x), sc[mt][h][1] = __uint_as_float(v.y);
            } else {
                const uint32_t v = lds32(at);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    sc[mt][h][k] = ue8m0_byte(v, k);
            }
        }
#pragma unroll
    for (int gr = 0; gr < kMvCols / F::G; ++gr) {
        float d[2][NT][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    d[mt][nt][q] = 0.f;
#pragma unroll
        for (int bb = 0; bb < BPG; ++bb) {
            const int b = gr * BPG + bb;
            uint32_t a[2][2][4];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t w = lds32(st + mv_chunk(mt * 16 + h * 8 + g, b) + t * 4);
                    if constexpr (FMT == MVLLM_FMT_INT4_G64)
                        int4x8_to_f16x8(w, a[mt][h][0], a[mt][h][1], a[mt][h][2], a[mt][h][3]);
                    else
                        e2m1x8_to_f16x8(w, a[mt][h][0], a[mt][h][1], a[mt][h][2], a[mt][h][3]);
                }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint4 v = lds128(xs + (nt * 8 + g) * pitch + b * 64 + t * 16);
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    mma_f16_16816(d[mt][nt], a[mt][0][0], a[mt][1][0], a[mt][0][1], a[mt][1][1],
                                  v.x, v.y, d[mt][nt]);
                    mma_f16_16816(d[mt][nt], a[mt][0][2], a[mt][1][2], a[mt][0][3], a[mt][1][3],
                                  v.z, v.w, d[mt][nt]);
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if constexpr (T == 1) {
                const float2 e = *reinterpret_cast<const float2 *>(ex + gr * RP + nt * 8 + 2 * t);
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    acc[mt][nt][0] = fmaf(d[mt][nt][0] * e.x, sc[mt][0][gr], acc[mt][nt][0]);
                    acc[mt][nt][1] = fmaf(d[mt][nt][1] * e.y, sc[mt][0][gr], acc[mt][nt][1]);
                    acc[mt][nt][2] = fmaf(d[mt][nt][2] * e.x, sc[mt][1][gr], acc[mt][nt][2]);
                    acc[mt][nt][3] = fmaf(d[mt][nt][3] * e.y, sc[mt][1][gr], acc[mt][nt][3]);
                }
            } else { // columns 2t, 2t + 1: the two parts of row 4 nt + t
                const float e = ex[gr * RP + nt * 4 + t];
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    acc[mt][nt][0] = fmaf((d[mt][nt][0] + d[mt][nt][1]) * e, sc[mt][0][gr],
                                          acc[mt][nt][0]);
                    acc[mt][nt][2] = fmaf((d[mt][nt][2] + d[mt][nt][3]) * e, sc[mt][1][gr],
                                          acc[mt][nt][2]);
                }
            }
        }
    }
}

// Gradient product of one stage: W^T, 128 columns x 32 rows.  A lane loads 8
// columns (4 bytes) of rows t, t + 4, t + 8, t + 12 of each 16 and pairs two
// rows' halfwords, after which the nibble extraction yields (row, row + 4)
// pairs of one column: the transposition costs 4 byte permutes per 32
// weights.  MXFP4's scale multiplies the bf16 weight, exact as a power of
// two; int4's f32 scale multiplies the row's value, before it is split.
template <int FMT, typename TX, int NT>
__device__ __forceinline__ void mv_gradient(uint32_t st, uint32_t xs, int pitch,
                                            float (&acc)[2][4][NT][4]) {
    using F = MvFormat<FMT>;
    constexpr bool I4 = FMT == MVLLM_FMT_INT4_G64;
    constexpr int T = MvTerms<FMT, TX, true>::T, RP = 8 * NT / T;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        uint32_t sw[4][I4 ? 2 : 1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t at = st + kMvRows * 64 + (kb * 16 + t + 4 * j) * F::SB;
            if constexpr (I4) {
                const uint2 v = lds64(at);
                sw[j][0] = v.x, sw[j][1] = v.y;
            } else {
                sw[j][0] = lds32(at);
            }
        }
        uint32_t bx[NT][2]; // MXFP4: the same for every column
        float4 bv[NT];      // int4: the rows' values
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if constexpr (I4) {
                const int r = (nt * 8 + g) / T;
                bv[nt] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r < RP) {
                    const uint4 v = lds128(xs + r * pitch + kb * 64 + t * 16);
                    bv[nt] = make_float4(__uint_as_float(v.x), __uint_as_float(v.y),
                                         __uint_as_float(v.z), __uint_as_float(v.w));
                }
            } else {
                const uint2 v = lds64(xs + (nt * 8 + g) * pitch + kb * 32 + t * 8);
                bx[nt][0] = v.x, bx[nt][1] = v.y;
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                r[j] = lds32(st + mv_chunk(kb * 16 + t + 4 * j, h * 2 + (g >> 2)) + (g & 3) * 4);
            // p[0]: columns 0..3 of rows (t, t + 4), p[1]: columns 4..7;
            // p[2], p[3] of rows (t + 8, t + 12).
            const uint32_t p[4] = {mv_prmt(r[0], r[1], 0x5410u), mv_prmt(r[0], r[1], 0x7632u),
                                   mv_prmt(r[2], r[3], 0x5410u), mv_prmt(r[2], r[3], 0x7632u)};
            uint32_t m[2] = {}, m2[2] = {};
            bool high = false;
            uint32_t b[NT][2];
            if constexpr (I4) {
                float s[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    s[j] = __uint_as_float(sw[j][h]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int term = (nt * 8 + g) % T;
                    b[nt][0] = pack_bf16(mv_term<T>(bv[nt].x * s[0], term),
                                         mv_term<T>(bv[nt].y * s[1], term));
                    b[nt][1] = pack_bf16(mv_term<T>(bv[nt].z * s[2], term),
                                         mv_term<T>(bv[nt].w * s[3], term));
                }
            } else {
                // 2^(code - 1) = 2^126 * scale as bf16 (code 0: 0), the
                // weight's bits being 2^-126 of its value; codes above 128
                // take 2^126 and then the scale.
                uint32_t c[4];
                const int k = h * 2 + (g >> 2);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    c[j] = (sw[j][0] >> (8 * k)) & 255u;
                    high |= c[j] > 128u;
                }
                high = __any_sync(0xffffffffu, high);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t lo = c[2 * j], hi = c[2 * j + 1];
                    const uint32_t a0 = high ? 253u : lo ? lo + 126u : 0u;
                    const uint32_t a1 = high ? 253u : hi ? hi + 126u : 0u;
                    m[j] = (a0 << 7) | (a1 << 23);
                    m2[j] = (lo << 7) | (hi << 23);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    b[nt][0] = bx[nt][0], b[nt][1] = bx[nt][1];
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t a[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (I4) {
                        const uint32_t v = ((p[j] >> (4 * q)) & 0x000f000fu) | 0x43004300u;
                        a[j] = sub_bf16x2(v, 0x43084308u); // (128 + code) - 136
                    } else {
                        const uint32_t mag = q == 0   ? p[j] << 6
                                             : q == 1 ? p[j] << 2
                                             : q == 2 ? p[j] >> 2
                                                      : p[j] >> 6;
                        const uint32_t v = (mag & 0x01c001c0u) |
                                           ((p[j] << (12 - 4 * q)) & 0x80008000u);
                        a[j] = mul_bf16x2(v, m[j >> 1]);
                    }
                }
                if (!I4 && high) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        a[j] = mul_bf16x2(a[j], m2[j >> 1]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_bf16_16816(acc[h][q][nt], a[0], a[1], a[2], a[3], b[nt][0], b[nt][1]);
            }
        }
    }
}

// Ring stages of a warp.
template <int NT> constexpr int mv_ring() { return NT == 4 ? 3 : 4; }
// The partial sums share the ring's memory (no copy of the next unit is in
// flight over the reduction) where both would not fit.
template <int NT, bool GRAD> constexpr bool mv_alias() { return GRAD || NT == 4; }
// f32 elements of one warp's partial sums.
template <int FMT, typename TX, int NT, bool GRAD> constexpr int mv_red_pitch() {
    return GRAD ? 129 : 36;
}
template <int FMT, typename TX, int NT, bool GRAD> constexpr int mv_red_size() {
    return (GRAD ? 8 * NT : 8 * NT / MvTerms<FMT, TX, GRAD>::T) *
           mv_red_pitch<FMT, TX, NT, GRAD>();
}
template <int FMT, typename TX, bool GRAD> __host__ __device__ constexpr int mv_x_pitch(int cols) {
    // Row pitch of the staged x: the lanes of one shared-memory phase fall
    // into different banks.
    if (!GRAD)
        return cols * 2 + 64;
    if (FMT == MVLLM_FMT_INT4_G64)
        return (cols * 4 + 127) / 128 * 128 + 64;
    return (cols * 2 + 127) / 128 * 128 + 32;
}

struct MvUnit {
    const uint8_t *w, *s;
    int item, r0, n, out0;
    bool w_al, s_al;
};

// One CTA of a cluster.  A unit is (rows of one matrix, at most RP of them) x
// (a range of outputs); the cluster's CTAs split the reduction, each CTA's
// warps split the range (wo) and the CTA's part of the reduction (wk).  Every
// warp streams its own tiles through its own ring, so the main loop has no
// barrier; the partial sums of a unit's wk x cluster parts meet in (distributed)
// shared memory and are added in a fixed order.
template <int FMT, typename TX, int NT, bool GRAD>
__global__ void __launch_bounds__(kMvThreads, 1)
    matvec_q4_kernel(const MatvecArgs a, const MatvecPlan pl, const TX *__restrict__ x,
                     int64_t ldx, void *__restrict__ y, int64_t ldy) {
    using F = MvFormat<FMT>;
    constexpr int T = MvTerms<FMT, TX, GRAD>::T, RP = 8 * NT / T, ST = mv_ring<NT>();
    constexpr int TILE = GRAD ? kMvCols : kMvRows, STEP = GRAD ? kMvRows : kMvCols;
    constexpr int RPITCH = mv_red_pitch<FMT, TX, NT, GRAD>();
    constexpr int RSIZE = mv_red_size<FMT, TX, NT, GRAD>();
    extern __shared__ __align__(128) uint8_t mv_smem[];
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int rank, ranks, cluster, clusters;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    asm("mov.u32 %0, %%clusterid.x;" : "=r"(cluster));
    asm("mov.u32 %0, %%nclusterid.x;" : "=r"(clusters));
    float *ex = reinterpret_cast<float *>(mv_smem + pl.off_ex);
    float *red = reinterpret_cast<float *>(mv_smem + pl.off_red);
    int *list = reinterpret_cast<int *>(mv_smem + pl.off_list); // passes before each expert
    int items;
    if (a.wt) {
        int n[2];
        __shared__ int wsum[kMvWarps];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int e = 2 * int(threadIdx.x) + k;
            const uint8_t *w, *s;
            int r0 = 0, r1 = 0;
            n[k] = e < a.nb && matvec_expert(a, e, w, s, r0, r1) ? (r1 - r0 + RP - 1) / RP : 0;
        }
        int v = n[0] + n[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            v += lane >= o ? u : 0;
        }
        if (lane == 31)
            wsum[warp] = v;
        __syncthreads();
        int before = 0;
        for (int k = 0; k < kMvWarps; ++k)
            before += k < warp ? wsum[k] : 0;
        const int first = before + v - n[0] - n[1];
        if (2 * int(threadIdx.x) <= a.nb)
            list[2 * threadIdx.x] = first;
        if (2 * int(threadIdx.x) + 1 <= a.nb)
            list[2 * threadIdx.x + 1] = first + n[0];
        if (threadIdx.x == kMvThreads - 1 && a.nb == kMvMaxExperts)
            list[kMvMaxExperts] = first + n[0] + n[1];
        __syncthreads();
        items = list[a.nb];
    } else {
        items = (a.rows + RP - 1) / RP;
    }
    const int64_t total = int64_t(items) * pl.nranges;
    const int rows_w = GRAD ? pl.K : pl.N; // rows of the matrices (O)

    auto decode = [&](int64_t u) {
        MvUnit q;
        q.item = int(u / pl.nranges);
        q.out0 = int(u - int64_t(q.item) * pl.nranges) * pl.range;
        int r0 = 0, r1 = 0, pass = q.item;
        if (a.wt) {
            int lo = 0, hi = a.nb; // the last expert with list[e] <= item has it
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (list[mid] <= q.item)
                    lo = mid;
                else
                    hi = mid;
            }
            pass -= list[lo];
            matvec_expert(a, lo, q.w, q.s, r0, r1);
        } else {
            matvec_expert(a, 0, q.w, q.s, r0, r1);
        }
        q.r0 = r0 + pass * RP;
        q.n = min(RP, r1 - q.r0);
        q.w_al = (reinterpret_cast<uintptr_t>(q.w) & 15u) == 0 && (a.I & 31) == 0;
        q.s_al = (reinterpret_cast<uintptr_t>(q.s) & 3u) == 0 &&
                 (FMT == MVLLM_FMT_INT4_G64 || (a.I & 127) == 0);
        return q;
    };
    // This warp's part of a unit: a tile of outputs and every wk-th stage of
    // the CTA's slice.
    const int wo = warp / pl.wk, wk = warp - wo * pl.wk;
    const int steps = (pl.K + STEP - 1) / STEP;
    const int k0 = min(rank * pl.slice, steps), nk = min(pl.slice, steps - k0);
    auto mine = [&](const MvUnit &q) {
        const int out = q.out0 + wo * TILE;
        const int end = min(pl.N, q.out0 + pl.range);
        return wo < pl.wo && out < end && q.w && nk > wk ? (nk - wk + pl.wk - 1) / pl.wk : 0;
    };
    const uint32_t ring = smem_u32(mv_smem) + warp * ST * F::STAGE;
    int head = 0; // ring slot of this warp's next stage to compute
    auto issue = [&](const MvUnit &q, int i, int n) {
        if (i < n) {
            const int step = k0 + wk + i * pl.wk, out = q.out0 + wo * TILE;
            int slot = head + i;
            slot %= ST;
            mv_fill<FMT>(ring + slot * F::STAGE, q.w, q.s, rows_w, a.I,
                         GRAD ? step * STEP : out, GRAD ? out / kMvCols : step, q.w_al, q.s_al);
        }
        mv_commit();
    };
    auto prologue = [&](const MvUnit &q) {
        const int n = mine(q);
        for (int i = 0; i < ST - 1; ++i)
            issue(q, i, n);
    };

    const int cols = pl.chunk * STEP, pitch = mv_x_pitch<FMT, TX, GRAD>(cols);
    const uint32_t xs = smem_u32(mv_smem + pl.off_x);
    int staged = -1; // the item whose only chunk is staged
    MvUnit cur{};
    if (cluster < total) {
        cur = decode(cluster);
        prologue(cur);
    }
    for (int64_t u = cluster; u < total; u += clusters) {
        const int n = mine(cur);
        float accf[GRAD ? 1 : 2][NT][4];
        float accg[GRAD ? 2 : 1][GRAD ? 4 : 1][NT][4];
        if constexpr (GRAD) {
#pragma unroll
            for (int i = 0; i < 8 * NT * 4; ++i)
                (&accg[0][0][0][0])[i] = 0.f;
        } else {
#pragma unroll
            for (int i = 0; i < 2 * NT * 4; ++i)
                (&accf[0][0][0])[i] = 0.f;
        }
        int i = 0;
        for (int c0 = 0; c0 < nk; c0 += pl.chunk) {
            if (cur.w && staged != cur.item) { // uniform over the CTA
                __syncthreads(); // the last readers of x are done
                mv_stage_x<FMT, TX, NT, GRAD>(mv_smem + pl.off_x, ex, pitch, x, ldx, cur.r0,
                                              cur.n, (k0 + c0) * STEP, cols, pl.K, pl.x_vec);
                __syncthreads();
                if (nk <= pl.chunk)
                    staged = cur.item;
            }
            for (; i < n; ++i) {
                const int step = wk + i * pl.wk - c0; // within the chunk
                if (step >= pl.chunk)
                    break;
                mv_wait<ST - 2>();
                __syncwarp();
                issue(cur, i + ST - 1, n); // into the slot computed last
                const uint32_t st = ring + ((head + i) % ST) * F::STAGE;
                if constexpr (GRAD)
                    mv_gradient<FMT, TX, NT>(
                        st, xs + step * STEP * (FMT == MVLLM_FMT_INT4_G64 ? 4 : 2), pitch, accg);
                else
                    mv_forward<FMT, TX, NT>(st, xs + step * STEP * 2,
                                            ex + step * (STEP / F::G) * RP, pitch, accf);
            }
        }
        head = (head + n) % ST;
        __syncwarp();
        MvUnit next{};
        if (u + clusters < total)
            next = decode(u + clusters);
        if constexpr (!mv_alias<NT, GRAD>()) {
            if (u + clusters < total)
                prologue(next);
        } else {
            mv_wait<0>();
            __syncthreads(); // the ring is done with before the sums overlay it
        }
        // Partial sums [column][output] of this warp.
        float *mr = red + warp * RSIZE;
        const int g = lane >> 2, t = lane & 3;
        if constexpr (GRAD) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float(&d)[4] = accg[h][q][nt];
                        float *at = mr + (nt * 8 + 2 * t) * RPITCH + h * 64 + 8 * g + q;
                        at[0] = d[0], at[RPITCH] = d[1];
                        at[4] = d[2], at[RPITCH + 4] = d[3];
                    }
        } else {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float(&d)[4] = accf[mt][nt];
                    float *at = mr + (T == 1 ? nt * 8 + 2 * t : nt * 4 + t) * RPITCH + mt * 16 + g;
                    at[0] = d[0], at[8] = d[2];
                    if (T == 1)
                        at[RPITCH] = d[1], at[RPITCH + 8] = d[3];
                }
        }
        mv_cluster_sync();
        // Each CTA adds up and writes its share of the unit's outputs.
        const int outs = min(pl.range, pl.N - cur.out0);
        for (int id = rank * kMvThreads + threadIdx.x; id < outs * cur.n;
             id += ranks * kMvThreads) {
            const int r = id / outs, o = id - r * outs;
            const int w0 = (o / TILE) * pl.wk;
            const uint32_t at = smem_u32(red + w0 * RSIZE + (GRAD ? r * T : r) * RPITCH + o % TILE);
            float v = 0.f;
            for (int c = 0; c < ranks; ++c) {
                const uint32_t ra = mv_cluster_addr(at, c);
                for (int k = 0; k < pl.wk; ++k)
#pragma unroll
                    for (int q = 0; q < (GRAD ? T : 1); ++q)
                        v += ld_cluster_f32(ra + 4 * (k * RSIZE + q * RPITCH));
            }
            const int64_t to = int64_t(cur.r0 + r) * ldy + cur.out0 + o;
            if (pl.y_f32)
                static_cast<float *>(y)[to] = v;
            else
                static_cast<__nv_bfloat16 *>(y)[to] = __float2bfloat16_rn(v);
        }
        mv_cluster_sync(); // the sums are read before they are overwritten
        cur = next;
        if constexpr (mv_alias<NT, GRAD>()) {
            if (u + clusters < total)
                prologue(cur);
        }
    }
}

} // namespace mvb

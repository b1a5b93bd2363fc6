// matvec_q4.cuh -- products of few rows with 4-bit weights and their
// gradient, for one matrix or for the expert-sorted rows of many.
//
//   forward   y[r, o]  = sum_i W[o, i] x[r, i]
//   gradient  dx[r, i] = sum_o W[o, i] dy[r, o]
// with W[o, i] = q[o, i] s[o, i / G] decoded from the packed formats (int4
// with a f32 scale per G = 64 columns, MXFP4 with a ue8m0 scale per G = 32).
// Sums are f32.
//
// The weights are read once per pass of up to 32 rows, 4.5 bits each, so the
// floor is their bytes; each decodes to an operand of m16n8k16 matrix
// instructions, which take the rows as the narrow side.  One row of 7168 ->
// 65536 streams at 4.8 TB/s, 73% of a copy; 7168 -> 16384 (60 MB) takes 17 to
// 18 us for 1 row, 20 for 8, 32 for 16 and 64 for 32.  Beyond the memory it is
// the decoding that bounds: 490 to 550 instructions per stage of a warp for 8
// rows, 1260 for 32 (1100 in the gradient, 8 rows), issued on 54 to 57% and 38%
// (43 to 52%) of the cycles; the matrix pipe is busy for 26 to 31%.  Short
// products are bound by their start: 6.9 us for 8 MB, of which the rows' way to
// the operands is about half.
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

// Warps of a CTA (one CTA per SM) and stages of a warp's ring.  The forward
// product is bound by the instructions of the dequantisation and wants as many
// warps to interleave as registers and the staged rows leave room for: with 16
// warps 16 rows take 7168 -> 16384 in 38 us in place of 32 (registers spill),
// with 12 warps 32 rows in 84 in place of 64 (the staged rows come in more
// chunks).  The gradient holds 64 or 128 sums per lane; 12 warps with rings of
// three stages spill, 513 us in place of 397 on 160 experts of 1536 x 6144 (int4;
// MXFP4 342 in place of 326).
template <int NT, bool GRAD> constexpr int mv_warps() {
    return GRAD || NT == 4 ? 8 : NT == 2 ? 12 : 16;
}
template <int NT, bool GRAD> constexpr int mv_ring() { return GRAD ? 4 : 2; }
constexpr int kMvSmem = 226 * 1024; // dynamic part of the 227 KB
constexpr int kMvRows = 32, kMvCols = 256; // weights of a warp's stage
constexpr int kMvMaxExperts = 1024;
constexpr int kMvMaxSide = 1 << 30; // rows and columns: steps past them stay in 32 bits

// How a launch cuts its work, filled by the host (MvHost::plan).
struct MatvecPlan {
    int N, K;      // outputs and reduction length: (O, I) forward, (I, O) gradient
    int range;     // outputs of a unit
    int nranges;   // units that cover N
    int wo, wk;    // tiles of a range, parts of each along the reduction
    int slice;     // stages of the reduction per CTA of the cluster
    int chunk;     // stages whose rows are staged in shared memory at a time
    int x_vec;     // rows of x start on 16-byte boundaries
    int y_vec;     // rows of y on boundaries of four elements
    int rows_most; // rows that one matrix can have
    int y_f32;
    int try_common; // a main loop long enough to pay for the survey of the rows
    int off_x, off_ex, off_red, off_mail, off_list; // shared memory (ring at 0)
};

// Per-format geometry of a stage.
template <int FMT> struct MvFormat {
    static constexpr int G = FMT == MVLLM_FMT_INT4_G64 ? 64 : 32; // columns of a scale
    static constexpr int SB = FMT == MVLLM_FMT_INT4_G64 ? 16 : 8; // scale bytes of a stage row
    // A row's scales take 16 bytes of a stage: MXFP4's 8 come as the aligned 16
    // that hold them, at (column-step & 1) * 8.  (Copied by 8 bytes they go
    // through L1, which had no room for the lines of 512 rows: 3.3 against
    // 5.5 TB/s on 48 experts of 7168 x 2048.)
    static constexpr int STAGE = kMvRows * (kMvCols / 2 + 16);
};

// Operand columns that an x element is split over; 8 * NT of them hold
// 8 * NT / T rows.
template <int FMT, typename TX, bool GRAD> struct MvTerms {
    static constexpr bool F32 = sizeof(TX) == 4;
    // forward: f16 parts, 11 bits each, scaled per group: bf16 fits one, f32
    // takes two (22 bits).  Gradient: bf16 parts, 8 bits each: bf16 rows of
    // an MXFP4 matrix fit one, f32 takes three (24 bits).  int4's f32 scales
    // multiply the rows first; a product's three parts (24 bits) go through one
    // column, one after another.
    static constexpr int T =
        !GRAD ? (F32 ? 2 : 1) : F32 && FMT != MVLLM_FMT_INT4_G64 ? 3 : 1;
};

__device__ __forceinline__ void cp_async16_at(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4_at(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
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
// The aligned forms want a warp's lanes together, which a loop whose trip count
// differs between them does not leave.
__device__ __forceinline__ void mv_cluster_wait() {
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mv_cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    mv_cluster_wait();
}
__device__ __forceinline__ uint32_t mv_cluster_addr(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void st_cluster_f32x4(uint32_t addr, const float (&v)[4]) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(v[0]),
                 "f"(v[1]), "f"(v[2]), "f"(v[3])
                 : "memory");
}

// A stage in shared memory: 32 weight rows of 128 bytes, 16-byte chunk c of
// row r at chunk c ^ f(r), then the rows' scales.  f gives the 8 rows x 16
// bytes (4 rows x 32 bytes) that the forward (gradient) lanes read together 8
// different bank groups.
__device__ __forceinline__ uint32_t mv_chunk(int row, int c) {
    const int f = ((row & 3) << 1) | ((row >> 2) & 1);
    return row * 128 + ((c ^ f) << 4);
}

__device__ __forceinline__ void cp_async8_at(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

// A warp's walk over a matrix [rows, I] in stages of 32 rows x 256 columns,
// along the columns (forward) or down the rows (gradient): 128 contiguous
// bytes of a row at a time.  (With 64, at the same bytes in flight, the
// stream ran at 3 TB/s.)  A lane copies 16 bytes of rows lane / 8 + 0, 4, ..
// 28 and the scales of row `lane`.  Bytes past the matrix's rows or columns
// become 0, their scales too.  Aligned matrices are copied asynchronously,
// others through registers, byte by byte where their addresses ask for it.
template <int FMT, bool GRAD> struct MvWalk {
    using F = MvFormat<FMT>;
    static constexpr int SW = FMT == MVLLM_FMT_INT4_G64 ? 4 : 1; // bytes of a scale
    const uint8_t *w, *s; // this lane's weight chunk and scale of the next stage
    int64_t dw;           // bytes from one stage's weights to the next one's
    int ds;               // and scales (times 32 rows: below 2^31)
    int rb, ng;           // bytes and scale groups of a row
    int row, col;         // first row and column-step of the next stage
    int rows, every;      // rows of the matrix; steps from a stage to the next
    int inside;           // stages ahead that lie in the matrix as a whole
    int s_al;             // 16, 8 or 4: scales can be copied by so many bytes; 0: one by one

    // From row `row_` and column-step `col_` on, every `every_`-th step.
    __device__ __forceinline__ void start(const uint8_t *w0, const uint8_t *s0, int rows_, int I,
                                          int row_, int col_, int every_) {
        const int lane = threadIdx.x & 31;
        rb = (I + 1) >> 1, ng = (I + F::G - 1) / F::G;
        row = row_, col = col_, rows = rows_, every = every_;
        const bool w_al = ((reinterpret_cast<uintptr_t>(w0) | unsigned(rb)) & 15u) == 0;
        const unsigned sa = unsigned(reinterpret_cast<uintptr_t>(s0)) | unsigned(ng * SW);
        s_al = (sa & 15) == 0 ? 16 : (sa & 7) == 0 ? 8 : (sa & 3) == 0 ? 4 : 0;
        w = w0 + int64_t(row + (lane >> 3)) * rb + int64_t(col) * (kMvCols / 2) + (lane & 7) * 16;
        s = s0 + (int64_t(row + lane) * ng + int64_t(col) * (kMvCols / F::G)) * SW;
        dw = GRAD ? int64_t(every) * kMvRows * rb : int64_t(every) * (kMvCols / 2);
        ds = GRAD ? every * kMvRows : every; // row or group steps
        const int full_rows = rows - row, full_cols = rb / (kMvCols / 2) - col;
        if (GRAD)
            inside = full_cols >= 1 ? (full_rows / kMvRows + every - 1) / every : 0;
        else
            inside = full_rows >= kMvRows ? (full_cols + every - 1) / every : 0;
        inside = !w_al ? -1 : max(inside, 0); // -1: not asynchronously either
    }
    // Copies the next stage.
    __device__ __forceinline__ void fill(uint32_t st) {
        const int lane = threadIdx.x & 31;
        const int half = F::SB == 8 ? (col & 1) * 8 : 0;
        const uint32_t sd = st + kMvRows * 128 + lane * 16;
        if (inside > 0) { // uniform over the warp
            const uint32_t d0 = st + mv_chunk(lane >> 3, lane & 7);
            const uint32_t d1 = st + mv_chunk((lane >> 3) + 4, lane & 7) - 512;
#pragma unroll
            for (int q = 0; q < 8; ++q)
                cp_async16_at((q & 1 ? d1 : d0) + 512 * q, w + uint64_t(uint32_t(4 * rb)) * q);
            if (s_al == 16)
                cp_async16_at(sd, s - half);
            else if (F::SB == 8 && s_al == 8)
                cp_async8_at(sd + half, s);
            else
                edge_scales(sd + half, s, ng, row, col, rows, s_al != 0);
            --inside;
        } else {
            edge_weights(st, w, rb, row, col, rows, inside == 0);
            edge_scales(sd + half, s, ng, row, col, rows, s_al != 0);
        }
        w += dw;
        s += int64_t(ds) * (GRAD ? ng * SW : F::SB);
        if (GRAD)
            row += every * kMvRows;
        else
            col += every;
    }
    // A stage at the matrix's edges, or of a matrix that cannot be copied by 16
    // bytes (`async` false).
    static __device__ __noinline__ void edge_weights(uint32_t st, const uint8_t *w, int rb,
                                                     int row, int col, int rows, bool async) {
        const int lane = threadIdx.x & 31;
        const int at = col * (kMvCols / 2) + (lane & 7) * 16;
        const int left_rows = rows - row - (lane >> 3);
        if (async) {
            for (int q = 0; q < 8; ++q) {
                const uint32_t to = st + mv_chunk((lane >> 3) + 4 * q, lane & 7);
                if (at < rb && 4 * q < left_rows)
                    cp_async16_at(to, w + int64_t(4 * q) * rb);
                else
                    asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(to), "r"(0)
                                 : "memory");
            }
        } else {
            for (int q = 0; q < 8; ++q)
                for (int k = 0; k < 4; ++k) {
                    uint32_t v = 0;
                    if (4 * q < left_rows) {
                        const uint8_t *p = w + int64_t(4 * q) * rb + 4 * k;
                        const int left = rb - at - 4 * k;
                        if (left >= 4 && (reinterpret_cast<uintptr_t>(p) & 3u) == 0)
                            v = *reinterpret_cast<const uint32_t *>(p);
                        else
                            for (int b = 0; b < 4 && b < left; ++b)
                                v |= uint32_t(p[b]) << (8 * b);
                    }
                    sts32(st + mv_chunk((lane >> 3) + 4 * q, lane & 7) + 4 * k, v);
                }
        }
    }
    static __device__ __noinline__ void edge_scales(uint32_t sd, const uint8_t *s, int ng, int row,
                                                    int col, int rows, bool async) {
        const int lane = threadIdx.x & 31;
        const int g0 = col * (kMvCols / F::G);
        const int left = row + lane < rows ? min(ng - g0, kMvCols / F::G) * SW : 0; // bytes
        for (int k = 0; k < F::SB / 4; ++k) {
            if (async && left >= 4 * k + 4) { // whole words
                cp_async4_at(sd + 4 * k, s + 4 * k);
            } else {
                uint32_t v = 0;
                for (int b = 0; b < 4; ++b)
                    if (4 * k + b < left)
                        v |= uint32_t(s[4 * k + b]) << (8 * b);
                sts32(sd + 4 * k, v);
            }
        }
    }
};

// Walks the groups of 8 elements of the rows to stage: group `tid` first, then
// every THREADS-th, as (row, group of the row).
template <int THREADS> struct MvGroups {
    int r, q, per;
    __device__ __forceinline__ explicit MvGroups(int per_) : r(0), q(threadIdx.x), per(per_) {
        settle();
    }
    __device__ __forceinline__ void settle() {
        while (q >= per)
            q -= per, ++r;
    }
    __device__ __forceinline__ void next() {
        q += THREADS;
        settle();
    }
};

// The gradient's rows: a thread's first HOLD groups, loaded before the weights'
// copies are issued; behind them in the memory system the rows would arrive
// some microseconds later, and the main loop waits for them.
template <typename TX, int NT> struct MvHeld {
    static constexpr int THREADS = 32 * mv_warps<NT, true>();
    static constexpr int HOLD = sizeof(TX) == 4 ? 4 : 8;
    Raw8<TX> raw[HOLD];
    __device__ __forceinline__ void load(const TX *x, int64_t ldx, int r0, int n, int c0, int cols,
                                         int K, bool vec) {
        MvGroups<THREADS> at(cols / 8);
#pragma unroll
        for (int h = 0; h < HOLD; ++h, at.next())
            if (at.r < n)
                raw[h].load(x + int64_t(r0 + at.r) * ldx, c0 + at.q * 8, K, vec);
    }
    // f(raw, r, q) for every group of the n rows, the held ones from registers.
    template <typename F>
    __device__ __forceinline__ void each(const TX *x, int64_t ldx, int r0, int n, int c0, int cols,
                                         int K, bool vec, bool have, F f) const {
        MvGroups<THREADS> at(cols / 8);
#pragma unroll
        for (int h = 0; h < HOLD; ++h, at.next()) {
            if (at.r < n) {
                Raw8<TX> now = raw[h];
                if (!have)
                    now.load(x + int64_t(r0 + at.r) * ldx, c0 + at.q * 8, K, vec);
                f(now, at.r, at.q);
            }
        }
        for (; at.r < n; at.next()) {
            Raw8<TX> now;
            now.load(x + int64_t(r0 + at.r) * ldx, c0 + at.q * 8, K, vec);
            f(now, at.r, at.q);
        }
    }
};

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
    static_assert(T == 1 || T == 3, "parts");
    if (T == 1)
        return v;
    const bool fin = fabsf(v) <= 3.402823466e38f;
    const float h = fin ? trunc_bf16(v) : v;
    const float r = fin ? v - h : 0.f;
    const float m = trunc_bf16(r);
    return term == 0 ? h : term == 1 ? m : r - m;
}

__device__ __forceinline__ float finite_max(const float (&v)[8]) {
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k)
        m = fmaxf(m, fabsf(v[k])); // passes NaN over
    if (m > 3.402823466e38f) {
        m = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float a = fabsf(v[k]);
            m = a <= 3.402823466e38f ? fmaxf(m, a) : m;
        }
    }
    return m;
}
// The power of two that brings m into [2^14, 2^15) (m = 0: 1), clamped so
// that it and its reciprocal are normal f32: its exponent.
__device__ __forceinline__ int mv_shift(float m) {
    const int e = int(__float_as_uint(m) >> 23) - 127;
    return m > 0.f ? min(14 - e, 126) : 0;
}
__device__ __forceinline__ float exp2_int(int e) {
    return __uint_as_float(uint32_t(127 + e) << 23);
}

// Stages rows [r0, r0 + n) of x, columns c0 .. c0 + cols, as the forward
// product's B operand: f16 parts of x * 2^e, [n T][cols] in 8-column chunks
// (int4: in its nibble pair order), and 2^-e in ex.  f16's 30 binades hold a
// row of activations with one e for all its columns; that is checked: where
// every scale group's largest finite value (or zero) lies within 2^-12 of its
// row's, and that is below 2^31, `common` is returned and ex[row] = 2^-e, else
// e goes by group, ex[group][row].  Either way the largest scaled value of a
// group whose largest is at least 2^-112 is at least 4 (below, e stops at
// 126), and what the parts leave of an element is at most 2^-22 of it (nothing,
// for bf16) or half of f16's last step.  That is 2^-25 for bf16, 2^-27 of the
// group's largest; f32's second part is held times 2^11, so 2^-36 there, 2^-38
// of the group's largest.
//
// The factors come in where no sum leaves f32's range before its result does:
// by group, d 2^-e first and then the weights' scale; where a group's largest
// is 2^112 or more (`wide`) 2^-e in two steps, before and after the scale.  A
// common 2^-e follows after all columns, which is checked at the end: sums that
// are not finite are taken again by group.  (Up to 2^31, what a scale below
// 2^-126 loses before the factor stays below f32's smallest normal value.)
//
// The elements come first, as they are, to the places of their parts, which
// take as many bytes (mv_fetch_rows, asynchronous where rows are aligned);
// mv_stage_forward then replaces them.
template <int FMT, typename TX, int NT>
__device__ __forceinline__ void mv_fetch_rows(uint8_t *xs, int pitch, const TX *x, int64_t ldx,
                                              int r0, int n, int c0, int cols, int K, bool vec) {
    constexpr int T = MvTerms<FMT, TX, false>::T;
    static_assert(sizeof(TX) == 2 * T, "raw elements fit their parts' places");
    for (MvGroups<32 * mv_warps<NT, false>()> at(cols / 8); at.r < n; at.next()) {
        const TX *row = x + int64_t(r0 + at.r) * ldx;
        const int c = c0 + at.q * 8;
        uint8_t *to = xs + at.r * T * pitch + at.q * 16;
        if (vec && c + 8 <= K) {
#pragma unroll
            for (int term = 0; term < T; ++term)
                cp_async16_at(smem_u32(to + term * pitch),
                              reinterpret_cast<const uint4 *>(row + c) + term);
        } else {
            Raw8<TX> raw;
            raw.load(row, c, K, vec);
#pragma unroll
            for (int term = 0; term < T; ++term)
                *reinterpret_cast<uint4 *>(to + term * pitch) = raw.u[term];
        }
    }
}
template <int FMT, typename TX, int NT>
__device__ __forceinline__ bool mv_stage_forward(uint8_t *xs, float *ex, int pitch, int n, int cols,
                                                 bool try_common, uint32_t *row_max, bool &wide) {
    constexpr int T = MvTerms<FMT, TX, false>::T, RP = 8 * NT / T;
    constexpr int GL = MvFormat<FMT>::G / 8; // lanes of a group
    using Groups = MvGroups<32 * mv_warps<NT, false>()>;
    const int lane = threadIdx.x & 31;
    auto read = [&](const Groups &at, float(&v)[8]) {
        Raw8<TX> raw;
#pragma unroll
        for (int term = 0; term < T; ++term)
            raw.u[term] =
                *reinterpret_cast<const uint4 *>(xs + (at.r * T + term) * pitch + at.q * 16);
        raw.get(v);
    };
    // row_max[r]: bits of the row's largest finite value; [RP + r]: of its
    // smallest nonzero group maximum.
    bool common = false;
    wide = false;
    if (try_common) {
        for (Groups at(cols / 8); at.r < n; at.next()) {
            float v[8];
            read(at, v);
            float m = finite_max(v);
#pragma unroll
            for (int o = 1; o < GL; o <<= 1)
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            // cols / 8 is a multiple of 32: a warp has one row; positive f32
            // order as their bits
            const uint32_t hi = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
            const uint32_t lo =
                __reduce_min_sync(0xffffffffu, m > 0.f ? __float_as_uint(m) : 0x7f800000u);
            if (lane == 0) {
                atomicMax(&row_max[at.r], hi);
                atomicMin(&row_max[RP + at.r], lo);
            }
        }
        __syncthreads();
        bool fits = true;
        if (int(threadIdx.x) < n) {
            const float m = __uint_as_float(row_max[threadIdx.x]);
            fits = __uint_as_float(row_max[RP + threadIdx.x]) >= m * 0x1p-12f && m < 0x1p31f;
            ex[threadIdx.x] = exp2_int(-mv_shift(m));
        }
        common = __syncthreads_and(fits);
    }
    for (Groups at(cols / 8); at.r < n; at.next()) {
        float v[8];
        read(at, v);
        int sh;
        if (common) {
            sh = mv_shift(__uint_as_float(row_max[at.r]));
        } else {
            float m = finite_max(v);
#pragma unroll
            for (int o = 1; o < GL; o <<= 1)
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            sh = mv_shift(m);
            wide |= m >= 0x1p112f;
            if ((at.q & (GL - 1)) == 0)
                ex[(at.q / GL) * RP + at.r] = exp2_int(-sh);
        }
        const float sc = exp2_int(sh);
        float l[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            v[k] *= sc;
            l[k] = fabsf(v[k]) <= 3.402823466e38f
                       ? (v[k] - __half2float(__float2half_rn(v[k]))) * 0x1p11f
                       : 0.f;
        }
#pragma unroll
        for (int term = 0; term < T; ++term) {
            const float(&p)[8] = term ? l : v;
            const uint4 w = FMT == MVLLM_FMT_INT4_G64
                                ? make_uint4(pack_f16(p[0], p[4]), pack_f16(p[1], p[5]),
                                             pack_f16(p[2], p[6]), pack_f16(p[3], p[7]))
                                : make_uint4(pack_f16(p[0], p[1]), pack_f16(p[2], p[3]),
                                             pack_f16(p[4], p[5]), pack_f16(p[6], p[7]));
            *reinterpret_cast<uint4 *>(xs + (at.r * T + term) * pitch + at.q * 16) = w;
        }
    }
    return common;
}

// The gradient's B operand: rows of dy as bf16 parts (MXFP4) or as they are
// (int4, whose scales multiply them first), the 16 rows of a matrix block in
// the order of lane t's four rows t, t + 4, t + 8, t + 12.
template <int FMT, typename TX, int NT>
__device__ __forceinline__ void mv_stage_gradient(uint8_t *xs, int pitch, const TX *x, int64_t ldx,
                                                  int r0, int n, int c0, int cols, int K, bool vec,
                                                  bool have, const MvHeld<TX, NT> &held) {
    constexpr bool I4 = FMT == MVLLM_FMT_INT4_G64; // split later
    constexpr int T = MvTerms<FMT, TX, true>::T;
    held.each(x, ldx, r0, n, c0, cols, K, vec, have, [&](const Raw8<TX> &raw, int r, int q) {
        float v[8];
        raw.get(v);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (v[k] != v[k])
                v[k] = __uint_as_float(0x7fc00000u);
        // elements k and k + 4 lie side by side at place 4 k (+ 2 in the
        // block's upper half)
        const int at = (q >> 1) * 16 + (q & 1) * 2;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (I4) {
                *reinterpret_cast<float2 *>(xs + r * pitch + (at + 4 * k) * 4) =
                    make_float2(v[k], v[k + 4]);
            } else {
#pragma unroll
                for (int term = 0; term < T; ++term)
                    *reinterpret_cast<uint32_t *>(xs + (r * T + term) * pitch + (at + 4 * k) * 2) =
                        pack_bf16(mv_term<T>(v[k], term), mv_term<T>(v[k + 4], term));
            }
        }
    });
}

// int4x8_to_f16x8 with one shift for eight codes, by the published reading of a
// nibble through f16's exponent (1024 + n in its low mantissa bits): a nibble in bits 4..7 of a
// halfword reads as 1024 + 16 n, which one multiply-add turns into n - 8.
__device__ __forceinline__ void mv_int4x8(uint32_t w, uint32_t (&h)[4]) {
    const uint32_t u = w >> 8, m0 = 0x000f000fu, m1 = 0x00f000f0u, one = 0x64006400u;
    uint32_t a, b, c, d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(a) : "r"(w), "r"(m0), "r"(one));
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(b) : "r"(w), "r"(m1), "r"(one));
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(c) : "r"(u), "r"(m0), "r"(one));
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(u), "r"(m1), "r"(one));
    // 1032, 1/16, -72
    const uint32_t bias = 0x64086408u, sixteenth = 0x2c002c00u, off = 0xd480d480u;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(h[0]) : "r"(a), "r"(bias));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(h[1]) : "r"(b), "r"(sixteenth), "r"(off));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(h[2]) : "r"(c), "r"(bias));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(h[3]) : "r"(d), "r"(sixteenth), "r"(off));
}

// Forward product of one stage: 32 weight rows x 256 columns on the staged
// columns from xc on.  A lane holds rows g and g + 8 of two 16-row tiles and,
// of every 32 columns, its own 8: their order along the MMA's K is the same
// for both operands, so no nibble moves between lanes.  Each scale group's
// sum starts from zero and is scaled into the f32 accumulator.
// The sum of an f32 row's two parts, the second 2^11 times what it stands for.
__device__ __forceinline__ float mv_both(float d0, float d1) { return fmaf(d1, 0x1p-11f, d0); }

enum MvFactor { kMvGroup, kMvCommon, kMvWide }; // where 2^-e comes in (mv_stage_forward)
template <int FMT, typename TX, int NT, MvFactor FACTOR>
__device__ __forceinline__ void mv_forward(uint32_t st, int half, const uint32_t (&xs)[NT],
                                           const float *ex,
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
            const uint32_t at = st + kMvRows * 128 + (mt * 16 + h * 8 + g) * 16 + half;
            if constexpr (FMT == MVLLM_FMT_INT4_G64) {
                const uint4 v = lds128(at);
                sc[mt][h][0] = __uint_as_float(v.x), sc[mt][h][1] = __uint_as_float(v.y);
                sc[mt][h][2] = __uint_as_float(v.z), sc[mt][h][3] = __uint_as_float(v.w);
            } else {
                const uint2 v = lds64(at);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    sc[mt][h][k] = ue8m0_byte(v.x, k);
                    sc[mt][h][4 + k] = ue8m0_byte(v.y, k);
                }
            }
        }
#pragma unroll
    for (int gr = 0; gr < kMvCols / F::G; ++gr) {
        float d[2][NT][4];
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
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
                        mv_int4x8(w, a[mt][h]);
                    else
                        e2m1x8_to_f16x8(w, a[mt][h][0], a[mt][h][1], a[mt][h][2], a[mt][h][3]);
                }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint4 v = lds128(xs[nt] + b * 64);
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    if (bb == 0)
                        mma_f16_16816(d[mt][nt], a[mt][0][0], a[mt][1][0], a[mt][0][1],
                                      a[mt][1][1], v.x, v.y, zero);
                    else
                        mma_f16_16816(d[mt][nt], a[mt][0][0], a[mt][1][0], a[mt][0][1],
                                      a[mt][1][1], v.x, v.y, d[mt][nt]);
                    mma_f16_16816(d[mt][nt], a[mt][0][2], a[mt][1][2], a[mt][0][3], a[mt][1][3],
                                  v.z, v.w, d[mt][nt]);
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if constexpr (FACTOR == kMvCommon) { // the columns' factors follow at the end
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    ffma2(acc[mt][nt][0], acc[mt][nt][1], d[mt][nt][0], d[mt][nt][1],
                          sc[mt][0][gr]);
                    ffma2(acc[mt][nt][2], acc[mt][nt][3], d[mt][nt][2], d[mt][nt][3],
                          sc[mt][1][gr]);
                }
            } else if constexpr (FACTOR == kMvWide) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (T == 2 && (q & 1))
                        continue;
                    const float e = ex[gr * RP + (T == 1 ? nt * 8 + 2 * t + (q & 1) : nt * 4 + t)];
                    const float e0 = fminf(e, 0x1p64f), e1 = fmaxf(e * 0x1p-64f, 1.f);
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        const float v = T == 1 ? d[mt][nt][q]
                                               : mv_both(d[mt][nt][q], d[mt][nt][q + 1]);
                        acc[mt][nt][q] = fmaf(v * e0 * sc[mt][q >> 1][gr], e1, acc[mt][nt][q]);
                    }
                }
            } else if constexpr (T == 1) {
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
                    acc[mt][nt][0] = fmaf(mv_both(d[mt][nt][0], d[mt][nt][1]) * e, sc[mt][0][gr],
                                          acc[mt][nt][0]);
                    acc[mt][nt][2] = fmaf(mv_both(d[mt][nt][2], d[mt][nt][3]) * e, sc[mt][1][gr],
                                          acc[mt][nt][2]);
                }
            }
        }
    }
}

// Gradient product of one stage: W^T, 256 columns x 32 rows.  A lane loads 8
// columns (4 bytes) of rows t, t + 4, t + 8, t + 12 of each 16 and pairs two
// rows' halfwords, after which the nibble extraction yields (row, row + 4)
// pairs of one column: the transposition costs 4 byte permutes per 32
// weights.
//
// p[0]: columns 0..3 of rows (t, t + 4), p[1]: columns 4..7; p[2], p[3] of rows
// (t + 8, t + 12); of the rows from kb * 16 on, column block h.
__device__ __forceinline__ void mv_gradient_pairs(uint32_t st, int kb, int h, uint32_t (&p)[4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint32_t r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        r[j] = lds32(st + mv_chunk(kb * 16 + t + 4 * j, h * 2 + (g >> 2)) + (g & 3) * 4);
    p[0] = mv_prmt(r[0], r[1], 0x5410u), p[1] = mv_prmt(r[0], r[1], 0x7632u);
    p[2] = mv_prmt(r[2], r[3], 0x5410u), p[3] = mv_prmt(r[2], r[3], 0x7632u);
}

// A stage's sums start from zero and are added to the task's in f32: the matrix
// unit cuts off what lies below a sum's last bit, each time towards zero, which
// over 16384 rows of far magnitudes left 1.2e-6 of the result where this leaves
// 1.4e-7.

// int4's f32 scale multiplies the row's value, and the product's three parts
// (its upper 16 bits, those of what is left, the rest: 24 bits in all) are a
// matrix instruction each, smallest first.  (Two parts, 16 to 17 bits, show in a
// bf16 result: ten times as many values one step off, 309 in place of 392 us on
// 512 rows of 160 experts of 1536 x 6144.)  A product that is not finite comes
// out as NaN; the caller notices the NaN in its sums and repeats the unit with
// CAREFUL, which keeps such a product whole in its first part.  One of finite
// factors is three times bf16's largest value there: infinite with any weight
// but 0, and 0 with that.
template <bool CAREFUL>
__device__ __forceinline__ void mv_gradient_int4(uint32_t st, uint32_t xs,
                                                 float (&acc)[4][4][1][4]) {
    const int t = threadIdx.x & 3;
    float v[2][4]; // the rows' values
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        const uint4 x = lds128(xs + kb * 64);
        v[kb][0] = __uint_as_float(x.x), v[kb][1] = __uint_as_float(x.y);
        v[kb][2] = __uint_as_float(x.z), v[kb][3] = __uint_as_float(x.w);
    }
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        uint32_t a[4][2][4], b[2][3][2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            float o[3][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float s = __uint_as_float(
                    lds32(st + kMvRows * 128 + 4 * h + (kb * 16 + t + 4 * j) * 16));
                const float m = v[kb][j] * s;
                if constexpr (CAREFUL) {
                    const bool over = fabsf(v[kb][j]) <= 3.402823466e38f &&
                                      fabsf(s) <= 3.402823466e38f && fabsf(m) > 3.402823466e38f;
#pragma unroll
                    for (int k = 0; k < 3; ++k) // bf16's largest value
                        o[k][j] = over ? copysignf(0x1.fep127f, m) : mv_term<3>(m, k);
                } else { // the packing takes the upper halves
                    o[0][j] = m;
                    o[1][j] = m - trunc_bf16(m);
                    o[2][j] = o[1][j] - trunc_bf16(o[1][j]);
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                b[kb][0][j] = mv_prmt(__float_as_uint(o[0][2 * j]),
                                      __float_as_uint(o[0][2 * j + 1]), 0x7632u);
                b[kb][1][j] = mv_prmt(__float_as_uint(o[1][2 * j]),
                                      __float_as_uint(o[1][2 * j + 1]), 0x7632u);
                b[kb][2][j] = pack_bf16(o[2][2 * j], o[2][2 * j + 1]);
            }
            uint32_t p[4];
            mv_gradient_pairs(st, kb, h, p);
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) // (128 + code) - 136
                    a[q][kb][j] = sub_bf16x2(((p[j] >> (4 * q)) & 0x000f000fu) | 0x43004300u,
                                             0x43084308u);
        }
        float d[4][4] = {};
#pragma unroll
        for (int k = 2; k >= 0; --k)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    mma_bf16_16816(d[q], a[q][kb][0], a[q][kb][1], a[q][kb][2], a[q][kb][3],
                                   b[kb][k][0], b[kb][k][1]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            ffma2(acc[h][q][0][0], acc[h][q][0][1], d[q][0], d[q][1], 1.f);
            ffma2(acc[h][q][0][2], acc[h][q][0][3], d[q][2], d[q][3], 1.f);
        }
    }
}

// MXFP4's scale multiplies the bf16 weight, exact as a power of two.  CAREFUL
// covers scale codes 0 and above 128, which the short form of the scale's bits
// does not.
template <int NT, bool CAREFUL>
__device__ __forceinline__ void mv_gradient_mxfp4(uint32_t st, int half, const uint32_t (&xs)[NT],
                                                  float (&acc)[4][4][NT][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint32_t b[2][NT][2]; // the same for every column
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint2 v = lds64(xs[nt] + kb * 32);
            b[kb][nt][0] = v.x, b[kb][nt][1] = v.y;
        }
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        uint32_t p[2][4], m[2][2], m2[2][2] = {};
        // 2^(code - 1) = 2^126 * scale as bf16, the weight's bits being 2^-126 of
        // its value: the code's exponent field plus 126.  Codes above 128 take
        // 2^126 and then the scale, 0 is 0.
        const uint32_t sel = ((h & 1) * 2 + (g >> 2)) * 0x11u;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            mv_gradient_pairs(st, kb, h, p[kb]);
            const uint32_t codes = st + kMvRows * 128 + (kb * 16 + t) * 16 + half + 4 * (h >> 1);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                // byte k of the two rows' codes in the two halfwords
                const uint32_t c = mv_prmt(lds32(codes + 128 * j), lds32(codes + 128 * j + 64),
                                           sel | ((sel | 0x44u) << 8)) &
                                   0x00ff00ffu;
                if constexpr (CAREFUL) {
                    const uint32_t lo = c & 255u, hi = c >> 16;
                    m[kb][j] = (lo ? 253u << 7 : 0u) | (hi ? 253u << 23 : 0u);
                    m2[kb][j] = (lo << 7) | (hi << 23);
                } else {
                    m[kb][j] = c * 128u + ((126u << 7) | (126u << 23));
                }
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float d[NT][4] = {};
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                uint32_t a[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w = p[kb][j];
                    const uint32_t mag = q == 0   ? w << 6
                                         : q == 1 ? w << 2
                                         : q == 2 ? w >> 2
                                                  : w >> 6;
                    const uint32_t v = (mag & 0x01c001c0u) | ((w << (12 - 4 * q)) & 0x80008000u);
                    a[j] = mul_bf16x2(v, m[kb][j >> 1]);
                    if constexpr (CAREFUL)
                        a[j] = mul_bf16x2(a[j], m2[kb][j >> 1]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_bf16_16816(d[nt], a[0], a[1], a[2], a[3], b[kb][nt][0], b[kb][nt][1]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                ffma2(acc[h][q][nt][0], acc[h][q][nt][1], d[nt][0], d[nt][1], 1.f);
                ffma2(acc[h][q][nt][2], acc[h][q][nt][3], d[nt][2], d[nt][3], 1.f);
            }
        }
    }
}

// Whether a stage of MXFP4 has a scale code of 0 or above 127 (lane = row).
__device__ __forceinline__ bool mv_odd_codes(uint32_t st, int half) {
    const uint2 v = lds64(st + kMvRows * 128 + (threadIdx.x & 31) * 16 + half);
    const uint32_t odd = v.x | v.y | ((v.x - 0x01010101u) & ~v.x) | ((v.y - 0x01010101u) & ~v.y);
    return __any_sync(0xffffffffu, (odd & 0x80808080u) != 0);
}

// The gradient's partial sums share the ring's memory (no copy of the next unit
// is in flight over the reduction): both would not fit.
template <bool GRAD> constexpr bool mv_alias() { return GRAD; }
// f32 elements of one task's partial sums.
template <int FMT, typename TX, int NT, bool GRAD> constexpr int mv_red_pitch() {
    return GRAD ? kMvCols + 1 : 36;
}
template <int FMT, typename TX, int NT, bool GRAD> constexpr int mv_red_size() {
    return (GRAD ? 8 * NT : 8 * NT / MvTerms<FMT, TX, GRAD>::T) *
           mv_red_pitch<FMT, TX, NT, GRAD>();
}
template <int FMT, typename TX, bool GRAD, typename Int>
__host__ __device__ constexpr Int mv_x_pitch(Int cols) {
    // Row pitch of the staged x: the lanes of one shared-memory phase fall
    // into different banks.
    if (!GRAD)
        return cols * 2 + 64;
    if (FMT == MVLLM_FMT_INT4_G64)
        return (cols * 4 + 127) / 128 * 128 + 64;
    return (cols * 2 + 127) / 128 * 128 + 32;
}

__device__ __forceinline__ void mv_store(void *y, int f32, int64_t at, float v) {
    if (f32)
        static_cast<float *>(y)[at] = v;
    else
        static_cast<__nv_bfloat16 *>(y)[at] = __float2bfloat16_rn(v);
}

// A task's partial sums to shared memory, [row of x][output] (f32 rows: their
// two parts added), times the rows' factors where those were left out (`check`
// becomes NaN where a sum before them is not finite); on top of what an earlier
// chunk left there when `add`.
template <int T, int RPITCH, int NT>
__device__ __forceinline__ void mv_put(float *to, const float (&acc)[2][NT][4], const float *ex,
                                       bool add, float &check) {
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float d[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
                d[q] = acc[mt][nt][q];
            if (T == 1) {
                if (ex) {
                    check = fmaf(d[0] + d[1] + d[2] + d[3], 0.f, check);
                    const float2 e = *reinterpret_cast<const float2 *>(ex + nt * 8 + 2 * t);
                    d[0] *= e.x, d[1] *= e.y, d[2] *= e.x, d[3] *= e.y;
                }
                float *at = to + (nt * 8 + 2 * t) * RPITCH + mt * 16 + g;
                at[0] = add ? at[0] + d[0] : d[0];
                at[8] = add ? at[8] + d[2] : d[2];
                at[RPITCH] = add ? at[RPITCH] + d[1] : d[1];
                at[RPITCH + 8] = add ? at[RPITCH + 8] + d[3] : d[3];
            } else {
                if (ex) {
                    const float e = ex[nt * 4 + t], s0 = mv_both(d[0], d[1]),
                                s1 = mv_both(d[2], d[3]);
                    check = fmaf(s0 + s1, 0.f, check);
                    d[0] = s0 * e, d[2] = s1 * e;
                }
                float *at = to + (nt * 4 + t) * RPITCH + mt * 16 + g;
                at[0] = add ? at[0] + d[0] : d[0];
                at[8] = add ? at[8] + d[2] : d[2];
            }
        }
}
// The gradient's: [part of a row][output].
template <int RPITCH, int NT>
__device__ __forceinline__ void mv_put_gradient(float *to, const float (&acc)[4][4][NT][4]) {
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float(&d)[4] = acc[h][q][nt];
                float *at = to + (nt * 8 + 2 * t) * RPITCH + h * 64 + 8 * g + q;
                at[0] = d[0], at[RPITCH] = d[1];
                at[4] = d[2], at[RPITCH + 4] = d[3];
            }
}

struct MvUnit {
    const uint8_t *w, *s;
    int item, r0, n, out0;
};

// One CTA of a cluster.  A unit is (rows of one matrix, at most RP of them) x
// (a range of outputs); the cluster's CTAs split the reduction.  A CTA's tasks
// are the range's tiles x wk parts of its slice of the reduction; its warps
// take them in turn, each streaming its tasks' stages through its own ring, so
// the main loop has no barrier (a stage takes a warp about 2 us).  The wk x
// cluster partial sums of an output meet in (distributed) shared memory and are
// added in a fixed order.
template <int FMT, typename TX, int NT, bool GRAD>
__global__ void __launch_bounds__(32 * mv_warps<NT, GRAD>(), 1)
    matvec_q4_kernel(const MatvecArgs a, const MatvecPlan pl, const TX *__restrict__ x,
                     int64_t ldx, void *__restrict__ y, int64_t ldy) {
    using F = MvFormat<FMT>;
    constexpr int T = MvTerms<FMT, TX, GRAD>::T, RP = 8 * NT / T, ST = mv_ring<NT, GRAD>();
    constexpr int kMvWarps = mv_warps<NT, GRAD>(), kMvThreads = 32 * kMvWarps;
    constexpr int TILE = GRAD ? kMvCols : kMvRows, STEP = GRAD ? kMvRows : kMvCols;
    constexpr int RPITCH = mv_red_pitch<FMT, TX, NT, GRAD>();
    constexpr int RSIZE = mv_red_size<FMT, TX, NT, GRAD>();
    extern __shared__ __align__(128) uint8_t mv_smem[];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int rank, ranks, cluster, clusters;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    asm("mov.u32 %0, %%clusterid.x;" : "=r"(cluster));
    asm("mov.u32 %0, %%nclusterid.x;" : "=r"(clusters));
    // A peer's shared memory is there once the peer has started: every thread
    // says so here and waits for the others before the first unit's sums.
    if (ranks > 1)
        asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    float *ex = reinterpret_cast<float *>(mv_smem + pl.off_ex);
    float *red = reinterpret_cast<float *>(mv_smem + pl.off_red);
    int *list = reinterpret_cast<int *>(mv_smem + pl.off_list); // passes before each expert
    int items;
    if (a.wt) {
        constexpr int PER = (kMvMaxExperts + kMvThreads - 1) / kMvThreads;
        __shared__ int wsum[kMvWarps];
        int n[PER], v = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int e = PER * int(threadIdx.x) + k;
            const uint8_t *w, *s;
            int r0 = 0, r1 = 0;
            n[k] = e < a.nb && matvec_expert(a, e, w, s, r0, r1) ? (r1 - r0 + RP - 1) / RP : 0;
            v += n[k];
        }
        int first = -v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            v += lane >= o ? u : 0;
        }
        if (lane == 31)
            wsum[warp] = v;
        __syncthreads();
        first += v;
        for (int k = 0; k < warp; ++k)
            first += wsum[k];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int e = PER * int(threadIdx.x) + k;
            if (e < a.nb)
                list[e] = first;
            first += n[k];
            if (e == a.nb - 1)
                list[a.nb] = first;
        }
        __syncthreads();
        items = list[a.nb];
    } else {
        items = (a.rows + RP - 1) / RP;
    }
    const int total = items * pl.nranges; // below the elements of y
    const int rows_w = GRAD ? pl.K : pl.N; // rows of the matrices (O)

    auto decode = [&](int u) {
        MvUnit q;
        q.item = u / pl.nranges;
        q.out0 = (u - q.item * pl.nranges) * pl.range;
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
        return q;
    };
    const int steps = (pl.K + STEP - 1) / STEP;
    const int k0 = min(rank * pl.slice, steps), nk = min(pl.slice, steps - k0);
    const uint32_t ring = smem_u32(mv_smem) + warp * ST * F::STAGE;
    // Tasks of a unit, and the stages of chunk c0 that part kk of one takes.
    auto tasks_of = [&](const MvUnit &q) {
        return q.w ? (min(pl.range, pl.N - q.out0) + TILE - 1) / TILE * pl.wk : 0;
    };
    auto stages_of = [&](int c0, int kk) {
        const int len = min(pl.chunk, nk - c0);
        return len > kk ? (len - kk + pl.wk - 1) / pl.wk : 0;
    };
    // The copies run ahead of the products through the same order: chunks,
    // this warp's tasks, the task's stages.
    MvWalk<FMT, GRAD> walk;
    int w_c0 = 0, w_task = 0, w_i = 0, w_n = 0, w_tasks = 0, filled = 0, used = 0;
    const uint8_t *w_w = nullptr, *w_s = nullptr;
    int w_out = 0;
    auto enter = [&] { // the walk's current task
        const int kk = w_task % pl.wk;
        w_i = 0, w_n = stages_of(w_c0, kk);
        const int out = w_out + w_task / pl.wk * TILE, at = k0 + w_c0 + kk;
        walk.start(w_w, w_s, rows_w, a.I, GRAD ? at * STEP : out, GRAD ? out / kMvCols : at,
                   pl.wk);
    };
    auto issue = [&] {
        while (w_i >= w_n && w_c0 < nk) { // the next task that has a stage
            w_task += kMvWarps;
            if (w_task >= w_tasks) {
                w_task = warp;
                w_c0 += pl.chunk;
                if (w_c0 >= nk)
                    break;
            }
            enter();
        }
        if (w_i < w_n) {
            walk.fill(ring + (filled % ST) * F::STAGE);
            ++w_i;
        }
        ++filled;
        mv_commit();
    };
    auto prologue = [&](const MvUnit &q) {
        w_w = q.w, w_s = q.s, w_out = q.out0, w_tasks = tasks_of(q);
        w_c0 = 0, w_task = warp, w_i = w_n = 0;
        filled = used;
        if (warp < w_tasks)
            enter();
        else
            w_c0 = nk; // nothing to copy
        issue();
    };

    const int cols = pl.chunk * STEP, pitch = mv_x_pitch<FMT, TX, GRAD>(cols);
    const uint32_t xs = smem_u32(mv_smem + pl.off_x);
    // Where this lane reads its operand columns.  A column without a row reads
    // the last one's again: its results are not written.
    constexpr int XB = GRAD ? (FMT == MVLLM_FMT_INT4_G64 ? 4 : 2) : 2; // bytes of an element
    uint32_t xcol[NT];
    int staged = -1;     // the item whose only chunk is staged
    MvFactor factor = kMvGroup; // how its rows are scaled
    int turn = 0;        // the mail buffer of this unit
    __shared__ uint32_t row_max[GRAD ? 1 : 2 * RP];
    MvHeld<TX, NT> held; // gradient
    // The first rows of a unit that has to be staged.
    auto fetch = [&](const MvUnit &q) {
        if (q.w && staged != q.item) {
            if constexpr (GRAD) {
                held.load(x, ldx, q.r0, q.n, k0 * STEP, cols, pl.K, pl.x_vec);
            } else {
                mv_fetch_rows<FMT, TX, NT>(mv_smem + pl.off_x, pitch, x, ldx, q.r0, q.n, k0 * STEP,
                                           cols, pl.K, pl.x_vec);
                if (threadIdx.x < RP)
                    row_max[threadIdx.x] = 0u, row_max[RP + threadIdx.x] = 0x7f800000u;
            }
        }
        mv_commit();
    };
    MvUnit cur{};
    // A cluster's units follow one another, so that an item's rows are staged
    // once for its ranges (48 experts of 5 rows, 7168 -> 2048: 111 us; 130 with
    // the clusters taking units in turn).
    const int each = total / clusters, more = total - each * clusters;
    const int u0 = each * cluster + min(cluster, more), u1 = u0 + each + (cluster < more);
    if (u0 < u1) {
        cur = decode(u0);
        fetch(cur);
        prologue(cur);
    }
    for (int u = u0; u < u1; ++u) {
        const int tasks = tasks_of(cur);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int col = min(nt * 8 + (lane >> 2), cur.n * T - 1);
            xcol[nt] = xs + col * pitch + (lane & 3) * (GRAD ? 4 * XB : 16);
        }
        // The gradient's one task per warp keeps its sums to the end of the
        // unit; the forward's tasks leave theirs in shared memory one by one.
        float accg[GRAD ? 4 : 1][GRAD ? 4 : 1][NT][4];
        MvUnit next{};
        float check = 0.f; // NaN where a sum before its factor is not finite
        for (bool careful = false;; careful = true) {
            bool refilled = false;
            if constexpr (GRAD) {
#pragma unroll
                for (int i = 0; i < 16 * NT * 4; ++i)
                    (&accg[0][0][0][0])[i] = 0.f;
            }
            for (int c0 = 0; c0 < nk; c0 += pl.chunk) {
                if (cur.w && staged != cur.item) { // uniform over the CTA
                    bool wide = false;
                    if constexpr (GRAD) {
                        __syncthreads(); // the last readers of x are done
                        mv_stage_gradient<FMT, TX, NT>(mv_smem + pl.off_x, pitch, x, ldx, cur.r0,
                                                       cur.n, (k0 + c0) * STEP, cols, pl.K,
                                                       pl.x_vec, c0 == 0, held);
                    } else {
                        if (c0 > 0) {
                            __syncthreads();
                            mv_fetch_rows<FMT, TX, NT>(mv_smem + pl.off_x, pitch, x, ldx, cur.r0,
                                                       cur.n, (k0 + c0) * STEP, cols, pl.K,
                                                       pl.x_vec);
                            mv_commit();
                            mv_wait<0>();
                        } else {
                            // the first unit's rows were asked for before its
                            // weights, the others' after
                            if (u == u0)
                                mv_wait<1>();
                            else
                                mv_wait<0>();
                        }
                        __syncthreads();
                        factor = mv_stage_forward<FMT, TX, NT>(
                                     mv_smem + pl.off_x, ex, pitch, cur.n, cols,
                                     pl.try_common && nk <= pl.chunk, row_max, wide)
                                     ? kMvCommon
                                     : kMvGroup;
                    }
                    if (__syncthreads_or(wide))
                        factor = kMvWide;
                    if (nk <= pl.chunk)
                        staged = cur.item;
                }
                // The ring's other stages, now that the rows are staged: the first
                // kept the memory system busy meanwhile, more would only have
                // queued in front of them.
                for (int k = refilled ? ST : 1; k < ST - 1; ++k)
                    issue();
                refilled = true;
                for (int task = warp; task < tasks; task += kMvWarps) {
                    const int kk = task % pl.wk, n = stages_of(c0, kk);
                    float accf[GRAD ? 1 : 2][NT][4] = {};
                    for (int i = 0; i < n; ++i) {
                        mv_wait<ST - 2>();
                        __syncwarp();
                        issue(); // into the slot computed last
                        const uint32_t st = ring + (used++ % ST) * F::STAGE;
                        const int step = kk + i * pl.wk; // within the chunk
                        const int colstep = GRAD ? (cur.out0 + task / pl.wk * TILE) / kMvCols
                                                 : k0 + c0 + step;
                        const int half = F::SB == 8 ? (colstep & 1) * 8 : 0;
                        uint32_t xat[NT];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            xat[nt] = xcol[nt] + step * (STEP * XB);
                        if constexpr (GRAD && FMT == MVLLM_FMT_INT4_G64) {
                            if (careful)
                                mv_gradient_int4<true>(st, xat[0], accg);
                            else
                                mv_gradient_int4<false>(st, xat[0], accg);
                        } else if constexpr (GRAD) {
                            if (mv_odd_codes(st, half))
                                mv_gradient_mxfp4<NT, true>(st, half, xat, accg);
                            else
                                mv_gradient_mxfp4<NT, false>(st, half, xat, accg);
                        } else {
                            const float *at = ex + step * (STEP / F::G) * RP;
                            if (factor == kMvCommon)
                                mv_forward<FMT, TX, NT, kMvCommon>(st, half, xat, ex, accf);
                            else if (factor == kMvGroup)
                                mv_forward<FMT, TX, NT, kMvGroup>(st, half, xat, at, accf);
                            else
                                mv_forward<FMT, TX, NT, kMvWide>(st, half, xat, at, accf);
                        }
                    }
                    __syncwarp();
                    if constexpr (!GRAD)
                        mv_put<T, RPITCH>(red + task * RSIZE, accf,
                                          factor == kMvCommon ? ex : nullptr, c0 > 0, check);
                }
            }
            if constexpr (!GRAD) {
                // A warp that is done goes on to the next unit's weights; its rows
                // wait until their places are free.
                __syncwarp();
                if (u + 1 < u1) {
                    next = decode(u + 1);
                    prologue(next);
                }
                if (!__syncthreads_or(check != check))
                    break;
                // Again with the rows' common factors as every group's.
                for (int i = RP + threadIdx.x; i < cols / F::G * RP; i += kMvThreads)
                    ex[i] = ex[i % RP];
                factor = kMvGroup, check = 0.f;
                mv_wait<0>(); // the stage just asked for: its place is needed
                __syncthreads();
                prologue(cur);
                continue;
            }
            if (FMT != MVLLM_FMT_INT4_G64 || careful)
                break;
            float nan = 0.f; // NaN where a sum is, or where infinities meet
#pragma unroll
            for (int i = 0; i < (GRAD ? 16 * NT * 4 : 0); ++i)
                nan += (&accg[0][0][0][0])[i];
            if (!__syncthreads_or(nan != nan))
                break;
            prologue(cur);
        }
        if constexpr (GRAD) {
            if (u + 1 < u1)
                next = decode(u + 1);
            mv_wait<0>();
            __syncthreads(); // the ring is done with before the sums overlay it
            if (warp < tasks)
                mv_put_gradient<RPITCH>(red + warp * RSIZE, accg);
            __syncthreads();
        } else if (u + 1 < u1) {
            fetch(next);
        }
        // The CTA's own wk partial sums (and the gradient's parts) first.  With
        // one CTA per cluster that is the result; else it goes to the CTA that
        // owns the block, and one cluster barrier later each CTA adds up what it
        // was sent.  Two buffers take
        // turns, so that a unit's values cannot meet the next one's.
        // An item is (row, block of 32 outputs), eight lanes of four outputs each;
        // warps take four at a time.  It is owned by rank item % ranks, there in
        // slot item / ranks * ranks + sender.  (Distributed shared memory takes
        // 16 bytes a lane better than 4: 16 rows of 7168 -> 16384 in 31 us then, 35
        // with four times the stores.)
        const int outs = min(pl.range, pl.N - cur.out0), blocks = (outs + 31) / 32;
        const int all = blocks * cur.n, sub = lane >> 3, o4 = (lane & 7) * 4;
        const int slots = (pl.range / 32 * RP + ranks - 1) / ranks * ranks; // of a mail buffer
        const uint32_t mail = smem_u32(mv_smem + pl.off_mail) + turn * slots * 128;
        const int parts = cur.w ? pl.wk : 0, mask = ranks - 1;
        auto out = [&](int r, int o, const float(&v)[4]) {
            const int64_t at = int64_t(cur.r0 + r) * ldy + cur.out0 + o;
            if (pl.y_vec && o + 4 <= outs) {
                if (pl.y_f32)
                    store_row<4>(static_cast<float *>(y) + at, v);
                else
                    store_row<4>(static_cast<__nv_bfloat16 *>(y) + at, v);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (o + q < outs)
                        mv_store(y, pl.y_f32, at + q, v[q]);
            }
        };
        if (ranks > 1 && u == u0)
            mv_cluster_wait();
        for (int item = warp * 4 + sub; item < all; item += kMvWarps * 4) {
            const int r = item / blocks, o = (item - r * blocks) * 32 + o4;
            const float *at =
                red + (o / TILE) * pl.wk * RSIZE + o % TILE + r * ((GRAD ? T : 1) * RPITCH);
            float v[4] = {};
            for (int k = 0; k < parts; ++k) {
                if constexpr (GRAD) {
#pragma unroll
                    for (int q = 0; q < T; ++q)
#pragma unroll
                        for (int s = 0; s < 4; ++s)
                            v[s] += at[k * RSIZE + q * RPITCH + s];
                } else {
                    const float4 p = *reinterpret_cast<const float4 *>(at + k * RSIZE);
                    v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w;
                }
            }
            if (ranks > 1)
                st_cluster_f32x4(
                    mv_cluster_addr(mail + ((item & ~mask) + rank) * 128 + o4 * 4, item & mask), v);
            else
                out(r, o, v);
        }
        if (ranks > 1) {
            mv_cluster_sync();
            for (int item = (warp * 4 + sub) * ranks + rank; item < all;
                 item += kMvWarps * 4 * ranks) {
                const int r = item / blocks, o = (item - r * blocks) * 32 + o4;
                const uint32_t at = mail + (item & ~mask) * 128 + o4 * 4;
                float v[4] = {};
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    if (c < ranks) {
                        const uint4 p = lds128(at + c * 128);
                        v[0] += __uint_as_float(p.x), v[1] += __uint_as_float(p.y);
                        v[2] += __uint_as_float(p.z), v[3] += __uint_as_float(p.w);
                    }
                }
                out(r, o, v);
            }
            turn ^= 1;
        } else {
            __syncthreads();
        }
        cur = next;
        if (GRAD && u + 1 < u1) {
            fetch(cur);
            prologue(cur);
        }
    }
    if (ranks > 1 && u0 >= u1) // without units the first wait is still owed
        mv_cluster_wait();
}

} // namespace mvb

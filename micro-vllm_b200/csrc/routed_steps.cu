// routed_steps.cu -- host entries of the routed layer's separate steps:
// dispatch, combine and the router, with their gradients.
#include "host.hpp"
#include "route_grad.cuh"

#include <algorithm>

using namespace mvb;

namespace {

bool row_dtype(int d) { return d == MVLLM_DTYPE_F32 || d == MVLLM_DTYPE_BF16; }
size_t dtype_bytes(int d) { return d == MVLLM_DTYPE_F32 ? 4 : 2; }

// Largest power of two (at most 16) that divides the address, the pitch and
// the row length, all in bytes.
unsigned row_align(const void *p, int64_t ld, int D, int dtype) {
    const uint64_t b = dtype_bytes(dtype);
    const uint64_t v = reinterpret_cast<uintptr_t>(p) | uint64_t(ld) * b | uint64_t(D) * b | 16u;
    return unsigned(v & (~v + 1));
}

// Elements per lane: 16 bytes of the widest-loaded type where everything is
// aligned for it, 4 bytes' worth, or one element.
int row_vec(unsigned align, size_t bytes) {
    return align >= 16 ? int(16 / bytes) : align >= 4 ? int(4 / bytes) : 1;
}

constexpr int64_t kMaxGrid = 0x7fffffff;
constexpr int kMaxRow = 1 << 30; // elements of a row: steps past its end stay in 32 bits

// Segments of a row of `total` lane-words for T tokens: as few as give `wanted`
// of them in all, each a multiple of `piece` words.
struct Segments {
    int n, words;
    Segments(int T, int total, int piece, int wanted) {
        const int most = (total + piece - 1) / piece;
        const int64_t want = (int64_t(wanted) + T - 1) / T;
        n = int(std::max<int64_t>(1, std::min<int64_t>(most, want)));
        words = (most + n - 1) / n * piece;
        n = (total + words - 1) / words;
    }
};

} // namespace

extern "C" {

int mvllm_moe_dispatch_dev(void *stream, const void *x, int dtype, int64_t ldx,
                           const int *tok_pos, int T, int KK, int D, void *xs, int64_t ldxs,
                           int rows_cap) {
    if ((T > 0 && (!x || !tok_pos || (!xs && rows_cap > 0))) || T < 0 || KK < 1 ||
        KK > kMaxSlots || D < 1 || D > kMaxRow || ldx < 0 || ldxs < D || rows_cap < 0 ||
        !row_dtype(dtype))
        return host_fail(MVLLM_ERR_INVALID, "dispatch_dev: invalid arguments");
    DeviceScope dev;
    if (int rc = dev.enter())
        return rc;
    if (T == 0 || rows_cap == 0)
        return MVLLM_OK;
    const unsigned al = std::min(row_align(x, ldx, D, dtype), row_align(xs, ldxs, D, dtype));
    const int64_t b = dtype_bytes(dtype), w = al >= 16 ? 16 : al >= 4 ? 4 : 2;
    // A lane's words: one of 16 bytes, four narrower ones (4096 tokens to 8
    // positions each, 2051 bf16: 32 us, 74 by one).
    const int words = int(D * b / w), piece = w == 16 ? 32 : 128;
    const int pieces = (words + piece - 1) / piece;
    const int64_t units = int64_t(T) * pieces, grid = (units + 7) / 8;
    if (grid > kMaxGrid)
        return host_fail(MVLLM_ERR_INVALID, "dispatch_dev: T too large");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
#define MVB_DISPATCH(W, Q)                                                                     \
    MVB_TRY(launch_serial(dispatch_rows_kernel<W, Q>, dim3(unsigned(grid)), dim3(256), 0, st,  \
                          static_cast<const W *>(x), ldx *b / w, tok_pos, units, pieces, KK,   \
                          words, static_cast<W *>(xs), ldxs *b / w, rows_cap))
    if (w == 16)
        MVB_DISPATCH(uint4, 1);
    else if (w == 4)
        MVB_DISPATCH(uint32_t, 4);
    else
        MVB_DISPATCH(uint16_t, 4);
#undef MVB_DISPATCH
    return MVLLM_OK;
}

} // extern "C"

namespace {

template <typename TY, typename TO>
int combine_launch(cudaStream_t st, int sms, int n, const TY *y, int64_t ldy, int cap,
                   const float *rw, const int *tok_pos, int T, int KK, int D, TO *out,
                   int64_t ldo, int accumulate) {
    // 64 warps per SM: whole rows leave 64 tokens of 8 rows of 7168 bf16 at 30 us
    // in place of 4.0; the finest cut costs 4096 tokens 93 in place of 85.
    const Segments s(T, (D + n - 1) / n, 32, sms * 64);
    const int64_t units = int64_t(T) * s.n, grid = (units + 7) / 8;
    if (grid > kMaxGrid)
        return host_fail(MVLLM_ERR_INVALID, "combine: T too large");
#define MVB_COMBINE(N)                                                                         \
    MVB_TRY(launch_serial(combine_rows_kernel<TY, TO, N>, dim3(unsigned(grid)), dim3(256), 0,  \
                          st, y, ldy, cap, rw, tok_pos, units, s.n, s.words * N, KK, D, out,   \
                          ldo, accumulate))
    if (n == 16 / int(sizeof(TY)))
        MVB_COMBINE(16 / int(sizeof(TY)));
    else if (n == 4 / int(sizeof(TY)) && n > 1)
        MVB_COMBINE(4 / int(sizeof(TY)));
    else
        MVB_COMBINE(1);
#undef MVB_COMBINE
    return MVLLM_OK;
}

int combine_any(const char *who, void *stream, const void *y, int y_dtype, int64_t ldy, int cap,
                const float *rw, const int *tok_pos, int T, int KK, int D, void *out,
                int out_dtype, int64_t ldo, int accumulate) {
    if ((T > 0 && ((!y && cap > 0) || !tok_pos || !out)) || T < 0 || KK < 1 || KK > kMaxSlots ||
        D < 1 || D > kMaxRow || ldy < 0 || ldo < D || cap < 0 || !row_dtype(y_dtype) ||
        !row_dtype(out_dtype))
        return host_fail(MVLLM_ERR_INVALID, "%s: invalid arguments", who);
    DeviceScope dev;
    if (int rc = dev.enter())
        return rc;
    if (T == 0)
        return MVLLM_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // N elements a lane for both matrices: y's vector, unless out's rows are
    // aligned for less.
    const int ey = int(dtype_bytes(y_dtype)), eo = int(dtype_bytes(out_dtype));
    int n = row_vec(row_align(y, ldy, D, y_dtype), ey);
    const unsigned ao = row_align(out, ldo, D, out_dtype);
    if (ao < std::min(16u, unsigned(n * eo)))
        n = std::min(n, row_vec(ao, ey));
    if (ao < std::min(16u, unsigned(n * eo)))
        n = 1;
    const bool fy = y_dtype == MVLLM_DTYPE_F32, fo = out_dtype == MVLLM_DTYPE_F32;
    using bf = __nv_bfloat16;
    if (fy && fo)
        return combine_launch(st, dev.sms, n, static_cast<const float *>(y), ldy, cap, rw,
                              tok_pos, T, KK, D, static_cast<float *>(out), ldo, accumulate);
    if (fy)
        return combine_launch(st, dev.sms, n, static_cast<const float *>(y), ldy, cap, rw,
                              tok_pos, T, KK, D, static_cast<bf *>(out), ldo, accumulate);
    if (fo)
        return combine_launch(st, dev.sms, n, static_cast<const bf *>(y), ldy, cap, rw,
                              tok_pos, T, KK, D, static_cast<float *>(out), ldo, accumulate);
    return combine_launch(st, dev.sms, n, static_cast<const bf *>(y), ldy, cap, rw, tok_pos,
                          T, KK, D, static_cast<bf *>(out), ldo, accumulate);
}

template <typename TD, typename TY>
int combine_grad_launch(cudaStream_t st, int n, const TD *dout, int64_t lddo, const TY *y,
                        int64_t ldy, int cap, const float *rw, const int *tok_pos,
                        const int *idx, int T, int K, int KK, int D, TY *dy, int64_t lddy,
                        float *dwt) {
#define MVB_CGRAD(N)                                                                           \
    MVB_TRY(launch_serial(combine_grad_kernel<TD, TY, N>, dim3(unsigned(T)), dim3(256), 0, st, \
                          dout, lddo, y, ldy, cap, rw, tok_pos, idx, K, KK, D, dy, lddy, dwt))
    if (n == 16 / int(sizeof(TY)))
        MVB_CGRAD(16 / int(sizeof(TY)));
    else if (n == 4 / int(sizeof(TY)) && n > 1)
        MVB_CGRAD(4 / int(sizeof(TY)));
    else
        MVB_CGRAD(1);
#undef MVB_CGRAD
    return MVLLM_OK;
}

} // namespace

extern "C" {

int mvllm_moe_dispatch_grad_dev(void *stream, const void *dxs, int dxs_dtype, int64_t lddxs,
                                int rows_cap, const int *tok_pos, int T, int KK, int D, void *dx,
                                int dx_dtype, int64_t lddx, int accumulate) {
    return combine_any("dispatch_grad_dev", stream, dxs, dxs_dtype, lddxs, rows_cap, nullptr,
                       tok_pos, T, KK, D, dx, dx_dtype, lddx, accumulate);
}

int mvllm_moe_combine_dev(void *stream, const void *y, int y_dtype, int64_t ldy, int rows_cap,
                          const float *rw, const int *tok_pos, int T, int KK, int D, void *out,
                          int out_dtype, int64_t ldo, int accumulate) {
    if (T > 0 && rows_cap > 0 && !rw)
        return host_fail(MVLLM_ERR_INVALID, "combine_dev: invalid arguments");
    return combine_any("combine_dev", stream, y, y_dtype, ldy, rows_cap, rw, tok_pos, T, KK, D,
                       out, out_dtype, ldo, accumulate);
}

int mvllm_moe_combine_grad_dev(void *stream, const void *dout, int dout_dtype, int64_t lddo,
                               const void *y, int y_dtype, int64_t ldy, int rows_cap,
                               const float *rw, const int *tok_pos, const int *idx, int T, int K,
                               int KK, int D, void *dy, int64_t lddy, float *dwt) {
    if ((T > 0 && (!dout || !tok_pos || !idx || !dwt || (rows_cap > 0 && (!y || !rw || !dy)))) ||
        T < 0 || K < 1 || KK < K || KK > kMaxSlots || D < 1 || D > kMaxRow || lddo < 0 ||
        ldy < 0 || lddy < D || rows_cap < 0 || !row_dtype(dout_dtype) || !row_dtype(y_dtype))
        return host_fail(MVLLM_ERR_INVALID, "combine_grad_dev: invalid arguments");
    DeviceScope dev;
    if (int rc = dev.enter())
        return rc;
    if (T == 0)
        return MVLLM_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int ey = int(dtype_bytes(y_dtype)), ed = int(dtype_bytes(dout_dtype));
    int n = row_vec(std::min(row_align(y, ldy, D, y_dtype), row_align(dy, lddy, D, y_dtype)), ey);
    const unsigned ad = row_align(dout, lddo, D, dout_dtype);
    if (ad < std::min(16u, unsigned(n * ed)))
        n = std::min(n, row_vec(ad, ey));
    if (ad < std::min(16u, unsigned(n * ed)))
        n = 1;
    using bf = __nv_bfloat16;
    const bool fd = dout_dtype == MVLLM_DTYPE_F32, fy = y_dtype == MVLLM_DTYPE_F32;
    if (fd && fy)
        return combine_grad_launch(st, n, static_cast<const float *>(dout), lddo,
                                   static_cast<const float *>(y), ldy, rows_cap, rw, tok_pos, idx,
                                   T, K, KK, D, static_cast<float *>(dy), lddy, dwt);
    if (fd)
        return combine_grad_launch(st, n, static_cast<const float *>(dout), lddo,
                                   static_cast<const bf *>(y), ldy, rows_cap, rw, tok_pos, idx, T,
                                   K, KK, D, static_cast<bf *>(dy), lddy, dwt);
    if (fy)
        return combine_grad_launch(st, n, static_cast<const bf *>(dout), lddo,
                                   static_cast<const float *>(y), ldy, rows_cap, rw, tok_pos, idx,
                                   T, K, KK, D, static_cast<float *>(dy), lddy, dwt);
    return combine_grad_launch(st, n, static_cast<const bf *>(dout), lddo,
                               static_cast<const bf *>(y), ldy, rows_cap, rw, tok_pos, idx, T, K,
                               KK, D, static_cast<bf *>(dy), lddy, dwt);
}

} // extern "C"

namespace {

template <typename TO>
int route_dx(cudaStream_t st, const RouteGradArgs &a, int sms, TO *dx, int64_t lddx) {
    const int type = sizeof(TO) == 4 ? MVLLM_DTYPE_F32 : MVLLM_DTYPE_BF16;
    const bool vec = std::min(row_align(a.router, a.H, a.H, MVLLM_DTYPE_F32), 16u) == 16 &&
                     row_align(dx, lddx, a.H, type) >= 4 * sizeof(TO);
    const int n = vec ? 4 : 1;
    // As few segments as make four CTAs per SM: 48 tokens of H 7168 take 5.9 us
    // in place of 17.8 in one segment each.
    const Segments s(a.T, a.H / n, kRgThreads, sms * 4);
    const int64_t grid = int64_t(a.T) * s.n;
    if (grid > kMaxGrid)
        return host_fail(MVLLM_ERR_INVALID, "route_grad_dev: T too large");
    if (vec)
        MVB_TRY(launch_serial(route_dx_kernel<TO, 4>, dim3(unsigned(grid)), dim3(kRgThreads), 0, st,
                              a, s.n, s.words * n, dx, lddx));
    else
        MVB_TRY(launch_serial(route_dx_kernel<TO, 1>, dim3(unsigned(grid)), dim3(kRgThreads), 0, st,
                              a, s.n, s.words * n, dx, lddx));
    return MVLLM_OK;
}

template <typename TX>
int route_dw(cudaStream_t st, const RouteGradArgs &a, int sms, const TX *x, int64_t ldx,
             const int *nr, const int *xoff, const int *rows, float *drouter) {
    const int64_t groups = ((a.H + kRgCols - 1) / kRgCols + 7) / 8;
    const int64_t most = (int64_t(a.cap) / kRgRows + a.E) * groups;
    const unsigned grid = unsigned(std::min<int64_t>(int64_t(sms) * 4, most));
    const unsigned b = sizeof(TX);
    const int vec = ((reinterpret_cast<uintptr_t>(x) | uint64_t(ldx) * b) & 15u) == 0;
    MVB_TRY(launch_serial(route_dw_kernel<TX>, dim3(grid), dim3(256), 0, st, a, x, ldx, vec, nr,
                          xoff, rows, drouter));
    return MVLLM_OK;
}

} // namespace

extern "C" {

size_t mvllm_moe_route_grad_workspace(int T, int H, int E, int K) {
    if (T < 0 || H < 1 || E < 1 || K < 1)
        return 0;
    const size_t slots = size_t(T) * K, ncol = (size_t(H) + kRgCols - 1) / kRgCols;
    // dz by position, counters, partial sums of each row block, all on 256-byte
    // boundaries
    return (slots + E * ncol + 1 + (slots / kRgRows + E) * H) * sizeof(float) + 4 * 256;
}

int mvllm_moe_route_grad_dev(void *stream, const void *x, int x_dtype, int64_t ldx, int T, int H,
                             const float *router, int E, int K, const int *idx,
                             const float *scores, const float *dwt, int score_fn,
                             float routed_scale, const int *nr, const int *xoff, const int *rows,
                             const int *tok_pos, int KK, void *dx, int dx_dtype, int64_t lddx,
                             float *drouter, int accumulate, void *workspace,
                             size_t workspace_bytes) {
    if ((T > 0 && (!x || !idx || !scores || !dwt || !rows || !tok_pos || (!dx && !drouter))) ||
        !router || !nr || !xoff || T < 0 || H < 1 || H > kMaxRow || E < 1 || E > 1024 || K < 1 ||
        K > 32 || KK < K || KK > kMaxSlots || ldx < 0 || (dx && lddx < H) || !row_dtype(x_dtype) ||
        (dx && !row_dtype(dx_dtype)) ||
        (score_fn != MVLLM_SCORE_SIGMOID && score_fn != MVLLM_SCORE_SQRT_SOFTPLUS) ||
        int64_t(T) * KK > kMaxGrid ||
        (int64_t(T) * K / kRgRows + E) * (H / kRgCols + 8) > kMaxGrid)
        return host_fail(MVLLM_ERR_INVALID, "route_grad_dev: invalid arguments");
    if (!workspace || workspace_bytes < mvllm_moe_route_grad_workspace(T, H, E, K))
        return host_fail(MVLLM_ERR_WORKSPACE, "route_grad_dev: workspace %zu < %zu",
                         workspace_bytes, mvllm_moe_route_grad_workspace(T, H, E, K));
    DeviceScope dev;
    if (int rc = dev.enter())
        return rc;
    if (T == 0 && !drouter)
        return MVLLM_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    RouteGradArgs a{};
    a.idx = idx, a.scores = scores, a.dwt = dwt, a.tok_pos = tok_pos, a.router = router;
    a.T = T, a.K = K, a.KK = KK, a.E = E, a.H = H, a.cap = T * K;
    a.score_fn = score_fn, a.accumulate = accumulate, a.scale = routed_scale;
    const size_t slots = size_t(T) * K;
    const int ncol = (H + kRgCols - 1) / kRgCols;
    uintptr_t at = reinterpret_cast<uintptr_t>(workspace);
    auto take = [&](size_t n) {
        at = (at + 255) & ~uintptr_t(255);
        float *p = reinterpret_cast<float *>(at);
        at += n * sizeof(float);
        return p;
    };
    if (drouter) {
        a.dzp = take(slots);
        a.arrived = reinterpret_cast<int *>(take(size_t(E) * ncol + 1));
        a.partial = take((slots / kRgRows + E) * H);
        a.counters = E * ncol + 1;
        // Long row blocks leave fewer partial sums, short ones more items to
        // share: 64 rows, doubled up to 256 while 24 items per SM remain.
        // (65536 slots evenly over 384 experts, H 7168, by 256 rows: 97 us; 32768 of 64,
        // H 2048: 28 by 64 or 128, 36 by 256; 512 rows cost uneven experts 12 us
        // more.)
        a.block = kRgRows;
        while (a.block < 256 && int64_t(slots / (2 * a.block)) * ncol >= 24 * dev.sms)
            a.block *= 2;
    }
    if (T > 0 && dx) { // dz on the way
        const int rc = dx_dtype == MVLLM_DTYPE_F32
                           ? route_dx(st, a, dev.sms, static_cast<float *>(dx), lddx)
                           : route_dx(st, a, dev.sms, static_cast<__nv_bfloat16 *>(dx), lddx);
        if (rc)
            return rc;
    } else {
        const unsigned warps = std::max(T, a.counters / 32 + 1);
        MVB_TRY(launch_serial(route_dz_kernel, dim3((warps + 7) / 8), dim3(256), 0, st, a));
    }
    if (drouter) {
        const int rc =
            x_dtype == MVLLM_DTYPE_F32
                ? route_dw(st, a, dev.sms, static_cast<const float *>(x), ldx, nr, xoff, rows,
                           drouter)
                : route_dw(st, a, dev.sms, static_cast<const __nv_bfloat16 *>(x), ldx, nr, xoff,
                           rows, drouter);
        if (rc)
            return rc;
    }
    return MVLLM_OK;
}

} // extern "C"

// matvec_q4.cu -- host entries of the few-row products with 4-bit weights.
#include "host.hpp"
#include "matvec_q4.cuh"

#include <algorithm>
#include <array>
#include <cmath>
#include <map>
#include <mutex>
#include <tuple>

using namespace mvb;

namespace {

using bf = __nv_bfloat16;

// Clusters of `ranks` CTAs that fit the device at once (one CTA per SM),
// asked once per device, kernel and shared-memory size.
int max_clusters(const void *kern, int threads, int ranks, int smem, int device, int *out) {
    static std::mutex mu;
    static std::map<std::tuple<int, const void *, int, int>, int> seen;
    std::lock_guard<std::mutex> lk(mu);
    auto key = std::make_tuple(device, kern, ranks, smem);
    auto it = seen.find(key);
    if (it == seen.end()) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(ranks);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = ranks, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        int n = 0;
        MVB_TRY(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
        it = seen.emplace(key, std::max(n, 1)).first;
    }
    *out = it->second;
    return MVLLM_OK;
}

// Passes over nb matrices for `rows` rows, rp a pass: experts' rows are taken
// to be Poisson distributed, an expert's passes being the k >= 0 with more
// than k rp rows.
double expected_passes(int rows, int nb, int rp) {
    if (nb == 1)
        return (rows + rp - 1) / rp;
    const double mean = double(rows) / nb;
    double p = std::exp(-mean), below = 0.0, passes = 0.0;
    if (p < 1e-200)
        return nb * (mean / rp + 0.5);
    for (int k = 0, n = 0; below < 0.999 && n < rows; ++k) {
        for (; n <= k * rp; ++n) // below: at most k rp rows
            below += p, p *= mean / (n + 1);
        passes += std::max(0.0, 1.0 - below);
    }
    return std::min<double>(rows, std::max(1.0, nb * passes));
}

// A plan, its launch and the rule's estimate of its time.
struct MvCut {
    MatvecPlan p{};
    int ranks = 1, grid = 1;
    double ns = 1e30;
};

template <int FMT, typename TX, int NT, bool GRAD> struct MvHost {
    using F = MvFormat<FMT>;
    static constexpr int T = MvTerms<FMT, TX, GRAD>::T, RP = 8 * NT / T;
    static constexpr int TILE = GRAD ? kMvCols : kMvRows, STEP = GRAD ? kMvRows : kMvCols;
    static constexpr int WARPS = mv_warps<NT, GRAD>(), THREADS = 32 * WARPS;
    static constexpr int RING = WARPS * mv_ring<NT, GRAD>() * F::STAGE;
    static constexpr int RED = mv_red_size<FMT, TX, NT, GRAD>() * 4; // bytes of a task's sums

    // Shared memory for `chunk` staged stages, whose rows may pass 2^31 bytes;
    // fills the plan's offsets, which hold where the answer fits the SM.
    static int64_t layout(MatvecPlan &p, int chunk, int ranks, int nb) {
        const int64_t cols = int64_t(chunk) * STEP;
        const int n = std::min(RP, p.rows_most), red = p.wo * p.wk * RED;
        int64_t at = mv_alias<GRAD>() ? std::max(RING, red) : RING;
        p.off_red = 0;
        if (!mv_alias<GRAD>())
            p.off_red = int(at), at += red;
        at = (at + 127) & ~127;
        p.off_x = int(at);
        at += n * T * mv_x_pitch<FMT, TX, GRAD>(cols);
        p.off_ex = int(at), at += GRAD ? 0 : cols / F::G * RP * 4;
        p.off_mail = int(at); // two buffers
        if (ranks > 1)
            at += 2 * ((p.wo * TILE / 32 * RP + ranks - 1) / ranks) * ranks * 128;
        p.off_list = int(at), at += (nb + 1) * 4;
        p.chunk = chunk;
        return at;
    }

    // How the work is cut.  The candidates are clusters of 1, 2, 4 or 8 CTAs
    // along the reduction, ranges of wo tiles and wk parts of each.  The rule
    // estimates each one's time: the rounds that its units need, in each the
    // stages that a CTA's warps take one after another, at the rate of its
    // share of the memory or of what its warps dequantise, and the unit's own
    // cost, with the partial sums it adds up; and the rows that are staged.
    // The constants (ns, bytes and elements per ns of a CTA) are a fit by hand to
    // times of 272 shapes of both formats and directions, 1 to 1024 rows, about 60
    // cuts of each: the answer was 3% slower than the best on average.  (Rows
    // staged at 20 elements per ns and 1500 ns a unit, first guesses, left 11%
    // and up to twice the time.)  int4's gradient, three matrix instructions a
    // product, has its own rate and unit cost from 7 shapes, 1 to 768 rows, where
    // the answer is 0 to 16% slower than the best.
    static int plan(MvCut &cut, int nb, const DeviceScope &dev) {
        MatvecPlan &p = cut.p;
        const double items = expected_passes(p.rows_most, nb, RP);
        const int tiles = (p.N + TILE - 1) / TILE, steps = (p.K + STEP - 1) / STEP;
        const double compute = // of a CTA's warps
            GRAD ? (FMT == MVLLM_FMT_INT4_G64 ? 18.0 : NT == 1 ? 25.0 : 21.0)
                 : (NT == 1 ? 42.0 : NT == 2 ? 28.0 : 17.0);
        const double fill = GRAD ? 1.05 : 0.58;        // of its warps that reach it
        const double latency = GRAD ? 1200.0 : 580.0;  // of a stage, at least
        const double staging = GRAD ? (sizeof(TX) == 4 ? 2.9 : 13.0)
                                    : (sizeof(TX) == 4 ? 4.1 : 7.8);
        const double rows_most = std::min<double>(RP, (p.rows_most + nb - 1) / nb);
        const int most = GRAD ? WARPS : 64;
        MatvecPlan q = p;
        for (int c = 1; c <= 8; c *= 2) {
            const int slice = (steps + c - 1) / c;
            if (c > 1 && slice * (c - 1) >= steps)
                break;
            int nc = dev.sms;
            if (c > 1)
                if (int rc = max_clusters(kernel(), THREADS, c, kMvSmem, dev.device, &nc))
                    return rc;
            for (int wo = 1; wo <= std::min(most, tiles); ++wo) {
                for (int wk = 1; wo * wk <= most && wk <= slice && wk <= WARPS; ++wk) {
                    q.wo = wo, q.wk = wk;
                    int chunk = slice;
                    while (chunk > 1 && layout(q, chunk, c, nb) > kMvSmem)
                        chunk = chunk > 8 ? chunk * 7 / 8 : chunk - 1;
                    if (layout(q, chunk, c, nb) > kMvSmem)
                        continue;
                    const int tasks = wo * wk, active = std::min(tasks, WARPS);
                    const int serial = (tasks + WARPS - 1) / WARPS * ((slice + wk - 1) / wk);
                    const int nr = (tiles + wo - 1) / wo;
                    const double units = items * nr, busy = std::min<double>(units, nc);
                    const double rounds = std::ceil(units / nc);
                    const double chunks = (slice + chunk - 1) / chunk;
                    const double rate = std::min(
                        compute * std::min(1.0, active / (fill * WARPS)), 6000.0 / (busy * c));
                    const double stage = std::max(active * F::STAGE / rate, latency);
                    const double sums = wo * TILE * rows_most;
                    const double unit =
                        GRAD ? (FMT == MVLLM_FMT_INT4_G64 ? 1500.0 : 750.0) +
                                   sums * (0.09 * wk * T + 0.39) + (c > 1 ? 650.0 : 0.0)
                             : 2800.0 + sums * 0.215 + (c > 1 ? 320.0 : 0.0);
                    // rows are staged once for the ranges that a cluster has of an
                    // item, or, in chunks, for every unit
                    const double rows = rows_most * slice * STEP / staging + (GRAD ? 380.0 : 120.0);
                    const double stagings =
                        chunks > 1 ? rounds : std::min(rounds, std::ceil(items / nc) + (nb > 1));
                    const double t =
                        rounds * (serial * stage + unit + (GRAD ? 6500.0 : 4000.0) * (chunks - 1)) +
                        stagings * rows;
                    if (t < cut.ns) {
                        cut.ns = t;
                        p.wo = wo, p.wk = wk, p.range = wo * TILE, p.nranges = nr;
                        p.slice = slice, p.chunk = chunk;
                        // the survey of the rows costs about as much as it
                        // saves a warp in four stages
                        p.try_common = chunks == 1 && (nb > 1 ? 1 : rounds) * serial > 4;
                        cut.ranks = c, cut.grid = int(std::ceil(busy)) * c;
                    }
                }
            }
        }
        return MVLLM_OK;
    }

    // The rule's answer by sizes: asking it takes the host 5 to 60 us, as long as
    // a small product; a new number of rows is a new size.
    static int cut_for(const MatvecPlan &p, int nb, const DeviceScope &dev, MvCut &cut) {
        static std::mutex mu;
        static std::map<std::array<int, 5>, MvCut> seen;
        static int sized = -1; // the device whose kernel may take the memory
        const std::array<int, 5> key = {dev.device, p.N, p.K, p.rows_most, nb};
        std::lock_guard<std::mutex> lk(mu);
        if (sized != dev.device) {
            MVB_TRY(cudaFuncSetAttribute(kernel(), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kMvSmem));
            sized = dev.device;
        }
        auto it = seen.find(key);
        if (it == seen.end()) {
            MvCut c{p};
            if (int rc = plan(c, nb, dev))
                return rc;
            if (seen.size() >= 4096) // a caller of ever new sizes
                seen.clear();
            it = seen.emplace(key, c).first;
        }
        cut = it->second;
        cut.p.y_f32 = p.y_f32, cut.p.x_vec = p.x_vec, cut.p.y_vec = p.y_vec;
        return MVLLM_OK;
    }
    static const void *kernel() {
        return reinterpret_cast<const void *>(matvec_q4_kernel<FMT, TX, NT, GRAD>);
    }

    // Launches a cut, or describes it in `told` (mvllm_matvec_q4_plan).
    static int launch(cudaStream_t st, const MatvecArgs &a, MvCut cut, const void *x, int64_t ldx,
                      void *y, int64_t ldy, int *told) {
        MatvecPlan &p = cut.p;
        const int ranks = cut.ranks;
        if (told) {
            const int is[8] = {RP, ranks, p.range, p.wk, p.slice, p.chunk, p.try_common, cut.grid};
            std::copy(is, is + 8, told);
            return MVLLM_OK;
        }
        const int64_t smem = layout(p, p.chunk, ranks, a.nb);
        if (p.range < 1 || smem > kMvSmem)
            return host_fail(MVLLM_ERR_UNSUPPORTED, "matvec_q4: %lld bytes of shared memory",
                             static_cast<long long>(smem));
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(cut.grid);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = size_t(smem);
        cfg.stream = st;
        cudaLaunchAttribute at[2];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        at[1].id = cudaLaunchAttributeClusterDimension;
        at[1].val.clusterDim.x = ranks, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 2;
        MVB_TRY(cudaLaunchKernelEx(&cfg, matvec_q4_kernel<FMT, TX, NT, GRAD>, a, p,
                                   static_cast<const TX *>(x), ldx, y, ldy));
        return MVLLM_OK;
    }
};

// Rows that a pass over a matrix takes: all rows of a single matrix where 8,
// 16 or 32 operand columns (gradient: 8 or 16; int4's: 8, its parts' sums need
// the registers) hold them, as many as that for more.  Experts, whose rows
// differ, take the width whose plan has the lowest estimate: 48 experts of 16
// rows on average, 7168 -> 2048, take 208 us by 16 rows a pass and 252 by 32,
// 160 experts of 20, 6144 -> 1536, 499 and 600.
template <int FMT, typename TX, bool GRAD>
int matvec_rows(cudaStream_t st, const MatvecArgs &a, const MatvecPlan &p, const DeviceScope &dev,
                const void *x, int64_t ldx, void *y, int64_t ldy, int *told) {
    constexpr int T = MvTerms<FMT, TX, GRAD>::T;
    constexpr bool NARROW = GRAD && FMT == MVLLM_FMT_INT4_G64;
    using One = MvHost<FMT, TX, 1, GRAD>;
    using Two = MvHost<FMT, TX, NARROW ? 1 : 2, GRAD>;
    using Four = MvHost<FMT, TX, NARROW ? 1 : GRAD ? 2 : 4, GRAD>;
    MvCut one, two, four;
    const bool some = a.nb > 1, wide = !GRAD && (some || a.rows > 16 / T);
    if (NARROW || some || a.rows <= 8 / T)
        if (int rc = One::cut_for(p, a.nb, dev, one))
            return rc;
    if (!NARROW && (some || (a.rows > 8 / T && !wide)))
        if (int rc = Two::cut_for(p, a.nb, dev, two))
            return rc;
    if (wide)
        if (int rc = Four::cut_for(p, a.nb, dev, four))
            return rc;
    if (one.ns <= two.ns && one.ns <= four.ns)
        return One::launch(st, a, one, x, ldx, y, ldy, told);
    if (two.ns <= four.ns)
        return Two::launch(st, a, two, x, ldx, y, ldy, told);
    return Four::launch(st, a, four, x, ldx, y, ldy, told);
}

template <int FMT, typename TX>
int matvec_way(cudaStream_t st, bool grad, const MatvecArgs &a, const MatvecPlan &p,
               const DeviceScope &dev, const void *x, int64_t ldx, void *y, int64_t ldy,
               int *told) {
    if (!grad)
        return matvec_rows<FMT, TX, false>(st, a, p, dev, x, ldx, y, ldy, told);
    return matvec_rows<FMT, TX, true>(st, a, p, dev, x, ldx, y, ldy, told);
}

int matvec_type(cudaStream_t st, bool grad, const MatvecArgs &a, const MatvecPlan &p,
                const DeviceScope &dev, const void *x, bool fx, int64_t ldx, void *y, int64_t ldy,
                int *told) {
    if (a.fmt == MVLLM_FMT_INT4_G64)
        return fx ? matvec_way<MVLLM_FMT_INT4_G64, float>(st, grad, a, p, dev, x, ldx, y, ldy, told)
                  : matvec_way<MVLLM_FMT_INT4_G64, bf>(st, grad, a, p, dev, x, ldx, y, ldy, told);
    return fx ? matvec_way<MVLLM_FMT_MXFP4, float>(st, grad, a, p, dev, x, ldx, y, ldy, told)
              : matvec_way<MVLLM_FMT_MXFP4, bf>(st, grad, a, p, dev, x, ldx, y, ldy, told);
}

bool matvec_sizes(const MatvecArgs &a, int x_dtype) {
    return (a.fmt == MVLLM_FMT_INT4_G64 || a.fmt == MVLLM_FMT_MXFP4) && a.I >= 1 && a.O >= 1 &&
           a.I <= kMvMaxSide && a.O <= kMvMaxSide && a.rows >= 0 && a.rows <= kMvMaxSide &&
           (x_dtype == MVLLM_DTYPE_F32 || x_dtype == MVLLM_DTYPE_BF16);
}

int matvec_any(const char *who, void *stream, bool grad, const MatvecArgs &a, const void *x,
               int x_dtype, int64_t ldx, void *y, int y_dtype, int64_t ldy) {
    const int out = grad ? a.I : a.O;
    if (!matvec_sizes(a, x_dtype) || (a.rows > 0 && (!x || !y)) || ldx < 0 || ldy < out ||
        (y_dtype != MVLLM_DTYPE_F32 && y_dtype != MVLLM_DTYPE_BF16))
        return host_fail(MVLLM_ERR_INVALID, "%s: invalid arguments", who);
    DeviceScope dev;
    if (int rc = dev.enter())
        return rc;
    if (a.rows == 0)
        return MVLLM_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    MatvecPlan p{};
    p.N = out, p.K = grad ? a.O : a.I;
    p.y_f32 = y_dtype == MVLLM_DTYPE_F32;
    p.rows_most = a.rows;
    const uint64_t ey = p.y_f32 ? 4 : 2;
    p.y_vec = ((reinterpret_cast<uintptr_t>(y) | (a.rows > 1 ? uint64_t(ldy) * ey : 0)) &
               (4 * ey - 1)) == 0;
    const bool fx = x_dtype == MVLLM_DTYPE_F32;
    const uint64_t pitch = a.rows > 1 ? uint64_t(ldx) * (fx ? 4 : 2) : 0;
    p.x_vec = ((reinterpret_cast<uintptr_t>(x) | pitch) & 15u) == 0;
    try { // the plans' tables allocate
        return matvec_type(st, grad, a, p, dev, x, fx, ldx, y, ldy, nullptr);
    } catch (...) {
        return host_fail(MVLLM_ERR_NOMEM, "%s: out of host memory", who);
    }
}

int matvec_one(const char *who, void *stream, bool grad, int fmt, const void *x, int x_dtype,
               int64_t ldx, const void *w, const void *s, int S, int I, int O, void *y,
               int y_dtype, int64_t ldy) {
    if (!w || !s || (fmt == MVLLM_FMT_INT4_G64 && (reinterpret_cast<uintptr_t>(s) & 3u)))
        return host_fail(MVLLM_ERR_INVALID, "%s: invalid arguments", who);
    MatvecArgs a{};
    a.fmt = fmt, a.I = I, a.O = O, a.w = w, a.s = s, a.rows = S, a.nb = 1;
    return matvec_any(who, stream, grad, a, x, x_dtype, ldx, y, y_dtype, ldy);
}

int matvec_experts(const char *who, void *stream, bool grad, int fmt, int nb, const void *x,
                   int x_dtype, int64_t ldx, int rows_cap, const int *nr, const int *xoff,
                   const void *const *wt, const void *const *st, int I, int O, void *y,
                   int y_dtype, int64_t ldy) {
    if (!wt || !st || !nr || !xoff || nb < 1 || nb > kMvMaxExperts)
        return host_fail(MVLLM_ERR_INVALID, "%s: invalid arguments", who);
    MatvecArgs a{};
    a.fmt = fmt, a.I = I, a.O = O, a.wt = wt, a.st = st, a.nr = nr, a.xoff = xoff;
    a.rows = rows_cap, a.nb = nb;
    return matvec_any(who, stream, grad, a, x, x_dtype, ldx, y, y_dtype, ldy);
}

} // namespace

extern "C" {

int mvllm_matvec_q4_plan(int fmt, int grad, int x_dtype, int nb, int rows, int I, int O,
                         int *plan) {
    MatvecArgs a{};
    a.fmt = fmt, a.I = I, a.O = O, a.rows = rows, a.nb = nb;
    if (!matvec_sizes(a, x_dtype) || rows < 1 || nb < 1 || nb > kMvMaxExperts || !plan)
        return host_fail(MVLLM_ERR_INVALID, "matvec_q4_plan: invalid arguments");
    DeviceScope dev;
    if (int rc = dev.enter())
        return rc;
    MatvecPlan p{};
    p.N = grad ? I : O, p.K = grad ? O : I, p.rows_most = rows;
    try {
        return matvec_type(nullptr, grad != 0, a, p, dev, nullptr, x_dtype == MVLLM_DTYPE_F32, 0,
                           nullptr, 0, plan);
    } catch (...) {
        return host_fail(MVLLM_ERR_NOMEM, "matvec_q4_plan: out of host memory");
    }
}

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

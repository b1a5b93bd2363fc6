"""Paths of the few-row products that only some plans or values take, on the
device."""
import pytest

torch = pytest.importorskip("torch")

import routed_cases as rc  # noqa: E402

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
INT4, MXFP4 = rc.INT4, rc.MXFP4


@pytest.mark.parametrize("fmt", [INT4, MXFP4])
def test_split_reduction_without_weights(moe, fmt):
    """Long reductions of few outputs are split over a cluster's CTAs; experts
    without a matrix have nothing to do before their sums (zeros) meet there,
    right at the start."""
    E, I, O = 6, 16384, 64
    w, s = rc.packed(torch.Generator().manual_seed(1), fmt, O, I, "cuda")
    none = torch.zeros(E, dtype=torch.int64, device="cuda")
    some, scales = none.clone(), torch.full_like(none, s.data_ptr())
    some[E - 1] = w.data_ptr()
    nr = torch.ones(E, dtype=torch.int32, device="cuda")
    xoff = torch.arange(E, dtype=torch.int32, device="cuda")
    W = rc.decode(w, s, fmt, I)
    for rows_in, rows_out, M, call in ((I, O, W.T, moe.expert_matvec_q4_dev),
                                       (O, I, W, moe.expert_matvec_q4_grad_dev)):
        x = torch.randn(E, rows_in, generator=torch.Generator().manual_seed(2)).cuda()
        first = None
        for _ in range(50):
            y = torch.full((E, rows_out), 7.0, device="cuda")
            call(fmt, x, none, scales, nr, xoff, y)
            assert (y == 0).all()
            call(fmt, x, some, scales, nr, xoff, y)
            assert (y[:-1] == 0).all()
            first = y.clone() if first is None else first
            assert torch.equal(y, first), "the sums repeat to the bit"
        want, size = x[-1].double() @ M, x[-1].double().abs() @ M.abs()
        assert ((first[-1].double() - want).abs() <= (rows_in / 16 + 64) * 2.0 ** -22 * size).all()


@pytest.mark.parametrize("fmt", [INT4, MXFP4])
@pytest.mark.parametrize("S,I,O", [(1, 7168, 2048), (3, 1000, 130), (7, 2050, 66), (16, 1536, 6144),
                                   (40, 512, 1024)])
def test_bf16_results_are_the_f32_ones_rounded(moe, S, I, O, fmt):
    """The sums do not depend on the type they are rounded to: bf16 rows give
    the same f32 sums whether these are stored or rounded once."""
    gen = torch.Generator().manual_seed(S + I + O)
    w, s = rc.packed(gen, fmt, O, I, "cuda")
    for n, m, call in ((I, O, moe.matvec_q4_dev), (O, I, moe.matvec_q4_grad_dev)):
        x = torch.randn(S, n, generator=gen).cuda().to(BF16)
        wide, narrow = torch.empty(S, m, device="cuda"), torch.empty(S, m, device="cuda").to(BF16)
        call(fmt, x, w, s, wide)
        call(fmt, x, w, s, narrow)
        assert torch.equal(narrow, wide.to(BF16))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("fmt", [INT4, MXFP4])
@pytest.mark.parametrize("n", [7168, 16384])
def test_long_sums_are_as_exact_as_f32_products(moe, n, fmt, dtype):
    """Sums over long rows, f32 results: the error in norm against 64 bits is no
    larger than that of an f32 product of the decoded weights (1.5 times, the
    spread of an error that is random)."""
    S, m = 6, 512
    gen = torch.Generator().manual_seed(n)
    x = torch.randn(S, n, generator=gen).cuda().to(dtype)
    for O, I, call in ((m, n, moe.matvec_q4_dev), (n, m, moe.matvec_q4_grad_dev)):
        w, s = rc.packed(gen, fmt, O, I, "cuda", spread=0)
        W = rc.decode(w, s, fmt, I)
        W = W.T if O == m else W
        y = torch.empty(S, m, device="cuda")
        call(fmt, x, w, s, y)
        want, plain = x.double() @ W, x.float() @ W.float()
        assert (y.double() - want).norm() <= 1.5 * (plain.double() - want).norm()


def rows_of(gen, exponents, n, dtype):
    """Rows of normal values, each times its power of two."""
    x = torch.randn(len(exponents), n, generator=gen)
    return (x * torch.exp2(torch.tensor(exponents, dtype=torch.float32))[:, None]).cuda().to(dtype)


def close(got, x, M, what):
    """Terms pass through at most length / 16 + 64 additions, each off by 2^-22
    of the magnitudes or, where they are that small, by half of f32's last step,
    2^-149; the result rounds once."""
    want, size = x.double() @ M, x.double().abs() @ M.abs()
    n = (x.shape[1] / 16 + 64) * (2.0 ** -22 * size + 2.0 ** -150)
    off = (got.double() - want).abs()
    assert (off <= n + rc.half_step(got.dtype) * (want.abs() + n)).all(), what


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("fmt", [INT4, MXFP4])
@pytest.mark.parametrize("rows,scale", [([-100, -20, 0, 2], 109), ([0, -3], 116),
                                        ([120, 100, 0, -30], -117), ([30, 31, 33], -60),
                                        ([-126, -120], 30), ([118], -126)])
@pytest.mark.parametrize("I,O", [(7168, 16384), (1024, 96)])
def test_finite_results_of_far_scales(moe, I, O, rows, scale, fmt, dtype):
    """Rows and scales at the two ends of f32's range whose results lie inside
    it: the sums on the way stay finite too, in a product whose rows are
    surveyed and in a short one."""
    gen = torch.Generator().manual_seed(I + scale)
    w, s = rc.packed(gen, fmt, O, I, "cuda", spread=0)
    if fmt == INT4:
        s = s * 2.0 ** 6 * 2.0 ** scale if scale < 120 else s
    else:
        s.fill_(127 + scale)
    x = rows_of(gen, rows, I, dtype)
    y = torch.empty(len(rows), O, device="cuda")
    moe.matvec_q4_dev(fmt, x, w, s, y)
    W = rc.decode(w, s, fmt, I)
    want = x.double() @ W.T
    live = want.abs() < 3e38
    assert live.float().mean() > 0.9 and torch.isfinite(y[live]).all()
    close(torch.where(live, y.double(), want), x, W.T, "forward")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("fmt", [INT4, MXFP4])
@pytest.mark.parametrize("I,O", [(7168, 16384), (192, 40)])
def test_group_sums_beyond_f32(moe, I, O, fmt, dtype):
    """Rows whose products with the codes leave f32's range before the scale
    brings them back, beside rows that a factor in two steps must not lose."""
    gen = torch.Generator().manual_seed(I)
    w, s = rc.packed(gen, fmt, O, I, "cuda", spread=0)
    w.fill_(0x77 if fmt == MXFP4 else 0xFF)  # every weight 6, or 7
    if fmt == INT4:
        s.fill_(2.0 ** -118)
    else:
        s.fill_(9)
    x = torch.ones(4, I)
    x[0] *= 2.0 ** 127
    x[1] *= -(2.0 ** 126)
    x[1, 64:] = 2.0 ** -100  # one group apart from the others
    x[2] = torch.randn(I, generator=gen)
    x[3] = 2.0 ** 90
    x = x.cuda().to(dtype)
    y = torch.empty(4, O, device="cuda")
    moe.matvec_q4_dev(fmt, x, w, s, y)
    assert torch.isfinite(y).all()
    close(y, x, rc.decode(w, s, fmt, I).T, "forward")


@pytest.mark.parametrize("fmt", [INT4, MXFP4])
def test_reductions_past_the_address_arithmetic(moe, fmt):
    """Rows whose staged form would pass 2^31 bytes: they are staged in chunks."""
    n, m, S = (1 << 25) + 40, 6, 32
    g = torch.Generator(device="cuda").manual_seed(3)
    for O, I, call in ((m, n, moe.matvec_q4_dev), (n, m, moe.matvec_q4_grad_dev)):
        w = torch.randint(0, 256, (O, (I + 1) // 2), generator=g, dtype=torch.uint8, device="cuda")
        if fmt == INT4:
            s = torch.rand(O, (I + 63) // 64, generator=g, device="cuda") * 0.01 + 1e-4
        else:
            s = torch.randint(113, 126, (O, (I + 31) // 32), generator=g, dtype=torch.uint8,
                              device="cuda")
        W = rc.decode(w, s, fmt, I)
        x = torch.randn(S, n, generator=g, device="cuda").to(BF16)
        y = torch.empty(S, m, device="cuda")
        call(fmt, x, w, s, y)
        close(y, x, W.T if O == m else W, f"outputs {O}")
        del W, x


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradient_products_beyond_f32_meet_zero_weights(moe, dtype):
    """Finite rows and int4 scales whose product passes f32's range: infinite in
    the columns that have weights, 0 where all weights are 0."""
    S, I, O = 3, 320, 64
    code = torch.arange(I) % 16
    w = (code[0::2] | (code[1::2] << 4)).to(torch.uint8).expand(O, -1).contiguous().cuda()
    s = torch.full((O, I // 64), 2.0 ** 100, device="cuda")
    dy = torch.ones(S, O) * 2.0 ** -110
    dy[1] = 2.0 ** 60
    dy[2, 1:] = 0  # one product alone
    dy[2, 0] = -(2.0 ** 28)
    dx = torch.empty(S, I, device="cuda")
    moe.matvec_q4_grad_dev(INT4, dy.cuda().to(dtype), w, s, dx)
    sign = (code - 8).sign().float().cuda()
    inf = torch.where(sign == 0, torch.zeros_like(sign), sign * float("inf"))
    assert torch.equal(dx[1], inf) and torch.equal(dx[2], -inf)
    assert torch.equal(dx[0], (code - 8).cuda() * (O * 2.0 ** -10))


def exact_as_f32(got, x, M, what):
    """No further off in norm, row by row, than an f32 product of the decoded
    weights (1.5 times) or one rounding of the result."""
    want, plain = x.double() @ M, x.float() @ M.float()
    off, most = (got.double() - want).norm(dim=1), 1.5 * (plain.double() - want).norm(dim=1)
    assert (off <= most + 2.0 ** -24 * want.norm(dim=1)).all(), what


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("fmt", [INT4, MXFP4])
@pytest.mark.parametrize("S,n,m", [(8, 7168, 512), (40, 16384, 512), (3, 65536, 256)])
def test_sums_of_far_magnitudes(moe, S, n, m, fmt, dtype):
    """Rows and scales over 24 binades: no bits of a sum are cut off on the way."""
    gen = torch.Generator().manual_seed(n)
    x = torch.randn(S, n, generator=gen) * torch.exp2(
        torch.randint(-6, 7, (S, n), generator=gen).float())
    x = x.cuda().to(dtype)
    for O, I, call in ((m, n, moe.matvec_q4_dev), (n, m, moe.matvec_q4_grad_dev)):
        w, s = rc.packed(gen, fmt, O, I, "cuda", spread=6)
        W = rc.decode(w, s, fmt, I)
        y = torch.empty(S, m, device="cuda")
        call(fmt, x, w, s, y)
        exact_as_f32(y, x, W.T if O == m else W, f"outputs {O}")


def product(moe, fmt, x, y, w, s, grad):
    (moe.matvec_q4_grad_dev if grad else moe.matvec_q4_dev)(fmt, x, w, s, y)


def plan_of(moe, fmt, dtype, S, I, O, nb=1, grad=False):
    return moe.matvec_q4_plan(fmt, moe.DTYPE_F32 if dtype == F32 else moe.DTYPE_BF16, S, I, O, nb,
                              grad)


# Type, rows, sizes, and the rows of a pass of a plan that surveys the rows.
SURVEYED = [(BF16, 1, 7168, 16384, 8), (BF16, 12, 7168, 16384, 16), (BF16, 32, 1024, 65536, 32),
            (F32, 4, 7168, 16384, 4), (F32, 8, 7168, 16384, 8), (F32, 12, 7168, 16384, 16),
            (F32, 32, 1024, 65536, 16)]


@pytest.mark.parametrize("fmt", [INT4, MXFP4])
@pytest.mark.parametrize("dtype,S,I,O,rows", SURVEYED)
def test_surveyed_rows(moe, dtype, S, I, O, rows, fmt):
    """A plan that gives a row one scale where the row's range allows it: rows
    that fit, one that does not, rows of zeros, and rows that are not finite."""
    plan = plan_of(moe, fmt, dtype, S, I, O)
    assert plan["surveyed"] and plan["rows"] == rows and plan["held"] == plan["stages"]
    gen = torch.Generator().manual_seed(S + I)
    w, s = rc.packed(gen, fmt, O, I, "cuda", spread=1)
    M = rc.decode(w, s, fmt, I).T
    x = torch.randn(S, I, generator=gen).cuda()
    y = torch.empty(S, O, device="cuda")
    for kind in ("fits", "zeros", "does not", "not finite"):
        z = x.clone()
        if kind != "fits":
            z[:, 64:192] = 0  # whole groups
            z[S // 2] = z[S // 2] if S == 1 else 0
        if kind == "does not":
            z[S - 1, 256:320] *= 2.0 ** -14
        z = z.to(dtype)
        if kind == "not finite":
            z[S - 1, 300] = float("inf")
            z[0, 301] = float("nan")
        moe.matvec_q4_dev(fmt, z, w, s, y)
        if kind != "not finite":
            exact_as_f32(y, z, M, kind)
        else:
            assert torch.isnan(y[0]).all()
            want = z.double() @ M
            if S > 1:
                exact_as_f32(y[1:-1], z[1:-1], M, kind)
                assert torch.equal(torch.isnan(y[-1]), torch.isnan(want[-1]))
                live = ~torch.isnan(want[-1])
                assert torch.equal(y[-1][live].double(), want[-1][live])


# Type, rows, sizes and direction whose plan stages the rows in chunks.
CHUNKED = [(BF16, 32, 16384, 4096, False), (BF16, 64, 16384, 4096, False),
           (F32, 16, 7168, 16384, False), (F32, 64, 16384, 4096, False),
           (BF16, 32, 1536, 32768, True), (F32, 32, 512, 65536, True),
           (BF16, 12, 4096, 16384, True)]


@pytest.mark.parametrize("fmt", [INT4, MXFP4])
@pytest.mark.parametrize("dtype,S,I,O,grad", CHUNKED)
def test_rows_in_chunks(moe, dtype, S, I, O, grad, fmt):
    if fmt == INT4 or not grad:
        plan = plan_of(moe, fmt, dtype, S, I, O, grad=grad)
        assert plan["held"] < plan["stages"]
    gen = torch.Generator().manual_seed(S + I)
    w, s = rc.packed(gen, fmt, O, I, "cuda", spread=1)
    W = rc.decode(w, s, fmt, I)
    n, m, M = (O, I, W) if grad else (I, O, W.T)
    x = torch.randn(S, n, generator=gen)
    x[:, ::7] *= 2.0 ** 9
    x[1] = 0
    x = x.cuda().to(dtype)
    y = torch.empty(S, m, device="cuda")
    product(moe, fmt, x, y, w, s, grad)
    exact_as_f32(y, x, M, "chunks")


@pytest.mark.parametrize("fmt", [INT4, MXFP4])
@pytest.mark.parametrize("dtype,S", [(BF16, 64), (BF16, 200), (F32, 64), (F32, 200)])
def test_many_experts_rows(moe, dtype, S, fmt):
    """Uneven segments of 16 experts, forward and gradient."""
    E, I, O = 16, 7168, 2048
    gen = torch.Generator().manual_seed(S)
    w, s = rc.packed(gen, fmt, E * O, I, "cuda", spread=1)
    tab, sct = (torch.tensor([t[e * O].data_ptr() for e in range(E)], device="cuda")
                for t in (w, s))
    nr = torch.bincount(torch.randint(0, E, (S,), generator=gen), minlength=E)
    nr[3], nr[5] = nr[3] + nr[5], 0
    xoff = (torch.cumsum(nr, 0) - nr).tolist()
    n32, o32 = nr.int().cuda(), torch.tensor(xoff, dtype=torch.int32, device="cuda")
    for n, m, call in ((I, O, moe.expert_matvec_q4_dev), (O, I, moe.expert_matvec_q4_grad_dev)):
        x = torch.randn(S, n, generator=gen).cuda().to(dtype)
        y = torch.full((S, m), 7.0, device="cuda")
        call(fmt, x, tab, sct, n32, o32, y)
        for e in range(E):
            part = slice(xoff[e], xoff[e] + int(nr[e]))
            W = rc.decode(w[e * O:(e + 1) * O], s[e * O:(e + 1) * O], fmt, I)
            if int(nr[e]):
                exact_as_f32(y[part], x[part], W.T if m == O else W, f"expert {e}")


@pytest.mark.parametrize("dtype,below", [(F32, 24), (BF16, 18)])
@pytest.mark.parametrize("fmt", [INT4, MXFP4])
@pytest.mark.parametrize("S,I,O", [(1, 32, 40), (5, 1000, 96), (4, 7168, 16384), (40, 512, 96)])
def test_small_values_beside_an_outlier(moe, S, I, O, fmt, dtype, below):
    """In every scale group one value that its weights, all 0, leave out, and the
    others far below it: these keep their bits."""
    gen = torch.Generator().manual_seed(I)
    w, s = rc.packed(gen, fmt, O, I, "cuda", spread=0)
    x = torch.randn(S, I, generator=gen) * 2.0 ** -below
    x[:, ::32] = 1.0
    at = torch.arange(0, (I + 1) // 2, 16, device="cuda")  # the bytes of columns 0, 32, ..
    w[:, at] = (w[:, at] & 0xF0) | (8 if fmt == INT4 else 0)
    x = x.cuda().to(dtype)
    y = torch.empty(S, O, device="cuda")
    moe.matvec_q4_dev(fmt, x, w, s, y)
    close(y, x, rc.decode(w, s, fmt, I).T, "forward")
    exact = x.double() @ rc.decode(w, s, fmt, I).T
    # 22 bits of each value: random, and below 2^-20 of a sum's norm
    assert (y.double() - exact).norm() <= 2.0 ** -20 * exact.norm()

"""Few-row products with 4-bit weights on the device against 64-bit forms.

Tolerance: a term passes through at most (length / 16 + 64) f32 additions,
each (in the tensor cores too) off by at most 2^-22 of the magnitudes summed;
rows of f32 are split into parts whose remainder is below 2^-22; the result
rounds once to the output's type.
"""
import pytest

torch = pytest.importorskip("torch")

import routed_cases as rc  # noqa: E402

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
INT4, MXFP4 = rc.INT4, rc.MXFP4


def bound(length, size, want, out_type):
    n = (length / 16 + 64) * 2.0 ** -22 * size
    return n + rc.half_step(out_type) * (want.abs() + n)


def check(got, x, W, length, what):
    """got = x W^T, W [outputs, inputs] f64."""
    want, size = x.double() @ W.T, x.double().abs() @ W.T.abs()
    off, most = (got.double() - want).abs(), bound(length, size, want, got.dtype)
    if not got.numel():
        return
    bad = ~(off <= most)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{(off / most.clamp_min(1e-300)).max():.2f} of the bound, first at "
                           f"{torch.nonzero(bad)[0].tolist()}")


SHAPES = [(1, 1, 1), (1, 64, 32), (1, 7168, 2048), (2, 33, 7), (3, 1000, 130), (4, 512, 96),
          (5, 2050, 66), (7, 65, 129), (8, 6144, 1536), (9, 128, 1000), (16, 1024, 512),
          (17, 4096, 48), (33, 320, 320), (64, 7168, 272), (1, 16384, 40), (6, 31, 4100)]


@pytest.mark.parametrize("dtype,out_type", [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("fmt", [INT4, MXFP4])
@pytest.mark.parametrize("S,I,O", SHAPES)
def test_matvec_and_gradient(moe, S, I, O, fmt, dtype, out_type):
    gen = torch.Generator().manual_seed(S * 7 + I * 3 + O)
    w, s = rc.packed(gen, fmt, O, I, "cuda")
    W = rc.decode(w, s, fmt, I)
    x = torch.randn(S, I, generator=gen).cuda().to(dtype)
    y = torch.full((S, O), 7.0, dtype=out_type, device="cuda")
    moe.matvec_q4_dev(fmt, x, w, s, y)
    check(y, x, W, I, "forward")
    dy = torch.randn(S, O, generator=gen).cuda().to(dtype)
    dx = torch.full((S, I), 7.0, dtype=out_type, device="cuda")
    moe.matvec_q4_grad_dev(fmt, dy, w, s, dx)
    check(dx, dy, W.T, O, "gradient")
    # the adjoint's identity <dy, W x> = <W^T dy, x>, a difference quotient of
    # a linear map, on the device's own outputs
    if out_type == F32:
        a = (dy.double() * y.double()).sum()
        b = (dx.double() * x.double()).sum()
        size = (dy.double().abs() @ W.abs() * x.double().abs()).sum()
        assert abs(a - b) <= (I / 16 + O / 16 + 130) * 2.0 ** -22 * size


@pytest.mark.parametrize("fmt", [INT4, MXFP4])
def test_wide_ranges(moe, fmt):
    """Rows and scales over many magnitudes, zeros among them: small values
    beside large ones keep the precision that the sums' size allows."""
    S, I, O = 5, 1024, 128
    gen = torch.Generator().manual_seed(3)
    w, s = rc.packed(gen, fmt, O, I, "cuda", spread=30)
    if fmt == MXFP4:
        s[::7, ::3] = 0  # code 0 decodes to 0
    else:
        s[::7, ::3] = 0.0
    W = rc.decode(w, s, fmt, I)
    for dtype in (F32, BF16):
        for power in (-60, -20, 0, 20, 50):
            x = torch.randn(S, I, generator=gen) * torch.exp2(
                torch.randint(-12, 13, (S, I), generator=gen).float())
            x[1], x[:, ::5] = 0, 0
            x = (x * 2.0 ** power).cuda().to(dtype)
            y = torch.empty(S, O, device="cuda")
            moe.matvec_q4_dev(fmt, x, w, s, y)
            check(y, x, W, I, f"forward 2^{power}")
            dy = x[:, :O].contiguous()
            dx = torch.empty(S, I, device="cuda")
            moe.matvec_q4_grad_dev(fmt, dy, w, s, dx)
            check(dx, dy, W.T, O, f"gradient 2^{power}")


@pytest.mark.parametrize("fmt", [INT4, MXFP4])
def test_non_finite_rows(moe, fmt):
    """A row's NaN or infinity makes that row NaN or infinite where its weight
    meets it, and leaves the other rows alone."""
    S, I, O = 4, 256, 64
    gen = torch.Generator().manual_seed(5)
    w, s = rc.packed(gen, fmt, O, I, "cuda")
    W = rc.decode(w, s, fmt, I)
    for dtype in (F32, BF16):
        x = torch.randn(S, I, generator=gen).cuda().to(dtype)
        x[1, 17], x[2, 100], x[3, 200] = float("nan"), float("inf"), float("-inf")
        y, dx = torch.empty(S, O, device="cuda"), torch.empty(S, I, device="cuda")
        moe.matvec_q4_dev(fmt, x, w, s, y)
        check(y[:1], x[:1], W, I, "the finite row")
        assert torch.isnan(y[1]).all()
        want = x.double() @ W.T
        for r in (2, 3):
            assert torch.equal(torch.isnan(y[r]), torch.isnan(want[r]))
            live = ~torch.isnan(want[r])
            assert torch.equal(y[r][live].double(), want[r][live])
        dy = x[:, :O].contiguous()
        dy[2, 40], dy[3, 3] = float("inf"), float("-inf")
        moe.matvec_q4_grad_dev(fmt, dy, w, s, dx)
        check(dx[:1], dy[:1], W.T, O, "the finite row")
        want = dy.double() @ W
        for r in (1, 2, 3):
            assert torch.equal(torch.isnan(dx[r]), torch.isnan(want[r]))
            live = torch.isinf(want[r])
            assert torch.equal(dx[r][live].double(), want[r][live])


def experts(gen, fmt, E, O, I, offset=0):
    """Packed experts in one buffer each, starting `offset` bytes in."""
    keep, ws, ss = [], [], []
    for _ in range(E):
        w, s = rc.packed(gen, fmt, O, I, "cuda")
        raw = torch.empty(w.numel() + offset + 16, dtype=torch.uint8, device="cuda")
        part = raw[offset:offset + w.numel()].view(w.shape)
        part.copy_(w)
        keep.append((raw, part, s))
        ws.append(part.data_ptr())
        ss.append(s.data_ptr())
    i64 = dict(dtype=torch.int64, device="cuda")
    return keep, torch.tensor(ws, **i64), torch.tensor(ss, **i64)


@pytest.mark.parametrize("offset", [0, 4, 1])
@pytest.mark.parametrize("dtype,out_type", [(F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("fmt", [INT4, MXFP4])
@pytest.mark.parametrize("I,O,nr", [(64, 32, [3]), (512, 256, [0, 1, 0, 9, 2]),
                                    (330, 77, [5, 0, 20, 1]), (1024, 640, [1] * 20 + [40, 0, 8])])
def test_expert_rows(moe, I, O, nr, fmt, dtype, out_type, offset):
    gen = torch.Generator().manual_seed(I + O + len(nr))
    E, R = len(nr), sum(nr)
    keep, wt, st = experts(gen, fmt, E, O, I, offset)
    null = 1 if E > 1 else None  # an expert without weights has rows of zeros
    if null is not None:
        wt[null] = 0
    n = torch.tensor(nr, dtype=torch.int32, device="cuda")
    xoff = (torch.cumsum(n, 0) - n).int()
    cap = R + 3
    for rows_in, rows_out, call in ((I, O, moe.expert_matvec_q4_dev),
                                    (O, I, moe.expert_matvec_q4_grad_dev)):
        x = torch.randn(cap, rows_in, generator=gen).cuda().to(dtype)
        y = torch.full((cap, rows_out), 7.0, dtype=out_type, device="cuda")
        call(fmt, x, wt, st, n, xoff, y)
        assert (y[R:] == 7).all(), "rows behind the last segment are left alone"
        at = 0
        for e in range(E):
            W = rc.decode(keep[e][1], keep[e][2], fmt, I)
            W = 0 * W if e == null else W
            check(y[at:at + nr[e]], x[at:at + nr[e]], W if rows_out == O else W.T, rows_in,
                  f"expert {e}")
            at += nr[e]
        # a batch of rows beyond the buffer is clipped to it
        short = torch.full((max(1, R - 2), rows_out), 7.0, dtype=out_type, device="cuda")
        call(fmt, x[:short.shape[0]], wt, st, n, xoff, short)
        at = 0
        for e in range(E):
            W = rc.decode(keep[e][1], keep[e][2], fmt, I)
            W = 0 * W if e == null else W
            end = min(at + nr[e], short.shape[0])
            check(short[at:end], x[at:end], W if rows_out == O else W.T, rows_in, f"cut {e}")
            at = end


@pytest.mark.parametrize("fmt", [INT4, MXFP4])
def test_pitched_rows_and_views(moe, fmt):
    S, I, O = 6, 320, 96
    gen = torch.Generator().manual_seed(11)
    w, s = rc.packed(gen, fmt, O, I, "cuda")
    W = rc.decode(w, s, fmt, I)
    for dtype in (F32, BF16):
        for shift in (0, 1, 8):
            x = torch.randn(S, I + 24, generator=gen).cuda().to(dtype)[:, shift:shift + I]
            big = torch.full((S, O + 9), 7.0, dtype=dtype, device="cuda")
            y = big[:, shift:shift + O]
            moe.matvec_q4_dev(fmt, x, w, s, y)
            check(y, x, W, I, "forward")
            assert (big[:, :shift] == 7).all() and (big[:, shift + O:] == 7).all()
            dy = torch.randn(S, O + 24, generator=gen).cuda().to(dtype)[:, shift:shift + O]
            big = torch.full((S, I + 9), 7.0, dtype=dtype, device="cuda")
            dx = big[:, shift:shift + I]
            moe.matvec_q4_grad_dev(fmt, dy, w, s, dx)
            check(dx, dy, W.T, O, "gradient")
            assert (big[:, :shift] == 7).all() and (big[:, shift + I:] == 7).all()
        # one row for every output row
        row = torch.randn(1, I, generator=gen).cuda().to(dtype).expand(S, I)
        y = torch.empty(S, O, device="cuda")
        moe.matvec_q4_dev(fmt, row, w, s, y)
        check(y, row, W, I, "broadcast")


@pytest.mark.parametrize("fmt", [INT4, MXFP4])
def test_repeat_stream_and_graph(moe, fmt):
    S, I, O = 8, 2048, 768
    gen = torch.Generator().manual_seed(13)
    w, s = rc.packed(gen, fmt, O, I, "cuda")
    x, dy = torch.randn(S, I, generator=gen).cuda(), torch.randn(S, O, generator=gen).cuda()

    def step(o):
        moe.matvec_q4_dev(fmt, x, w, s, o[0])
        moe.matvec_q4_grad_dev(fmt, dy, w, s, o[1])

    outs = [[torch.zeros(S, O, device="cuda"), torch.zeros(S, I, device="cuda")] for _ in range(3)]
    step(outs[0])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(outs[1])
        graph = torch.cuda.CUDAGraph()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            step(outs[2])
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(*outs):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_no_rows(moe):
    w, s = rc.packed(torch.Generator().manual_seed(1), INT4, 32, 64, "cuda")
    moe.matvec_q4_dev(INT4, torch.zeros(0, 64, device="cuda"), w, s,
                      torch.zeros(0, 32, device="cuda"))
    moe.matvec_q4_grad_dev(INT4, torch.zeros(0, 32, device="cuda"), w, s,
                           torch.zeros(0, 64, device="cuda"))


def test_agrees_with_the_serial_product(moe):
    """The same matrix and rows through matmul_dev, the library's serial form."""
    S, I, O = 4, 1024, 160
    gen = torch.Generator().manual_seed(17)
    for fmt in (INT4, MXFP4):
        w, s = rc.packed(gen, fmt, O, I, "cuda")
        x = torch.randn(S, I, generator=gen).cuda()
        a, b = torch.empty(S, O, device="cuda"), torch.empty(S, O, device="cuda")
        moe.matvec_q4_dev(fmt, x, w, s, a)
        moe.matmul_dev(fmt, b, x, w, s)
        W = rc.decode(w, s, fmt, I)
        size = x.double().abs() @ W.T.abs()
        assert ((a - b).double().abs() <= (I / 16 + 64 + I * 0.5) * 2.0 ** -22 * size).all()


@pytest.mark.parametrize("fmt", [INT4, MXFP4])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_f32_results_keep_f32_precision(moe, fmt, dtype):
    """With f32 results the parts of an element keep at least 22 bits (one
    exact part for bf16 where the scale is a power of two): every term is off
    by at most 2^-22, the sums' roundings by about as much, and random errors
    add up to less in norm: 2^-20 of the result's."""
    S, I, O = 6, 2048, 640
    gen = torch.Generator().manual_seed(23)
    w, s = rc.packed(gen, fmt, O, I, "cuda", spread=2)
    W = rc.decode(w, s, fmt, I)
    x, dy = (torch.randn(S, n, generator=gen).cuda().to(dtype) for n in (I, O))
    y, dx = torch.empty(S, O, device="cuda"), torch.empty(S, I, device="cuda")
    moe.matvec_q4_dev(fmt, x, w, s, y)
    moe.matvec_q4_grad_dev(fmt, dy, w, s, dx)
    for got, want in ((y, x.double() @ W.T), (dx, dy.double() @ W)):
        assert (got.double() - want).norm() <= 2.0 ** -20 * want.norm()


@pytest.mark.parametrize("fmt", [INT4, MXFP4])
def test_products_beyond_f32(moe, fmt):
    """Finite rows and scales whose product passes f32's range: infinities of
    the right sign, not NaN, and the other rows as ever."""
    S, I, O = 3, 320, 128
    gen = torch.Generator().manual_seed(29)
    w, s = rc.packed(gen, fmt, O, I, "cuda", spread=0)
    w.fill_(0x77 if fmt == MXFP4 else 0xFF)  # every weight 6, or 7
    if fmt == INT4:
        s.fill_(2.0 ** 100)
    else:
        s.fill_(227)
    W = rc.decode(w, s, fmt, I)
    for dtype in (F32, BF16):
        dy = torch.ones(S, O, device="cuda", dtype=dtype) * 2.0 ** -110
        dy[1] = 2.0 ** 60
        dx = torch.empty(S, I, device="cuda")
        moe.matvec_q4_grad_dev(fmt, dy, w, s, dx)
        assert torch.isposinf(dx[1]).all()
        check(dx[[0, 2]], dy[[0, 2]], W.T, O, "gradient")
        x = torch.ones(S, I, device="cuda", dtype=dtype) * 2.0 ** -110
        x[1] = -2.0 ** 60
        y = torch.empty(S, O, device="cuda")
        moe.matvec_q4_dev(fmt, x, w, s, y)
        assert torch.isneginf(y[1]).all()
        check(y[[0, 2]], x[[0, 2]], W, I, "forward")

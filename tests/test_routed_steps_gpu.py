"""Dispatch, combine and router gradients on the device against 64-bit forms.

Tolerances, from the roundings alone (u = 2^-24, r = the output type's half
step): a sum of n f32 terms is off by at most n u times the sum of the terms'
magnitudes, and its rounding to the output by r times its value.  A dot
product over D columns is at least 32 interleaved partial sums, so no term
passes through more than D / 32 + 48 additions.
"""
import pytest

torch = pytest.importorskip("torch")

import routed_cases as rc  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def bits(t):
    return t.contiguous().view(torch.int32 if t.dtype == F32 else torch.int16)


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} values off, worst "
                           f"{(off / bound.clamp_min(1e-300)).max():.2f} of the bound")


def case(moe, T, K, E, ns=0, repeats=False, dropped=0.2):
    gen = torch.Generator().manual_seed(T * 131 + K * 17 + E + ns)
    idx, wt = rc.routing(gen, T, K, E, dropped, repeats)
    idx, wt = idx.cuda(), wt.cuda()
    plan = rc.device_plan(moe, idx, wt, E, ns)
    g = torch.Generator(device="cuda").manual_seed(T + K)
    return idx, wt, plan, g, int(plan["n_rows"].item())


def matrix(g, rows, D, dtype, extra=0, shift=0):
    """A row matrix inside a wider one: pitch D + extra, starting `shift` in."""
    big = torch.randn(rows, D + extra + shift, generator=g, device="cuda").to(dtype)
    return big[:, shift:shift + D]


SHAPES = [(1, 1, 1, 1, 0), (1, 8, 256, 7168, 0), (3, 2, 4, 64, 0), (5, 3, 7, 1, 0),
          (37, 6, 160, 2051, 0), (64, 8, 16, 250, 1), (130, 4, 64, 1000, 1), (300, 8, 384, 96, 0),
          (9, 32, 40, 520, 1), (2000, 2, 8, 36, 0)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,K,E,D,ns", SHAPES)
def test_dispatch(moe, T, K, E, D, ns, dtype):
    idx, wt, plan, g, R = case(moe, T, K, E, ns)
    x = matrix(g, T, D, dtype)
    xs = matrix(g, T * (K + ns) + 3, D, dtype)
    before = xs.clone()
    moe.dispatch_dev(x, plan["tok_pos"], xs)
    assert torch.equal(bits(xs[:R]), bits(x[plan["rows"][:R].long()]))
    assert torch.equal(bits(xs[R:]), bits(before[R:])), "rows behind the last are left alone"


@pytest.mark.parametrize("out_type", [F32, BF16])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,K,E,D,ns", SHAPES)
def test_combine_and_dispatch_gradient(moe, T, K, E, D, ns, dtype, out_type):
    idx, wt, plan, g, R = case(moe, T, K, E, ns, repeats=True)
    y = matrix(g, T * (K + ns), D, dtype)
    y[R:] = float("nan")  # rows no position names are not read into anything
    n = K + ns + 2
    for rw in (plan["rw"], None):
        for accumulate in (False, True):
            out = matrix(g, T, D, out_type)
            first = out.double() if accumulate else torch.zeros(T, D, dtype=torch.float64).cuda()
            if rw is None:
                moe.dispatch_grad_dev(y, plan["tok_pos"], out, accumulate)
            else:
                moe.combine_dev(y, rw, plan["tok_pos"], out, accumulate)
            want, size = rc.combine(y[:R], rw, plan, T)
            want, size = want + first, size + first.abs()
            within(out, want, n * U * size + rc.half_step(out_type) * (want.abs() + n * U * size),
                   f"rw={rw is not None} accumulate={accumulate}")


@pytest.mark.parametrize("dtype,grad_type", [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("T,K,E,D,ns", SHAPES)
def test_combine_gradient(moe, T, K, E, D, ns, dtype, grad_type):
    idx, wt, plan, g, R = case(moe, T, K, E, ns, repeats=True)
    y, dout = matrix(g, T * (K + ns), D, dtype), matrix(g, T, D, grad_type)
    dy, dwt = matrix(g, T * (K + ns), D, dtype), torch.full((T, K), 7.0, device="cuda")
    before = dy.clone()
    moe.combine_grad_dev(dout, y, plan["rw"], plan["tok_pos"], idx, dy, dwt)
    seen = dout.double()[plan["rows"][:R].long()]
    want = seen * plan["rw"][:R, None].double()
    within(dy[:R], want, (U + rc.half_step(dtype)) * 1.01 * want.abs() + 1e-40, "dy")
    assert torch.equal(bits(dy[R:]), bits(before[R:]))
    dots, size = (seen * y[:R].double()).sum(1), (seen * y[:R].double()).abs().sum(1)
    want = torch.zeros(T, K, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    at = plan["tok_pos"].long()
    for k in range(K):
        for j in range(k, -1, -1):  # the first slot with the same id
            same = (idx[:, j] == idx[:, k]) & (at[:, j] >= 0)
            want[same, k], bound[same, k] = dots[at[same, j]], size[at[same, j]]
    within(dwt, want, (D / 32 + 48) * U * bound, "dwt")


ROUTER = [(1, 16, 2, 1), (1, 1024, 16, 4), (33, 7168, 256, 8), (64, 1024, 16, 4), (50, 37, 5, 3),
          (700, 250, 384, 8), (3000, 64, 2, 2), (257, 130, 1024, 32)]


@pytest.mark.parametrize("score_fn", [0, 1])
@pytest.mark.parametrize("dtype,dx_type", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("T,H,E,K", ROUTER)
def test_router_gradient(moe, T, H, E, K, dtype, dx_type, score_fn):
    g = torch.Generator(device="cuda").manual_seed(T + H + E)
    x = matrix(g, T, H, dtype)
    router = torch.randn(E, H, generator=g, device="cuda") / H ** 0.5
    idx = torch.empty(T, K, dtype=torch.int32, device="cuda")
    wt, dwt = torch.empty(T, K, device="cuda"), torch.randn(T, K, generator=g, device="cuda")
    scores, choice = (torch.empty(T, E, device="cuda") for _ in range(2))
    bias = torch.randn(E, generator=g, device="cuda") * 0.1
    scale = 2.5
    moe.route_ex_dev(x.contiguous(), router, bias, K, idx, wt, scores, choice, score_fn, scale)
    off = torch.rand(T, generator=g, device="cuda") < 0.2  # padding: no id at all
    idx[off], wt[off] = -1, 0
    plan = rc.device_plan(moe, idx, wt, E)
    args = (x, router, idx, scores, dwt, plan["nr"], plan["xoff"], plan["rows"], plan["tok_pos"])
    want_x, want_r, _ = rc.route_grad(x, router, idx, scores, dwt, score_fn, scale)
    size_x, size_r = rc.route_grad_bounds(x, router, idx, scores, dwt, score_fn, scale)
    # dz: sums of K terms, two divisions, the slope (expm1 within 2 ulp) and
    # four products: (2 K + 16) roundings of magnitudes that size_* carries.
    n = 2 * K + 16
    for accumulate in (False, True):
        dx, dr = matrix(g, T, H, dx_type), torch.randn(E, H, generator=g, device="cuda")
        fx, fr = (dx.double(), dr.double()) if accumulate else (0 * dx.double(), 0 * dr.double())
        moe.route_grad_dev(*args, dx, dr, score_fn=score_fn, routed_scale=scale,
                           accumulate=accumulate)
        wx, bx = want_x + fx, (n + K + 1) * U * (size_x + fx.abs())
        within(dx, wx, bx + rc.half_step(dx_type) * (wx.abs() + bx), f"dx {accumulate}")
        longest = int(plan["nr"].max())  # rows of the longest segment
        within(dr, want_r + fr, (n + longest + 1) * U * (size_r + fr.abs()), f"drouter {accumulate}")
    # either output alone
    one, two = torch.empty_like(dx), torch.empty_like(dr)
    moe.route_grad_dev(*args, one, None, score_fn=score_fn, routed_scale=scale)
    moe.route_grad_dev(*args, None, two, score_fn=score_fn, routed_scale=scale)
    both = torch.empty_like(dx), torch.empty_like(dr)
    moe.route_grad_dev(*args, *both, score_fn=score_fn, routed_scale=scale)
    assert torch.equal(bits(one), bits(both[0])) and torch.equal(bits(two), bits(both[1]))


@pytest.mark.parametrize("extra,shift", [(8, 0), (3, 0), (0, 1), (5, 2)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pitches_and_alignments(moe, dtype, extra, shift):
    T, K, E, D = 41, 4, 12, 192
    idx, wt, plan, g, R = case(moe, T, K, E)
    x, xs = matrix(g, T, D, dtype, extra, shift), matrix(g, T * K, D, dtype, extra, shift)
    moe.dispatch_dev(x, plan["tok_pos"], xs)
    assert torch.equal(bits(xs[:R]), bits(x[plan["rows"][:R].long()]))
    other = F32 if dtype == BF16 else BF16
    for out_type in (dtype, other):
        out = matrix(g, T, D, out_type, shift, extra)
        moe.combine_dev(xs, plan["rw"], plan["tok_pos"], out)
        want, size = rc.combine(xs[:R], plan["rw"], plan, T)
        within(out, want, (K + 2) * U * size + rc.half_step(out_type) * (want.abs() + size * U * K),
               "combine")
        dy, dwt = matrix(g, T * K, D, dtype, shift, extra), torch.empty(T, K, device="cuda")
        flat = torch.empty(T * K, D, dtype=dtype, device="cuda")
        flat_wt = torch.empty(T, K, device="cuda")
        moe.combine_grad_dev(out, xs, plan["rw"], plan["tok_pos"], idx, dy, dwt)
        moe.combine_grad_dev(out.contiguous(), xs.contiguous(), plan["rw"], plan["tok_pos"], idx,
                             flat, flat_wt)
        assert torch.equal(bits(dy[:R]), bits(flat[:R]))
        size = (out.double()[plan["rows"][:R].long()] * xs[:R].double()).abs().sum(1)
        assert float((dwt - flat_wt).abs().max()) <= 2 * (D / 32 + 48) * U * float(size.max())


def test_one_row_for_all_tokens(moe):
    """A gradient broadcast over the tokens has row pitch 0."""
    T, K, E, D = 20, 2, 6, 64
    idx, wt, plan, g, R = case(moe, T, K, E)
    one = torch.randn(1, D, generator=g, device="cuda")
    y = matrix(g, T * K, D, F32)
    dy, dwt = torch.zeros_like(y), torch.empty(T, K, device="cuda")
    dy2, dwt2 = torch.zeros_like(y), torch.empty(T, K, device="cuda")
    moe.combine_grad_dev(one.expand(T, D), y, plan["rw"], plan["tok_pos"], idx, dy, dwt)
    moe.combine_grad_dev(one.repeat(T, 1), y, plan["rw"], plan["tok_pos"], idx, dy2, dwt2)
    assert torch.equal(dy, dy2) and torch.equal(dwt, dwt2)


def test_non_finite_rows_stay_in_their_tokens(moe):
    """Infinities and NaN reach the tokens that own them and no others."""
    T, K, E, D = 33, 4, 8, 72
    idx, wt, plan, g, R = case(moe, T, K, E)
    x = matrix(g, T, D, BF16)
    x[3], x[4, 5] = float("nan"), float("inf")
    xs = torch.zeros(T * K, D, dtype=BF16, device="cuda")
    moe.dispatch_dev(x, plan["tok_pos"], xs)
    assert torch.equal(bits(xs[:R]), bits(x[plan["rows"][:R].long()]))
    out = torch.empty(T, D, device="cuda")
    moe.combine_dev(xs, plan["rw"], plan["tok_pos"], out)
    has = (plan["tok_pos"] >= 0).any(1)
    assert torch.equal(~torch.isfinite(out), ~torch.isfinite(x.float()) & has[:, None])


def test_positions_outside_the_rows_count_as_none(moe):
    T, K, E, D = 16, 2, 4, 32
    idx, wt, plan, g, R = case(moe, T, K, E, dropped=0.0)
    cap = R // 2
    x, xs = matrix(g, T, D, F32), torch.full((cap, D), 5.0, device="cuda")
    moe.dispatch_dev(x, plan["tok_pos"], xs)
    assert torch.equal(xs, x[plan["rows"][:cap].long()])
    out = torch.empty(T, D, device="cuda")
    moe.combine_dev(xs, plan["rw"], plan["tok_pos"], out)
    cut = dict(tok_pos=torch.where(plan["tok_pos"] < cap, plan["tok_pos"], -1))
    want, size = rc.combine(xs, plan["rw"], cut, T)
    within(out, want, (K + 2) * U * (size + want.abs()), "cut")


def test_large_offsets(moe):
    """Rows whose element offsets pass 2^31."""
    D, T, K, E = 65536, 2, 2, 4
    cap = (1 << 31) // D + 64
    idx = torch.tensor([[0, 3], [3, 1]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([[0, cap - 1], [cap - 2, cap - 3]], dtype=torch.int32, device="cuda")
    rw = torch.zeros(cap, device="cuda")
    rw[pos.long().flatten()] = torch.tensor([1.0, 2.0, 3.0, 4.0], device="cuda")
    x = torch.randn(T, D, device="cuda").to(BF16)
    xs = torch.zeros(cap, D, dtype=BF16, device="cuda")
    moe.dispatch_dev(x, pos, xs)
    assert torch.equal(xs[0], x[0]) and torch.equal(xs[cap - 1], x[0])
    assert torch.equal(xs[cap - 2], x[1]) and torch.equal(xs[cap - 3], x[1])
    out = torch.empty(T, D, device="cuda")
    moe.combine_dev(xs, rw, pos, out)
    assert torch.equal(out, x.float() * torch.tensor([[3.0], [7.0]], device="cuda"))
    dy, dwt = torch.zeros_like(xs), torch.empty(T, K, device="cuda")
    moe.combine_grad_dev(x, xs, rw, pos, idx, dy, dwt)
    for t, k, w in ((0, 0, 1.0), (0, 1, 2.0), (1, 0, 3.0), (1, 1, 4.0)):
        assert torch.equal(dy[int(pos[t, k])], (x[t].float() * w).to(BF16))
        dot = (x[t].double() ** 2).sum()
        assert abs(dwt[t, k].double() - dot) <= (D / 32 + 48) * U * dot


def test_results_repeat_and_capture(moe):
    """The same bits again, on another stream, and from a replayed graph."""
    T, K, E, H = 600, 8, 64, 520
    idx, wt, plan, g, R = case(moe, T, K, E)
    x, y, dout = matrix(g, T, H, BF16), matrix(g, T * K, H, BF16), matrix(g, T, H, BF16)
    router, scores = torch.randn(E, H, generator=g, device="cuda"), torch.rand(
        T, E, generator=g, device="cuda")
    dwt_in = torch.randn(T, K, generator=g, device="cuda")
    ws = torch.empty(moe.route_grad_workspace_bytes(T, H, E, K), dtype=torch.uint8, device="cuda")

    def outputs():
        return [torch.zeros(T * K, H, dtype=BF16, device="cuda"), torch.zeros(T, H, device="cuda"),
                torch.zeros(T * K, H, dtype=BF16, device="cuda"), torch.zeros(T, K, device="cuda"),
                torch.zeros(T, H, dtype=BF16, device="cuda"), torch.zeros(E, H, device="cuda"),
                torch.zeros(T, H, device="cuda")]

    def step(o):
        moe.dispatch_dev(x, plan["tok_pos"], o[0])
        moe.combine_dev(y, plan["rw"], plan["tok_pos"], o[1])
        moe.combine_grad_dev(dout, y, plan["rw"], plan["tok_pos"], idx, o[2], o[3])
        moe.route_grad_dev(x, router, idx, scores, dwt_in, plan["nr"], plan["xoff"], plan["rows"],
                           plan["tok_pos"], o[4], o[5], ws)
        moe.dispatch_grad_dev(o[2], plan["tok_pos"], o[6])

    first, second, third = outputs(), outputs(), outputs()
    step(first)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(second)
        graph = torch.cuda.CUDAGraph()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            step(third)
    for o in third:
        o.fill_(9)
    third[0].zero_(), third[2].zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_empty_batch(moe):
    E, H, K = 4, 32, 2
    z = dict(device="cuda")
    pos = torch.zeros(0, K, dtype=torch.int32, **z)
    x, xs = torch.zeros(0, H, **z), torch.full((5, H), 3.0, **z)
    moe.dispatch_dev(x, pos, xs)
    assert (xs == 3).all()
    moe.combine_dev(xs, torch.zeros(5, **z), pos, x)
    moe.dispatch_grad_dev(xs, pos, x)
    i0 = torch.zeros(0, K, dtype=torch.int32, **z)
    f0 = torch.zeros(0, K, **z)
    moe.combine_grad_dev(x, xs, torch.zeros(5, **z), pos, i0, xs, f0)
    zero = torch.zeros(E, dtype=torch.int32, **z)
    dr = torch.full((E, H), 3.0, **z)
    moe.route_grad_dev(x, torch.zeros(E, H, **z), i0, torch.zeros(0, E, **z), f0, zero, zero,
                       torch.zeros(0, dtype=torch.int32, **z), pos, x, dr)
    assert (dr == 0).all(), "no token: the router's gradient is zero"
    dr.fill_(3.0)
    moe.route_grad_dev(x, torch.zeros(E, H, **z), i0, torch.zeros(0, E, **z), f0, zero, zero,
                       torch.zeros(0, dtype=torch.int32, **z), pos, x, dr, accumulate=True)
    assert (dr == 3).all()

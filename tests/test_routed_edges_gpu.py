"""Edges of the routed steps' entries on the device: tiny scores, weights
shorter than the rows, a given stream, the Python entries' refusals."""
import pytest

torch = pytest.importorskip("torch")

import routed_cases as rc  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16 = torch.bfloat16


@pytest.mark.parametrize("score_fn", [0, 1])
@pytest.mark.parametrize("size", [1e-3, 1e-12, 1e-19, 1e-30, 1e-36])
def test_router_gradient_of_tiny_scores(moe, size, score_fn):
    """A token all of whose scores are tiny has ordinary weights and an
    ordinary gradient.  Of its factors m / M, the difference and s' / m none
    leaves f32's range; each is off by (2 K + 16) roundings at most."""
    T, H, E, K = 12, 40, 9, 3
    g = torch.Generator(device="cuda").manual_seed(5)
    x, router = (torch.randn(n, H, generator=g, device="cuda") for n in (T, E))
    scores = (torch.rand(T, E, generator=g, device="cuda") + 0.5) * size
    dwt = torch.randn(T, K, generator=g, device="cuda")
    idx = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:K]
                       for t in range(T)]).int().cuda()
    m = scores.gather(1, idx.long())
    plan = rc.device_plan(moe, idx, m / m.sum(1, keepdim=True), E)
    dx, dr = torch.empty_like(x), torch.empty_like(router)
    moe.route_grad_dev(x, router, idx, scores, dwt, plan["nr"], plan["xoff"], plan["rows"],
                       plan["tok_pos"], dx, dr, score_fn=score_fn)
    m = m.double()
    w, gd = m / m.sum(1, keepdim=True), dwt.double()
    slope = 1 - m if score_fn == 0 else torch.where(
        m > 1e-5, -torch.expm1(-m * m) / (2 * m * m), 0.5 - m * m / 4)
    G = (gd * w).sum(1, keepdim=True)
    parts = []
    for diff in (gd - G, gd.abs() + (gd * w).abs().sum(1, keepdim=True)):
        dz = torch.zeros(T, E, dtype=torch.float64, device="cuda")
        parts.append(dz.scatter_(1, idx.long(), diff * w * slope))
    n = 2 * K + 16
    for got, want, bound in ((dx, parts[0] @ router.double(), parts[1] @ router.double().abs()),
                             (dr, parts[0].T @ x.double(), parts[1].T @ x.double().abs())):
        assert torch.isfinite(got).all() and torch.count_nonzero(want)
        assert ((got.double() - want).abs() <= (n + T + 1) * U * bound).all()


def test_weights_shorter_than_the_rows(moe):
    """Positions behind the weights count as no slot."""
    T, K, E, D = 20, 2, 5, 48
    gen = torch.Generator().manual_seed(1)
    idx, wt = rc.routing(gen, T, K, E, 0.0)
    idx, wt = idx.cuda(), wt.cuda()
    plan = rc.device_plan(moe, idx, wt, E)
    cap = T * K + 9
    y = torch.randn(cap, D, device="cuda")
    with pytest.raises(ValueError, match="rw"):
        moe.combine_dev(y, plan["rw"][:T * K - 1], plan["tok_pos"], torch.empty(T, D).cuda())
    far = plan["tok_pos"].clone()
    far[far == 0] = T * K + 4  # a row of y that has no weight
    out, dy = torch.empty(T, D, device="cuda"), torch.full_like(y, 3.0)
    dwt = torch.empty(T, K, device="cuda")
    moe.combine_dev(y, plan["rw"], far, out)
    cut = dict(tok_pos=torch.where(far < T * K, far, -1))
    want, size = rc.combine(y, plan["rw"], cut, T)
    assert ((out.double() - want).abs() <= (K + 2) * U * size).all()
    moe.combine_grad_dev(out, y, plan["rw"], far, idx, dy, dwt)
    assert (dy[T * K:] == 3).all() and (dy[0] == 3).all()
    assert (dwt[plan["tok_pos"] == 0] == 0).all()


def test_a_given_stream(moe):
    """Every entry on a stream that is not the current one, the workspace left
    to the entry."""
    T, K, E, D = 90, 4, 16, 256
    gen = torch.Generator().manual_seed(2)
    idx, wt = rc.routing(gen, T, K, E)
    idx, wt = idx.cuda(), wt.cuda()
    plan = rc.device_plan(moe, idx, wt, E)
    pos = plan["tok_pos"]
    x = torch.randn(T, D, device="cuda").to(BF16)
    router, scores = torch.randn(E, D, device="cuda"), torch.rand(T, E, device="cuda")
    w, s = rc.packed(gen, rc.INT4, 64, D, "cuda")
    wp = torch.full((E,), w.data_ptr(), dtype=torch.int64, device="cuda")
    sp = torch.full((E,), s.data_ptr(), dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()

    def run(stream):
        xs, y = torch.zeros(T * K, D, device="cuda").to(BF16), torch.zeros(T * K, 64).cuda()
        out, dy, dwt = torch.zeros(T, 64).cuda(), torch.zeros_like(y), torch.zeros(T, K).cuda()
        dxs, dx, dr = torch.zeros_like(xs), torch.zeros_like(x), torch.zeros_like(router)
        one, back = torch.zeros(T, 64).cuda(), torch.zeros_like(x)
        torch.cuda.synchronize()
        moe.dispatch_dev(x, pos, xs, stream=stream)
        moe.expert_matvec_q4_dev(rc.INT4, xs, wp, sp, plan["nr"], plan["xoff"], y, stream=stream)
        moe.combine_dev(y, plan["rw"], pos, out, stream=stream)
        moe.combine_grad_dev(out, y, plan["rw"], pos, idx, dy, dwt, stream=stream)
        moe.expert_matvec_q4_grad_dev(rc.INT4, dy, wp, sp, plan["nr"], plan["xoff"], dxs,
                                      stream=stream)
        moe.dispatch_grad_dev(dxs, pos, dx, stream=stream)
        moe.route_grad_dev(x, router, idx, scores, dwt, plan["nr"], plan["xoff"], plan["rows"],
                           pos, dx, dr, accumulate=True, stream=stream)
        moe.matvec_q4_dev(rc.INT4, x, w, s, one, stream=stream)
        moe.matvec_q4_grad_dev(rc.INT4, one, w, s, back, stream=stream)
        (stream or torch.cuda.current_stream()).synchronize()
        return xs, y, out, dy, dwt, dxs, dx, dr, one, back

    for a, b in zip(run(None), run(side)):
        assert torch.count_nonzero(a) and torch.equal(a, b)


def test_nothing_to_do(moe):
    """No token and no router gradient asked for; one of the outputs alone."""
    z = dict(device="cuda")
    i0, f0 = torch.zeros(0, 2, dtype=torch.int32, **z), torch.zeros(0, 2, **z)
    zero, x = torch.zeros(4, dtype=torch.int32, **z), torch.zeros(0, 8, **z)
    moe.route_grad_dev(x, torch.zeros(4, 8, **z), i0, torch.zeros(0, 4, **z), f0, zero, zero,
                       torch.zeros(0, dtype=torch.int32, **z), i0, x.clone(), None)
    w, s = rc.packed(torch.Generator(), rc.MXFP4, 8, 32, "cuda")
    moe.matvec_q4_dev(rc.MXFP4, torch.zeros(0, 32, **z), w, s, torch.zeros(0, 8, **z))
    moe.matvec_q4_grad_dev(rc.MXFP4, torch.zeros(0, 8, **z), w, s, torch.zeros(0, 32, **z))
    torch.cuda.synchronize()


def test_python_refusals(moe):
    z = dict(device="cuda")
    T, K, E, D = 4, 2, 3, 16
    x, xs = torch.zeros(T, D, **z), torch.zeros(T * K, D, **z)
    pos, rw = torch.zeros(T, K, dtype=torch.int32, **z), torch.zeros(T * K, **z)
    wt = torch.zeros(T, K, **z)

    def no(match, call, *args, **kw):
        with pytest.raises(ValueError, match=match):
            call(*args, **kw)

    no("dtype of x", moe.dispatch_dev, x.bfloat16(), pos, xs)
    no("float16", moe.dispatch_dev, x.half(), pos, xs.half())
    no("tok_pos", moe.dispatch_dev, x, pos.long(), xs)
    no("tok_pos", moe.dispatch_dev, x, pos.flatten(), xs)
    no("shape", moe.dispatch_dev, x[:3], pos, xs)
    no("shape", moe.dispatch_dev, x, pos, torch.zeros(T * K, D + 1, **z))
    no("overlap", moe.dispatch_dev, x, pos, torch.zeros(1, D, **z).expand(T * K, D))
    no("contiguous", moe.dispatch_dev, torch.zeros(D, T, **z).t(), pos, xs)
    no("CUDA tensor", moe.dispatch_dev, x.cpu(), pos, xs)
    no("2-D", moe.dispatch_dev, x, pos, xs[0])
    no("rw", moe.combine_dev, xs, rw.double(), pos, x)
    no("out", moe.combine_dev, xs, rw, pos, x[:2])
    no("dy", moe.combine_grad_dev, x, xs, rw, pos, pos, xs.bfloat16(), wt)
    no("dwt", moe.combine_grad_dev, x, xs, rw, pos, pos, xs, wt[:1])
    zero = torch.zeros(E, dtype=torch.int32, **z)
    args = [x, torch.zeros(E, D, **z), pos, torch.zeros(T, E, **z), wt, zero, zero, pos.flatten(),
            pos, x.clone(), torch.zeros(E, D, **z)]
    for at, name in ((0, "x"), (1, "scores"), (2, "idx"), (3, "scores"), (4, "dwt"), (5, "nr"),
                     (7, "rows"), (9, "dx"), (10, "drouter")):
        bad = list(args)
        bad[at] = bad[at][:1]
        no(name, moe.route_grad_dev, *bad)
    no("workspace", moe.route_grad_dev, *args, workspace=torch.zeros(1 << 16, dtype=torch.uint8))
    no("workspace", moe.route_grad_dev, *args,
       workspace=torch.zeros(1 << 16, dtype=torch.uint8, **z)[::2])
    with pytest.raises(RuntimeError, match="workspace"):
        moe.route_grad_dev(*args, workspace=torch.zeros(16, dtype=torch.uint8, **z))
    w, s = rc.packed(torch.Generator(), rc.INT4, 8, D, "cuda")
    y = torch.zeros(T, 8, **z)
    no("w:", moe.matvec_q4_dev, rc.INT4, x, w[:7], s, y)
    no("scales", moe.matvec_q4_dev, rc.MXFP4, x, w, s, y)
    no("shape", moe.matvec_q4_dev, rc.INT4, x, w, s, y[:3])
    no("overlap", moe.matvec_q4_dev, rc.INT4, x, w, s, y[:1].expand(T, 8))
    no("2-D", moe.matvec_q4_grad_dev, rc.INT4, y, w, s, x[0])
    tab = torch.zeros(E, dtype=torch.int64, **z)
    no("xoff", moe.expert_matvec_q4_dev, rc.INT4, x, tab, tab, zero, zero[:1], y)
    no("w:", moe.expert_matvec_q4_dev, rc.INT4, x, tab[:1], tab, zero, zero, y)
    no("int64", moe.expert_matvec_q4_dev, rc.INT4, x, zero, tab, zero, zero, y)
    no("fmt", moe.expert_matvec_q4_grad_dev, 8, y, tab, tab, zero, zero, x)
    torch.cuda.synchronize()


@pytest.mark.parametrize("fmt", [rc.INT4, rc.MXFP4])
def test_matrices_past_two_gigabytes(moe, fmt):
    """Offsets of packed weights beyond 2^31 bytes.  Some outputs of the
    forward product, and a gradient that only some weight rows enter, against
    64 bits: length / 16 + 64 additions off by 2^-22 of the magnitudes, as for
    the other products, and the factors' f16 or bf16 parts."""
    O, I, S = 70000, 65536, 2
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randint(0, 256, (O, I // 2), generator=g, dtype=torch.uint8, device="cuda")
    if fmt == rc.INT4:
        s = torch.rand(O, I // 64, generator=g, device="cuda") * 0.01 + 1e-4
    else:
        s = torch.randint(113, 126, (O, I // 32), generator=g, dtype=torch.uint8, device="cuda")
    at = torch.tensor([0, 1, 33333, 65535, 65536, 69997, O - 1], device="cuda")
    W = rc.decode(w[at], s[at], fmt, I)
    x = torch.randn(S, I, generator=g, device="cuda")
    y = torch.empty(S, O, device="cuda")
    moe.matvec_q4_dev(fmt, x, w, s, y)
    want, size = x.double() @ W.T, x.double().abs() @ W.T.abs()
    assert ((y[:, at].double() - want).abs() <= (I / 16 + 64) * 2.0 ** -22 * size).all()
    dy, dx = torch.zeros(S, O, device="cuda"), torch.empty(S, I, device="cuda")
    dy[:, at] = torch.randn(S, len(at), generator=g, device="cuda")
    moe.matvec_q4_grad_dev(fmt, dy, w, s, dx)
    want, size = dy[:, at].double() @ W, dy[:, at].double().abs() @ W.abs()
    assert ((dx.double() - want).abs() <= (O / 16 + 64) * 2.0 ** -22 * size).all()


def test_calls_at_the_same_time(moe):
    """Two streams and two host threads, sizes that no call has had before."""
    import threading
    gen = torch.Generator().manual_seed(8)
    E, T, K = 12, 75, 3
    cases = []
    for I, O in ((1184, 736), (864, 1248)):
        w, s = rc.packed(gen, rc.INT4, E * O, I, "cuda")
        tab = torch.tensor([w[e * O].data_ptr() for e in range(E)], device="cuda")
        sct = torch.tensor([s[e * O].data_ptr() for e in range(E)], device="cuda")
        idx, wt = rc.routing(gen, T, K, E)
        plan = rc.device_plan(moe, idx.cuda(), wt.cuda(), E)
        x = torch.randn(T * K, I, generator=gen).cuda()
        cases.append((w, s, tab, sct, plan, x, torch.randn(T * K, O, generator=gen).cuda()))
    torch.cuda.synchronize()

    def step(c, stream, out):
        w, s, tab, sct, plan, x, dy = c
        y, dx = torch.zeros_like(dy), torch.zeros_like(x)
        stream.wait_stream(torch.cuda.current_stream())
        for _ in range(20):
            moe.expert_matvec_q4_dev(rc.INT4, x, tab, sct, plan["nr"], plan["xoff"], y,
                                     stream=stream)
            moe.expert_matvec_q4_grad_dev(rc.INT4, dy, tab, sct, plan["nr"], plan["xoff"], dx,
                                          stream=stream)
        stream.synchronize()
        out.append((y, dx))

    together = [[], []]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    threads = [threading.Thread(target=step, args=(cases[i], streams[i], together[i]))
               for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        alone = []
        step(cases[i], streams[i], alone)
        for a, b in zip(together[i][0], alone[0]):
            assert torch.count_nonzero(a) and torch.equal(a, b)


def test_first_call_of_a_size_captured(moe):
    """Nothing that a size's first call does on the host disturbs a capture."""
    gen = torch.Generator().manual_seed(9)
    S, I, O = 5, 1376, 928
    w, s = rc.packed(gen, rc.MXFP4, O, I, "cuda")
    x, dy = torch.randn(S, I, generator=gen).cuda(), torch.randn(S, O, generator=gen).cuda()
    outs = [[torch.zeros(S, O, device="cuda"), torch.zeros(S, I, device="cuda")] for _ in range(2)]

    def step(o):
        moe.matvec_q4_dev(rc.MXFP4, x, w, s, o[0])
        moe.matvec_q4_grad_dev(rc.MXFP4, dy, w, s, o[1])

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(outs[0])
    graph.replay()
    step(outs[1])
    torch.cuda.synchronize()
    for a, b in zip(*outs):
        assert torch.count_nonzero(a) and torch.equal(a, b)

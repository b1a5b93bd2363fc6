"""Row steps and router gradients on the device: calls that the permutation's
own output does not lead to, and sizes that single branches wait for."""
import pytest

torch = pytest.importorskip("torch")

import routed_cases as rc  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("KK", [2, 8, 33, 64])
def test_a_position_named_twice(moe, KK):
    """Slots of a token that share a position each count: every place of the
    sorted list holds a position of the token's own."""
    T, D, cap = 40, 96, 50
    g = torch.Generator(device="cuda").manual_seed(KK)
    pos = torch.randint(-2, cap + 2, (T, KK), generator=g, device="cuda", dtype=torch.int32)
    pos[0], pos[1, :2] = 7, 49  # all slots the same; a pair
    pos[2] = -1
    y, rw = torch.randn(cap, D, generator=g, device="cuda"), torch.rand(cap, device="cuda")
    live = dict(tok_pos=torch.where(pos < cap, pos, -1))
    for weights in (rw, None):
        out = torch.empty(T, D, device="cuda")
        if weights is None:
            moe.dispatch_grad_dev(y, pos, out)
        else:
            moe.combine_dev(y, rw, pos, out)
        want, size = rc.combine(y, weights, live, T)
        assert ((out.double() - want).abs() <= (KK + 2) * U * size).all()


def routed(moe, T, K, E, H, ns=0, repeats=False, dtype=F32, seed=0):
    """Inputs of the router's gradient for given ids, and the permutation."""
    gen = torch.Generator().manual_seed(T + E + seed)
    g = torch.Generator(device="cuda").manual_seed(T + H)
    logits = torch.rand(T, E, generator=g, device="cuda")
    idx = torch.topk(logits, K, dim=1).indices.int()
    off = torch.rand(T, generator=gen) < 0.1
    idx[off.cuda()] = -1
    if repeats:
        idx[::2, K - 1] = idx[::2, 0]
        idx[::5, 1] = idx[::5, 0]
        idx[1] = idx[1, 0]  # all slots the same
    scores = torch.rand(T, E, generator=g, device="cuda") * 0.9 + 0.05
    m = scores.gather(1, idx.clamp_min(0).long()) * (idx >= 0)
    wt = m / m.sum(1, keepdim=True).clamp_min(1e-9)
    return dict(x=torch.randn(T, H, generator=g, device="cuda").to(dtype),
                router=torch.randn(E, H, generator=g, device="cuda") / H ** 0.5, idx=idx,
                scores=scores, dwt=torch.randn(T, K, generator=g, device="cuda"),
                plan=rc.device_plan(moe, idx, wt.contiguous(), E, ns))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("score_fn", [0, 1])
@pytest.mark.parametrize("T,K,E,H,ns,repeats", [(8192, 8, 64, 2048, 0, False),
                                                (8192, 8, 48, 4096, 0, False),
                                                (300, 4, 24, 520, 0, True),
                                                (300, 4, 24, 520, 1, False),
                                                (77, 8, 9, 300, 1, True)])
def test_router_gradient_paths(moe, T, K, E, H, ns, repeats, score_fn, dtype):
    """Row blocks of 128 and 256 (the first two sizes), ids that repeat within a
    token, permutations with a shared expert; bounds as for the other router
    tests: (2 K + 16) roundings of dz, then the products' sums."""
    c = routed(moe, T, K, E, H, ns, repeats, dtype)
    p = c["plan"]
    args = [c[k] for k in ("x", "router", "idx", "scores", "dwt")]
    dx = torch.empty(T, H, device="cuda")
    dr = torch.empty(E, H, device="cuda")
    moe.route_grad_dev(*args, p["nr"], p["xoff"], p["rows"], p["tok_pos"], dx, dr,
                       score_fn=score_fn, routed_scale=2.5)
    want_x, want_r, _ = rc.route_grad(*args, score_fn, 2.5)
    size_x, size_r = rc.route_grad_bounds(*args, score_fn, 2.5)
    n = 2 * K + 16
    assert ((dx.double() - want_x).abs() <= (n + K + 1) * U * size_x).all()
    longest = int(p["nr"][:E].max())
    assert ((dr.double() - want_r).abs() <= (n + longest + 1) * U * size_r).all()
    # sums of random signs are far below their bound: the norms say more
    assert (dx.double() - want_x).norm() <= n * U * want_x.norm()
    assert (dr.double() - want_r).norm() <= n * U * want_r.norm()


@pytest.mark.parametrize("T,K", [(1, 1), (2, 8), (3, 64), (40, 7)])
def test_few_tokens_of_wide_rows(moe, T, K):
    """Decode-sized combines and their gradient over rows of any width."""
    E = 80
    for D in (7168, 7169, 5):
        gen = torch.Generator().manual_seed(T + D)
        idx, wt = rc.routing(gen, T, K, E, 0.1)
        idx, wt = idx.cuda(), wt.cuda()
        plan = rc.device_plan(moe, idx, wt, E)
        R = int(plan["n_rows"].item())
        for dtype in (F32, BF16):
            y = torch.randn(T * K, D, generator=gen).cuda().to(dtype)
            dout = torch.randn(T, D, generator=gen).cuda().to(dtype)
            out, dy, dwt = torch.empty(T, D).cuda(), torch.zeros_like(y), torch.empty(T, K).cuda()
            moe.combine_dev(y, plan["rw"], plan["tok_pos"], out)
            want, size = rc.combine(y, plan["rw"], plan, T)
            assert ((out.double() - want).abs() <= (K + 2) * U * size).all()
            moe.combine_grad_dev(dout, y, plan["rw"], plan["tok_pos"], idx, dy, dwt)
            seen = dout.double()[plan["rows"][:R].long()]
            want = seen * plan["rw"][:R, None].double()
            assert ((dy[:R].double() - want).abs() <=
                    (U + rc.half_step(dtype)) * 1.01 * want.abs() + 1e-40).all()
            assert (dy[R:] == 0).all()
            dots, size = (seen * y[:R].double()).sum(1), (seen * y[:R].double()).abs().sum(1)
            t, k, at = rc.slots(plan)
            assert ((dwt[t, k].double() - dots[at]).abs() <= (D / 32 + 48) * U * size[at]).all()


@pytest.mark.parametrize("score_fn", [0, 1])
def test_tokens_whose_weights_are_constant(moe, score_fn):
    """Where the chosen scores' sum is 0 or NaN the forward pass gives every
    choice the same weight: such a token has no gradient, the others theirs."""
    T, K, E, H = 24, 3, 8, 64
    c = routed(moe, T, K, E, H)
    args = [c[k] for k in ("x", "router", "idx", "scores", "dwt")]
    idx, scores = c["idx"].long(), c["scores"]
    chosen = [t for t in range(T) if int(idx[t, 0]) >= 0]
    a, b = chosen[2], chosen[7]
    scores[a, idx[a]] = 0.0
    scores[b, idx[b, 1]] = float("nan")
    two = torch.tensor([a, b], device="cuda")
    choice = torch.zeros(2, E, device="cuda").scatter_(1, idx[two], 1.0)
    ids, wt = torch.empty(2, K, dtype=torch.int32, device="cuda"), torch.empty(2, K, device="cuda")
    moe.topk_dev(choice, K, ids, wt, mix=scores[two].contiguous())
    assert torch.equal(wt, torch.full_like(wt, 1 / K)), "the forward pass"
    p = c["plan"]
    dx, dr = torch.full((T, H), 7.0, device="cuda"), torch.empty(E, H, device="cuda")
    moe.route_grad_dev(*args, p["nr"], p["xoff"], p["rows"], p["tok_pos"], dx, dr,
                       score_fn=score_fn)
    assert (dx[a] == 0).all() and (dx[b] == 0).all()
    clean = scores.clone()
    clean[a] = clean[b] = 0.5
    dwt = c["dwt"].clone()
    dwt[a] = dwt[b] = 0
    want_x, want_r, _ = rc.route_grad(c["x"], c["router"], c["idx"], clean, dwt, score_fn, 1.0)
    n = (2 * K + 16) * U
    assert (dx.double() - want_x).norm() <= n * want_x.norm()
    assert (dr.double() - want_r).norm() <= n * want_r.norm()

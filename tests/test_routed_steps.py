"""The routed layer's separate steps without a GPU: what their entries refuse,
and the 64-bit forms that the device tests compare with, against automatic
differentiation and difference quotients."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import build as mvbuild  # noqa: E402
import routed_cases as rc  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    mvbuild.build()
    import mvllm_moe
    return mvllm_moe


P = C.c_void_p(4096)  # an address that is never followed


def refused(lib, name, good, bads, code=None):
    """Every change of one argument is refused before any device work; the
    unchanged call gets as far as asking for a device."""
    fn = getattr(lib.lib(), name)
    if not lib.available():
        assert fn(*good) == lib.ERR_NOT_INIT, name
    for at, value in bads:
        args = list(good)
        args[at] = value
        got = fn(*args)
        assert got == (code or lib.ERR_INVALID), (name, at, value, got, lib.last_error())


def test_dispatch_refusals(lib):
    # stream, x, dtype, ldx, tok_pos, T, KK, D, xs, ldxs, cap
    refused(lib, "mvllm_moe_dispatch_dev", [None, P, 1, 64, P, 4, 2, 64, P, 64, 8],
            [(1, None), (2, 2), (2, -1), (3, -1), (4, None), (5, -1), (6, 0), (6, 65), (7, 0),
             (8, None), (9, 63), (10, -1)])
    # stream, dxs, dtype, ld, cap, tok_pos, T, KK, D, dx, dtype, ld, accumulate
    refused(lib, "mvllm_moe_dispatch_grad_dev", [None, P, 1, 64, 8, P, 4, 2, 64, P, 0, 64, 0],
            [(1, None), (2, 7), (3, -1), (4, -1), (5, None), (6, -1), (7, 0), (7, 65), (8, 0),
             (9, None), (10, 7), (11, 63)])


def test_combine_refusals(lib):
    # stream, y, dtype, ld, cap, rw, tok_pos, T, KK, D, out, dtype, ld, accumulate
    refused(lib, "mvllm_moe_combine_dev", [None, P, 1, 64, 8, P, P, 4, 2, 64, P, 0, 64, 0],
            [(1, None), (2, 7), (3, -1), (4, -1), (5, None), (6, None), (7, -1), (8, 0), (8, 65),
             (9, 0), (10, None), (11, 7), (12, 63)])
    # stream, dout, dtype, ld, y, dtype, ld, cap, rw, tok_pos, idx, T, K, KK, D, dy, ld, dwt
    refused(lib, "mvllm_moe_combine_grad_dev",
            [None, P, 1, 64, P, 1, 64, 8, P, P, P, 4, 2, 2, 64, P, 64, P],
            [(1, None), (2, 7), (3, -1), (4, None), (5, 7), (6, -1), (7, -1), (8, None), (9, None),
             (10, None), (11, -1), (12, 0), (12, 3), (13, 1), (13, 65), (14, 0), (15, None),
             (16, 63), (17, None)])


def test_route_grad_refusals(lib):
    L = lib.lib()
    need = L.mvllm_moe_route_grad_workspace(4, 64, 8, 2)
    assert need > 0
    for bad in ((-1, 64, 8, 2), (4, 0, 8, 2), (4, 64, 0, 2), (4, 64, 8, 0)):
        assert L.mvllm_moe_route_grad_workspace(*bad) == 0
    # stream, x, dtype, ld, T, H, router, E, K, idx, scores, dwt, score_fn, scale, nr, xoff,
    # rows, tok_pos, KK, dx, dtype, ld, drouter, accumulate, workspace, bytes
    good = [None, P, 1, 64, 4, 64, P, 8, 2, P, P, P, 0, 1.0, P, P, P, P, 2, P, 0, 64, P, 0, P, need]
    refused(lib, "mvllm_moe_route_grad_dev", good,
            [(1, None), (2, 7), (3, -1), (4, -1), (5, 0), (6, None), (7, 0), (7, 1025), (8, 0),
             (8, 33), (9, None), (10, None), (11, None), (12, 2), (14, None), (15, None),
             (16, None), (17, None), (18, 1), (18, 65), (20, 7), (21, 63)])
    refused(lib, "mvllm_moe_route_grad_dev", good, [(24, None), (25, need - 1)],
            lib.ERR_WORKSPACE)
    neither = list(good)
    neither[19] = neither[22] = None
    assert L.mvllm_moe_route_grad_dev(*neither) == lib.ERR_INVALID


@pytest.mark.parametrize("way", ["", "_grad"])
def test_matvec_refusals(lib, way):
    # stream, fmt, x, dtype, ld, w, scales, S, I, O, y, dtype, ld
    refused(lib, f"mvllm_matvec_q4{way}_dev", [None, 4, P, 0, 64, P, P, 2, 64, 64, P, 0, 64],
            [(1, 0), (1, 8), (1, 9), (2, None), (3, 7), (4, -1), (5, None), (6, None), (7, -1),
             (8, 0), (9, 0), (10, None), (11, 7), (12, 63)])
    odd = C.c_void_p(4097)  # f32 scales at an odd address
    refused(lib, f"mvllm_matvec_q4{way}_dev", [None, 4, P, 0, 64, P, P, 2, 64, 64, P, 0, 64],
            [(6, odd)])
    # stream, fmt, nb, x, dtype, ld, cap, nr, xoff, w, scales, I, O, y, dtype, ld
    refused(lib, f"mvllm_moe_matvec_q4{way}_dev",
            [None, 7, 3, P, 0, 64, 8, P, P, P, P, 64, 64, P, 0, 64],
            [(1, 0), (2, 0), (2, 1025), (3, None), (4, 7), (5, -1), (6, -1), (7, None), (8, None),
             (9, None), (10, None), (11, 0), (12, 0), (13, None), (14, 7), (15, 63)])


def test_host_tensors_are_refused(lib):
    """The Python entries name the argument that does not fit."""
    x, pos = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    for call, args in ((lib.dispatch_dev, (x, pos, x)), (lib.dispatch_grad_dev, (x, pos, x)),
                       (lib.combine_dev, (x, x[0], pos, x)),
                       (lib.combine_grad_dev, (x, x, x[0], pos, pos, x, x))):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call(*args)
    w, s = torch.zeros(8, 4, dtype=torch.uint8), torch.zeros(8, 1)
    for call in (lib.matvec_q4_dev, lib.matvec_q4_grad_dev):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call(lib.FMT_INT4_G64, x, w, s, x)
        with pytest.raises(ValueError, match="fmt"):
            call(lib.FMT_F32, x, w, s, x)


def test_plan_by_definition():
    idx = torch.tensor([[2, 0, 2], [1, -1, 5], [0, 1, 2]], dtype=torch.int32)
    wt = torch.tensor([[.5, .25, .25], [1., .5, .5], [0., 2., -1.]])
    p = rc.cpu_plan(idx, wt, 3, n_shared=1)
    assert p["nr"].tolist() == [1, 2, 2, 3] and p["xoff"].tolist() == [0, 1, 3, 5]
    assert p["rows"].tolist() == [0, 1, 2, 0, 2, 0, 1, 2]
    assert p["rw"].tolist() == [.25, 1., 2., .75, -1., 1., 1., 1.]
    assert p["tok_pos"].tolist() == [[3, 0, -1, 5], [1, -1, -1, 6], [-1, 2, 4, 7]]


@pytest.mark.parametrize("score_fn", [0, 1])
def test_router_gradient_form(score_fn):
    """The closed form against automatic differentiation of the forward pass
    and against central differences."""
    g = torch.Generator().manual_seed(score_fn)
    T, H, E, K, scale = 6, 5, 7, 3, 2.5
    x = torch.randn(T, H, generator=g, dtype=torch.float64, requires_grad=True)
    router = torch.randn(E, H, generator=g, dtype=torch.float64, requires_grad=True)
    idx, _ = rc.routing(g, T, K, E, dropped=0.4)
    dwt = torch.randn(T, K, generator=g, dtype=torch.float64)

    def loss(a, b):
        return (rc.route_weights(a @ b.T, idx, score_fn, scale)[0] * dwt).sum()

    _, scores = rc.route_weights(x @ router.T, idx, score_fn, scale)
    want = torch.autograd.grad(loss(x, router), (x, router))
    dx, dr, _ = rc.route_grad(x.detach(), router.detach(), idx, scores.detach(), dwt, score_fn,
                              scale)
    assert torch.allclose(dx, want[0], rtol=1e-12, atol=1e-13)
    assert torch.allclose(dr, want[1], rtol=1e-12, atol=1e-13)
    with torch.no_grad():
        step, at = 1e-6, torch.randn(E, H, generator=g, dtype=torch.float64)
        slope = (loss(x, router + step * at) - loss(x, router - step * at)) / (2 * step)
        assert abs(slope - (dr * at).sum()) < 1e-8 * max(1.0, float(abs(slope)))


def test_combine_form():
    """Dispatch, combine and their gradients by automatic differentiation of
    the definition, row by row."""
    g = torch.Generator().manual_seed(3)
    T, K, E, D = 7, 3, 5, 4
    idx, wt = rc.routing(g, T, K, E, repeats=True)
    p = rc.cpu_plan(idx, wt, E)
    y = torch.randn(p["n"], D, generator=g, dtype=torch.float64, requires_grad=True)
    w = wt.double().requires_grad_()
    out = torch.zeros(T, D, dtype=torch.float64)
    for r in range(p["n"]):
        t = int(p["rows"][r])
        e = int(idx[t][(p["tok_pos"][t] == r).nonzero()[0, 0]])
        out = out.index_add(0, torch.tensor([t]), (y[r] * w[t][idx[t] == e].sum())[None])
    assert torch.allclose(out, rc.combine(y, p["rw"], p, T)[0], rtol=1e-6)
    dout = torch.randn(T, D, generator=g, dtype=torch.float64)
    dy, dw = torch.autograd.grad(out, (y, w), dout)
    assert torch.allclose(dy, p["rw"][:, None].double() * dout[p["rows"].long()], rtol=1e-6)
    dots = (dout[p["rows"].long()] * y).sum(1)
    for t in range(T):
        for k in range(K):
            at = [int(p["tok_pos"][t, j]) for j in range(K)
                  if idx[t, j] == idx[t, k] and p["tok_pos"][t, j] >= 0]
            assert torch.allclose(dw[t, k], dots[at[0]] if at else torch.tensor(0.0).double())


def test_sizes_beyond_the_arithmetic_are_refused(lib):
    big = (1 << 30) + 1
    refused(lib, "mvllm_moe_dispatch_dev", [None, P, 1, 64, P, 4, 2, 64, P, 2 * big, 8],
            [(7, big)])
    refused(lib, "mvllm_moe_dispatch_grad_dev",
            [None, P, 1, 64, 8, P, 4, 2, 64, P, 0, 2 * big, 0], [(8, big)])
    refused(lib, "mvllm_moe_combine_dev", [None, P, 1, 64, 8, P, P, 4, 2, 64, P, 0, 2 * big, 0],
            [(9, big)])
    refused(lib, "mvllm_moe_combine_grad_dev",
            [None, P, 1, 64, P, 1, 64, 8, P, P, P, 4, 2, 2, 64, P, 2 * big, P], [(14, big)])
    refused(lib, "mvllm_moe_route_grad_dev",
            [None, P, 1, 64, 4, 64, P, 8, 2, P, P, P, 0, 1.0, P, P, P, P, 2, P, 0, 2 * big, P, 0,
             P, 1 << 20], [(5, big), (4, 1 << 30)])
    for way in ("", "_grad"):
        refused(lib, f"mvllm_matvec_q4{way}_dev",
                [None, 4, P, 0, 64, P, P, 2, 64, 64, P, 0, 2 * big], [(7, big), (8, big), (9, big)])
        refused(lib, f"mvllm_moe_matvec_q4{way}_dev",
                [None, 7, 3, P, 0, 64, 8, P, P, P, P, 64, 64, P, 0, 2 * big],
                [(6, big), (11, big), (12, big)])

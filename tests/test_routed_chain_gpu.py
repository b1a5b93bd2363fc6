"""The routed layer's steps one after another, as a caller runs them: route,
permute, dispatch, the experts' products, combine, and the way back, against
64-bit automatic differentiation, and against the fused layer.

Tolerance of the chain: each of its eight f32 steps is off by at most
(L / 16 + 64) 2^-22 of the magnitudes it sums, L <= 512 terms, and sums of
random signs are about sqrt(2 L / pi) <= 18 times smaller than the sums of
their magnitudes: 8 * 96 * 2^-22 * 18 = 3.3e-3 of the result's norm.
"""
import pytest

torch = pytest.importorskip("torch")

import routed_cases as rc  # noqa: E402
from conftest import assert_close  # noqa: E402

pytestmark = pytest.mark.gpu
CHAIN = 3.3e-3


class Layer:
    """Two frozen 4-bit matrices per expert with a SiLU between, by the
    library's steps; every buffer is made once."""

    def __init__(self, moe, fmt, T, K, E, H, I, score_fn, seed):
        gen = torch.Generator().manual_seed(seed)
        self.moe, self.fmt, self.T, self.K, self.E, self.score_fn = moe, fmt, T, K, E, score_fn
        self.w1 = [rc.packed(gen, fmt, I, H, "cuda", spread=1) for _ in range(E)]
        self.w2 = [rc.packed(gen, fmt, H, I, "cuda", spread=1) for _ in range(E)]
        self.router = (torch.randn(E, H, generator=gen) / H ** 0.5).cuda()
        self.bias = (torch.randn(E, generator=gen) * 0.1).cuda()
        self.x = torch.randn(T, H, generator=gen).cuda()
        self.dout = torch.randn(T, H, generator=gen).cuda()
        self.off = (torch.rand(T, generator=gen) < 0.25).cuda()  # padded tokens
        i64, i32, cap = dict(dtype=torch.int64, device="cuda"), dict(
            dtype=torch.int32, device="cuda"), T * K
        self.tables = [torch.tensor([p[k].data_ptr() for p in w], **i64)
                       for w in (self.w1, self.w2) for k in (0, 1)]
        self.idx, self.wt = torch.zeros(T, K, **i32), torch.zeros(T, K, device="cuda")
        self.scores, self.choice = (torch.zeros(T, E, device="cuda") for _ in range(2))
        self.nr, self.xoff = torch.zeros(E, **i32), torch.zeros(E, **i32)
        self.rows, self.rw = torch.zeros(cap, **i32), torch.zeros(cap, device="cuda")
        self.pos, self.n = torch.zeros(T, K, **i32), torch.zeros(1, **i32)
        self.xs, self.y, self.dy, self.dxs = (torch.zeros(cap, H, device="cuda") for _ in range(4))
        self.h1, self.dh = (torch.zeros(cap, I, device="cuda") for _ in range(2))
        self.out, self.dx = (torch.zeros(T, H, device="cuda") for _ in range(2))
        self.drouter, self.dwt = torch.zeros(E, H, device="cuda"), torch.zeros(T, K, device="cuda")
        self.pws = torch.empty(moe.permute_workspace_bytes(T, K, E, 0), dtype=torch.uint8,
                               device="cuda")
        self.rws = torch.empty(moe.route_grad_workspace_bytes(T, H, E, K), dtype=torch.uint8,
                               device="cuda")

    def step(self):
        m, f = self.moe, self.fmt
        m.route_ex_dev(self.x, self.router, self.bias, self.K, self.idx, self.wt, self.scores,
                       self.choice, self.score_fn, 2.5)
        self.idx.masked_fill_(self.off[:, None], -1)
        self.wt.masked_fill_(self.off[:, None], 0.0)
        m.permute_dev(self.idx, self.wt, self.E, 0, self.nr, self.xoff, self.rows, self.rw,
                      self.pos, self.n, self.pws)
        m.dispatch_dev(self.x, self.pos, self.xs)
        m.expert_matvec_q4_dev(f, self.xs, *self.tables[:2], self.nr, self.xoff, self.h1)
        act = torch.nn.functional.silu(self.h1)
        m.expert_matvec_q4_dev(f, act, *self.tables[2:], self.nr, self.xoff, self.y)
        m.combine_dev(self.y, self.rw, self.pos, self.out)
        # back
        m.combine_grad_dev(self.dout, self.y, self.rw, self.pos, self.idx, self.dy, self.dwt)
        m.expert_matvec_q4_grad_dev(f, self.dy, *self.tables[2:], self.nr, self.xoff, self.dh)
        s = torch.sigmoid(self.h1)
        self.dh.mul_(s * (1 + self.h1 * (1 - s)))
        m.expert_matvec_q4_grad_dev(f, self.dh, *self.tables[:2], self.nr, self.xoff, self.dxs)
        m.dispatch_grad_dev(self.dxs, self.pos, self.dx)
        m.route_grad_dev(self.x, self.router, self.idx, self.scores, self.dwt, self.nr, self.xoff,
                         self.rows, self.pos, self.dx, None, self.rws, self.score_fn, 2.5,
                         accumulate=True)
        m.route_grad_dev(self.x, self.router, self.idx, self.scores, self.dwt, self.nr, self.xoff,
                         self.rows, self.pos, None, self.drouter, self.rws, self.score_fn, 2.5)

    def want(self, H, I):
        """The same from f64 and automatic differentiation, for the ids the
        device chose."""
        x = self.x.double().requires_grad_()
        router = self.router.double().requires_grad_()
        wt, _ = rc.route_weights(x @ router.T, self.idx, self.score_fn, 2.5)
        out = torch.zeros(self.T, H, dtype=torch.float64, device="cuda")
        for e in range(self.E):
            t, k = torch.nonzero(self.idx == e, as_tuple=True)
            if not len(t):
                continue
            a, b = (rc.decode(*w[e], self.fmt, n) for w, n in ((self.w1, H), (self.w2, I)))
            out = out.index_add(0, t, wt[t, k][:, None] *
                                (torch.nn.functional.silu(x[t] @ a.T) @ b.T))
        return out, *torch.autograd.grad(out, (x, router), self.dout.double())


@pytest.mark.parametrize("fmt,score_fn", [(rc.INT4, 0), (rc.MXFP4, 1)])
@pytest.mark.parametrize("T,K,E,H,I", [(1, 2, 4, 128, 96), (37, 4, 16, 256, 512),
                                       (150, 8, 24, 200, 130)])
def test_forward_and_backward(moe, T, K, E, H, I, fmt, score_fn):
    layer = Layer(moe, fmt, T, K, E, H, I, score_fn, T + E)
    layer.step()
    for name, got, want in zip(("out", "dx", "drouter"), (layer.out, layer.dx, layer.drouter),
                               layer.want(H, I)):
        norm = want.norm()
        assert (got.double() - want).norm() <= CHAIN * norm + 1e-30, name


def test_captured_step_repeats(moe):
    """The whole step in a graph: the eager result's bits, replay by replay,
    with new inputs in the same buffers."""
    H, I = 256, 512
    layer = Layer(moe, rc.MXFP4, 64, 4, 16, H, I, 0, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step()
        side.synchronize()
        first = [t.clone() for t in (layer.out, layer.dx, layer.drouter)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            layer.step()
        for _ in range(2):
            graph.replay()
            side.synchronize()
            for a, b in zip(first, (layer.out, layer.dx, layer.drouter)):
                assert torch.equal(a, b)
        layer.x.copy_(torch.flip(layer.x, (0,)))
        graph.replay()
        side.synchronize()
        again = [t.clone() for t in (layer.out, layer.dx, layer.drouter)]
        layer.step()
        side.synchronize()
        for a, b in zip(again, (layer.out, layer.dx, layer.drouter)):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("fmt", [rc.INT4, rc.MXFP4])
def test_agrees_with_the_fused_layer(moe, fmt):
    """Dispatch, gate and up products, SiLU, down product and combine give what
    mvllm_moe_layer_dev gives (within its tolerance)."""
    T, K, E, D, I = 24, 4, 8, 512, 512
    gen = torch.Generator().manual_seed(9)
    packs = [[rc.packed(gen, fmt, I, D, "cuda", spread=0) for _ in range(E)],
             [rc.packed(gen, fmt, I, D, "cuda", spread=0) for _ in range(E)],
             [rc.packed(gen, fmt, D, I, "cuda", spread=0) for _ in range(E)]]
    for m in packs:
        for _, s in m:
            if fmt == rc.INT4:
                s.mul_(0.5)
            else:
                s.sub_(2)
    table = [torch.tensor([p[j].data_ptr() for p in m], dtype=torch.int64, device="cuda")
             for j in (0, 1) for m in packs]
    idx, wt = rc.routing(gen, T, K, E)
    idx, wt = idx.cuda(), wt.cuda()
    x = torch.randn(T, D, generator=gen).cuda().to(torch.bfloat16)
    want = torch.zeros(T, D, device="cuda")
    ws = torch.empty(moe.layer_workspace_bytes(T, K, E, 0, D, I, fmt), dtype=torch.uint8,
                     device="cuda")
    moe.layer_dev(T, K, E, 0, D, I, fmt, idx, wt, x, table, want, moe.ACT_SILU, 0.0, 0.0, ws)
    assert moe.layer_error(ws) == 0
    plan = rc.device_plan(moe, idx, wt, E)
    xs = torch.zeros(T * K, D, dtype=torch.bfloat16, device="cuda")
    moe.dispatch_dev(x, plan["tok_pos"], xs)
    gate, up = (torch.zeros(T * K, I, device="cuda") for _ in range(2))
    for out, w in ((gate, 0), (up, 1)):
        moe.expert_matvec_q4_dev(fmt, xs, table[w], table[3 + w], plan["nr"], plan["xoff"], out)
    y = torch.zeros(T * K, D, device="cuda")
    moe.expert_matvec_q4_dev(fmt, torch.nn.functional.silu(gate) * up, table[2], table[5],
                             plan["nr"], plan["xoff"], y)
    out = torch.empty(T, D, device="cuda")
    moe.combine_dev(y, plan["rw"], plan["tok_pos"], out)
    assert_close(out.cpu().numpy(), want.cpu().numpy(), "steps against the fused layer")
    assert torch.count_nonzero(want)  # the relative error above says something

"""The routed layer opened up, as cases that can be timed and checked.

Four operators, each with its gradient:

* dispatch: token rows to the positions of the expert-sorted order that
  ``permute_dev`` plans, and the gradient of the token rows;
* combine: the weighted sum of a token's expert rows, and the gradients of
  the rows and of the routing weights;
* matvec: products of few rows with 4-bit weights (int4 with a f32 scale per
  64 columns, or MXFP4), for one matrix or for rows sorted by expert, and the
  gradient of the rows;
* router: the gradients that the routing weights send back to the token rows
  and to the router's matrix.

``own`` False: the plain forms in elementary torch operations.  ``own`` True:
the calls a user makes of the library.
"""
import math
import os
import sys

import torch

own = False

INT4, MXFP4 = 4, 7
SIGMOID, SQRT_SOFTPLUS = 0, 1
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}


def listed():
    return [
        # One decode step of 32 sequences: 256 rows, where the launch counts.
        dict(name="dispatch decode", op="dispatch", dir="forward", dtype="bf16", T=32, K=8, E=256,
             D=7168, skew=0.0, padded=0.0),
        # A training or prefill step of 8192 tokens over 384 experts.
        dict(name="dispatch step", op="dispatch", dir="forward", dtype="bf16", T=8192, K=8, E=384,
             D=7168, skew=0.0, padded=0.0),
        # A padded batch with a row length that no vector width divides.
        dict(name="dispatch gradient odd", op="dispatch", dir="gradient", dtype="f32", T=1537, K=6,
             E=160, D=2051, skew=1.1, padded=0.2),
        # One decode step's way back to the residual stream, in f32.
        dict(name="combine decode", op="combine", dir="forward", dtype="f32", T=8, K=8, E=256,
             D=7168, skew=0.0, padded=0.0),
        # Prefill of 4096 tokens under skewed routing, bf16 rows.
        dict(name="combine prefill", op="combine", dir="forward", dtype="bf16", T=4096, K=8, E=256,
             D=7168, skew=1.1, padded=0.0),
        # The backward pass of the same step: rows and routing weights.
        dict(name="combine gradient", op="combine", dir="gradient", dtype="bf16", T=4096, K=8,
             E=256, D=7168, skew=1.1, padded=0.1),
        # A dense projection for one token.
        dict(name="matvec one token", op="matvec", dir="forward", dtype="bf16", out="f32", fmt=MXFP4,
             E=1, S=1, I=7168, O=2048, skew=0.0),
        # A wide dense projection for a batch of sequences, f32 throughout.
        dict(name="matvec batch f32", op="matvec", dir="forward", dtype="f32", out="f32", fmt=INT4,
             E=1, S=16, I=6144, O=12288, skew=0.0),
        # One rank's 48 experts of 384 in a decode step: 256 rows, uneven.
        dict(name="experts decode", op="matvec", dir="forward", dtype="bf16", out="bf16", fmt=MXFP4,
             E=48, S=256, I=7168, O=2048, skew=0.5),
        # Gradients through frozen int4 experts, as adapters below them need.
        dict(name="experts gradient", op="matvec", dir="gradient", dtype="bf16", out="bf16",
             fmt=INT4, E=160, S=512, I=6144, O=1536, skew=0.0),
        # The router of a small layer.
        dict(name="router small", op="router", dir="gradient", dtype="f32", T=64, K=4, E=16, D=1024,
             skew=0.0, score=SIGMOID, scale=1.0),
        # The router of the large layer over a whole step.
        dict(name="router step", op="router", dir="gradient", dtype="bf16", T=8192, K=8, E=384,
             D=7168, skew=1.1, score=SQRT_SOFTPLUS, scale=2.5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi, step):
    """A length over [lo, hi]: two in three a multiple of `step`, the rest as they fall."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.34 else max(step, n // step * step)


def draw(rng):
    op = rng.choice(["dispatch", "combine", "matvec", "matvec", "router"])
    dtype = rng.choice(["f32", "bf16"])
    way = rng.choice(["forward", "gradient"])
    if op == "matvec":
        E = rng.choice([1, 1, 1, 8, 16, 48])
        I, O = _width(rng, 64, 16384, 128), _width(rng, 64, 16384, 32)
        most = 704_643_072 // E  # the weights of "experts decode"
        if I * O > most:
            O = max(64, most // I)
        S = _log(rng, 1, 64) if E == 1 else _log(rng, 1, 6 * E)
        return dict(op=op, dir=way, dtype=dtype, out=rng.choice([dtype, "f32"]),
                    fmt=rng.choice([INT4, MXFP4]), E=E, S=S, I=I, O=O,
                    skew=rng.choice([0.0, 1.1]) if E > 1 else 0.0)
    E = rng.choice([16, 64, 160, 256, 384])
    K = rng.choice([2, 4, 6, 8] if op == "router" else [1, 2, 4, 6, 8])  # one choice has weight 1
    most = 8192 // ((2 if dtype == "f32" else 1) * (2 if op == "combine" else 1))
    T, D = _log(rng, 1, most), _width(rng, 64, 7168, 64)
    if op == "router":
        return dict(op=op, dir="gradient", dtype=dtype, T=T, K=K, E=E, D=D,
                    skew=rng.choice([0.0, 1.1]), score=rng.choice([SIGMOID, SQRT_SOFTPLUS]),
                    scale=rng.choice([1.0, 2.5]))
    return dict(op=op, dir=way, dtype=dtype, T=T, K=K, E=E, D=D, skew=rng.choice([0.0, 1.1]),
                padded=rng.choice([0.0, 0.25]))


# ---- inputs -----------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _popularity(gen, E, skew):
    """Log odds of the experts: Zipf of this exponent over a random order."""
    rank = torch.randperm(E, generator=gen, device="cuda")
    return -skew * torch.log1p(rank.float())


def _plan(idx, wt, E):
    """What permute_dev writes for these ids: counts, segment starts, token and
    weight of each sorted row, and the sorted position of each slot."""
    T, K = idx.shape
    live = (idx >= 0) & (wt != 0)
    key = torch.where(live, idx.long() * T + torch.arange(T, device="cuda")[:, None],
                      torch.full_like(idx, E, dtype=torch.long) * T)
    order = torch.argsort(key.reshape(-1), stable=True)
    R = int(live.sum())
    rows = torch.zeros(T * K, dtype=torch.int32, device="cuda")
    rw = torch.zeros(T * K, device="cuda")
    tok_pos = torch.full((T * K,), -1, dtype=torch.int32, device="cuda")
    first = order[:R]
    rows[:R] = (first // K).int()
    rw[:R] = wt.reshape(-1)[first]
    tok_pos[first] = torch.arange(R, dtype=torch.int32, device="cuda")
    nr = torch.bincount(idx[live].long(), minlength=E).int()
    xoff = (torch.cumsum(nr, 0) - nr).int()
    return dict(nr=nr, xoff=xoff, rows=rows, rw=rw, tok_pos=tok_pos.reshape(T, K), R=R)


def _routing(gen, c, logits):
    """Ids, scores and weights of a routed batch."""
    score, scale = c.get("score", SIGMOID), c.get("scale", 1.0)
    s = torch.sigmoid(logits) if score == SIGMOID else torch.log1p(torch.exp(logits)).sqrt()
    pick = logits + _popularity(gen, c["E"], c["skew"]) * 2
    idx = torch.topk(pick, c["K"], dim=1).indices.int()
    mix = s.gather(1, idx.long())
    wt = mix / mix.sum(1, keepdim=True) * scale
    if c.get("padded"):
        off = torch.rand(c["T"], generator=gen, device="cuda") < c["padded"]
        idx = torch.where(off[:, None], torch.full_like(idx, -1), idx)
        wt = torch.where(off[:, None], torch.zeros_like(wt), wt)
    return idx.contiguous(), s, wt.contiguous()


def _pack(w, fmt):
    """Packed codes and scales of f32 weights [rows, columns]."""
    rows, cols = w.shape
    group = 64 if fmt == INT4 else 32
    n = -(-cols // group)
    g = torch.zeros(rows, n * group, device=w.device)
    g[:, :cols] = w
    g = g.reshape(rows, n, group)
    most = g.abs().amax(2)
    if fmt == INT4:
        scales = most / 7
        code = torch.round(g / scales.clamp_min(1e-20)[:, :, None]).clamp(-8, 7) + 8
        code = code.reshape(rows, -1)[:, :cols].to(torch.uint8)
    else:
        scales = torch.ceil(torch.log2((most / 6).clamp_min(1e-20))).clamp(-126, 126)
        a = (g / torch.exp2(scales)[:, :, None]).reshape(rows, -1)[:, :cols]
        edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
        code = torch.bucketize(a.abs(), edges).to(torch.uint8) + 8 * (a < 0).to(torch.uint8)
        scales = (scales + 127).to(torch.uint8)
    if cols % 2:
        code = torch.cat([code, torch.zeros(rows, 1, dtype=torch.uint8, device=w.device)], 1)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), scales.contiguous()


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[c["dtype"]]
    if c["op"] == "matvec":
        E, S, I, O = c["E"], c["S"], c["I"], c["O"]
        parts = [_pack(_normal(gen, O, I) * 0.02, c["fmt"]) for _ in range(E)]
        w, s = torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])
        odds = torch.softmax(_popularity(gen, E, c["skew"]), 0)
        own_e = torch.sort(torch.multinomial(odds, S, replacement=True, generator=gen)).values
        nr = torch.bincount(own_e, minlength=E)
        xoff = torch.cumsum(nr, 0) - nr
        rows_in, rows_out = (I, O) if c["dir"] == "forward" else (O, I)
        return dict(case=c, w=w, s=s, x=_normal(gen, S, rows_in).to(t),
                    y=torch.zeros(S, rows_out, dtype=TYPES[c["out"]], device="cuda"),
                    expert=own_e, place=torch.arange(S, device="cuda") - xoff[own_e],
                    most=int(nr.max()), nr=nr.int(), xoff=xoff.int(),
                    w_table=torch.tensor([a.data_ptr() for a in w], device="cuda"),
                    s_table=torch.tensor([a.data_ptr() for a in s], device="cuda"))
    T, K, E, D = c["T"], c["K"], c["E"], c["D"]
    if c["op"] == "router":
        x = _normal(gen, T, D).to(t)
        router = _normal(gen, E, D) / math.sqrt(D)
        idx, scores, wt = _routing(gen, c, x.float() @ router.T)
        return dict(case=c, x=x, router=router, idx=idx, scores=scores.contiguous(),
                    dwt=_normal(gen, T, K), dx=torch.zeros(T, D, dtype=t, device="cuda"),
                    drouter=torch.zeros(E, D, device="cuda"), plan=_plan(idx, wt, E))
    idx, _, wt = _routing(gen, c, _normal(gen, T, E))
    plan = _plan(idx, wt, E)
    rows = torch.zeros(T * K, D, dtype=t, device="cuda")
    d = dict(case=c, idx=idx, plan=plan)
    if c["op"] == "dispatch":
        if c["dir"] == "forward":
            return dict(d, x=_normal(gen, T, D).to(t), xs=rows)
        rows[:plan["R"]] = _normal(gen, plan["R"], D).to(t)
        return dict(d, dxs=rows, dx=torch.zeros(T, D, dtype=t, device="cuda"))
    rows[:plan["R"]] = _normal(gen, plan["R"], D).to(t)
    if c["dir"] == "forward":
        return dict(d, y=rows, out=torch.zeros(T, D, device="cuda"))
    return dict(d, y=rows, dout=_normal(gen, T, D).to(t), dy=torch.zeros_like(rows),
                dwt=torch.zeros(T, K, device="cuda"))


# ---- one pass ---------------------------------------------------------------
_library = None


def _moe():
    """The library, initialised on the current device as a program does once."""
    global _library
    if _library is None:
        here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(here, "micro-vllm_b200"))
        import mvllm_moe
        mvllm_moe.init(torch.cuda.current_device())
        _library = mvllm_moe
    return _library


def run(state):
    op, way = state["case"]["op"], state["case"]["dir"]
    if op == "dispatch":
        return _dispatch(state) if way == "forward" else _dispatch_gradient(state)
    if op == "combine":
        return _combine(state) if way == "forward" else _combine_gradient(state)
    if op == "router":
        return _router_gradient(state)
    return _matvec(state) if way == "forward" else _matvec_gradient(state)


def _dispatch(s):
    p, xs = s["plan"], s["xs"]
    if own:
        _moe().dispatch_dev(s["x"], p["tok_pos"], xs)
        return xs
    xs[:p["R"]] = s["x"].float()[p["rows"][:p["R"]]].to(xs.dtype)
    return xs


def _dispatch_gradient(s):
    p = s["plan"]
    if own:
        _moe().dispatch_grad_dev(s["dxs"], p["tok_pos"], s["dx"])
        return s["dx"]
    at = p["tok_pos"]
    rows = s["dxs"].float()[at.clamp_min(0)] * (at >= 0)[:, :, None]
    return rows.sum(1).to(s["dx"].dtype)


def _combine(s):
    p = s["plan"]
    if own:
        _moe().combine_dev(s["y"], p["rw"], p["tok_pos"], s["out"])
        return s["out"]
    at = p["tok_pos"]
    w = p["rw"][at.clamp_min(0)] * (at >= 0)
    return (s["y"].float()[at.clamp_min(0)] * w[:, :, None]).sum(1)


def _combine_gradient(s):
    p, R = s["plan"], s["plan"]["R"]
    if own:
        _moe().combine_grad_dev(s["dout"], s["y"], p["rw"], p["tok_pos"], s["idx"], s["dy"],
                                s["dwt"])
        return s["dy"], s["dwt"]
    g = s["dout"].float()[p["rows"][:R]]
    s["dy"][:R] = (g * p["rw"][:R, None]).to(s["dy"].dtype)
    drw = torch.cat([(g * s["y"][:R].float()).sum(1), g.new_zeros(1)])
    return s["dy"], drw[p["tok_pos"]]  # -1, a slot without a row, takes the zero at the end


def _weights(s):
    """The f32 weights [E, O, I] of the packed ones."""
    c, w = s["case"], s["w"]
    code = torch.stack([w & 15, w >> 4], 3).reshape(c["E"], c["O"], -1)[:, :, :c["I"]]
    if c["fmt"] == INT4:
        value, scale, group = code.float() - 8, s["s"], 64
    else:
        e2m1 = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6],
                            device=w.device)
        value, scale, group = e2m1[code.int()], torch.exp2(s["s"].float() - 127), 32
    return value * scale.repeat_interleave(group, 2)[:, :, :c["I"]]


def _product(s, weights):
    """Each row times its expert's matrix: rows padded to one batch per expert."""
    c = s["case"]
    x = s["x"].float()
    batch = x.new_zeros(c["E"], s["most"], x.shape[1])
    batch[s["expert"], s["place"]] = x
    return torch.bmm(batch, weights)[s["expert"], s["place"]].to(s["y"].dtype)


def _matvec(s):
    c = s["case"]
    if own:
        if c["E"] == 1:
            _moe().matvec_q4_dev(c["fmt"], s["x"], s["w"][0], s["s"][0], s["y"])
        else:
            _moe().expert_matvec_q4_dev(c["fmt"], s["x"], s["w_table"], s["s_table"], s["nr"],
                                        s["xoff"], s["y"])
        return s["y"]
    return _product(s, _weights(s).transpose(1, 2))


def _matvec_gradient(s):
    c = s["case"]
    if own:
        if c["E"] == 1:
            _moe().matvec_q4_grad_dev(c["fmt"], s["x"], s["w"][0], s["s"][0], s["y"])
        else:
            _moe().expert_matvec_q4_grad_dev(c["fmt"], s["x"], s["w_table"], s["s_table"],
                                             s["nr"], s["xoff"], s["y"])
        return s["y"]
    return _product(s, _weights(s))


def _router_gradient(s):
    c, p = s["case"], s["plan"]
    if own:
        moe = _moe()
        if "scratch" not in s:  # a program sizes it once and keeps it
            need = moe.route_grad_workspace_bytes(c["T"], c["D"], c["E"], c["K"])
            s["scratch"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        moe.route_grad_dev(s["x"], s["router"], s["idx"], s["scores"], s["dwt"], p["nr"],
                           p["xoff"], p["rows"], p["tok_pos"], s["dx"], s["drouter"],
                           s["scratch"], score_fn=c["score"], routed_scale=c["scale"])
        return s["dx"], s["drouter"]
    at = s["idx"].long()
    mix = s["scores"].gather(1, at)
    total = mix.sum(1, keepdim=True)
    g = s["dwt"] * c["scale"]
    dmix = (g - (g * mix / total).sum(1, keepdim=True)) / total
    if c["score"] == SIGMOID:
        dz = dmix * mix * (1 - mix)
    else:
        dz = dmix * -torch.expm1(-mix * mix) / (2 * mix)
    dlogits = torch.zeros_like(s["scores"]).scatter_(1, at, dz)
    return (dlogits @ s["router"]).to(s["dx"].dtype), dlogits.T @ s["x"].float()


# ---- what one pass cannot do without ----------------------------------------
def work(case):
    c = case
    b = BYTES[c["dtype"]]
    if c["op"] == "matvec":
        per_row = -(-c["I"] // 2) + (-(-c["I"] // 64) * 4 if c["fmt"] == INT4 else -(-c["I"] // 32))
        touched = c["E"] * (1 - (1 - 1 / c["E"]) ** c["S"])  # experts that have a row
        ends = (c["I"], c["O"]) if c["dir"] == "forward" else (c["O"], c["I"])
        return {"bytes": touched * c["O"] * per_row + c["S"] * (ends[0] * b + ends[1] * BYTES[c["out"]]),
                "flops": 2.0 * c["S"] * c["I"] * c["O"]}
    T, K, E, D = c["T"], c["K"], c["E"], c["D"]
    if c["op"] == "router":
        return {"bytes": 2.0 * T * D * b + 8.0 * E * D + 16.0 * T * K, "flops": 4.0 * T * K * D}
    live = T * (1 - c["padded"])
    rows, plan = live * K * D, 4.0 * T * K
    if c["op"] == "dispatch":
        tokens = (live if c["dir"] == "forward" else T) * D
        return {"bytes": (tokens + rows) * b + plan, "flops": 0.0 if c["dir"] == "forward" else rows}
    if c["dir"] == "forward":
        return {"bytes": rows * b + 4.0 * T * D + 2 * plan, "flops": 2.0 * rows}
    return {"bytes": (live * D + 2 * rows) * b + 4 * plan, "flops": 3.0 * rows}


# ---- the definitions in 64 bits ---------------------------------------------
def _decoded(w, s, fmt, I):
    """One matrix of the packed codes, from the formats' bit fields."""
    byte = w.long()
    code = torch.empty(w.shape[0], 2 * w.shape[1], dtype=torch.long, device=w.device)
    code[:, 0::2], code[:, 1::2] = byte % 16, byte // 16
    code = code[:, :I]
    column = torch.arange(I, device=w.device)
    if fmt == INT4:
        return (code - 8).double() * s.double()[:, column // 64]
    exponent, mantissa = (code % 8) // 2, code % 2
    size = torch.where(exponent == 0, mantissa * 0.5,
                       torch.exp2(exponent.double() - 1) * (1 + mantissa * 0.5))
    sign = torch.where(code >= 8, -1.0, 1.0).double()
    return sign * size * torch.exp2(s.double() - 127)[:, column // 32]


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "matvec":
        out = torch.zeros(c["S"], s["y"].shape[1], dtype=torch.float64, device="cuda")
        starts, counts = s["xoff"].tolist(), s["nr"].tolist()
        for e in range(c["E"]):
            if counts[e]:
                m = _decoded(s["w"][e], s["s"][e], c["fmt"], c["I"])
                part = slice(starts[e], starts[e] + counts[e])
                out[part] = s["x"][part].double() @ (m.T if c["dir"] == "forward" else m)
        return out
    p = s["plan"]
    R, T, K = p["R"], c["T"], c["K"]
    if c["op"] == "router":
        ids = s["idx"].long()
        top = torch.gather(s["scores"], 1, ids).double()
        norm = top.sum(1)
        dots = (s["dwt"].double() * top).sum(1) / norm
        back = c["scale"] * (s["dwt"].double() - dots[:, None]) / norm[:, None]
        slope = top - top ** 2 if c["score"] == SIGMOID else (1 - torch.exp(-top ** 2)) / top / 2
        full = torch.zeros(T, c["E"], dtype=torch.float64, device="cuda")
        full[torch.arange(T, device="cuda")[:, None], ids] = back * slope
        return full @ s["router"].double(), full.T @ s["x"].double()
    token = p["rows"][:R].long()
    if c["op"] == "dispatch":
        if c["dir"] == "forward":
            out = torch.zeros(T * K, c["D"], dtype=torch.float64, device="cuda")
            out[:R] = s["x"][token].double()
            return out
        out = torch.zeros(T, c["D"], dtype=torch.float64, device="cuda")
        return out.index_add_(0, token, s["dxs"][:R].double())
    if c["dir"] == "forward":
        out = torch.zeros(T, c["D"], dtype=torch.float64, device="cuda")
        return out.index_add_(0, token, s["y"][:R].double() * p["rw"][:R].double()[:, None])
    seen = s["dout"].double()[token]
    dw = torch.zeros(T, K, dtype=torch.float64, device="cuda")
    dots = (seen * s["y"][:R].double()).sum(1)
    for k in range(K):
        at = p["tok_pos"][:, k].long()
        dw[at >= 0, k] = dots[at[at >= 0]]
    dy = torch.zeros(T * K, c["D"], dtype=torch.float64, device="cuda")
    dy[:R] = seen * p["rw"][:R].double()[:, None]
    return dy, dw

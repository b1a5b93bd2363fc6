"""Plain 64-bit forms of the routed layer's separate steps (torch, CPU or GPU)
and the inputs their tests share."""
import torch

INT4, MXFP4 = 4, 7
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def half_step(dtype):
    """The largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def decode(w, s, fmt, I):
    """f64 weights [O, I] of packed codes w and scales s."""
    code = torch.stack([w & 15, w >> 4], -1).reshape(w.shape[0], -1)[:, :I].long()
    group = 64 if fmt == INT4 else 32
    if fmt == INT4:
        value, scale = (code - 8).double(), s.double()
    else:
        table = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=w.device)
        value, scale = table[code], torch.exp2(s.double() - 127)
        scale = torch.where(s == 0, torch.zeros_like(scale), scale)  # code 0 decodes to 0
    return value * scale.repeat_interleave(group, 1)[:, :I]


def packed(gen, fmt, O, I, dev, spread=6):
    """Random codes (all of them) and scales over a range of magnitudes."""
    w = torch.randint(0, 256, (O, (I + 1) // 2), generator=gen, dtype=torch.uint8)
    if fmt == INT4:
        s = torch.rand(O, (I + 63) // 64, generator=gen) * 0.01 + 1e-4
        s *= torch.exp2(torch.randint(-spread, spread + 1, s.shape, generator=gen).float())
    else:
        s = torch.randint(119 - spread, 119 + spread + 1, (O, (I + 31) // 32), generator=gen,
                          dtype=torch.uint8)
    return w.to(dev), s.to(dev)


def slots(plan):
    """(token, slot, position) of every slot that has a row."""
    t, j = torch.nonzero(plan["tok_pos"] >= 0, as_tuple=True)
    return t, j, plan["tok_pos"][t, j].long()


def combine(y, rw, plan, T):
    """out[t] = sum rw[p] y[p], and the sum of magnitudes beside it."""
    t, _, p = slots(plan)
    term = y.double()[p] * (rw.double()[p, None] if rw is not None else 1.0)
    out = torch.zeros(T, y.shape[1], dtype=torch.float64, device=y.device)
    return out.index_add(0, t, term), out.index_add(0, t, term.abs())


def route_weights(z, idx, score_fn, scale):
    """The weights [T, K] of given ids from f64 logits, and the scores."""
    s = torch.sigmoid(z) if score_fn == 0 else torch.nn.functional.softplus(z).sqrt()
    live = idx >= 0
    m = s.gather(1, idx.clamp_min(0).long()) * live
    total = m.sum(1, keepdim=True)
    return m / torch.where(total > 0, total, torch.ones_like(total)) * scale, s


def route_grad(x, router, idx, scores, dwt, score_fn, scale):
    """dx, drouter and the dense gradient of the logits, in f64."""
    live = (idx >= 0) & (idx < router.shape[0])
    at = idx.clamp(0, router.shape[0] - 1).long()
    m = scores.double().gather(1, at).clamp_min(0) * live
    M = m.sum(1, keepdim=True)
    g = dwt.double() * scale
    dm = torch.where((m > 0), (g - (g * m).sum(1, keepdim=True) / M) / M, torch.zeros_like(m))
    slope = m * (1 - m) if score_fn == 0 else -torch.expm1(-m * m) / (2 * m.clamp_min(1e-300))
    dz = torch.zeros(scores.shape, dtype=torch.float64, device=x.device)
    dz.scatter_add_(1, at, torch.where(live, dm * slope, torch.zeros_like(dm)))
    return dz @ router.double(), dz.T @ x.double(), dz


def route_grad_bounds(x, router, idx, scores, dwt, score_fn, scale):
    """The magnitudes that the roundings of dz scale with, carried through the
    two products: |dz| with every difference taken as a sum."""
    live = (idx >= 0) & (idx < router.shape[0])
    at = idx.clamp(0, router.shape[0] - 1).long()
    m = scores.double().gather(1, at).clamp_min(0) * live
    M = m.sum(1, keepdim=True)
    g = (dwt.double() * scale).abs()
    dm = torch.where((m > 0), (g + (g * m).sum(1, keepdim=True) / M) / M, torch.zeros_like(m))
    slope = m * (1 + m) if score_fn == 0 else (-torch.expm1(-m * m) / (2 * m.clamp_min(1e-300)))
    dz = torch.zeros(scores.shape, dtype=torch.float64, device=x.device)
    dz.scatter_add_(1, at, torch.where(live, dm * slope, torch.zeros_like(dm)))
    return dz @ router.double().abs(), dz.T @ x.double().abs()


def cpu_plan(idx, wt, E, n_shared=0):
    """The permutation's outputs from its definition, row by row."""
    T, K = idx.shape
    KK = K + n_shared
    seg = [[] for _ in range(E + n_shared)]
    for t in range(T):
        for k in range(K):
            e = int(idx[t, k])
            if not 0 <= e < E or e in idx[t, :k].tolist():
                continue
            w = float(wt[t][idx[t] == e].sum())
            if w != 0:
                seg[e].append((t, k, w))
        if n_shared:
            seg[E].append((t, K, 1.0))
    rows, rw, tok_pos, nr = [], [], torch.full((T, KK), -1, dtype=torch.int32), []
    for part in seg:
        nr.append(len(part))
        for t, k, w in part:
            tok_pos[t, k] = len(rows)
            rows.append(t)
            rw.append(w)
    nr = torch.tensor(nr, dtype=torch.int32)
    return dict(nr=nr, xoff=(torch.cumsum(nr, 0) - nr).int(),
                rows=torch.tensor(rows, dtype=torch.int32), rw=torch.tensor(rw),
                tok_pos=tok_pos, n=len(rows))


def device_plan(moe, idx, wt, E, n_shared=0):
    """The permutation from the library."""
    T, K = idx.shape
    KK, i32 = K + n_shared, dict(dtype=torch.int32, device="cuda")
    p = dict(nr=torch.zeros(E + n_shared, **i32), xoff=torch.zeros(E + n_shared, **i32),
             rows=torch.zeros(T * KK, **i32), rw=torch.zeros(T * KK, device="cuda"),
             tok_pos=torch.zeros(T, KK, **i32), n_rows=torch.zeros(1, **i32))
    ws = torch.empty(moe.permute_workspace_bytes(T, K, E, n_shared), dtype=torch.uint8,
                     device="cuda")
    moe.permute_dev(idx, wt, E, n_shared, p["nr"], p["xoff"], p["rows"], p["rw"], p["tok_pos"],
                    p["n_rows"], ws)
    return p


def routing(gen, T, K, E, dropped=0.2, repeats=False):
    """Ids (some tokens with none at all, some slots -1) and weights."""
    idx = torch.stack([torch.randperm(E, generator=gen)[:K] for _ in range(T)]).int()
    wt = torch.rand(T, K, generator=gen) + 0.1
    idx[torch.rand(T, K, generator=gen) < dropped / 2] = -1
    idx[torch.rand(T, generator=gen) < dropped] = -1
    if repeats and K > 1:
        idx[::3, K - 1] = idx[::3, 0]
    return idx, wt

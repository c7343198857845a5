"""Cases of the sorted-token operators and the 4-bit products: what is measured, the plain torch
form of each operator, and its definition in 64 bits.

op "permute"           ids [T, k] and rows x [T, H] -> rows sorted by expert, and the plan
op "permute_backward"  gradient of the sorted rows -> gradient of x
op "combine"           expert rows back to tokens with the routing weights (+ a shared expert's rows)
op "combine_backward"  gradient of the combined rows -> gradients of the expert rows and the weights
op "q4_dense"          y = x W^T, W in 4-bit codes with group scales
op "q4_experts"        the same for rows sorted by expert, each with its expert's matrix
op "q4_gate_up"        two such products of the unsorted rows and their clamped SwiGLU

4-bit matrices: codes uint8 [.., N, K/2] (element 2j of a row in the low nibble of byte j), scales
[.., K/G, N] fp16 or bf16, zero points uint8 [.., K/G, N] or none (8): w = s * (q - z).
"""

import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
SORTED = ("permute", "permute_backward", "combine", "combine_backward")
LIMIT = 10.0


def listed():
    glm = dict(k=8, E=256, H=6144)          # the layer shape of the C1-C4 configurations
    small = dict(k=4, E=16)                 # the C0 gate's routing
    return [
        # one decoded token: every microsecond here is latency
        dict(name="permute_t1", op="permute", T=1, dtype="bf16", dropped=0.0, skew=0.0, **glm),
        # the largest prefill batch, Zipf-skewed experts
        dict(name="permute_t8192", op="permute", T=8192, dtype="bf16", dropped=0.0, skew=1.1, **glm),
        # a padded fp16 batch (a third of the lanes carry no expert) with rows of an odd length
        dict(name="permute_odd", op="permute", T=1021, H=1023, dtype="f16", dropped=0.3, skew=0.0, **small),
        # training: the gradient of a prefill-sized batch, and a small fp32 one
        dict(name="permute_back_t4096", op="permute_backward", T=4096, dtype="bf16", dropped=0.0, skew=1.1, **glm),
        dict(name="permute_back_t33", op="permute_backward", T=33, H=1024, dtype="f32", dropped=0.3, skew=0.0, **small),
        # bf16 expert rows back to their tokens, with the shared expert: prefill and decode
        dict(name="combine_t4096", op="combine", T=4096, dtype="bf16", shared=True, dropped=0.0, skew=1.1, **glm),
        # gradients of the way back: a full training batch, and rows of an odd length with dropped lanes
        dict(name="combine_back_t8192", op="combine_backward", T=8192, dtype="bf16", dropped=0.0, skew=1.1, **glm),
        dict(name="combine_back_odd", op="combine_backward", T=257, H=1023, dtype="f32", dropped=0.3, skew=0.0, **small),
        # an output head for one token: as much weight traffic as a 4-bit product meets
        dict(name="q4_head_n1", op="q4_dense", n=1, N=131072, K=6144, G=128, dtype="bf16", sdtype="bf16", zeros=False),
        # one dense expert matrix for a small batch, with zero points
        dict(name="q4_dense_n16", op="q4_dense", n=16, N=2048, K=6144, G=64, dtype="f16", sdtype="f16", zeros=True),
        # one token through its experts' gate and up matrices
        dict(name="q4_gate_up_t1", op="q4_gate_up", T=1, k=8, E=256, N=2048, K=6144, G=32, dtype="bf16",
             sdtype="f16", zeros=False, skew=0.0),
        # a decode batch through the experts' down matrices
        dict(name="q4_down_t32", op="q4_experts", T=32, k=8, E=256, N=6144, K=2048, G=64, dtype="bf16",
             sdtype="bf16", zeros=True, skew=0.0),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(SORTED + ("q4_dense", "q4_experts", "q4_gate_up"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op in SORTED:
        H = _spread(rng, 64, 8192)
        if rng.random() < 0.6:
            H = max(64, H // 64 * 64)
        E = _spread(rng, 4, 512)
        k = min(E, rng.choice((1, 2, 4, 6, 8, 8, 16)))
        T = min(_spread(rng, 1, 16384), max(1, 8192 * 8 * 6144 * 2 // (k * H * SIZE[dtype])))
        c = dict(op=op, T=T, k=k, E=E, H=H, dtype=dtype, dropped=rng.choice((0.0, 0.0, 0.3)),
                 skew=rng.choice((0.0, 1.1)))
        if op == "combine":
            c["shared"] = rng.random() < 0.5
        return c
    G = rng.choice((32, 64, 128))
    K = G * _spread(rng, max(1, 256 // G), 8192 // G)
    N = 16 * _spread(rng, 16, 512)
    c = dict(op=op, N=N, K=K, G=G, dtype=dtype, sdtype=rng.choice(("bf16", "f16")), zeros=rng.random() < 0.5)
    if op == "q4_dense":
        return dict(c, n=_spread(rng, 1, 256))
    E = _spread(rng, 4, max(4, min(256, 256 * 2048 * 6144 // (N * K))))
    k = min(E, rng.choice((1, 2, 4, 8)))
    return dict(c, T=_spread(rng, 1, 64), k=k, E=E, skew=rng.choice((0.0, 1.1)))


# ------------------------------------------------------------------------------------ inputs
def _ids(c, g, dev):
    """Distinct expert ids a token; skew s > 0 draws them with popularity rank^-s."""
    T, E, k = c["T"], c["E"], c["k"]
    score = -torch.log(-torch.log(torch.rand(T, E, generator=g, device=dev).clamp_(1e-12, 1 - 1e-7)))
    if c["skew"]:
        score += -c["skew"] * torch.log1p(torch.randperm(E, generator=g, device=dev).float())
    idx = score.topk(k, dim=1).indices.to(torch.int32)
    if c.get("dropped"):
        idx[torch.rand(T, k, generator=g, device=dev) < c["dropped"]] = -1
    return idx


def _plan(idx, E):
    """(perm_tok, pos_of, offsets, counts) by a stable sort of the flat lanes."""
    T, k = idx.shape
    flat = idx.reshape(-1).long()
    key, order = torch.where(flat < 0, E, flat).sort(stable=True)
    counts = torch.zeros(E + 1, dtype=torch.long, device=idx.device).index_add_(0, key, torch.ones_like(key))[:E]
    offsets = torch.zeros(E + 1, dtype=torch.long, device=idx.device)
    offsets[1:] = counts.cumsum(0)
    pos = torch.empty_like(order)
    pos[order] = torch.arange(T * k, device=idx.device)
    pos_of = torch.where(flat < 0, -1, pos)
    perm_tok = torch.where(key < E, order // k, -1)
    return tuple(v.to(torch.int32) for v in (perm_tok, pos_of, offsets, counts))


def _randn(shape, dtype, g, dev):
    return torch.randn(shape, generator=g, device=dev, dtype=torch.float32 if dtype == torch.float32 else dtype)


def _q4(c, lead, g, dev):
    """Codes, scales and zero points of stacked matrices: weights of about N(0, 0.02)."""
    N, K, G = c["N"], c["K"], c["G"]
    q = torch.randint(0, 256, (*lead, N, K // 2), generator=g, device=dev, dtype=torch.uint8)
    s = (0.002 + 0.004 * torch.rand((*lead, K // G, N), generator=g, device=dev)).to(DT[c["sdtype"]])
    z = torch.randint(5, 11, (*lead, K // G, N), generator=g, device=dev, dtype=torch.uint8) if c["zeros"] else None
    return q, s, z


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = DT[c["dtype"]]
    if c["op"] in SORTED:
        T, k, E, H = c["T"], c["k"], c["E"], c["H"]
        idx = _ids(c, g, dev)
        st = dict(case=c, idx=idx)
        if c["op"] == "permute":
            st["x"] = _randn((T, H), dt, g, dev)
            st["xs"] = torch.zeros((T * k, H), dtype=dt, device=dev)
            return st
        st["perm_tok"], st["pos_of"], st["offsets"], _ = _plan(idx, E)
        if c["op"] == "permute_backward":
            st["dxs"] = _randn((T * k, H), dt, g, dev)
            return st
        st["y"] = _randn((T * k, H), dt, g, dev)
        w = torch.sigmoid(torch.randn((T, k), generator=g, device=dev))
        st["w"] = w / w.sum(1, keepdim=True) * 2.5
        if c["op"] == "combine":
            st["y_shared"] = _randn((T, H), dt, g, dev) if c["shared"] else None
        else:
            st["dout"] = _randn((T, H), dt, g, dev)
            st["dy"] = torch.zeros((T * k, H), dtype=dt, device=dev)
        return st
    if c["op"] == "q4_dense":
        return dict(case=c, x=_randn((c["n"], c["K"]), dt, g, dev), w=_q4(c, (), g, dev))
    idx = _ids(c, g, dev)
    perm_tok, _, offsets, _ = _plan(idx, c["E"])
    st = dict(case=c, perm_tok=perm_tok, offsets=offsets, w=_q4(c, (c["E"],), g, dev))
    if c["op"] == "q4_gate_up":
        st["up"] = _q4(c, (c["E"],), g, dev)
        st["x"] = _randn((c["T"], c["K"]), dt, g, dev)
    else:
        st["x"] = _randn((c["T"] * c["k"], c["K"]), dt, g, dev)
    return st


# ------------------------------------------------------------------------------------ plain forms
def _dequant(q, s, z, G):
    """fp32 [.., N, K] of codes, scales and zero points."""
    c = torch.stack((q & 15, q >> 4), dim=-1).flatten(-2).float()
    c = c.unflatten(-1, (-1, G))
    c = c - (8.0 if z is None else z.float().transpose(-1, -2).unsqueeze(-1))
    return (c * s.float().transpose(-1, -2).unsqueeze(-1)).flatten(-2)


def _experts(x, w, c, expert, row):
    """y[r] = W[expert[r]] x[r] in fp32; row[r]: the row's place among its expert's rows."""
    if x.shape[0] <= c["E"]:  # each row's own copy of its matrix
        m = _dequant(w[0][expert], w[1][expert], None if w[2] is None else w[2][expert], c["G"])
        return torch.bmm(m, x.float().unsqueeze(-1)).squeeze(-1)
    pad = torch.zeros((c["E"], c["T"], c["K"]), device=x.device)
    pad[expert, row] = x.float()
    return torch.bmm(pad, _dequant(*w, c["G"]).transpose(1, 2))[expert, row]


def _rows(st, c):
    """(expert, place among the expert's rows) of each sorted row."""
    r = torch.arange(c["T"] * c["k"], device=st["x"].device)
    off = st["offsets"].long()
    e = torch.searchsorted(off[1:].contiguous(), r, right=True)
    return e, r - off[e]


def _plain(st):
    c = st["case"]
    op, dt = c["op"], DT[c["dtype"]]
    if op == "permute":
        plan = _plan(st["idx"], c["E"])
        xs = st["x"][plan[0].clamp(min=0).long()]
        return {"xs": torch.where(plan[0].unsqueeze(1) >= 0, xs, torch.zeros((), dtype=dt, device=xs.device)),
                "perm_tok": plan[0], "pos_of": plan[1], "offsets": plan[2], "counts": plan[3]}
    if op in SORTED:
        T, k, H = c["T"], c["k"], c["H"]
        pos = st["pos_of"].long()
        kept = (pos >= 0).view(T, k)
        at = pos.clamp(min=0)
        if op == "permute_backward":
            v = st["dxs"].float()[at].view(T, k, H)
            return {"dx": torch.where(kept.unsqueeze(-1), v, 0.0).sum(1).to(dt)}
        v = st["y"].float()[at].view(T, k, H)
        if op == "combine":
            out = torch.where(kept.unsqueeze(-1), v * st["w"].unsqueeze(-1), 0.0).sum(1)
            return {"out": (out if st["y_shared"] is None else out + st["y_shared"].float()).to(dt)}
        d = st["dout"].float().unsqueeze(1)
        dy = torch.zeros((T * k + 1, H), dtype=dt, device=pos.device)
        dy[torch.where(pos < 0, T * k, pos)] = (d * st["w"].unsqueeze(-1)).to(dt).view(T * k, H)
        return {"dy": dy[:T * k], "dw": torch.where(kept, (d * v).sum(-1), 0.0)}
    if op == "q4_dense":
        return {"y": (st["x"].float() @ _dequant(*st["w"], c["G"]).T).to(dt)}
    e, row = _rows(st, c)
    if op == "q4_experts":
        return {"y": _experts(st["x"], st["w"], c, e, row).to(dt)}
    x = st["x"][st["perm_tok"].long()]
    g = _experts(x, st["w"], c, e, row).clamp(max=LIMIT)
    u = _experts(x, st["up"], c, e, row).clamp(-LIMIT, LIMIT)
    return {"y": (g / (1.0 + torch.exp(-g)) * u).to(dt)}


# ------------------------------------------------------------------------------------ the framework's calls
def _own(st):
    from vybforge_b200 import moe

    c = st["case"]
    op = c["op"]
    if op == "permute":
        xs, plan = moe.permute(st["x"], st["idx"], c["E"], out=st["xs"])
        return {"xs": xs, "perm_tok": plan.perm_tok, "pos_of": plan.pos_of, "offsets": plan.offsets,
                "counts": plan.counts}
    if op == "permute_backward":
        return {"dx": moe.permute_backward(st["dxs"], st["pos_of"], c["T"], c["k"])}
    if op == "combine":
        return {"out": moe.combine(st["y"], st["pos_of"], st["w"], c["T"], c["k"], y_shared=st["y_shared"],
                                   out_dtype=DT[c["dtype"]])}
    if op == "combine_backward":
        dy, dw = moe.combine_backward(st["dout"], st["y"], st["pos_of"], st["w"], c["T"], c["k"], dy=st["dy"])
        return {"dy": dy, "dw": dw}
    w = moe.Q4Matrix(*st["w"])
    if op == "q4_dense":
        return {"y": moe.q4_matvec(st["x"], w)}
    if op == "q4_experts":
        return {"y": moe.q4_matvec(st["x"], w, offsets=st["offsets"])}
    return {"y": moe.q4_matvec(st["x"], w, up=moe.Q4Matrix(*st["up"]), limit=LIMIT, offsets=st["offsets"],
                               row_map=st["perm_tok"])}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------ work
def work(case):
    c = case
    s = SIZE[c["dtype"]]
    if c["op"] in SORTED:
        lanes = c["T"] * c["k"]
        rows = lanes * (1.0 - c["dropped"])
        one = c["T"] * c["H"] * s
        if c["op"] == "permute":
            return {"bytes": one + rows * c["H"] * s + 12 * lanes + 8 * c["E"], "flops": 0}
        if c["op"] == "permute_backward":
            return {"bytes": one + rows * c["H"] * s + 4 * lanes, "flops": rows * c["H"]}
        if c["op"] == "combine":
            return {"bytes": one * (2 if c["shared"] else 1) + rows * c["H"] * s + 8 * lanes,
                    "flops": 2 * rows * c["H"]}
        return {"bytes": one + 2 * rows * c["H"] * s + 12 * lanes, "flops": 3 * rows * c["H"]}
    N, K = c["N"], c["K"]
    matrix = N * K // 2 + N * (K // c["G"]) * (3 if c["zeros"] else 2)
    if c["op"] == "q4_dense":
        return {"bytes": matrix + c["n"] * (N + K) * s, "flops": 2 * c["n"] * N * K}
    rows = c["T"] * c["k"]
    touched = c["E"] * (1.0 - (1.0 - c["k"] / c["E"]) ** c["T"])  # expected, ids without skew
    if c["op"] == "q4_experts":
        return {"bytes": touched * matrix + rows * (N + K) * s + 4 * c["E"], "flops": 2 * rows * N * K}
    return {"bytes": 2 * touched * matrix + rows * N * s + c["T"] * K * s + 4 * (rows + c["E"]),
            "flops": 4 * rows * N * K}


# ------------------------------------------------------------------------------------ definitions in 64 bits
def _matrix64(w, e, G):
    """fp64 [N, K] of matrix e (None: the only one)."""
    q, s, z = (None if v is None else v if e is None else v[e] for v in w)
    m = torch.empty((q.shape[0], 2 * q.shape[1]), dtype=torch.float64, device=q.device)
    m[:, 0::2] = (q % 16).double()
    m[:, 1::2] = (q // 16).double()
    m -= 8.0 if z is None else z.double().T.repeat_interleave(G, dim=1)
    return m.mul_(s.double().T.repeat_interleave(G, dim=1))


def exact(case, seed):
    c, st = case, prepare(case, seed)
    op = c["op"]
    if op in SORTED:
        T, k, E, H = c["T"], c["k"], c["E"], c["H"]
        flat = st["idx"].reshape(-1).long()
        # rank of a lane: kept lanes of lower experts, then earlier lanes of its own
        hot = torch.zeros((T * k, E), dtype=torch.int32, device=flat.device)
        kept = (flat >= 0).nonzero().squeeze(1)
        hot[kept, flat[kept]] = 1
        counts = hot.sum(0)
        offsets = torch.cat((counts.new_zeros(1), counts.cumsum(0)))
        pos = torch.full((T * k,), -1, dtype=torch.long, device=flat.device)
        pos[kept] = offsets[flat[kept]] + hot.cumsum(0)[kept, flat[kept]] - 1
        tok = torch.arange(T, device=flat.device).repeat_interleave(k)
        if op == "permute":
            xs = torch.zeros((T * k, H), dtype=torch.float64, device=flat.device)
            xs[pos[kept]] = st["x"].double()[tok[kept]]
            perm = torch.full_like(pos, -1)
            perm[pos[kept]] = tok[kept]
            return {"xs": xs, "perm_tok": perm, "pos_of": pos, "offsets": offsets, "counts": counts}
        if op == "permute_backward":
            dx = torch.zeros((T, H), dtype=torch.float64, device=flat.device)
            return {"dx": dx.index_add_(0, tok[kept], st["dxs"][pos[kept]].double())}
        wl = st["w"].reshape(-1).double()
        if op == "combine":
            out = torch.zeros((T, H), dtype=torch.float64, device=flat.device)
            if st["y_shared"] is not None:
                out += st["y_shared"].double()
            return {"out": out.index_add_(0, tok[kept], st["y"][pos[kept]].double() * wl[kept, None])}
        dy = torch.zeros((T * k, H), dtype=torch.float64, device=flat.device)
        d = st["dout"].double()[tok[kept]]
        dy[pos[kept]] = d * wl[kept, None]
        dw = torch.zeros(T * k, dtype=torch.float64, device=flat.device)
        dw[kept] = torch.einsum("rh,rh->r", d, st["y"][pos[kept]].double())
        return {"dy": dy, "dw": dw.view(T, k)}
    if op == "q4_dense":
        parts = [slice(a, a + 16384) for a in range(0, c["N"], 16384)]
        w = st["w"]
        cut = [(w[0][p], w[1][:, p], None if w[2] is None else w[2][:, p]) for p in parts]
        return {"y": torch.cat([st["x"].double() @ _matrix64(v, None, c["G"]).T for v in cut], dim=1)}
    off = st["offsets"].tolist()
    y = torch.empty((c["T"] * c["k"], c["N"]), dtype=torch.float64, device="cuda")
    for e in range(c["E"]):
        rows = slice(off[e], off[e + 1])
        if off[e] == off[e + 1]:
            continue
        if op == "q4_experts":
            y[rows] = st["x"][rows].double() @ _matrix64(st["w"], e, c["G"]).T
            continue
        x = st["x"][st["perm_tok"][rows].long()].double()
        a = (x @ _matrix64(st["w"], e, c["G"]).T).clamp(max=LIMIT)
        b = (x @ _matrix64(st["up"], e, c["G"]).T).clamp(-LIMIT, LIMIT)
        y[rows] = a * torch.sigmoid(a) * b
    return {"y": y}

"""The operators of the 8-bit floating point expert layer and of the token sort: their cases, their plain forms in
elementary torch operations, and their values in 64 bits.

  linear   y = x W^T with W in e4m3 (4 exponent, 3 mantissa bits) and one float32 scale for each 128 x 128 block; each
           row of x is quantised to e4m3 in groups of 128 with a power-of-two scale. Prompts and single tokens.
  experts  the routed expert layer on such tables: y = sum_j w_j Wd_e swiglu(Wg_e x, Wu_e x), e = idx_j, the SwiGLU
           output quantised like x before the down product. Prompts and single tokens.
  sort     tokens copied into expert order (rows of each expert in blocks of tm, padding rows zero), forward and backward.
  join     the rows back in token order, weighted and summed over the token's experts, forward and backward to the rows
           and to the weights.

A group's scale is the least power of two s (at least 2^-100) with max|x| <= 448 s, so that x / s is exact; a group with
an infinity or a NaN has the scale NaN and stands for NaN.
"""
import math
import os
import sys

import torch

own = False

LIMIT = 10.0                    # the SwiGLU clamp of the layer tests
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
LEAST = 448.0 * 2.0 ** -100     # the group maximum below which the scale stays at 2^-100


def listed():
    return [
        # one decoded token through the fused QKV projection: the latency of a single row
        {"name": "linear 1 token", "op": "linear", "N": 1, "K": 5120, "rows": 12288, "x": "bf16", "y": "bf16"},
        # a decode batch through the same projection
        {"name": "linear 64 tokens", "op": "linear", "N": 64, "K": 5120, "rows": 12288, "x": "bf16", "y": "bf16"},
        # a ragged piece through a matrix whose last blocks are cut, float32 in and out
        {"name": "linear odd sizes", "op": "linear", "N": 77, "K": 5000, "rows": 1411, "x": "fp32", "y": "fp32"},
        # a prompt of 4096 tokens through the attention output projection
        {"name": "linear 4096 tokens", "op": "linear", "N": 4096, "K": 12288, "rows": 5120, "x": "bf16", "y": "bf16"},
        # one decoded token through the routed experts
        {"name": "experts 1 token", "op": "experts", "N": 1, "E": 160, "H": 5120, "I": 1536, "k": 8, "empty": 0.0},
        # a decode batch of 8
        {"name": "experts 8 tokens", "op": "experts", "N": 8, "E": 160, "H": 5120, "I": 1536, "k": 8, "empty": 0.0},
        # a padded batch over a rank's share of experts, with sizes that end inside a block and empty slots
        {"name": "experts odd sizes", "op": "experts", "N": 141, "E": 20, "H": 2000, "I": 700, "k": 4, "empty": 0.1},
        # a prompt of 4096 tokens
        {"name": "experts 4096 tokens", "op": "experts", "N": 4096, "E": 160, "H": 5120, "I": 1536, "k": 8, "empty": 0.0},
        # a training micro-batch of few tokens, odd width, blocks of 16 rows, some slots empty
        {"name": "sort 50 tokens", "op": "sort", "N": 50, "E": 20, "H": 1411, "k": 4, "tm": 16, "x": "fp16", "empty": 0.1},
        # a training batch of 4096 tokens
        {"name": "sort 4096 tokens", "op": "sort", "N": 4096, "E": 160, "H": 5120, "k": 8, "tm": 1, "x": "bf16", "empty": 0.0},
        # the small batch's way back, float32
        {"name": "join 50 tokens", "op": "join", "N": 50, "E": 20, "H": 1411, "k": 4, "tm": 16, "x": "fp32", "empty": 0.1},
        # the large batch's way back
        {"name": "join 4096 tokens", "op": "join", "N": 4096, "E": 160, "H": 5120, "k": 8, "tm": 1, "x": "bf16", "empty": 0.0},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["linear", "experts", "sort", "join"])
    if op == "linear":
        rows, K = _log(rng, 200, 16000), _log(rng, 200, 14000)
        if rng.random() < 0.5:
            rows, K = -(-rows // 128) * 128, -(-K // 128) * 128
        N = min(_log(rng, 1, 8192), 4096 * 5120 * 12288 // (rows * K))
        t = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return {"op": op, "N": max(1, N), "K": K, "rows": rows, "x": t, "y": t}
    k = rng.choice([1, 2, 4, 6, 8])
    if op == "experts":
        E, H, I = _log(rng, 8, 160), _log(rng, 300, 5120), _log(rng, 200, 2048)
        if rng.random() < 0.5:
            H, I = -(-H // 128) * 128, -(-I // 128) * 128
        N = min(_log(rng, 1, 8192), 4096 * 8 * 5120 * 1536 // (k * H * I))
        return {"op": op, "N": max(1, N), "E": E, "H": H, "I": I, "k": k, "empty": rng.choice([0.0, 0.0, 0.2])}
    E, H = _log(rng, 8, 256), _log(rng, 64, 8192)
    if rng.random() < 0.5:
        H = -(-H // 64) * 64
    t = rng.choice(["bf16", "fp16", "fp32"])
    N = min(_log(rng, 1, 16384), 4096 * 8 * 5120 * 2 // (k * H * (4 if t == "fp32" else 2)))
    return {"op": op, "N": max(1, N), "E": E, "H": H, "k": k, "tm": rng.choice([1, 1, 8, 32, 128]), "x": t,
            "empty": rng.choice([0.0, 0.0, 0.2])}


def _table(g, lead, rows, K):
    """Weights N(0, 0.02) as a checkpoint holds them: e4m3 values whose row stride is a multiple of 16 bytes, and a
    float32 scale for each 128 x 128 block (the last ones cut)."""
    rb, kb = -(-rows // 128), -(-K // 128)
    w = torch.zeros(lead + (rb * 128, kb * 128), device="cuda")
    w[..., :rows, :K] = torch.randn(lead + (rows, K), device="cuda", generator=g) * 0.02
    w = w.view(lead + (rb, 128, kb, 128))
    s = w.abs().amax(dim=(-3, -1)) / 448.0
    w = (w / s[..., :, None, :, None]).view(lead + (rb * 128, kb * 128))[..., :rows, :K]
    q = torch.zeros(lead + (rows, -(-K // 16) * 16), dtype=torch.uint8, device="cuda")
    q[..., :K] = w.to(E4M3).view(torch.uint8)
    return q.view(E4M3)[..., :K], s


def _activations(g, N, K, dtype):
    """N(0, 1) with some rows larger, as behind a norm with learned gains."""
    x = torch.randn(N, K, device="cuda", generator=g)
    return (x * torch.exp(torch.randn(N, 1, device="cuda", generator=g))).to(dtype)


def _routing(g, N, E, k, empty):
    """Top-k of random logits, softmax over the chosen; some slots empty (negative), as in a padded batch."""
    v, idx = torch.randn(N, E, device="cuda", generator=g).topk(k, dim=1)
    w = torch.softmax(v, dim=1)
    if empty:
        gone = torch.rand(N, k, device="cuda", generator=g) < empty
        idx = torch.where(gone, -1, idx)
    return idx.to(torch.int32).contiguous(), w.contiguous()


def _rows(T, k, E, tm):
    """Rows of the sorted order: all slots, and where blocks are padded room for each expert's last block."""
    return T * k if tm == 1 else (-(-T * k // tm) + E) * tm


def _sorted_order(idx, E, tm):
    """(tok_row [R], row_slot [T, k]): the token of each sorted row (-1: padding) and each slot's row (-1: empty)."""
    T, k = idx.shape
    R = _rows(T, k, E, tm)
    e = torch.where(idx < 0, E, idx.long()).flatten()
    counts = torch.zeros(E + 1, dtype=torch.long, device=idx.device).index_add_(0, e, torch.ones_like(e))
    padded = (counts + tm - 1) // tm * tm
    start, first = padded.cumsum(0) - padded, counts.cumsum(0) - counts
    order = e.argsort(stable=True)
    rank = torch.empty_like(order)
    rank[order] = torch.arange(T * k, device=idx.device)
    row = torch.where(e < E, start[e] + rank - first[e], R)
    tok = torch.full((R + 1,), -1, dtype=torch.int32, device=idx.device)
    tok[row] = (torch.arange(T * k, device=idx.device) // k).to(torch.int32)
    return tok[:R].contiguous(), torch.where(row < R, row, -1).to(torch.int32).view(T, k)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    N, op = case["N"], case["op"]
    st = dict(case)
    if op == "linear":
        st["q"], st["s"] = _table(g, (), case["rows"], case["K"])
        st["xv"] = _activations(g, N, case["K"], TYPES[case["x"]])
        return st
    E, H, k = case["E"], case["H"], case["k"]
    st["idx"], st["w"] = _routing(g, N, E, k, case["empty"])
    if op == "experts":
        I = case["I"]
        st["gate"], st["up"], st["down"] = _table(g, (E,), I, H), _table(g, (E,), I, H), _table(g, (E,), H, I)
        st["xv"] = _activations(g, N, H, torch.bfloat16)
        return st
    dt, R = TYPES[case["x"]], _rows(N, k, E, case["tm"])
    if op == "sort":
        st["xv"] = torch.randn(N, H, device="cuda", generator=g).to(dt)
        st["dxs"] = torch.randn(R, H, device="cuda", generator=g).to(dt)
        return st
    tok_row, row_slot = _sorted_order(st["idx"], E, case["tm"])
    st["plan"] = {"tok_row": tok_row, "row_slot": row_slot}   # what the sort left
    st["ys"] = torch.randn(R, H, device="cuda", generator=g).to(dt)
    st["dy"] = torch.randn(N, H, device="cuda", generator=g).to(dt)
    return st


# ------------------------------------------------------------------------------------------------- the plain forms
def _quantised(x):
    """The values that x [.., K] stands for after e4m3 quantisation in groups of 128, in float32."""
    K = x.shape[-1]
    kb = -(-K // 128)
    v = torch.nn.functional.pad(x.float(), (0, kb * 128 - K)).unflatten(-1, (kb, 128))
    top = v.abs().amax(-1, keepdim=True)
    m, ex = torch.frexp(top.clamp_min(LEAST))
    s = ((ex - 8 - (m <= 0.875).to(ex.dtype) + 127) << 23).view(torch.float32)
    s = torch.where(torch.isfinite(top), s, math.nan)
    return ((v / s).to(E4M3).float() * s).flatten(-2)[..., :K]


def _values(q, s):
    """The values of an e4m3 table [.., rows, K] with scales [.., rows / 128, K / 128], in float32."""
    rows, K = q.shape[-2:]
    return q.float() * s.repeat_interleave(128, -2)[..., :rows, :].repeat_interleave(128, -1)[..., :K]


def _of(table, act):
    q, s = table
    return q.view(torch.uint8)[act].view(E4M3), s[act]


def _linear(st):
    return (_quantised(st["xv"]) @ _values(st["q"], st["s"]).T).to(TYPES[st["y"]])


def _experts(st):
    idx, w = st["idx"], st["w"]
    N, k = idx.shape
    act, e = torch.unique(idx.clamp_min(0).long(), return_inverse=True)      # the experts in use
    e = torch.where(idx < 0, act.numel(), e).flatten()
    counts = torch.bincount(e, minlength=act.numel() + 1)
    order = e.argsort(stable=True)
    pos = torch.empty_like(order)
    pos[order] = torch.arange(N * k, device=idx.device)
    pos = pos - (counts.cumsum(0) - counts)[e]                                # place within the expert
    cap = int(counts[:-1].max())
    real = (e < act.numel()) & (pos < cap)
    at = torch.where(real, e * cap + pos, act.numel() * cap)
    xq = _quantised(st["xv"]).repeat_interleave(k, 0)
    xs = xq.new_zeros(act.numel() * cap + 1, xq.shape[1])
    xs[at] = xq
    xs = xs[:-1].view(act.numel(), cap, -1)
    h = torch.bmm(xs, _values(*_of(st["gate"], act)).transpose(1, 2)).clamp_max(LIMIT)
    u = torch.bmm(xs, _values(*_of(st["up"], act)).transpose(1, 2)).clamp(-LIMIT, LIMIT)
    h = _quantised(h / (1 + torch.exp(-h)) * u)
    y = torch.bmm(h, _values(*_of(st["down"], act)).transpose(1, 2)).flatten(0, 1)
    y = torch.where(real[:, None], y[at.clamp_max(act.numel() * cap - 1)], 0.0)
    return (y.view(N, k, -1) * w[..., None]).sum(1).to(torch.bfloat16)


def _sort(st):
    x, dxs = st["xv"], st["dxs"]
    tok_row, row_slot = _sorted_order(st["idx"], st["E"], st["tm"])
    xs = torch.where((tok_row >= 0)[:, None], x[tok_row.clamp_min(0).long()], 0.0)
    d = torch.where((row_slot >= 0)[..., None], dxs[row_slot.clamp_min(0).long()].float(), 0.0)
    return {"xs": xs.to(x.dtype), "tok_row": tok_row, "row_slot": row_slot, "dx": d.sum(1).to(x.dtype)}


def _join(st):
    ys, dy, w, slot = st["ys"], st["dy"].float(), st["w"], st["plan"]["row_slot"]
    R = ys.shape[0]
    real = slot >= 0
    wz = torch.where(real, w, 0.0)
    v = torch.where(real[..., None], ys[slot.clamp_min(0).long()].float(), 0.0)
    dys = torch.zeros(R + 1, ys.shape[1], device=ys.device)
    dys[torch.where(real, slot, R).long()] = wz[..., None] * dy[:, None, :]
    return {"y": (wz[..., None] * v).sum(1).to(ys.dtype), "dys": dys[:R].to(ys.dtype), "dw": (v * dy[:, None, :]).sum(-1)}


# ------------------------------------------------------------------------------------------- the framework's calls
def _package():
    path = os.path.join(os.getcwd(), "kaggle-llm-endpoint_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import cbmoe
    return cbmoe


def _own(st):
    cbmoe = _package()
    op = st["op"]
    if op == "linear":
        return cbmoe.ops.fp8_linear(st["q"], st["s"], st["xv"], out_dtype=TYPES[st["y"]])
    if op == "experts":
        if "layer" not in st:   # the tables and the fetch object that a program keeps for its layers
            st["layer"] = cbmoe.fp8.pack_layer(st["gate"], st["up"], st["down"])
            st["fetch"] = cbmoe.ResidentFetch(out_dtype=torch.bfloat16)
        return st["fetch"].apply(st["layer"], st["xv"], st["idx"], st["w"], 0, LIMIT)
    if op == "sort":
        x = st["xv"].detach().requires_grad_()
        plan = cbmoe.ops.route_plan(st["idx"], st["w"], st["E"], st["tm"])
        xs = cbmoe.moe_permute(x, plan)
        dx, = torch.autograd.grad(xs, x, st["dxs"])
        return {"xs": xs, "tok_row": plan["tok_row"][:xs.shape[0]], "row_slot": plan["row_slot"], "dx": dx}
    ys, w = st["ys"].detach().requires_grad_(), st["w"].detach().requires_grad_()
    y = cbmoe.moe_unpermute(ys, w, st["plan"])
    dys, dw = torch.autograd.grad(y, (ys, w), st["dy"])
    return {"y": y, "dys": dys, "dw": dw}


def run(state):
    if own:
        return _own(state)
    return {"linear": _linear, "experts": _experts, "sort": _sort, "join": _join}[state["op"]](state)


# --------------------------------------------------------------------------------------------------- work and exact
def work(case):
    N, op = case["N"], case["op"]
    if op == "linear":
        K, rows = case["K"], case["rows"]
        size = {"bf16": 2, "fp16": 2, "fp32": 4}
        b = rows * K + 4 * -(-rows // 128) * -(-K // 128) + N * K * size[case["x"]] + N * rows * size[case["y"]]
        return {"bytes": b, "flops": 2 * N * K * rows}
    E, H, k = case["E"], case["H"], case["k"]
    slots = N * k * (1 - case["empty"])
    if op == "experts":
        I = case["I"]
        used = E * (1 - (1 - k * (1 - case["empty"]) / E) ** N)      # experts that some token chose, on average
        return {"bytes": used * 3 * H * I + 4 * N * H + 8 * N * k, "flops": 2 * slots * 3 * H * I}
    b, R = (4 if case["x"] == "fp32" else 2) * H, _rows(N, k, E, case["tm"])
    if op == "sort":   # x read, the rows written; their gradients read, dx written; idx read, both orders written
        return {"bytes": 2 * N * b + (R + slots) * b + 8 * N * k + 4 * R, "flops": slots * H}
    # the rows and dy read, y and the rows' gradients written; the backward pass reads the rows again
    return {"bytes": (2 * N + 2 * slots + R) * b + 12 * N * k + 4 * R, "flops": 5 * slots * H}


def _group64(row):
    """One row's values after quantisation, in float64: group by group from the definition."""
    K = row.shape[-1]
    out = torch.empty_like(row)
    for k0 in range(0, K, 128):
        part = row[..., k0:k0 + 128]
        top = part.abs().amax(-1, keepdim=True).clamp_min(LEAST)
        p = torch.floor(torch.log2(top / 448.0)) - 1
        for _ in range(3):                                       # the least power of two that holds the largest value
            p = torch.where(448.0 * torch.exp2(p) < top, p + 1, p)
        s = torch.exp2(p)
        out[..., k0:k0 + 128] = (part / s).to(E4M3).double() * s
    return out


def _weights64(q, s):
    w = q.double()
    for i in range(s.shape[-2]):
        for j in range(s.shape[-1]):
            w[128 * i:128 * i + 128, 128 * j:128 * j + 128] *= s[i, j].double()
    return w


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        return _group64(st["xv"].double()) @ _weights64(st["q"], st["s"]).T
    idx, w = st["idx"].cpu(), st["w"].double()
    if op == "experts":
        x = _group64(st["xv"].double())
        y = torch.zeros_like(x)
        for e in range(case["E"]):
            t, j = torch.nonzero(idx == e, as_tuple=True)
            if not len(t):
                continue
            t, j = t.cuda(), j.cuda()
            gate, up, down = (_weights64(st[n][0][e], st[n][1][e]) for n in ("gate", "up", "down"))
            a, b = x[t] @ gate.T, x[t] @ up.T
            a, b = torch.clamp(a, max=LIMIT), torch.clamp(b, -LIMIT, LIMIT)
            y.index_add_(0, t, w[t, j][:, None] * (_group64(a * torch.sigmoid(a) * b) @ down.T))
        return y
    if op == "sort":
        x, dxs = st["xv"].double(), st["dxs"].double()
        xs, dx, row = torch.zeros_like(dxs), torch.zeros_like(x), 0
        for e in range(case["E"]):
            t = torch.nonzero(idx == e, as_tuple=True)[0].cuda()
            xs[row:row + len(t)] = x[t]
            dx.index_add_(0, t, dxs[row:row + len(t)])
            row += -(-len(t) // case["tm"]) * case["tm"]
        return {"xs": xs, "tok_row": None, "row_slot": None, "dx": dx}
    ys, dy = st["ys"].double(), st["dy"].double()
    y, dys, dw, row = torch.zeros_like(dy), torch.zeros_like(ys), torch.zeros_like(w), 0
    for e in range(case["E"]):
        t, j = (v.cuda() for v in torch.nonzero(idx == e, as_tuple=True))
        part = ys[row:row + len(t)]
        y.index_add_(0, t, w[t, j][:, None] * part)
        dys[row:row + len(t)] = w[t, j][:, None] * dy[t]
        dw[t, j] = (part * dy[t]).sum(1)
        row += -(-len(t) // case["tm"]) * case["tm"]
    return {"y": y, "dys": dys, "dw": dw}

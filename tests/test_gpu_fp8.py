"""e4m3 with block scales on the GPU against the float64 oracle: quantiser bit for bit, products and experts inside the
bounds that oracle/fp8.py derives (needs a B200: -m gpu)."""
import numpy as np
import pytest
import torch

from oracle import fp8, gen

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def half_eps(dtype):
    return torch.finfo(dtype).eps / 2


def f64(t):
    return t.detach().double().cpu().numpy()


def table(rng, rows, K, E=None):
    """Codes and scales of N(0, 0.02) weights on the GPU (rows padded to 16 bytes), and the same in NumPy."""
    n = 1 if E is None else E
    rb, kb = -(-rows // 128), -(-K // 128)
    w = np.zeros((n, rb * 128, kb * 128), np.float32)
    w[:, :rows, :K] = rng.standard_normal((n, rows, K)) * 0.02
    v = w.reshape(n, rb, 128, kb, 128)
    s = (np.abs(v).max(axis=(2, 4)) / 448).astype(np.float32)
    q = (v / s[:, :, None, :, None]).reshape(w.shape)[:, :rows, :K].astype(fp8.E4M3)
    import cbmoe
    tq = cbmoe.ops.fp8_pad_rows(torch.from_numpy(q.view(np.uint8)).cuda().view(torch.float8_e4m3fn))
    ts = torch.from_numpy(s).cuda()
    if E is None:
        return (tq[0], ts[0]), (q[0], s[0])
    return (tq, ts), [(q[e], s[e]) for e in range(n)]


def activations(rng, N, K, dtype):
    x = rng.standard_normal((N, K)) * np.exp(rng.standard_normal((N, 1)))
    return torch.from_numpy(x).to(dtype).cuda()


def no_device_errors():
    import cbmoe
    torch.cuda.synchronize()
    assert cbmoe.device_errors(clear=True) == 0


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("N,K", [(1, 1), (1, 128), (3, 127), (5, 129), (2, 16), (33, 1000), (4, 5120), (0, 256)])
def test_quantize_matches_oracle(dtype, N, K):
    import cbmoe
    rng = np.random.default_rng(N * 10007 + K)
    x = activations(rng, N, K, TYPES[dtype])
    q, s = cbmoe.ops.fp8_quantize(x)
    assert q.shape == (N, K) and q.dtype == torch.float8_e4m3fn and s.shape == (N, -(-K // 128))
    if N:
        want = fp8.group_scales(f64(x))
        assert np.array_equal(f64(s), want)
        assert np.array_equal(f64(q.float()), fp8.codes(f64(x), want))
    no_device_errors()


def test_quantize_values_at_the_edges():
    import cbmoe
    big = torch.finfo(torch.float32).max
    x = torch.zeros(9, 256)
    x[1, :128] = 1e-40
    x[2, 5], x[2, 6] = 448.0, -449.0
    x[3, 200] = big
    x[4, 3] = float("inf")
    x[5, 130] = float("nan")
    x[6, :] = torch.linspace(-448, 448, 256)
    x[7, 0], x[7, 1] = 1.0, 2.0 ** -9
    x[8, 0] = fp8.LEAST
    q, s = cbmoe.ops.fp8_quantize(x.cuda())
    want = fp8.group_scales(f64(x))
    assert np.array_equal(f64(s), want, equal_nan=True)
    assert np.array_equal(f64(q.float()), fp8.codes(f64(x), want), equal_nan=True)
    assert np.isnan(f64(q.float())[4, :128]).all() and np.isfinite(f64(q.float())[4, 128:]).all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_quantize_strided_rows(dtype):
    import cbmoe
    rng = np.random.default_rng(5)
    whole = activations(rng, 6, 700, TYPES[dtype])
    for x in (whole[:, 8:520], whole[:, 3:400], whole[::2], whole.t()[:64]):
        q, s = cbmoe.ops.fp8_quantize(x)
        want = fp8.group_scales(f64(x))
        assert np.array_equal(f64(s), want) and np.array_equal(f64(q.float()), fp8.codes(f64(x), want))


LINEAR = [(1, 128, 128), (1, 5120, 700), (2, 16, 1), (3, 100, 127), (8, 129, 128), (16, 1000, 129), (31, 257, 255),
          (32, 384, 256), (33, 640, 257), (64, 512, 512), (65, 128, 384), (77, 5000, 1411), (128, 896, 300),
          (129, 300, 640), (300, 1536, 513), (1, 1, 1), (1000, 256, 256)]


@pytest.mark.parametrize("N,K,rows", LINEAR)
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "fp32"), ("bf16", "fp32")])
def test_linear_matches_oracle(N, K, rows, dtype, out):
    import cbmoe
    rng = np.random.default_rng(N * 7 + K * 3 + rows)
    (q, s), (qn, sn) = table(rng, rows, K)
    x = activations(rng, N, K, TYPES[dtype])
    y = cbmoe.ops.fp8_linear(q, s, x, out_dtype=TYPES[out])
    assert y.shape == (N, rows) and y.dtype == TYPES[out]
    want, bound = fp8.linear(qn, sn, f64(x), half_eps(TYPES[out]))
    tiny = torch.finfo(TYPES[out]).tiny * half_eps(TYPES[out]) * 2          # fp16 results below its normal range
    assert (np.abs(f64(y) - want) <= bound + tiny).all()
    pair = cbmoe.ops.fp8_linear(q, s, cbmoe.ops.fp8_quantize(x), out_dtype=TYPES[out])
    assert torch.equal(pair, y)
    assert torch.equal(cbmoe.ops.fp8_linear(q, s, x, out_dtype=TYPES[out]), y)      # the same bits again
    no_device_errors()


def test_linear_many_rows():
    """A prompt's rows, several passes and several output tiles per CTA."""
    import cbmoe
    rng = np.random.default_rng(3)
    (q, s), (qn, sn) = table(rng, 2600, 768)
    x = activations(rng, 2500, 768, torch.bfloat16)
    y = cbmoe.ops.fp8_linear(q, s, x)
    want, bound = fp8.linear(qn, sn, f64(x), half_eps(torch.float32))
    assert (np.abs(f64(y) - want) <= bound).all()
    no_device_errors()


def test_linear_empty_batch_and_bad_rows():
    import cbmoe
    rng = np.random.default_rng(4)
    (q, s), (qn, sn) = table(rng, 200, 300)
    assert cbmoe.ops.fp8_linear(q, s, torch.zeros(0, 300, device="cuda")).shape == (0, 200)
    x = activations(rng, 40, 300, torch.bfloat16)
    x[7, 299], x[30, 0], x[31] = float("nan"), float("-inf"), 0
    y = f64(cbmoe.ops.fp8_linear(q, s, x))
    bad = np.zeros(40, bool)
    bad[[7, 30]] = True
    assert np.isnan(y[bad]).all() and np.isfinite(y[~bad]).all() and (y[31] == 0).all()
    xc = f64(x)
    xc[bad] = 0
    want, bound = fp8.linear(qn, sn, xc, half_eps(torch.float32))
    assert (np.abs(y - want)[~bad] <= bound[~bad]).all()


def test_linear_scales_of_any_value_and_bad_weights():
    """Scales are used as they are (not only powers of two); a NaN code makes its output column NaN, no other."""
    import cbmoe
    rng = np.random.default_rng(6)
    (q, s), (qn, sn) = table(rng, 256, 256)
    qn = qn.copy()
    s2 = (sn * np.exp(4 * rng.standard_normal(sn.shape))).astype(np.float32)
    raw = q.contiguous().view(torch.uint8).clone()
    raw[17, 200] = 0x7F
    x = activations(rng, 5, 256, torch.float16)
    y = f64(cbmoe.ops.fp8_linear(raw.view(torch.float8_e4m3fn), torch.from_numpy(s2).cuda(), x))
    want, bound = fp8.linear(qn, s2, f64(x), half_eps(torch.float32))
    keep = np.arange(256) != 17
    assert np.isnan(y[:, 17]).all() and (np.abs(y - want)[:, keep] <= bound[:, keep]).all()


def test_linear_on_streams_and_in_graphs():
    import cbmoe
    rng = np.random.default_rng(8)
    (q, s), (qn, sn) = table(rng, 1000, 1024)
    xs = [activations(rng, n, 1024, torch.bfloat16) for n in (1, 40, 200)]
    want = [cbmoe.ops.fp8_linear(q, s, x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for st, x in zip(streams, xs):                   # overlapping calls share no scratch
        with torch.cuda.stream(st):
            got.append([cbmoe.ops.fp8_linear(q, s, x) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(w, g) for w, gs in zip(want, got) for g in gs)
    graphs = []
    for x in xs:
        static = x.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = cbmoe.ops.fp8_linear(q, s, static)
        graphs.append((g, static, y))
    for _ in range(2):
        for g, _, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(w, y) for w, (_, _, y) in zip(want, graphs))
    for (g, static, y), x in zip(graphs, xs):        # other values in the captured input
        static.copy_(-x)
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(-w, y) for w, (_, _, y) in zip(want, graphs))
    no_device_errors()


def test_linear_refusals():
    import cbmoe
    rng = np.random.default_rng(9)
    (q, s), _ = table(rng, 130, 256)
    x = activations(rng, 2, 256, torch.bfloat16)
    f = cbmoe.ops.fp8_linear
    tight = torch.zeros(130, 250, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    s_tight = torch.ones(2, 2, device="cuda")
    for call in (lambda: f(q, s, x[:, :255]), lambda: f(q, s[:1], x), lambda: f(q, s.double(), x), lambda: f(q, s.t(), x),
                 lambda: f(q.float(), s, x), lambda: f(q, s, x.double()), lambda: f(q, s, x[0]),
                 lambda: f(q, s, x, out_dtype=torch.float64), lambda: f(tight, s_tight, x[:, :250]),
                 lambda: f(q, s, (x, s)), lambda: f(q, s, (q[:2], s[:1])), lambda: f(q[:0], s, x),
                 lambda: cbmoe.ops.fp8_quantize(x.double()), lambda: cbmoe.ops.fp8_quantize(x[:, :0]),
                 lambda: cbmoe.ops.fp8_quantize(x[0])):
        with pytest.raises(ValueError):
            call()
    assert f(cbmoe.ops.fp8_pad_rows(tight), s_tight, x[:, :250]).shape == (2, 130)


# ------------------------------------------------------------------------------------------------------ experts
def layer(rng, E, H, I):
    import cbmoe
    made = [table(rng, r, c, E) for r, c in ((I, H), (I, H), (H, I))]
    return cbmoe.fp8.pack_layer(*(m[0] for m in made)), [m[1] for m in made]


def apply(p, x, idx, w, out):
    import cbmoe
    return cbmoe.ResidentFetch(out_dtype=out).apply(p, x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda(), 0,
                                                    gen.LIMIT)


EXPERTS = [(1, 8, 256, 128, 2), (1, 4, 1280, 384, 4), (5, 4, 200, 100, 2), (33, 3, 256, 129, 3), (40, 2, 130, 257, 1),
           (150, 4, 384, 256, 2), (300, 2, 256, 128, 2), (70, 16, 512, 130, 4)]


@pytest.mark.parametrize("N,E,H,I,k", EXPERTS)
@pytest.mark.parametrize("out", ["bf16", "fp32"])
def test_experts_match_oracle(N, E, H, I, k, out):
    rng = np.random.default_rng(N + E + H + I)
    p, (gate, up, down) = layer(rng, E, H, I)
    x = activations(rng, N, H, torch.bfloat16)
    idx, w = gen.routing(rng, N, E, k)
    y = apply(p, x, idx, w, TYPES[out])
    assert y.shape == (N, H) and y.dtype == TYPES[out]
    want, bound = fp8.experts(gate, up, down, f64(x), idx, w.astype(np.float64), gen.LIMIT, half_eps(TYPES[out]))
    assert (np.abs(f64(y) - want) <= bound).all()
    # The bound adds worst cases; on the whole the result is nearer. Codes of h that may fall on either side of a border:
    # those within sum_bound * sqrt(K) ~ 2^-10.6 of one (K = 1280), 2^-10.6 / 2^-5 of all; each moves by 2^-3 of its value
    # at most, together sqrt(2^-5.6) * 2^-3 < 2^-5.7 of the norm; two bf16 roundings are below 2^-8 of it.
    assert np.linalg.norm(f64(y) - want) <= 2.0 ** -5.5 * np.linalg.norm(want)
    assert torch.equal(apply(p, x, idx, w, TYPES[out]), y)
    no_device_errors()


def test_experts_empty_slots_repeats_and_skew():
    """Empty slots add nothing; one expert may come twice in a token; all tokens may want one expert."""
    rng = np.random.default_rng(11)
    E, H, I, k, N = 6, 256, 200, 4, 90
    p, (gate, up, down) = layer(rng, E, H, I)
    x = activations(rng, N, H, torch.bfloat16)
    idx = rng.integers(0, E, (N, k)).astype(np.int32)
    idx[:, 0] = 3
    idx[rng.random((N, k)) < 0.3] = -1
    idx[17] = -1
    w = rng.random((N, k)).astype(np.float32)
    y = f64(apply(p, x, idx, w, torch.float32))
    want, bound = fp8.experts(gate, up, down, f64(x), idx, w.astype(np.float64), gen.LIMIT, half_eps(torch.float32))
    assert (np.abs(y - want) <= bound).all() and (y[17] == 0).all()
    none = apply(p, x, np.full((N, k), -1, np.int32), w, torch.bfloat16)
    assert (f64(none) == 0).all()
    assert apply(p, x[:0], idx[:0], w[:0], torch.bfloat16).shape == (0, H)
    no_device_errors()


def test_experts_bad_token_stays_its_own():
    rng = np.random.default_rng(12)
    E, H, I, k, N = 4, 256, 128, 2, 35
    p, _ = layer(rng, E, H, I)
    x = activations(rng, N, H, torch.bfloat16)
    idx, w = gen.routing(rng, N, E, k)
    good = apply(p, x, idx, w, torch.float32)
    x[3, 100], x[20, 0] = float("nan"), float("inf")
    y = apply(p, x, idx, w, torch.float32)
    bad = torch.zeros(N, dtype=torch.bool)
    bad[[3, 20]] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], good[~bad])


def test_experts_index_out_of_range_is_reported():
    import cbmoe
    rng = np.random.default_rng(13)
    p, _ = layer(rng, 4, 128, 128)
    x = activations(rng, 3, 128, torch.bfloat16)
    idx, w = gen.routing(rng, 3, 4, 2)
    want = apply(p, x, np.where(idx == idx[0, 0], -1, idx), w, torch.float32)
    idx[idx == idx[0, 0]] = 4
    y = apply(p, x, idx, w, torch.float32)
    torch.cuda.synchronize()
    assert cbmoe.device_errors(clear=True) == 2 and torch.equal(y, want)      # the slot is skipped


def test_experts_refusals():
    import cbmoe
    rng = np.random.default_rng(14)
    p, _ = layer(rng, 2, 256, 128)
    (gq, gs), (uq, us), (dq, ds) = p["gate_q"], p["up_q"], p["down_q"]
    for bad in (((gq, gs), (uq, us), (gq, gs)), ((gq, gs[:, :, :1]), (uq, us), (dq, ds)), ((gq, gs), (uq, us.half()), (dq, ds)),
                ((gq[0], gs), (uq, us), (dq, ds)), ((gq.float(), gs), (uq, us), (dq, ds))):
        with pytest.raises(ValueError):
            cbmoe.fp8.pack_layer(*bad)
    x = activations(rng, 2, 256, torch.bfloat16)
    idx, w = (torch.from_numpy(t).cuda() for t in gen.routing(rng, 2, 2, 2))
    with pytest.raises(ValueError):        # the tables hold FP8
        cbmoe.ResidentFetch(qtypes={0: {"gate_q": "CB3"}}).apply(p, x, idx, w, 0, 10.0)
    with pytest.raises(ValueError):
        cbmoe.ResidentFetch().layer(p, x, idx, w, 10.0)
    with pytest.raises(ValueError):
        cbmoe.ResidentFetch(out_dtype=torch.float64).apply(p, x, idx, w, 0, 10.0)


def test_experts_on_streams_and_in_graphs():
    """Overlapping calls and two captured graphs share no scratch; a replay takes new values of the captured inputs."""
    import cbmoe
    rng = np.random.default_rng(16)
    E, H, I, k = 6, 384, 256, 2
    p, _ = layer(rng, E, H, I)
    fetch = cbmoe.ResidentFetch(out_dtype=torch.bfloat16)
    made = []
    for N in (3, 50, 900):
        idx, w = (torch.from_numpy(t).cuda() for t in gen.routing(rng, N, E, k))
        made.append((activations(rng, N, H, torch.bfloat16), idx, w))
    call = lambda c: fetch.apply(p, c[0], c[1], c[2], 0, gen.LIMIT)
    want = [call(c) for c in made]
    torch.cuda.synchronize()
    got = []
    for c in made:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append([call(c) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(w, g) for w, gs in zip(want, got) for g in gs)
    graphs = []
    for c in made:
        g = torch.cuda.CUDAGraph()
        static = (c[0].clone(), c[1].clone(), c[2].clone())
        with torch.cuda.graph(g):
            y = call(static)
        graphs.append((g, static, y))
    for g, _, _ in graphs + graphs[::-1]:
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(w, y) for w, (_, _, y) in zip(want, graphs))
    g, static, y = graphs[1]
    static[1].copy_(made[1][1].flip(0))
    g.replay()
    assert torch.equal(y, call((made[1][0], made[1][1].flip(0), made[1][2])))
    no_device_errors()


def test_many_tiles_with_a_cut_remainder():
    """More tiles than pairs of SMs, the rest cut along K: whole and partial sums side by side, the same bits again."""
    import cbmoe
    rng = np.random.default_rng(17)
    (q, s), (qn, sn) = table(rng, 128 * 21, 1500)
    x = activations(rng, 2700, 1500, torch.float16)
    y = cbmoe.ops.fp8_linear(q, s, x)
    rows = rng.choice(2700, 64, replace=False)
    want, bound = fp8.linear(qn, sn, f64(x)[rows], half_eps(torch.float32))
    assert (np.abs(f64(y)[rows] - want) <= bound).all()
    assert torch.equal(cbmoe.ops.fp8_linear(q, s, x), y)
    no_device_errors()


def test_router_plan_products_and_join_are_the_layer():
    """The operators one after another, as a program with its own expert loop uses them, against the fused layer."""
    import cbmoe
    rng = np.random.default_rng(15)
    E, H, I, k, N, tm = 8, 384, 256, 2, 100, 32
    p, _ = layer(rng, E, H, I)
    x = activations(rng, N, H, torch.bfloat16)
    router = torch.from_numpy(rng.standard_normal((H, E)) * 0.05).to(torch.bfloat16).cuda()
    idx, w = cbmoe.moe_route(x, router, torch.zeros(E, device="cuda"), k)
    plan = cbmoe.ops.route_plan(idx, w, E, tm)
    xs = cbmoe.moe_permute(x, plan)
    counts = plan["counts"].tolist()
    ys = torch.zeros(xs.shape, dtype=torch.float32, device="cuda")
    (gq, gs), (uq, us), (dq, ds) = p["gate_q"], p["up_q"], p["down_q"]
    row = 0
    for e in range(E):
        n = counts[e]
        if n:
            xe = cbmoe.ops.fp8_quantize(xs[row:row + n])
            g, u = cbmoe.ops.fp8_linear(gq[e], gs[e], xe), cbmoe.ops.fp8_linear(uq[e], us[e], xe)
            g, u = g.clamp_max(gen.LIMIT), u.clamp(-gen.LIMIT, gen.LIMIT)
            ys[row:row + n] = cbmoe.ops.fp8_linear(dq[e], ds[e], g * torch.sigmoid(g) * u)
        row += -(-n // tm) * tm
    y = cbmoe.moe_unpermute(ys, w, plan)
    fused = cbmoe.ResidentFetch().apply(p, x, idx, w, 0, gen.LIMIT)
    # h is rounded to e4m3 from values that differ in the last fp32 bits: a code may fall on either side of a border
    # (2^-4 of that value). Per element of y: one of I = 256 terms; 2^-4 sqrt(1 / 256) of the norm is 2^-8.
    assert (y - fused).norm() <= 2.0 ** -8 * fused.norm()
    no_device_errors()


@pytest.mark.parametrize("N,E,H,I,k", EXPERTS + [(9, 3, 131, 140, 3), (40, 16, 260, 128, 8)])
@pytest.mark.parametrize("out", ["bf16", "fp16"])
def test_experts_round_once(N, E, H, I, k, out):
    """The slots' outputs stay in fp32 whatever the type of the result: 16 bits are the fp32 result rounded, no more."""
    rng = np.random.default_rng(N + E + H + I + 1)
    p, _ = layer(rng, E, H, I)
    x = activations(rng, N, H, torch.bfloat16)
    idx, w = gen.routing(rng, N, E, k)
    y = apply(p, x, idx, w, TYPES[out])
    assert torch.equal(y, apply(p, x, idx, w, torch.float32).to(TYPES[out]))
    no_device_errors()


def test_experts_slots_past_the_range_of_fp16():
    """Slots beyond 65504, of both signs, whose weighted sums fit fp16."""
    rng = np.random.default_rng(18)
    E, H, I, k, N = 4, 200, 100, 2, 24
    p, (gate, up, down) = layer(rng, E, H, I)
    grow = 2.0 ** 22
    p["down_q"] = (p["down_q"][0], p["down_q"][1] * grow)
    down = [(q, s * np.float32(grow)) for q, s in down]
    x = activations(rng, N, H, torch.bfloat16)
    idx, w = gen.routing(rng, N, E, k)
    one = np.ones((N, 1), np.float32)
    slots = np.stack([fp8.experts(gate, up, down, f64(x), idx[:, j:j + 1], one, gen.LIMIT, 0.0)[0] for j in range(k)])
    w = (w * np.float32(30000 / np.abs(slots).max())).astype(np.float32)
    assert (slots.min(axis=0) < -65504).any() and (slots.max(axis=0) > 65504).any()
    y = apply(p, x, idx, w, torch.float16)
    want, bound = fp8.experts(gate, up, down, f64(x), idx, w.astype(np.float64), gen.LIMIT, half_eps(torch.float16))
    # + half the least fp16 subnormal
    assert torch.isfinite(y).all() and (np.abs(f64(y) - want) <= bound + 2.0 ** -25).all()
    no_device_errors()


def test_inputs_that_require_a_gradient_are_refused():
    """The products have no backward pass: under autograd they would drop their part of the gradient without a word."""
    import cbmoe
    rng = np.random.default_rng(20)
    (q, s), _ = table(rng, 130, 256)
    x = activations(rng, 4, 256, torch.float32).requires_grad_()
    p, _ = layer(rng, 2, 256, 128)
    idx, w = (torch.from_numpy(t).cuda() for t in gen.routing(rng, 4, 2, 2))
    codes, scales = cbmoe.ops.fp8_quantize(x.detach())
    fetch = cbmoe.ResidentFetch()
    trained = w.clone().requires_grad_()
    calls = (lambda: cbmoe.ops.fp8_linear(q, s, x), lambda: cbmoe.ops.fp8_quantize(x),
             lambda: cbmoe.ops.fp8_linear(q, s.clone().requires_grad_(), x.detach()),
             lambda: cbmoe.ops.fp8_linear(q, s, (codes, scales.clone().requires_grad_())),
             lambda: fetch.apply(p, x, idx, w, 0, gen.LIMIT), lambda: fetch.apply(p, x.detach(), idx, trained, 0, gen.LIMIT))
    for call in calls:
        with pytest.raises(ValueError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
    assert not fetch.apply(p, x.detach(), idx, w, 0, gen.LIMIT).requires_grad
    no_device_errors()


@pytest.fixture(scope="module")
def wide_layer():
    """40 experts of 4 gate/up tiles (10 column blocks each): more tiles than SMs whatever the rows of a pass."""
    rng = np.random.default_rng(19)
    return layer(rng, 40, 1280, 512)


@pytest.mark.parametrize("N,skew,width", [(60, False, 32), (400, False, 64), (900, False, 128), (1500, False, 256),
                                          (60, True, 32), (1604, True, 256)])
def test_experts_with_more_tiles_than_sms(wide_layer, N, skew, width):
    """Passes of 32, 64, 128 and 256 rows, where a CTA (at 256 rows: a pair) takes several tiles one after another; pairs
    cut the gate/up tiles left over along K. Skewed: one expert has a slot of every token, a few rows past whole passes."""
    p, (gate, up, down) = wide_layer
    E, H, I, k = 40, 1280, 512, 4
    rng = np.random.default_rng(N + skew)
    x = activations(rng, N, H, torch.bfloat16)
    idx, w = gen.routing(rng, N, E, k)
    if skew:
        idx[idx == 7] = 8
        idx[:, 0] = 7
    slots = N * k / E
    assert width == (32 if slots <= 32 else 64 if slots <= 64 else 128 if slots <= 128 else 256)
    counts = np.bincount(idx.ravel(), minlength=E)
    tiles = int((-(-counts // width)).sum()) * (I // 128)
    workers = torch.cuda.get_device_properties(0).multi_processor_count // (2 if width == 256 else 1)
    assert tiles > workers and (width < 256 or tiles % workers)
    want, bound = fp8.experts(gate, up, down, f64(x), idx, w.astype(np.float64), gen.LIMIT, half_eps(torch.float32))
    y = apply(p, x, idx, w, torch.float32)
    assert (np.abs(f64(y) - want) <= bound).all()
    assert np.linalg.norm(f64(y) - want) <= 2.0 ** -5.5 * np.linalg.norm(want)     # as in test_experts_match_oracle
    assert torch.equal(apply(p, x, idx, w, torch.float32), y)
    no_device_errors()


@pytest.mark.parametrize("N,K,rows", [(3, 8192, 262400), (262400, 8192, 130), (70000, 130, 32768)])
def test_linear_past_32_bit_offsets(N, K, rows):
    """Weights, activations and outputs of more than 2^31 elements: the last rows are found where they lie."""
    import cbmoe
    g = torch.Generator(device="cuda").manual_seed(N)
    ld = -(-K // 16) * 16
    q = torch.randint(0, 0x7F, (rows, ld), dtype=torch.uint8, device="cuda", generator=g).view(torch.float8_e4m3fn)[:, :K]
    s = torch.rand(-(-rows // 128), -(-K // 128), device="cuda", generator=g) * 2.0 ** -10
    x = torch.randn(N, K, device="cuda", generator=g, dtype=torch.bfloat16)
    y = cbmoe.ops.fp8_linear(q, s, x, out_dtype=torch.bfloat16)
    n = torch.tensor(sorted({0, N // 2, N - 2, N - 1}), device="cuda")
    b = sorted({0, rows // 128 // 2, -(-rows // 128) - 1})                       # 128-row blocks
    for i in b:
        r = slice(128 * i, min(128 * i + 128, rows))
        want, bound = fp8.linear(f64(q[r].float()), f64(s[i:i + 1]), f64(x[n]), half_eps(torch.bfloat16))
        assert (np.abs(f64(y[n, r]) - want) <= bound).all()
    no_device_errors()


def test_weights_of_empty_slots_are_not_read():
    rng = np.random.default_rng(21)
    p, _ = layer(rng, 5, 200, 130)
    x = activations(rng, 40, 200, torch.bfloat16)
    idx, w = gen.routing(rng, 40, 5, 3)
    idx[rng.random(idx.shape) < 0.4] = -1
    want = apply(p, x, idx, w, torch.bfloat16)
    w[idx < 0] = np.nan
    y = apply(p, x, idx, w, torch.bfloat16)
    assert torch.isfinite(y).all() and torch.equal(y, want)
    no_device_errors()

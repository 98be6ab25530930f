"""Tokens into expert order and back, forward and backward, against the formulas in float64 (needs a B200: -m gpu)."""
import numpy as np
import pytest
import torch

from oracle import gen

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
#        T, E, k, H, tm
SIZES = [(1, 8, 2, 64, 1), (1, 160, 8, 5120, 1), (7, 4, 4, 1, 1), (50, 20, 4, 1411, 16), (33, 5, 3, 130, 8),
         (300, 32, 8, 264, 128), (40, 64, 17, 72, 1), (700, 16, 8, 96, 1), (3, 300, 1, 8, 32)]


def case(T, E, k, H, tm, dtype, empty, seed=0):
    import cbmoe
    rng = np.random.default_rng(T + E + k + H + tm + seed)
    idx, w = gen.routing(rng, T, E, k)
    if empty:
        idx[rng.random(idx.shape) < 0.3] = -1
        idx[T // 2] = -1
    idx, w = torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()
    plan = cbmoe.ops.route_plan(idx, w, E, tm)
    new = lambda *s: torch.from_numpy(rng.standard_normal(s)).to(TYPES[dtype]).cuda()
    return plan, idx, w, new


def rows_of(plan, T, k, E, tm):
    slot = plan["row_slot"].long().cpu()
    R = T * k if tm == 1 else (-(-T * k // tm) + E) * tm
    return slot, R


@pytest.mark.parametrize("T,E,k,H,tm", SIZES)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("empty", [False, True])
def test_permute_and_gradient(T, E, k, H, tm, dtype, empty):
    import cbmoe
    plan, idx, w, new = case(T, E, k, H, tm, dtype, empty)
    slot, R = rows_of(plan, T, k, E, tm)
    x = new(T, H).requires_grad_()
    xs = cbmoe.moe_permute(x, plan)
    assert xs.shape == (R, H) and xs.dtype == x.dtype
    want = torch.zeros(R, H, dtype=x.dtype)
    for j in range(k):
        t = torch.nonzero(slot[:, j] >= 0)[:, 0]
        want[slot[t, j]] = x.detach().cpu()[t]
    assert torch.equal(xs.detach().cpu(), want)
    g = new(R, H)
    dx, = torch.autograd.grad(xs, x, g)
    rows = torch.where((slot >= 0)[..., None], g.double().cpu()[slot.clamp_min(0)], 0.0)
    # k - 1 fp32 additions of the running sum, one rounding to the type
    bound = k * 2.0 ** -24 * rows.abs().sum(1) * 1.001
    he = torch.finfo(x.dtype).eps / 2
    assert ((dx.double().cpu() - rows.sum(1)).abs() <= bound + he * (rows.sum(1).abs() + bound) + 2.0 ** -25).all()


@pytest.mark.parametrize("T,E,k,H,tm", SIZES)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("empty", [False, True])
def test_unpermute_and_gradients(T, E, k, H, tm, dtype, empty):
    import cbmoe
    plan, idx, w, new = case(T, E, k, H, tm, dtype, empty)
    slot, R = rows_of(plan, T, k, E, tm)
    ys, wl = new(R, H).requires_grad_(), w.clone().requires_grad_()
    y = cbmoe.moe_unpermute(ys, wl, plan)
    assert y.shape == (T, H) and y.dtype == ys.dtype
    real = slot >= 0
    rows = torch.where(real[..., None], ys.detach().double().cpu()[slot.clamp_min(0)], 0.0)
    terms = w.double().cpu()[..., None] * rows
    he = torch.finfo(ys.dtype).eps / 2
    bound = k * 2.0 ** -24 * terms.abs().sum(1) * 1.001
    # 2^-25: half the least fp16 subnormal
    assert ((y.detach().double().cpu() - terms.sum(1)).abs() <= bound + he * (terms.sum(1).abs() + bound) + 2.0 ** -25).all()
    dy = new(T, H)
    dys, dw = torch.autograd.grad(y, (ys, wl), dy)
    want = torch.zeros(R, H, dtype=torch.float64)
    want[slot[real]] = (w.double().cpu()[..., None] * dy.double().cpu()[:, None])[real]
    # one fp32 product, one rounding to the type
    assert ((dys.double().cpu() - want).abs() <= (he + 2.0 ** -24) * 1.001 * want.abs() + 2.0 ** -25).all()
    prod = rows * dy.double().cpu()[:, None]
    # on the way of a term at most H / 128 + 8 multiply-adds of its thread, 5 and 4 additions across lanes and warps
    assert ((dw.double().cpu() - prod.sum(-1)).abs() <= (H / 128 + 18) * 2.0 ** -24 * prod.abs().sum(-1)).all()
    assert (dw.cpu()[~real] == 0).all()
    again = torch.autograd.grad(cbmoe.moe_unpermute(ys, wl, plan), (ys, wl), dy)
    assert torch.equal(again[0], dys) and torch.equal(again[1], dw)        # the same bits again


@pytest.mark.parametrize("H", [20, 132, 1282, 2564])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shift", [0, 1, 2, 4])
def test_units_of_a_row(H, dtype, shift):
    """Rows and pointers aligned to 2, 4, 8 and 16 bytes (views `shift` elements into their storage): the same values
    whatever the width of a load, and nothing written outside."""
    import cbmoe
    T, E, k, tm = 37, 6, 4, 8
    plan, idx, w, new = case(T, E, k, H, tm, dtype, True)
    slot, R = rows_of(plan, T, k, E, tm)

    def moved(t):
        flat = torch.empty(t.numel() + shift, dtype=t.dtype, device="cuda")
        flat[shift:] = t.flatten()
        return flat[shift:].view(t.shape)

    x, ys, dy = new(T, H), new(R, H), new(T, H)
    xs = cbmoe.moe_permute(moved(x), plan)
    want = torch.zeros(R, H, dtype=x.dtype)
    for j in range(k):
        t = torch.nonzero(slot[:, j] >= 0)[:, 0]
        want[slot[t, j]] = x.cpu()[t]
    assert torch.equal(xs.cpu(), want)
    a, wl = moved(ys).requires_grad_(), w.clone().requires_grad_()
    y = cbmoe.moe_unpermute(a, wl, plan)
    real = slot >= 0
    rows = torch.where(real[..., None], ys.double().cpu()[slot.clamp_min(0)], 0.0)
    terms = w.double().cpu()[..., None] * rows
    he = torch.finfo(ys.dtype).eps / 2
    bound = k * 2.0 ** -24 * terms.abs().sum(1) * 1.001
    assert ((y.detach().double().cpu() - terms.sum(1)).abs() <= bound + he * (terms.sum(1).abs() + bound) + 2.0 ** -25).all()
    dys, dw = torch.autograd.grad(y, (a, wl), moved(dy))
    want = torch.zeros(R, H, dtype=torch.float64)
    want[slot[real]] = (w.double().cpu()[..., None] * dy.double().cpu()[:, None])[real]
    assert ((dys.double().cpu() - want).abs() <= (he + 2.0 ** -24) * 1.001 * want.abs() + 2.0 ** -25).all()
    prod = rows * dy.double().cpu()[:, None]
    assert ((dw.double().cpu() - prod.sum(-1)).abs() <= (H / 128 + 18) * 2.0 ** -24 * prod.abs().sum(-1)).all()


def test_gradients_against_differences():
    """Both operators are linear in each argument, so a central difference along a direction is exact up to rounding."""
    import cbmoe
    plan, idx, w, new = case(20, 6, 3, 40, 4, "fp32", True)
    R = plan["tok_row"].numel()
    x, ys, a, b = new(20, 40).requires_grad_(), new(R, 40).requires_grad_(), new(R, 40), new(20, 40)
    wl = w.clone().requires_grad_()

    def check(f, leaf, dout):
        g, = torch.autograd.grad(f(leaf), leaf, dout)
        d = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(1)).cuda()
        with torch.no_grad():
            diff = ((f(leaf + d) - f(leaf - d)).double() * dout.double()).sum() / 2
        size = (g.double() * d.double()).abs().sum()
        assert (diff - (g.double() * d.double()).sum()).abs() <= 2.0 ** -20 * (size + dout.double().abs().sum())

    check(lambda t: cbmoe.moe_permute(t, plan), x, a)
    check(lambda t: cbmoe.moe_unpermute(t, wl, plan), ys, b)
    check(lambda t: cbmoe.moe_unpermute(ys, t, plan), wl, b)


def test_round_trip_and_partial_gradients():
    """permute -> a row-wise map -> unpermute: gradients reach x and w through both; frozen rows skip theirs."""
    import cbmoe
    plan, idx, w, new = case(64, 8, 2, 128, 8, "fp32", False)
    x, wl = new(64, 128).requires_grad_(), w.clone().requires_grad_()
    y = cbmoe.moe_unpermute(torch.tanh(cbmoe.moe_permute(x, plan)), wl, plan)
    g = new(64, 128)
    dx, dw = torch.autograd.grad(y, (x, wl), g)
    xd, wd = x.detach().double().requires_grad_(), w.double().requires_grad_()
    yd = wd.sum(1, keepdim=True) * torch.tanh(xd)
    rx, rw = torch.autograd.grad(yd, (xd, wd), g.double())
    assert (y.double() - yd).abs().max() <= 2.0 ** -20 and (dx.double() - rx).abs().max() <= 2.0 ** -18
    assert (dw.double() - rw).abs().max() <= 2.0 ** -16
    ys = cbmoe.moe_permute(x.detach(), plan)
    only_w, = torch.autograd.grad(cbmoe.moe_unpermute(ys, wl, plan), wl, g)
    ysl = ys.clone().requires_grad_()
    only_ys, = torch.autograd.grad(cbmoe.moe_unpermute(ysl, w, plan), ysl, g)
    both = torch.autograd.grad(cbmoe.moe_unpermute(ysl, wl, plan), (ysl, wl), g)
    assert torch.equal(only_ys, both[0]) and torch.equal(only_w, both[1])
    assert not cbmoe.moe_unpermute(ys, w, plan).requires_grad
    half = cbmoe.moe_unpermute(ys, wl.detach().half().requires_grad_(), plan)      # w of another type is taken in fp32
    assert half.dtype == torch.float32


def test_strided_inputs_streams_and_graphs():
    import cbmoe
    plan, idx, w, new = case(90, 8, 4, 96, 1, "bf16", False)
    big = new(96, 90 * 2)
    x = big.t()[::2]
    want = cbmoe.moe_permute(x.contiguous(), plan)
    assert torch.equal(cbmoe.moe_permute(x, plan), want)
    off = new(90 * 96 + 1)[1:].view(90, 96)                  # rows not 16-byte aligned: single elements
    assert torch.equal(cbmoe.moe_permute(off, plan), cbmoe.moe_permute(off.clone(), plan))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        xs = cbmoe.moe_permute(x, plan)
        y = cbmoe.moe_unpermute(xs, w, plan)
    torch.cuda.synchronize()
    assert torch.equal(xs, want)
    static, gy = x.contiguous().requires_grad_(), new(90, 96)
    eager = torch.autograd.grad(cbmoe.moe_unpermute(cbmoe.moe_permute(static, plan), w, plan), static, gy)[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yc = cbmoe.moe_unpermute(cbmoe.moe_permute(static, plan), w, plan)
        gc, = torch.autograd.grad(yc, static, gy)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(yc.detach(), y) and torch.equal(gc, eager)


def test_bad_rows_in_a_plan_are_skipped():
    """Rows outside the sorted range are empty slots to every kernel, so a bad plan reads and writes nothing outside."""
    import cbmoe
    plan, idx, w, new = case(10, 4, 2, 32, 1, "fp32", False)
    R = 20
    broken = {"tok_row": plan["tok_row"][:R].clone(), "row_slot": plan["row_slot"].clone()}
    broken["row_slot"][3, 1], broken["row_slot"][4, 0] = R, 1 << 30
    ys, wl = new(R, 32).requires_grad_(), w.clone().requires_grad_()
    y = cbmoe.moe_unpermute(ys, wl, broken)
    fixed = {**broken, "row_slot": torch.where(broken["row_slot"] >= R, -1, broken["row_slot"])}
    assert torch.equal(y, cbmoe.moe_unpermute(ys, wl, fixed))
    dw, = torch.autograd.grad(y, wl, torch.ones_like(y))
    assert dw[3, 1] == 0 and dw[4, 0] == 0 and torch.isfinite(dw).all()


def test_no_tokens():
    import cbmoe
    for tm in (1, 16):
        plan, idx, w, new = case(4, 4, 2, 32, tm, "bf16", False)
        none = {"tok_row": torch.full((4 * tm,), -1, dtype=torch.int32, device="cuda"),
                "row_slot": torch.zeros((0, 2), dtype=torch.int32, device="cuda")}
        x = torch.zeros(0, 32, device="cuda", requires_grad=True)
        xs = cbmoe.moe_permute(x, none)
        assert xs.shape == (4 * tm, 32) and (xs == 0).all()
        assert torch.autograd.grad(xs.sum(), x)[0].shape == (0, 32)
        ys = torch.ones(4 * tm, 32, device="cuda", requires_grad=True)
        y = cbmoe.moe_unpermute(ys, torch.zeros(0, 2, device="cuda"), none)
        assert y.shape == (0, 32) and (torch.autograd.grad(y.sum(), ys)[0] == 0).all()


def test_refusals():
    import cbmoe
    plan, idx, w, new = case(10, 4, 2, 32, 1, "bf16", False)
    x, ys = new(10, 32), new(20, 32)
    p, u = cbmoe.moe_permute, cbmoe.moe_unpermute
    for call in (lambda: p(x[:9], plan), lambda: p(x.double(), plan), lambda: p(x[0], plan), lambda: p(x[:, :0], plan),
                 lambda: u(ys[:19], w, plan), lambda: u(ys, w[:, :1], plan), lambda: u(ys, w.cpu(), plan),
                 lambda: u(ys.long(), w, plan), lambda: p(x, {**plan, "row_slot": plan["row_slot"].long()}),
                 lambda: p(x, {**plan, "tok_row": plan["tok_row"].cpu()}),
                 lambda: p(x, {**plan, "row_slot": plan["row_slot"].t()})):
        with pytest.raises(ValueError):
            call()


def test_rows_past_32_bit_offsets():
    """More than 2^31 elements of sorted rows: permute, its gradient and unpermute find the last rows where they lie."""
    import cbmoe
    T, H, E, k = 33000, 32776, 4, 2
    g = torch.Generator(device="cuda").manual_seed(3)
    idx = torch.randint(0, E, (T, k), device="cuda", generator=g, dtype=torch.int32)
    w = torch.ones(T, k, device="cuda")
    plan = cbmoe.ops.route_plan(idx, w, E, 1)
    x = torch.randint(-3, 4, (T, H), device="cuda", generator=g).to(torch.bfloat16)
    slot = plan["row_slot"].long()
    xs = cbmoe.moe_permute(x, plan)
    assert xs.shape == (T * k, H) and xs.numel() > 1 << 31
    for rows in torch.arange(T, device="cuda").split(4000):
        assert torch.equal(xs[slot[rows, 0]], x[rows]) and torch.equal(xs[slot[rows, 1]], x[rows])
    y = cbmoe.moe_unpermute(xs, w, plan)                      # whole numbers: x + x without rounding
    assert torch.equal(y, x + x)
    del y
    ys = xs.requires_grad_()
    wl = w.clone().requires_grad_()
    dys, dw = torch.autograd.grad(cbmoe.moe_unpermute(ys, wl, plan), (ys, wl), x)
    assert torch.equal(dys, xs.detach())
    want = torch.cat([x[r].float().square().sum(1) for r in torch.arange(T, device="cuda").split(4000)])
    assert torch.equal(dw, want[:, None].expand(T, k))        # sums of whole numbers below 2^24: exact


@pytest.mark.parametrize("dtype", list(TYPES))
def test_infinities_and_nans_in_masked_places(dtype):
    """Padding rows of ys and of permute's incoming gradient, and the weights of empty slots, are never read."""
    import cbmoe
    T, E, k, H, tm = 29, 5, 4, 70, 8
    plan, idx, w, new = case(T, E, k, H, tm, dtype, True)
    pad, empty = plan["tok_row"] < 0, plan["row_slot"] < 0
    x, ys, dy, g = new(T, H).requires_grad_(), new(pad.numel(), H), new(T, H), new(pad.numel(), H)
    bad_ys, bad_g, bad_w = ys.clone(), g.clone(), w.clone()
    bad_ys[pad], bad_g[pad] = float("nan"), float("-inf")
    bad_w[empty] = float("nan")
    ys[pad], w[empty] = 0, 0
    got = []
    for a, b, wl in ((ys, g, w), (bad_ys, bad_g, bad_w)):
        a, wl = a.clone().requires_grad_(), wl.clone().requires_grad_()
        y = cbmoe.moe_unpermute(a, wl, plan)
        got.append([y, *torch.autograd.grad(y, (a, wl), dy),
                    *torch.autograd.grad(cbmoe.moe_permute(x, plan), x, b)])
    assert all(torch.isfinite(t).all() and torch.equal(s, t) for s, t in zip(*got))

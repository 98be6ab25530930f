"""The e4m3 and token-order entry points refuse bad calls on the host, before any launch (no GPU needed): null device
pointers stand for tensors, 16 for an aligned one."""
import ctypes

import pytest
import torch

INVALID, WORKSPACE, UNSUPPORTED = -1, -3, -4
BF16, F16, F32, E4M3 = range(4)


@pytest.fixture(scope="module")
def L():
    import cbmoe
    return cbmoe.lib()


def test_quantize_refusals(L):
    f = L.cbmoe_fp8_quantize
    assert f(None, BF16, 0, 128, 128, None, 128, None, None) == 0                 # nothing to do
    assert f(None, BF16, 1, 128, 128, 16, 128, 16, None) == INVALID               # no x
    assert f(16, BF16, 1, 128, 128, None, 128, 16, None) == INVALID
    assert f(16, BF16, 1, 128, 128, 16, 128, None, None) == INVALID
    assert f(16, E4M3, 1, 128, 128, 16, 128, 16, None) == INVALID                 # codes are not quantised again
    assert f(16, BF16, 1, 0, 128, 16, 128, 16, None) == INVALID
    assert f(16, BF16, -1, 128, 128, 16, 128, 16, None) == INVALID
    assert f(16, BF16, 1, 128, 127, 16, 128, 16, None) == INVALID                 # row stride below K
    assert f(16, BF16, 1, 128, 128, 16, 127, 16, None) == INVALID


def linear(L, q=16, ldq=128, s=16, rows=4, K=128, x=16, x_type=BF16, ldx=128, xs=None, N=1, y=16, y_type=F32, ws=256,
           nbytes=1 << 30):
    return L.cbmoe_fp8_linear(q, ldq, s, rows, K, x, x_type, ldx, xs, N, y, y_type, ws, nbytes, None)


def test_linear_refusals(L):
    assert linear(L, N=0) == 0
    for bad in (dict(q=None), dict(s=None), dict(rows=0), dict(K=0), dict(N=-1), dict(ldq=120), dict(ldq=136), dict(q=24),
                dict(x=None), dict(y=None), dict(ldx=100), dict(x_type=4), dict(y_type=E4M3), dict(y_type=-1),
                dict(x_type=E4M3), dict(x_type=E4M3, xs=16, ldx=136), dict(x_type=E4M3, xs=16, x=24)):
        assert linear(L, **bad) == INVALID, bad
    assert linear(L, N=(1 << 30) + 1) == UNSUPPORTED
    assert linear(L, K=(1 << 24) + 16, ldq=1 << 25, ldx=1 << 25) == UNSUPPORTED
    assert linear(L, rows=0x7ffffe01) == INVALID
    assert linear(L, ws=None) == WORKSPACE
    assert linear(L, ws=264) == WORKSPACE                                         # not 256-byte aligned
    need = L.cbmoe_fp8_linear_workspace_bytes(1, 128, 4, BF16)
    assert need >= 128 + 4 and linear(L, nbytes=need - 1) == WORKSPACE
    assert L.cbmoe_fp8_linear_workspace_bytes(1, 0, 4, BF16) == 0
    assert L.cbmoe_fp8_linear_workspace_bytes(-1, 8, 4, BF16) == 0


def test_experts_refusals(L):
    from cbmoe._lib import Fp8Experts
    good = dict(E=4, H=256, I=128, gate=16, up=16, down=16, gate_s=16, up_s=16, down_s=16, ld_in=256, ld_down=128)

    def call(N=1, k=2, x=16, idx=16, w=16, y=16, y_type=F32, ws=256, nbytes=1 << 30, **kw):
        ex = Fp8Experts(**{**good, **kw})
        return L.cbmoe_fp8_experts_apply(ctypes.byref(ex), x, N, idx, w, k, 10.0, y, y_type, ws, nbytes, None)

    assert call(N=0) == 0
    for bad in (dict(E=0), dict(E=1025), dict(H=0), dict(I=0), dict(gate=None), dict(up=24), dict(down_s=None),
                dict(ld_in=250), dict(ld_in=240), dict(ld_down=136), dict(k=0), dict(k=65), dict(N=-1), dict(y_type=E4M3),
                dict(x=None), dict(idx=None), dict(w=None), dict(y=None)):
        assert call(**bad) == INVALID, bad
    assert call(ws=None) == WORKSPACE
    assert call(N=1 << 28, k=8) == UNSUPPORTED
    ex = Fp8Experts(**good)
    need = [L.cbmoe_fp8_experts_workspace_bytes(ctypes.byref(ex), n, 2, F32) for n in (1, 8, 64)]
    assert 0 < need[0] < need[1] < need[2]
    assert call(N=64, nbytes=need[2] - 1) == WORKSPACE


def test_token_order_refusals(L):
    def permute(x=16, t=BF16, T=2, H=8, slot=16, k=2, tok=16, R=4, xs=16):
        return L.cbmoe_permute(x, t, T, H, slot, k, tok, R, xs, None)

    assert permute(T=0, R=0) == 0
    for bad in (dict(t=E4M3), dict(T=-1), dict(H=0), dict(k=0), dict(R=-1), dict(x=None), dict(slot=None), dict(tok=None),
                dict(xs=None)):
        assert permute(**bad) == INVALID, bad

    def unpermute(ys=16, t=BF16, R=4, H=8, slot=16, w=16, T=2, k=2, y=16):
        return L.cbmoe_unpermute(ys, t, R, H, slot, w, T, k, y, None)

    assert unpermute(T=0) == 0
    for bad in (dict(t=7), dict(T=-1), dict(H=0), dict(k=0), dict(R=-1), dict(ys=None), dict(slot=None), dict(y=None)):
        assert unpermute(**bad) == INVALID, bad

    def backward(dy=16, ys=16, t=BF16, R=4, H=8, slot=16, tok=16, w=16, T=2, k=2, dys=16, dw=16):
        return L.cbmoe_unpermute_backward(dy, ys, t, R, H, slot, tok, w, T, k, dys, dw, None)

    assert backward(dys=None, dw=None) == 0 and backward(T=0, R=0) == 0
    for bad in (dict(t=7), dict(T=-1), dict(H=0), dict(k=0), dict(R=-1), dict(dy=None), dict(ys=None), dict(slot=None),
                dict(tok=None)):
        assert backward(**bad) == INVALID, bad


def test_tensors_off_the_gpu_are_refused():
    import cbmoe
    x = torch.zeros(2, 8)
    plan = {"tok_row": torch.zeros(4, dtype=torch.int32), "row_slot": torch.zeros(2, 2, dtype=torch.int32)}
    for call in (lambda: cbmoe.ops.fp8_quantize(x), lambda: cbmoe.moe_permute(x, plan),
                 lambda: cbmoe.moe_unpermute(x, torch.ones(2, 2), plan),
                 lambda: cbmoe.ops.fp8_linear(x.to(torch.float8_e4m3fn), x, x)):
        with pytest.raises(cbmoe.CbmoeError):
            call()


def test_row_padding_of_codes():
    from cbmoe import ops
    raw = torch.arange(60, dtype=torch.uint8)
    tight = raw.view(3, 20).view(torch.float8_e4m3fn)          # stride 20: padded copy
    q = ops.fp8_pad_rows(tight)
    assert q.shape == (3, 20) and ops.fp8_row_stride(q) == 32
    assert torch.equal(q.contiguous().view(torch.uint8), raw.view(3, 20))
    assert ops.fp8_pad_rows(q) is q
    whole = torch.zeros(2, 3, 32, dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert ops.fp8_row_stride(whole) == 32 and ops.fp8_pad_rows(whole) is whole
    assert ops.fp8_row_stride(whole[:, :2]) is None            # experts not dense
    assert ops.fp8_row_stride(whole[:, :, 16:]) == 32 and ops.fp8_row_stride(whole[:, :, 8:]) is None
    with pytest.raises(ValueError):
        ops.fp8_pad_rows(raw.view(3, 20))


def token_order(L, t):
    """The three entry points for elements of type t, with defaults that they take up to the launch."""
    def permute(x=16, T=2, H=8, slot=16, k=2, tok=16, R=4, xs=16):
        return L.cbmoe_permute(x, t, T, H, slot, k, tok, R, xs, None)

    def unpermute(ys=16, R=4, H=8, slot=16, w=16, T=2, k=2, y=16):
        return L.cbmoe_unpermute(ys, t, R, H, slot, w, T, k, y, None)

    def backward(dy=16, ys=16, R=4, H=8, slot=16, tok=16, w=16, T=2, k=2, dys=16, dw=16):
        return L.cbmoe_unpermute_backward(dy, ys, t, R, H, slot, tok, w, T, k, dys, dw, None)

    return permute, unpermute, backward


def test_misaligned_elements_are_refused(L):
    """A pointer off its element's alignment would be a misaligned address in the kernel."""
    from cbmoe._lib import Fp8Experts
    for t, size in ((BF16, 2), (F16, 2), (F32, 4)):
        permute, unpermute, backward = token_order(L, t)
        for f, typed, words in ((permute, ("x", "xs"), ("slot", "tok")), (unpermute, ("ys", "y"), ("slot", "w")),
                                (backward, ("dy", "ys", "dys"), ("slot", "tok", "w", "dw"))):
            for name in typed:
                assert f(**{name: 16 + size // 2}) == INVALID, (f, name)
            for name in words:
                assert f(**{name: 18}) == INVALID, (f, name)
        assert L.cbmoe_fp8_quantize(16 + size // 2, t, 1, 128, 128, 16, 128, 16, None) == INVALID
        assert linear(L, x=16 + size // 2, x_type=t) == INVALID
        assert linear(L, y=16 + size // 2, y_type=t) == INVALID
    assert L.cbmoe_fp8_quantize(16, BF16, 1, 128, 128, 17, 128, 18, None) == INVALID              # s
    assert linear(L, x_type=E4M3, xs=18) == INVALID
    ex = Fp8Experts(E=4, H=256, I=128, gate=16, up=16, down=16, gate_s=16, up_s=16, down_s=16, ld_in=256, ld_down=128)
    good = dict(x=16, idx=16, w=16, y=16, y_type=F32)
    for bad in (dict(x=17), dict(idx=18), dict(w=18), dict(y=18), dict(y=17, y_type=BF16)):
        a = {**good, **bad}
        assert L.cbmoe_fp8_experts_apply(ctypes.byref(ex), a["x"], 1, a["idx"], a["w"], 2, 10.0, a["y"], a["y_type"], 256,
                                         1 << 30, None) == INVALID, bad


def test_counts_past_32_bit_loops_are_refused(L):
    """The kernels' strided loops count in 32 bits: tokens, rows, widths and slots a token up to 2^31 - 2^16 stay in range."""
    most, past = 0x7fff0000, 0x7fff0001
    for t in (BF16, F16, F32):
        permute, unpermute, backward = token_order(L, t)
        for f in (permute, unpermute, backward):
            for name in ("T", "R", "H", "k"):
                assert f(**{name: past}) == UNSUPPORTED, (f, name)
        assert permute(T=most, R=0) == 0 and unpermute(T=0, R=most) == 0 and backward(T=most, dys=None, dw=None) == 0
        assert L.cbmoe_fp8_quantize(16, t, 1, (1 << 30) + 1, 1 << 31, 16, 1 << 31, 16, None) == UNSUPPORTED


def test_sizes_past_32_bits_are_refused():
    """Sizes that a C int would cut to other ones raise."""
    from cbmoe import _lib
    for sizes in ((1, (1 << 32) + 8), (1 << 31, 1), (0, 1 << 31)):
        with pytest.raises(ValueError):
            _lib.int_sizes(*sizes)
    _lib.int_sizes(0, 3, (1 << 31) - 1)

"""Tokens into expert order and back over a routing plan, with gradients: the row gather and the weighted combine of the
layer (resident.py:144-165) as operators, for expert products of the caller's own.

    plan = ops.route_plan(idx, w, E, tm)       # idx [T, k], w [T, k]
    xs = moe_permute(x, plan)                  # rows sorted by expert, each expert's rows in whole blocks of tm
    y = moe_unpermute(ys, w, plan)             # sum_j w[t, j] ys[row_slot[t, j]]

Types bf16, fp16, fp32, any width. Sums run in fp32 over a token's slots in order and are rounded once, so forward and
backward give the same bits on every call.
"""
import torch
from torch.autograd.function import once_differentiable

from ._lib import TYPES, check, int_sizes, lib, on_device, raw_stream, require_cuda


def _ptr(t):
    return None if t is None else t.data_ptr()


def _plan_rows(plan, device):
    """(tok_row [R], row_slot [T, k]) of a plan; with blocks of one row the R = T k rows that can be in use."""
    tok_row, row_slot = plan["tok_row"], plan["row_slot"]
    for name, t, dim in (("tok_row", tok_row, 1), ("row_slot", row_slot, 2)):
        if t.dtype is not torch.int32 or t.dim() != dim or not t.is_contiguous() or t.device != device:
            raise ValueError(f"plan[{name!r}] is contiguous int32 of {dim} dimension(s) on {device}, got {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
    int_sizes(*tok_row.shape, *row_slot.shape)
    if row_slot.shape[1] == 0:
        raise ValueError("the plan has no slots per token")
    blocks = plan.get("blk_expert")
    if blocks is not None and blocks.shape[0] == tok_row.shape[0]:
        tok_row = tok_row[:row_slot.numel()]
    return tok_row, row_slot


def _rows(name, t):
    require_cuda(t)
    if t.dim() != 2 or t.shape[1] == 0:
        raise ValueError(f"{name} is [rows, H], got {tuple(t.shape)}")
    int_sizes(*t.shape)
    if t.dtype not in TYPES:
        raise ValueError(f"{name} is bf16, fp16 or fp32, got {t.dtype}")


def _permute(x, tok_row, row_slot):
    (T, k), R, H = row_slot.shape, tok_row.numel(), x.shape[1]
    xs = torch.empty((R, H), dtype=x.dtype, device=x.device)
    with on_device(x):
        check(lib().cbmoe_permute(x.data_ptr(), TYPES[x.dtype], T, H, row_slot.data_ptr(), k, tok_row.data_ptr(), R,
                                  xs.data_ptr(), raw_stream(row_slot)), "cbmoe_permute")
    return xs


def _unpermute(ys, w, row_slot):
    (T, k), (R, H) = row_slot.shape, ys.shape
    y = torch.empty((T, H), dtype=ys.dtype, device=ys.device)
    with on_device(ys):
        check(lib().cbmoe_unpermute(ys.data_ptr(), TYPES[ys.dtype], R, H, row_slot.data_ptr(), _ptr(w), T, k,
                                    y.data_ptr(), raw_stream(row_slot)), "cbmoe_unpermute")
    return y


class _Permute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tok_row, row_slot):
        ctx.save_for_backward(row_slot)
        return _permute(x.contiguous(), tok_row, row_slot)

    @staticmethod
    @once_differentiable
    def backward(ctx, dxs):
        row_slot, = ctx.saved_tensors
        return _unpermute(dxs.contiguous(), None, row_slot), None, None


class _Unpermute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ys, w, tok_row, row_slot):
        ys, w = ys.contiguous(), w.contiguous()
        ctx.save_for_backward(ys if ctx.needs_input_grad[1] else None, w, tok_row, row_slot)
        ctx.rows = ys.shape[0]
        return _unpermute(ys, w, row_slot)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        ys, w, tok_row, row_slot = ctx.saved_tensors
        dy = dy.contiguous()
        (T, k), R, H = row_slot.shape, ctx.rows, dy.shape[1]
        need_ys, need_w = ctx.needs_input_grad[:2]
        dys = torch.empty((R, H), dtype=dy.dtype, device=dy.device) if need_ys else None
        dw = torch.empty((T, k), dtype=torch.float32, device=dy.device) if need_w else None
        with on_device(dy):
            check(lib().cbmoe_unpermute_backward(dy.data_ptr(), _ptr(ys), TYPES[dy.dtype], R, H, row_slot.data_ptr(),
                                                 tok_row.data_ptr(), w.data_ptr(), T, k, _ptr(dys), _ptr(dw),
                                                 raw_stream(row_slot)), "cbmoe_unpermute_backward")
        return dys, dw, None, None


def moe_permute(x, plan):
    """x [T, H] -> xs [R, H] in the plan's order: xs[row_slot[t, j]] = x[t], padding rows zero. `plan` as ops.route_plan
    returns it (tok_row, row_slot); R = tok_row's length, or T k with blocks of one row. Differentiable in x (a token's
    gradient is the fp32 sum over its rows)."""
    _rows("x", x)
    tok_row, row_slot = _plan_rows(plan, x.device)
    if row_slot.shape[0] != x.shape[0]:
        raise ValueError(f"the plan has {row_slot.shape[0]} tokens, x {x.shape[0]}")
    return _Permute.apply(x, tok_row, row_slot)


def moe_unpermute(ys, w, plan):
    """ys [R, H] in the plan's order, w [T, k] -> y [T, H] = sum_j w[t, j] ys[row_slot[t, j]] in ys's type; empty slots
    (negative experts) add nothing. Differentiable in ys (padding rows get zeros) and in w."""
    _rows("ys", ys)
    tok_row, row_slot = _plan_rows(plan, ys.device)
    if w.shape != row_slot.shape or w.device != ys.device:
        raise ValueError(f"w is {tuple(row_slot.shape)} on {ys.device}, got {tuple(w.shape)} on {w.device}")
    if ys.shape[0] != tok_row.numel():
        raise ValueError(f"the plan has {tok_row.numel()} rows, ys {ys.shape[0]}")
    return _Unpermute.apply(ys, w.to(torch.float32), tok_row, row_slot)

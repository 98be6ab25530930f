"""Tensor-level wrappers of the C ABI: load-time repacks, the routing plan, and the single-matrix ops.

Every function takes and returns torch tensors on the current CUDA device and enqueues on the current stream.
bf16 tensors cross the ABI as raw bit patterns; int/float tensors as-is.
"""
import ctypes

import torch

from ._lib import (E4M3, TYPES, check, int_sizes, lib, no_gradient, on_device, ptr, raw_stream, require_cuda,
                   stream_handle)

PLAN_FIELDS = ("counts", "row_start", "act", "n_act", "n_blocks", "n_pass", "blk_expert", "tok_row", "w_row",
               "row_slot", "pass_expert", "pass_row0", "pass_cnt")


def _contig(t, dtype):
    assert t.dtype == dtype, (t.dtype, dtype)
    return t.contiguous()


def pack_cb3(idx0, cb0, idx1=None, cb1=None):
    """CB3 tables idx uint32-as-int32 [E, rows, K*3/32], cb bf16 [E, rows, 8] (one matrix, or gate + up) ->
    (idx_k uint8, cb_k uint8) in the kernel layout. Replaces pack_chip_planes (resident.py:48-60)."""
    require_cuda(idx0, cb0, idx1, cb1)
    nmat = 1 if idx1 is None else 2
    E, rows, wpr = idx0.shape
    K = wpr * 32 // 3
    idx0, cb0 = _contig(idx0, torch.int32), _contig(cb0, torch.bfloat16)
    if nmat == 2:
        idx1, cb1 = _contig(idx1, torch.int32), _contig(cb1, torch.bfloat16)
        assert idx1.shape == idx0.shape and cb1.shape == cb0.shape
    L = lib()
    idx_k = torch.empty(L.cbmoe_cb3k_idx_bytes(E, rows, K, nmat), dtype=torch.uint8, device=idx0.device)
    cb_k = torch.empty(L.cbmoe_cb3k_cb_bytes(E, rows, nmat), dtype=torch.uint8, device=idx0.device)
    check(L.cbmoe_cb3k_repack(ptr(idx0), ptr(cb0), ptr(idx1), ptr(cb1), nmat, E, rows, K, ptr(idx_k), ptr(cb_k),
                              stream_handle()), "cbmoe_cb3k_repack")
    return idx_k, cb_k


def build_cb8(cb_k, nmat, E, rows):
    """CB3K codebooks -> CB8 tables (uint8: int8 hi / uint8 lo bytes + row factors) for the int8-digit decode kernels."""
    require_cuda(cb_k)
    out = torch.empty(lib().cbmoe_cb8_bytes(E, rows, nmat), dtype=torch.uint8, device=cb_k.device)
    check(lib().cbmoe_cb8_build(ptr(cb_k), nmat, E, rows, ptr(out), stream_handle()), "cbmoe_cb8_build")
    return out


def cb8_matvec(idx_k, cb8, rows, K, x, ws=None):
    """One matrix (expert 0 of a CB3K table) times x bf16 [N, K] -> fp32 [N, rows] on the int8-digit decode kernel.
    `ws`: the workspace (uint8, at least cbmoe_cb8_matvec_workspace_bytes); allocated when not given."""
    require_cuda(idx_k, cb8, x)
    N = x.shape[0]
    xb = x.to(torch.bfloat16).contiguous()
    y = torch.empty((N, rows), dtype=torch.float32, device=x.device)
    if ws is None:
        ws = torch.empty(max(1, lib().cbmoe_cb8_matvec_workspace_bytes(N, K)), dtype=torch.uint8, device=x.device)
    check(lib().cbmoe_cb8_matvec(ptr(idx_k), ptr(cb8), rows, K, ptr(xb), N, ptr(y), ptr(ws), ws.numel(),
                                 stream_handle()), "cbmoe_cb8_matvec")
    return y


def dequant_cb3k(idx_k, cb_k, nmat, E, rows, K):
    """Kernel-layout table -> bf16 [nmat, E, rows, K] through the kernels' register dequant."""
    require_cuda(idx_k, cb_k)
    out = torch.empty((nmat, E, rows, K), dtype=torch.bfloat16, device=idx_k.device)
    check(lib().cbmoe_cb3k_dequant(ptr(idx_k), ptr(cb_k), nmat, E, rows, K, ptr(out), stream_handle()),
          "cbmoe_cb3k_dequant")
    return out


def pack_w8(q0, q1=None):
    """int8 leaves q [K_in, rows_out] (quant8 "[in, out]"; one, or gate + up) -> W8K uint8."""
    require_cuda(q0, q1)
    nmat = 1 if q1 is None else 2
    K, rows = q0.shape
    q0 = _contig(q0, torch.int8)
    q1 = None if q1 is None else _contig(q1, torch.int8)
    out = torch.empty(lib().cbmoe_w8k_bytes(rows, K, nmat), dtype=torch.uint8, device=q0.device)
    check(lib().cbmoe_w8k_repack(ptr(q0), ptr(q1), nmat, K, rows, ptr(out), stream_handle()), "cbmoe_w8k_repack")
    return out


def dequant_w8k(qk, s0, s1, scale_axis, nmat, rows, K):
    require_cuda(qk, s0, s1)
    out = torch.empty((nmat, rows, K), dtype=torch.bfloat16, device=qk.device)
    check(lib().cbmoe_w8k_dequant(ptr(qk), ptr(s0.contiguous()), ptr(None if s1 is None else s1.contiguous()),
                                  scale_axis, nmat, rows, K, ptr(out), stream_handle()), "cbmoe_w8k_dequant")
    return out


def plan_layout(T, k, E, tm, pass_tokens):
    off = (ctypes.c_int64 * 14)()
    check(lib().cbmoe_plan_layout(T, k, E, tm, pass_tokens, off), "cbmoe_plan_layout")
    return list(off)


def route_plan(idx, w, E, tm, pass_tokens=8):
    """pallas_moe.ragged_plan (pallas_moe.py:564-592) on the GPU -> dict of int32/fp32 tensors (views of one
    buffer): blk_expert, n_blocks, tok_row, w_row, row_slot [T, k], and the decode lists."""
    require_cuda(idx, w)
    T, k = idx.shape
    off = plan_layout(T, k, E, tm, pass_tokens)
    buf = torch.empty(off[13], dtype=torch.int32, device=idx.device)
    check(lib().cbmoe_route_plan(ptr(_contig(idx, torch.int32)), ptr(_contig(w, torch.float32)), T, k, E, tm,
                                 pass_tokens, ptr(buf), off[13] * 4, stream_handle()), "cbmoe_route_plan")
    S = T * k
    G = -(-S // tm) + E
    P = -(-S // pass_tokens) + E
    used = (E, E, E, 1, 1, 1, G, G * tm, G * tm, S, P, P, P)
    sizes = []
    for i, n in enumerate(used):   # each field and what pads it to the next one: one split instead of a view per field
        sizes += [n, off[i + 1] - off[i] - n]
    out = dict(zip(PLAN_FIELDS, buf.split(sizes)[::2]))
    out["w_row"] = out["w_row"].view(torch.float32)
    out["row_slot"] = out["row_slot"].view(T, k)
    return out


def cb3_matvec(idx_k, cb_k, rows, K, x):
    """One CB3K matrix times x bf16 [N, K] -> fp32 [N, rows] (moe_matvec with every slot on one expert)."""
    require_cuda(idx_k, cb_k, x)
    x = _contig(x, torch.bfloat16)
    N = x.shape[0]
    y = torch.empty((N, rows), dtype=torch.float32, device=x.device)
    check(lib().cbmoe_cb3_matvec(ptr(idx_k), ptr(cb_k), rows, K, ptr(x), N, ptr(y), None, 0, stream_handle()),
          "cbmoe_cb3_matvec")
    return y


def w8_linear(qk, s, scale_axis, rows, K, x):
    """x bf16 [N, K] @ bf16(q * s) -> fp32 [N, rows] (quant8.dequant_tree + dot)."""
    require_cuda(qk, s, x)
    x = _contig(x, torch.bfloat16)
    N = x.shape[0]
    y = torch.empty((N, rows), dtype=torch.float32, device=x.device)
    check(lib().cbmoe_w8_linear(ptr(qk), ptr(_contig(s, torch.float32)), scale_axis, rows, K, ptr(x), N, ptr(y),
                                None, 0, stream_handle()), "cbmoe_w8_linear")
    return y


def w8_logits(qk, s, rows, K, x, ws=None):
    """The int8 lm_head (engine.py:345-351): x bf16 [N, K] times int8 columns (W8K, per-column scales s [rows])
    -> bf16 [N, rows] = bf16(f32(x @ q) * s), the scale after the dot."""
    require_cuda(qk, s, x)
    N = x.shape[0]
    xb = x.to(torch.bfloat16).contiguous()
    out = torch.empty((N, rows), dtype=torch.bfloat16, device=x.device)
    if ws is None:
        ws = torch.empty(max(1, lib().cbmoe_cb8_matvec_workspace_bytes(N, K)), dtype=torch.uint8, device=x.device)
    check(lib().cbmoe_w8_logits(ptr(qk), ptr(s.float().contiguous()), rows, K, ptr(xb), N, ptr(out), ptr(ws),
                                ws.numel(), stream_handle()), "cbmoe_w8_logits")
    return out


def _fp8_x(x):
    """(x 2-D with unit inner stride, its row stride in elements)."""
    if x.dim() != 2:
        raise ValueError(f"x is [N, K], got {tuple(x.shape)}")
    if x.stride(1) != 1 or x.stride(0) < x.shape[1]:
        x = x.contiguous()
    return x, max(x.stride(0), x.shape[1])


def fp8_quantize(x):
    """x [N, K] (bf16, fp16 or fp32) -> (q float8_e4m3fn [N, K], s fp32 [N, ceil(K / 128)]): per row and group of 128
    columns the scale is the least power of two s >= 2^-100 with max|x| <= 448 s, the codes e4m3(x / s). A group with
    an infinity or a NaN has the scale NaN. q is a view of rows padded to 16 bytes, as fp8_linear takes it. Has no
    gradient: an x that requires one is refused."""
    require_cuda(x)
    no_gradient("fp8_quantize", x)
    if x.dtype not in TYPES:
        raise ValueError(f"x is bf16, fp16 or fp32, got {x.dtype}")
    x, ldx = _fp8_x(x)
    N, K = x.shape
    int_sizes(N, K)
    if K == 0:
        raise ValueError("x has no columns")
    ld = -(-K // 16) * 16
    with on_device(x):
        q = torch.empty((N, ld), dtype=torch.float8_e4m3fn, device=x.device)
        s = torch.empty((N, -(-K // 128)), dtype=torch.float32, device=x.device)
        check(lib().cbmoe_fp8_quantize(x.data_ptr(), TYPES[x.dtype], N, K, ldx, q.data_ptr(), ld, s.data_ptr(), raw_stream(x)),
              "cbmoe_fp8_quantize")
    return q[:, :K], s


def fp8_pad_rows(q):
    """e4m3 codes [.., rows, K] in the layout the kernels read: unit inner stride, rows dense at a stride of a multiple
    of 16 bytes, first row 16-byte aligned. Returned as they are when they already are so; else a padded copy (load time)."""
    if q.dtype != torch.float8_e4m3fn or q.dim() < 2:
        raise ValueError(f"codes are float8_e4m3fn [.., rows, K], got {q.dtype} {tuple(q.shape)}")
    K = q.shape[-1]
    if fp8_row_stride(q) is not None:
        return q
    out = torch.zeros(q.shape[:-1] + (-(-K // 16) * 16,), dtype=torch.uint8, device=q.device)
    out[..., :K] = q.view(torch.uint8) if q.stride(-1) == 1 else q.contiguous().view(torch.uint8)
    return out.view(torch.float8_e4m3fn)[..., :K]


def fp8_row_stride(q):
    """Row stride (bytes) of codes laid out as the kernels read them (fp8_pad_rows), or None."""
    ld = q.stride(-2) if q.shape[-2] > 1 else -(-q.shape[-1] // 16) * 16
    if q.shape[-2] == 1 and q.dim() == 3 and q.shape[0] > 1:
        ld = q.stride(0)
    ok = (q.stride(-1) == 1 or q.shape[-1] == 1) and ld % 16 == 0 and ld >= q.shape[-1] and q.data_ptr() % 16 == 0
    if q.dim() == 3 and q.shape[0] > 1:
        ok = ok and q.stride(0) == ld * q.shape[1]
    return ld if ok else None


def fp8_table_stride(name, q, s, lead, rows, K, device):
    """Checks one table of block-scaled codes (q [*lead, rows, K] as fp8_pad_rows leaves it, s its scales); its row
    stride in bytes."""
    want = (*lead, -(-rows // 128), -(-K // 128))
    if q.dtype != torch.float8_e4m3fn or tuple(q.shape) != (*lead, rows, K):
        raise ValueError(f"{name}: codes are float8_e4m3fn {(*lead, rows, K)}, got {q.dtype} {tuple(q.shape)}")
    if s.dtype != torch.float32 or tuple(s.shape) != want or not s.is_contiguous():
        raise ValueError(f"{name}: scales are contiguous fp32 {want}, got {s.dtype} {tuple(s.shape)}")
    if q.device != device or s.device != device:
        raise ValueError(f"{name}: tensors on {q.device} and {s.device}, expected {device}")
    ld = fp8_row_stride(q)
    if ld is None:
        raise ValueError(f"{name}: rows are not 16-byte aligned at a stride of a multiple of 16: use fp8_pad_rows")
    return ld


def fp8_linear(q, s, x, out_dtype=torch.float32):
    """x [N, K] @ W^T -> [N, rows] in out_dtype (fp32, bf16, fp16), W = e4m3 codes q [rows, K] (fp8_pad_rows) times fp32
    scales s [ceil(rows / 128), ceil(K / 128)] of 128 x 128 blocks. x: bf16, fp16 or fp32, quantised per row in groups of
    128 as fp8_quantize does, or the pair (codes, scales) that fp8_quantize returned (one quantisation for several
    products). fp32 sums. Inference only: inputs that require a gradient are refused."""
    ready = isinstance(x, (tuple, list))
    xv, xs = x if ready else (x, None)
    require_cuda(q, s, xv, xs)
    no_gradient("fp8_linear", q, s, xv, xs)
    if q.dim() != 2 or xv.dim() != 2 or xv.shape[1] != q.shape[1] or q.shape[0] == 0 or q.shape[1] == 0:
        raise ValueError(f"q [rows, K] and x [N, K], got {tuple(q.shape)} and {tuple(xv.shape)}")
    if out_dtype not in TYPES:
        raise ValueError(f"out_dtype is fp32, bf16 or fp16, got {out_dtype}")
    (rows, K), N = q.shape, xv.shape[0]
    int_sizes(rows, K, N)
    ldq = fp8_table_stride("weights", q, s, (), rows, K, xv.device)
    if ready:
        if xv.dtype != torch.float8_e4m3fn:
            raise ValueError(f"a pair holds float8_e4m3fn codes, got {xv.dtype}")
        if xs.dtype != torch.float32 or tuple(xs.shape) != (N, -(-K // 128)) or xs.device != xv.device:
            raise ValueError(f"scales of x are fp32 {(N, -(-K // 128))} on {xv.device}, got {xs.dtype} {tuple(xs.shape)}")
        xv, xs = fp8_pad_rows(xv), xs.contiguous()
        ldx, code = (fp8_row_stride(xv) if N > 0 else K), E4M3
    else:
        if xv.dtype not in TYPES:
            raise ValueError(f"x is bf16, fp16 or fp32, got {xv.dtype}")
        xv, ldx = _fp8_x(xv)
        code = TYPES[xv.dtype]
    with on_device(xv):
        y = torch.empty((N, rows), dtype=out_dtype, device=xv.device)
        nbytes = lib().cbmoe_fp8_linear_workspace_bytes(N, K, rows, code)
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=xv.device)
        check(lib().cbmoe_fp8_linear(q.data_ptr(), ldq, s.data_ptr(), rows, K, xv.data_ptr(), code, ldx,
                                     None if xs is None else xs.data_ptr(), N, y.data_ptr(), TYPES[out_dtype],
                                     ws.data_ptr(), nbytes, raw_stream(xv)), "cbmoe_fp8_linear")
    return y

"""Routed experts in 8-bit floating point: e4m3 tables with an fp32 scale per 128 x 128 block, the form block-scaled
checkpoints ship (the reference's loader reads such safetensors, engine/glm53/checkpoint.py), behind
ResidentFetch.apply like the other table formats (resident.py:100-120), through cbmoe_fp8_experts_apply.

    p = fp8.pack_layer((gate_q, gate_s), (up_q, up_s), (down_q, down_s))
    y = ResidentFetch(out_dtype=torch.bfloat16).apply(p, x, idx, w, layer, limit)

Activations are quantised per row in groups of 128 (ops.fp8_quantize); so is the SwiGLU output before the down product.
"""
import torch

from . import ops
from ._lib import TYPES, Fp8Experts, check, int_sizes, lib, no_gradient, on_device, raw_stream, require_cuda

FP8 = "FP8"


def pack_layer(gate, up, down):
    """One layer's tables from (codes, scales) pairs on the GPU: gate and up float8_e4m3fn [E, I, H] with fp32 scales
    [E, ceil(I / 128), ceil(H / 128)], down [E, H, I] with [E, ceil(H / 128), ceil(I / 128)] -> the table dict
    ResidentFetch.apply takes. Codes whose rows are 16-byte aligned are kept as they are, others get a padded copy."""
    (gq, gs), (uq, us), (dq, ds) = gate, up, down
    require_cuda(gq, gs, uq, us, dq, ds)
    if gq.dim() != 3 or 0 in gq.shape:
        raise ValueError(f"gate codes are [E, I, H], got {tuple(gq.shape)}")
    E, I, H = gq.shape
    int_sizes(E, I, H)
    gq, uq, dq = (ops.fp8_pad_rows(t) for t in (gq, uq, dq))
    gs, us, ds = (t.contiguous() for t in (gs, us, ds))
    ld = [ops.fp8_table_stride(n, q, s, (E,), r, c, gq.device)
          for n, q, s, r, c in (("gate", gq, gs, I, H), ("up", uq, us, I, H), ("down", dq, ds, H, I))]
    if ld[0] != ld[1]:
        raise ValueError(f"gate and up have different row strides: {ld[0]} and {ld[1]}")
    return {"format": FP8, "E": E, "H": H, "I": I, "qtypes": dict.fromkeys(("gate_q", "up_q", "down_q"), FP8),
            "gate_q": (gq, gs), "up_q": (uq, us), "down_q": (dq, ds), "ld": (ld[0], ld[2])}


def experts_struct(p):
    (gq, gs), (uq, us), (dq, ds) = p["gate_q"], p["up_q"], p["down_q"]
    return Fp8Experts(p["E"], p["H"], p["I"], gq.data_ptr(), uq.data_ptr(), dq.data_ptr(), gs.data_ptr(), us.data_ptr(),
                      ds.data_ptr(), *p["ld"])


def apply(p, x, idx, w, limit, out_dtype=torch.float32):
    """x bf16 [N, H]; idx int32 [N, k]; w fp32 [N, k] -> the routed partial [N, H] in out_dtype (fp32, bf16, fp16).
    Inference only: inputs that require a gradient are refused."""
    no_gradient("the expert layer on FP8 tables", x, w, *(t for n in ("gate_q", "up_q", "down_q") for t in p[n]))
    N, k = idx.shape
    int_sizes(N, k)
    if out_dtype not in TYPES:
        raise ValueError(f"out_dtype is fp32, bf16 or fp16, got {out_dtype}")
    if not p["gate_q"][0].device == x.device == idx.device == w.device:
        raise ValueError(f"tables on {p['gate_q'][0].device}, x on {x.device}, idx on {idx.device}, w on {w.device}")
    ex = experts_struct(p)
    with on_device(x):
        y = torch.empty((N, p["H"]), dtype=out_dtype, device=x.device)
        # per call, from the caching allocator: calls on several streams and captured graphs share nothing
        nbytes = lib().cbmoe_fp8_experts_workspace_bytes(ex, N, k, TYPES[out_dtype])
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=x.device)
        check(lib().cbmoe_fp8_experts_apply(ex, x.data_ptr(), N, idx.data_ptr(), w.data_ptr(), k, float(limit),
                                            y.data_ptr(), TYPES[out_dtype], ws.data_ptr(), nbytes, raw_stream(x)),
              "cbmoe_fp8_experts_apply")
    return y

"""CPU oracle for the codebook-MoE expert path: TEST INFRASTRUCTURE, not product code.

Only `tests/`, `__graft_entry__.smoke()` and the CPU-baseline legs of `bench.py` may import this package, and only
as the checker or as the timed CPU baseline. The CUDA library never calls it and has no CPU fallback.

What it restates (reference = shallmall/kaggle-llm-endpoint, paths relative to launcher/glm53-flash/engine/glm53/):
  cb3.py   the CB3 expert format named by the benchmark configs (3-bit indices, little-endian in uint32, one
           8-entry bf16 codebook per row). The reference has NO implementation of CB3; its dequant follows the
           semantics of `planes.dequant_planes` / `moe_matvec_ref` (pallas_moe.py:310-323): gather -> dequant -> f32
           contraction.
  q8.py    int8 weight-only storage, quant8.py:26-32 (quantize_array) and quant8.py:91-99 (dequant_tree).
  moe.py   swiglu_clamped (model.py:119-122), the decode composition `_apply_kernel` (resident.py:110-120), the
           grouped prefill plan `ragged_plan` (pallas_moe.py:564-592) and the ragged GEMM semantics
           (pallas_moe.py:622-755, resident.py:144-165), the shared expert `mlp_partial` (model.py:125-127) and
           `moe_dense`'s sum (model.py:840-856).
  gen.py   seeded synthetic inputs with the benchmark configs' shapes and value distributions.
  iq.py    the reference's real expert formats IQ2_S / IQ3_S / IQ4_XS (iqquant.py:108-146, llama.cpp's published
           dequant; grid tables loaded from gguf-py at run time).
  fp8.py   e4m3 with block scales in float64: the activation quantiser, the block-scaled product and the routed experts
           on such tables, each with a bound on an fp32 evaluation's error. No counterpart in the reference.

Pinning: the format-independent pieces (ragged_plan, swiglu_clamped, quantize_array, dequant_tree, the decode and
ragged compositions) are pinned by fixtures generated by executing the reference's own functions on a NumPy-backed
jax stand-in (tests/golden/make_golden.py). CB3 itself has no reference implementation, so its dequant is pinned
only by the written spec and hand-computed known-answer vectors: for CB3, parity is unpinned by the reference.
The IQ formats are pinned bit for bit by the reference's own dequant executed on its GGUF samples and random
blocks (tests/golden/make_iq_golden.py -> iq_samples.npz) and by gguf-py 0.19.0.
"""

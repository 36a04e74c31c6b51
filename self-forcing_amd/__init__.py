"""MI355X (gfx950) Monarch / KV-cache attention for the causal Wan DiT.

Host-side mirror of the reference's attention operators; all compute runs in the HIP
library `libsfm_attn.so` built from `csrc/` (see `build.py`).  Sub-modules keep the
reference's module names:

    monarch_attn.monarch_attn_with_kv_cache / monarch_attn.monarch_attn
    attention.attention / attention.full_attention_with_kv_cache
    paged_attn.plan_pages / write_pages / paged_attention / select_pages (many requests, one paged cache)
    prologue.qk_prologue / prologue.rope_table
    causal_model.CausalWanModel (+ self-attention, block, head), pipeline.CausalInferencePipeline
    linear8.linear8 / linear8.pack / linear8.quantize (linear layers in 8-bit blocks and their gradients),
    block_ops.ln_affine / ln_modulate / gelu_tanh (forward and backward, with 8-bit checkpoints)
    vae_decode.WanVAEDecoder (streaming latent -> pixel decode; channels-last HIP convolutions and norms, conv_ops)
"""
from . import lib, monarch_attn, attention, prologue, causal_model, pipeline, vae_decode, linear, block_ops, linear8, paged_attn  # noqa: F401

__all__ = ["lib", "monarch_attn", "attention", "prologue", "causal_model", "pipeline", "vae_decode", "linear", "linear8",
           "paged_attn"]

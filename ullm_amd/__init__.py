"""ullm_amd -- MI355X (gfx950) attention path for uLLM.

Hand-written HIP kernels behind the C ABI of include/ullm_hip.h:
single-query GQA decode attention (split-KV), causal prefill attention
(MFMA), and the fused Q/K-norm + RoPE + KV-cache append.  The Python layer
here only binds that ABI (ctypes) and uses torch for device memory.
"""
from ._lib import UllmHipError, lib  # noqa: F401
from .attention import (  # noqa: F401
    GpuAttention,
    attn_decode,
    attn_prefill,
    attn_tree,
    attn_tree_paged,
    decode_workspace_bytes,
    key_weights,
    key_weights_paged,
    kv_accept,
    kv_accept_paged,
    kv_evict,
    kv_evict_paged,
    kv_pages_update,
    qkv_append,
    qkv_append_tree,
    qkv_append_tree_paged,
    rope_table,
    tree_masks,
    tree_verify,
)

__version__ = "0.1.0"

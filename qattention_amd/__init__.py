"""qattention_amd -- MI355X-native ancestor-sparse tree-verify attention.

Public API mirrors the reference module src.ragged_attn (saifmb0/QAttention):
see qattention_amd.ragged_attn.  Kernels are hand-written gfx950 HIP in
csrc/, exposed through the C ABI of include/qattn.h (libqattn.so).
"""
from .paged_kv import (  # noqa: F401
    append_paged_kv,
    compact_paged_kv,
    copy_kv_pages,
    prefix_attention_paged,
)
from .quantized_kv import (  # noqa: F401
    QuantizedKV,
    append_quantized_kv,
    prefix_attention_quantized,
    quantized_kv_cache,
    read_quantized_kv,
)
from .ragged_attn import (  # noqa: F401
    ancestor_table,
    build_paged_kv,
    fused_lse_merge,
    pack_inputs,
    prompt_attention,
    ragged_attention,
    ragged_attention_hybrid,
    ragged_attention_paged,
    ragged_attention_prefix,
    ragged_attention_sibling,
    ragged_attention_sibling_with_lse,
    ragged_attention_with_lse,
    ragged_attention_with_parents,
    set_layout_copies,
)

__version__ = "0.1.0"

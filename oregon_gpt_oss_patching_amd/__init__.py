"""MI355X-native flash attention (forward + backward) for the GPT-OSS attention
variant, with the Python surface of nlp-uoregon/oregon_gpt_oss_patching.

    from oregon_gpt_oss_patching_amd import triton_flash_attention
    from oregon_gpt_oss_patching_amd.patching import patch_flash_attention
"""
from .attention_kernel import (  # noqa: F401
    attention,
    attention_backward,
    attention_forward,
    doc_start_from_position_ids,
    hip_flash_attention,
    triton_flash_attention,
)
from .page_tables import (  # noqa: F401
    TokenMap,
    page_table_update,
    token_map,
)
from .paged_cache import (  # noqa: F401
    PagedCache,
    PagedState,
    paged_attention,
    paged_attention_forward,
    paged_cache,
    paged_cache_read,
    paged_cache_write,
    paged_cache_write_tokens,
)
from .rotary_positions import (  # noqa: F401
    Rotary,
    hip_rotary_pos_emb,
    rotary,
    rotary_frequencies,
    rotary_tables,
)

__all__ = ["attention", "attention_forward", "attention_backward", "doc_start_from_position_ids",
           "hip_flash_attention", "triton_flash_attention",
           "PagedCache", "PagedState", "paged_cache", "paged_cache_write", "paged_cache_write_tokens", "paged_cache_read", "paged_attention", "paged_attention_forward",
           "TokenMap", "page_table_update", "token_map", "Rotary", "rotary", "rotary_frequencies", "rotary_tables", "hip_rotary_pos_emb"]

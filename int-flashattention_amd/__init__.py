"""MI355X-native INT8 FlashAttention forward behind the reference's Python entry points.

    attention(q, k, v, causal, sm_scale)
    attention_int8(q, k, v, q_scale, k_scale, causal, sm_scale)
    attention_full_int8(q, k, v, q_scale, k_scale, v_scale, causal, sm_scale)

    rotary(x, positions, freqs), paged_kvcache_append(...), attention_paged_int8(...): a serving step over a paged int8 cache
    paged_latent_append(...), attention_paged_latent_int8(...), attention_latent(...): the same where keys and values
        come from one latent vector a token, and its prompts
    paged_reserve(...), paged_fork(...), paged_free(...), paged_compact(...), paged_copy(...): the pages of such caches

All of them launch hand-written HIP kernels (gfx950) through the C ABI of ``libintfa.so``; nothing here
computes attention in PyTorch.
"""
from .flash_atten_fp import attention
from .flash_atten_int8 import attention_int8
from .flash_atten_full_int8 import attention_full_int8
from ._host import debug_qk_int32, block_n
from .quant import quant_pertoken, quant_pertensor, quant_perblock_channel, kvcache_append
from .rotary import rotary, rotary_frequencies
from .paged import attention_paged_int8, paged_kvcache_append
from .latent import attention_latent, attention_paged_latent_int8, paged_latent_append
from .pages import paged_compact, paged_copy, paged_fork, paged_free, paged_reserve

__all__ = ["attention", "attention_int8", "attention_full_int8", "debug_qk_int32", "block_n", "quant_pertoken", "quant_pertensor",
           "quant_perblock_channel", "kvcache_append", "rotary", "rotary_frequencies", "paged_kvcache_append", "attention_paged_int8",
           "paged_latent_append", "attention_paged_latent_int8", "attention_latent",
           "paged_reserve", "paged_fork", "paged_free", "paged_compact", "paged_copy"]

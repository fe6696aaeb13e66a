"""Attention whose keys and values come from one latent vector a token.

The cache is a pool of pages, ``cache`` int8 [pages, page_size, latent_dim + rope_dim]: a token's latent vector (128, 256 or 512 numbers) and the rotary key (32 or 64) that all heads
share, with two fp32 scales a token, ``scale`` [pages, page_size, 2].  Pages and ``block_table`` are those of the other paged cache.
"""
from . import _host


def paged_latent_append(cache, scale, c_new, k_new, block_table, seqlens_k, freqs=None, *, interleaved=False, magnitude=1.0, seqlens_new=None,
                        norm_weight=None, norm_eps=1e-6):
    """Appends new tokens, ``c_new`` [Z, N_new, latent_dim] and ``k_new`` [Z, N_new, rope_dim] (both fp16 or both bf16), to the pages of their sequences, in place.

    Sequence z holds ``seqlens_k[z]`` tokens (int32 [Z] on the device); its new rows go to the positions from there on.  With ``norm_weight`` ([latent_dim] of the same type)
    the latent vectors are normalised on the way, c * weight / sqrt(mean(c^2) + norm_eps), and with ``freqs`` the rotary keys are rotated by their positions as ``rotary``
    does; neither is rounded to 16 bits in between.  ``seqlens_new`` (int32 [Z]): new rows of each sequence where they differ.  Rows past the table's last column, or
    of a page that the table does not name, are dropped.  The lengths are not advanced here.

    Each part of a token is rounded to its own scale, its largest magnitude over 127 (at least 2^-100).  NaN becomes 0 and infinities +-127, and neither counts for the scale.
    No other token of a page is touched."""
    return (_host._native or _host.native()).paged_latent_append(cache, scale, c_new, k_new, block_table, seqlens_k, freqs, interleaved, magnitude, seqlens_new,
                                                                 norm_weight, norm_eps)


def attention_paged_latent_int8(q_latent, q_rope, cache, scale, block_table, seqlens_k, causal, sm_scale, *, freqs=None, interleaved=False,
                                magnitude=1.0, seqlens_q=None, return_lse=False):
    """Attention of new tokens over the pages of their sequences, with queries taken into the latent space (the absorbed form): ``q_latent`` [Z, H, N, latent_dim] is what
    a head's query becomes by the matrix that would expand its keys, ``q_rope`` [Z, H, N, rope_dim] its rotary part, fp16 or bf16.  Every head's key is the whole row of the cache, its
    value the latent part.  Returns [Z, H, N, latent_dim] of the same type, to be taken through the matrix that would expand the values, and with ``return_lse`` also
    m + log2(l) of each row, fp32 [Z, H, N].

    ``seqlens_k``, ``causal``, ``freqs`` (for ``q_rope``), ``seqlens_q`` and rows that see no key: as in ``attention_paged_int8``; a forward pass alone, like it.
    Scales must be finite and not negative.  A query row enters in steps of 1/32512 of its largest element, keys and values as the numbers that the cache stands for.
    """
    return (_host._native or _host.native()).attention_latent_paged(q_latent, q_rope, cache, scale, block_table, seqlens_k, causal, sm_scale, freqs, interleaved,
                                                                    magnitude, seqlens_q, return_lse)


def attention_latent(q_nope, q_rope, k_nope, k_rope, v, causal, sm_scale, *, seqlens_q=None, seqlens_k=None, return_lse=False):
    """The same attention with keys and values expanded for every head, which prompts are cheaper with: ``q_nope`` [Z, H, N, dn], ``q_rope`` [Z, H, N, dr], ``k_nope`` [Z, H, N_k, dn],
    ``k_rope`` [Z, 1, N_k, dr] (shared by the heads), ``v`` [Z, H, N_k, dv], all fp16 or all bf16; (dn, dr, dv) is (128, 64, 128) or (64, 32, 64).  Slices of projections will do:
    only the last dimension has to be contiguous (rows of keys that overlap or are 2^24 elements and more apart are copied first).  N_k is less than 2^25.  Rotary parts come rotated (``rotary``).  Returns a new contiguous [Z, H, N, dv] tensor, and with ``return_lse`` also
    m + log2(l) of each row, fp32 [Z, H, N].

    ``seqlens_q`` and ``seqlens_k`` (int32 [Z] on the device): queries and keys of each sequence where they are fewer; nothing behind a sequence's keys is read.  With ``causal`` row i
    of m queries sees the first N_k - m + i + 1 of its N_k keys.  Rows past a sequence's queries and rows that see no key are zeros with an lse of -inf.
    Like the other attention entry points a forward pass alone.
    """
    return (_host._native or _host.native()).attention_latent(q_nope, q_rope, k_nope, k_rope, v, causal, sm_scale, seqlens_q, seqlens_k, return_lse)

"""A paged int8 key/value cache: the append of new tokens to it and the attention that reads it.

The cache is a pool of pages, ``k_cache`` and ``v_cache`` int8 [pages, H_kv, page_size, d] (views of one tensor will do: only d has to be
contiguous), with one fp32 scale per page and head, ``k_scale`` and ``v_scale`` [pages, H_kv].  Row z of ``block_table`` (int32 [Z, columns])
names the pages of sequence z in order; an entry outside the pool (-1) names none.
"""
from . import _host


def paged_kvcache_append(k_cache, k_scale, v_cache, v_scale, k_new, v_new, block_table, seqlens_k, freqs=None, *, interleaved=False,
                         magnitude=1.0, seqlens_new=None):
    """Appends new keys and values (fp16 or bf16 [Z, H_kv, N_new, d]) to the pages of their sequences, in place.

    Sequence z holds ``seqlens_k[z]`` tokens (int32 [Z] on the device); its new rows go to the positions from there on.  With
    ``freqs`` the keys are rotated by these positions on the way, as ``rotary`` does, without the rounding to 16 bits in between.
    ``seqlens_new`` (int32 [Z]): new rows of each sequence where they differ.  Rows past the table's last column, or of a page that the
    table does not name, are dropped.  The lengths are not advanced here: pass ``seqlens_k + N_new`` to the next call.

    A page's scale is the largest magnitude among its new rows over 127; a page that held rows of the sequence before keeps a larger scale,
    and where the new rows need a larger one its rows are requantised to it (rint(q * old / new)).  NaN becomes 0 and infinities +-127, and neither
    counts for the scale.  A page that rows go to must stand once in the table, in one sequence of the call."""
    return (_host._native or _host.native()).paged_kvcache_append(k_cache, k_scale, v_cache, v_scale, k_new, v_new, block_table, seqlens_k,
                                                                  freqs, interleaved, magnitude, seqlens_new)


def attention_paged_int8(q, k_cache, v_cache, k_scale, v_scale, block_table, seqlens_k, causal, sm_scale, *, freqs=None,
                         interleaved=False, magnitude=1.0, seqlens_q=None, return_lse=False):
    """Attention of new tokens q (fp16 or bf16 [Z, H, N, d], H a multiple of H_kv) over the pages of their sequences; returns a new
    contiguous [Z, H, N, d] tensor of q's dtype, and with ``return_lse`` also m + log2(l) of each row, fp32 [Z, H, N].

    ``seqlens_k`` (int32 [Z] on the device): keys of each sequence, the new tokens among them.  ``seqlens_q`` (int32 [Z]): new tokens of
    each sequence where they differ; rows past them are zeros.  Row i of m new tokens stands at position seqlens_k - m + i: with
    ``causal`` it sees the keys up to there, and with ``freqs`` the query is rotated by it first.  Rows that see no key are zeros with
    an lse of -inf; tokens of a page that the table does not name are hidden.
    Like the other attention entry points a forward pass alone: the result requires no gradient and carries no tangent, whatever q does.
    Page scales must not be negative, and have to be finite: one that is not reaches the rows computed together with those that see its page.
    """
    return (_host._native or _host.native()).attention_paged(q, k_cache, v_cache, k_scale, v_scale, block_table, seqlens_k, causal, sm_scale,
                                                             freqs, interleaved, magnitude, seqlens_q, return_lse)

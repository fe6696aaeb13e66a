"""The pages of a cache: which sequences hold them, and their copies.

``refs`` (int32 [pages] on the device) counts the entries of ``block_table`` (int32 [Z, columns]) that name each page; one with a count of 0 is free, and a cache
begins with ``refs`` all zeros and a table of -1.  ``caches`` are the tensors whose first axis is pages - keys, values, scales, latent rows, of as many layers as share
the table; of each, a page has to be contiguous (``kv[:, 0]`` of a [pages, 2, ...] tensor will do).  Everything happens on the device, in place and in the order of the
current stream: nothing is read back, and captured calls follow the counts, tables and lengths as they are then.

A server's step:  ``granted = paged_reserve(...)``, the appends of all layers with ``seqlens_new=granted``, ``seqlens_k += granted``, attention; ``paged_free`` when sequences end.
"""
from . import _host


def paged_copy(caches, src, dst):
    """Copies page ``src[i]`` over page ``dst[i]`` (int32 [n]) in every cache.  Pairs with either outside the pool are left out.  A page that is copied to must not
    stand in ``dst`` twice, nor in ``src``."""
    return (_host._native or _host.native()).paged_copy(caches, src, dst)


def paged_fork(refs, block_table, seqlens_k, parents, children):
    """Sequence ``children[i]`` goes on from ``parents[i]`` (int32 [n], at most 4096): it gets the parent's pages, which both hold from then on, and its length; the
    pages that it held before are let go.  All parents are read before any child is written, so beams may be exchanged; of equal children the last one counts, and pairs
    with either outside the table's rows are left out.  Nothing is copied: ``paged_reserve`` gives a sequence a page of its own before it writes."""
    return (_host._native or _host.native()).paged_fork(refs, block_table, seqlens_k, parents, children)


def paged_free(refs, block_table, seqlens_k, sequences, page_size, keep=None):
    """Sequences (int32 [n]; those outside the table's rows are left out) end, or with ``keep`` (int32 [n]) go back to their first ``keep[i]`` tokens: entries of the table
    behind those become -1 and the counts of their pages one less."""
    return (_host._native or _host.native()).paged_free(refs, block_table, seqlens_k, sequences, page_size, keep)


def paged_reserve(caches, refs, block_table, seqlens_k, seqlens_new, page_size):
    """Makes room for ``seqlens_new`` (int32 [Z], or an int for all) tokens behind the ``seqlens_k`` of each sequence (at most 8192 of them) and returns how many it made
    room for, int32 [Z]: fewer where the pages ran out or the table ends.  Pass that on as ``seqlens_new`` of the append.  Lengths are not changed.

    Columns that the tokens reach and that name no page get a free one: free pages are dealt in their order, to sequence 0 first.  A page among them that other sequences hold too is
    replaced by a copy in every cache; of sequences that all want a copy of a page in one call, the last keeps the page itself if nobody else holds it.
    (Once the pages have run out, sequences behind that are granted nothing in a page that others were to leave.)"""
    return (_host._native or _host.native()).paged_reserve(caches, refs, block_table, seqlens_k, seqlens_new, page_size)


def paged_compact(caches, refs, block_table):
    """Moves the used pages to the first places of their pools, with as few copies as that takes: of U used ones, those from place U onward go to the free places before it,
    both in their order.  Counts and table follow.  Returns where each page is now, int32 [pages], -1 for those that were free."""
    return (_host._native or _host.native()).paged_compact(caches, refs, block_table)

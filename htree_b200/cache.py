"""Generation around a paged key/value cache: where tokens go, putting them there, reading them back, and the attention that reads them.

A cache is two tensors k_cache [pages, page_size, H_kv, K] and v_cache [pages, page_size, H_kv, V] (any strides whose rows are dense and
16-byte aligned, so that a slice of a larger buffer will do), shared by all requests.  What belongs to whom is kept on the device:

    lengths      [B] int32        tokens that request b holds
    block_table  [B, M] int32     its pages, in order; -1 behind them
    pool, top    [P], [1] int32   the free pages are pool[:top]

A turn of generation, with drafted tokens or one token at a time:

    out = draft_attention(q, k, v, k_cache, v_cache, block_table, lengths, parents)      # in every layer
    ...                                                                                   # which drafts are accepted: path, counts
    slots, taken = cache_plan(lengths, counts, block_table, pool, top, page_size, n)      # once, for all layers
    cache_append(k, v, k_cache, v_cache, slots, path)                                     # in every layer

Drafts are not part of the cache until they are accepted, so a rejected one leaves nothing behind.  cache_gather turns the pages into the
contiguous k, v of htree_forward, for the layers or the lengths where htree attention takes over.

No call synchronises or reads a tensor on the host, and all can be captured into a CUDA graph; pages, slots and lengths that lie outside
the cache are left out and reported by check_status.  None of the calls has a derivative: inputs that require a gradient, or carry a tangent,
are refused.  The reference has no counterpart."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .ops import _status, _status_words


def _calls(t: torch.Tensor):
    """The C++ side of the calls, and the status word of the device (a call of a few microseconds: nothing is looked up twice)."""
    if not t.is_cuda:
        raise RuntimeError("htree_b200 runs on CUDA tensors only; there is no CPU implementation")
    g = _lib.glue()
    if not g:
        raise RuntimeError("the cache operators need the library that the torch glue is linked to: unset HTREE_B200_LIB")
    device = t.device
    status = _status_words.get(device)
    return g, _status(device) if status is None else status


def cache_plan(lengths: torch.Tensor, counts: torch.Tensor, block_table: torch.Tensor, pool: torch.Tensor, top: torch.Tensor,
               page_size: int, n: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Pages for new tokens: block tables and slot maps from request lengths.  Returns (slots [B, n] int64, taken [B] int32).

    counts[b] > 0: request b grows by that many tokens (at most n); 0: nothing; < 0: the request ends.  Ending requests give their pages
    back first, in row order; then, in row order, requests take pages from the pool's end as long as it holds what all up to them need.
    taken[b] is counts[b] where request b was served and 0 where it was not (no pages left, or, reported by check_status, more than n
    tokens or than its table row can name); slots[b, i] is the slot (page * page_size + place) of its i-th new token, -1 elsewhere.
    An entry below 0 among the pages of a request or the free ones is reported when it is given back and when it is asked for slots, which are -1.
    lengths, block_table, pool and top are updated in place."""
    g, status = _calls(block_table)
    return g.cache_plan(lengths, counts, block_table, pool, top, page_size, n, status)


def cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
                 index: Optional[torch.Tensor] = None) -> None:
    """Rows of k [B, N, H_kv, K] and v [B, N, H_kv, V] into their slots [B, n] (-1: not written): token i of request b, or token
    index[b, i] (int32), e.g. the accepted drafts.  Slots of one call have to differ: what a slot holds that several tokens share is not
    specified, a mixture of them included.  k and v must not lie in the cache themselves."""
    g, status = _calls(k_cache)
    g.cache_append(k, v, k_cache, v_cache, slots, index, status)


def cache_gather(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                 T: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first T tokens of every request as contiguous (k [B, T, H_kv, K], v [B, T, H_kv, V]), zeros behind a request's end."""
    g, status = _calls(k_cache)
    return g.cache_gather(k_cache, v_cache, block_table, lengths, T, status)


def draft_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, parents: Optional[torch.Tensor] = None, scale: Optional[float] = None, return_lse: bool = False):
    """Softmax attention of N drafted tokens per request over its cached tokens and over the drafts that lead to them.

    q [B, N, H, K] and the drafts' own k [B, N, H_kv, K], v [B, N, H_kv, V]; N = 1 is ordinary decoding.  parents [B, N] int32: the draft
    that draft i continues (below i), -1 where it continues the cached tokens, below -1 where there is no such draft (its rows come back
    as zeros).  Without parents every draft continues the one before it: several tokens at once, or a chunk of a prompt.  A draft reads all
    cached tokens, itself, its parent, its parent's parent and so on; what other drafts hold does not reach it.
    Returns out [B, N, H, V] in q's dtype; with return_lse also the log of the sum of the exponentials, [B, N, H] fp32, by which outputs over
    other keys can be joined.  Rows that read nothing, or whose every score is -inf, are zeros with -inf.  scale is K**-0.5 unless given.  Rows
    of up to 256 elements, trees of up to 1024 drafts, chains of any length."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    g, status = _calls(k_cache)
    out, lse = g.draft_attention(q, k, v, k_cache, v_cache, block_table, lengths, parents, scale, return_lse, status)
    return (out, lse) if return_lse else out


__all__ = ["cache_plan", "cache_append", "cache_gather", "draft_attention"]

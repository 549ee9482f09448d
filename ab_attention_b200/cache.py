"""A paged key/value cache, and the attention of new tokens over it.

A stream (text, or video generated frame by frame) keeps the keys and values of its
tokens in pages; each call brings a chunk of new tokens, from one to many, of a
batch of sequences. `append_kv` stores their keys and values (turning keys and
queries by their rotary positions on the way), `chunk_attention` attends from their
queries to everything stored, under a causal or block-causal rule with an optional
sliding window and sinks.

Tokens are packed: q, k, v are [tokens, heads, 128], and sequence s owns tokens
``starts[s]:starts[s + 1]`` (``starts`` never decreases). ``lengths[s]`` counts its keys once the chunk is stored, so
token i of n sits at position ``lengths[s] - n + i``; position p lies in page
``page_table[s, p // page_size]``, row ``p % page_size``. All three are int32 on the
device and are read there, so the calls never synchronise and can be captured into CUDA
graphs and replayed with new contents.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .rotary import VIDEO_AXES, _on_gpu


class KVCache(NamedTuple):
    """Keys and values of all pages, each [pages, kv_heads, page_size, 128] (bf16 or fp16).

    ``page_size`` is 16, 32, 64 or a multiple of 128. Any strides with contiguous rows on
    16-byte boundaries will do, so a [pages, page_size, kv_heads, 128] buffer can be passed transposed.
    """

    keys: torch.Tensor
    values: torch.Tensor


def kv_cache(pages: int, kv_heads: int, *, page_size: int = 128, dtype=torch.bfloat16, device="cuda") -> KVCache:
    """A cache of zeros."""
    shape = (pages, kv_heads, page_size, 128)
    return KVCache(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))


def append_kv(cache, k, v, page_table, starts, lengths, *, positions=None, axes=VIDEO_AXES, q=None):
    """Stores the new tokens' k and v [tokens, kv_heads, 128] in their pages, in one launch.

    With ``positions`` (int32 [tokens, axes]) the keys are turned by `apply_rotary`'s rule, and
    so are ``q`` [tokens, heads, 128] when given; the turned queries are returned (else None).
    A token whose place is outside the page table or the cache is not stored and sets the
    device error word (`_lib.device_status`); tokens behind the last sequence are not
    stored. Two tokens must not share a place (sequences may share pages they only read).
    """
    _on_gpu(k)
    sections, theta, paired, shared = axes
    turned = torch.ops.ab_attention.append(cache.keys, cache.values, k, v, page_table, starts, lengths, q, positions,
                                           sections, theta, shared, not paired)
    return None if q is None else turned


def chunk_attention(q, cache, page_table, starts, lengths, *, longest=None, window=None, sinks=0, block=1,
                    return_lse=False, out=None):
    """Attention (scale 128^-0.5) of the new tokens' q [tokens, heads, 128] over the cached keys.

    The query at position p sees key j when ``j < e`` and (``j >= e - window`` or ``j < sinks``),
    ``e = (p // block + 1) * block``: causal for block 1, and for a larger block every token
    sees to the end of its own block (a video frame). window=None: no limit (sinks then
    change nothing). A row that sees nothing gives zeros. Head h reads key head
    ``h // (heads // kv_heads)``.

    ``longest``: an upper bound of the tokens of any one sequence, known on the host (default:
    all tokens). Give it: a batch of short chunks takes another kernel than one long chunk. The other
    bound that a call is planned by is the table's width (the lengths are on the device): a table much wider
    than the longest sequence gives the same results, and a few short sequences take up to 2.4 times as long. A
    sequence with more tokens is not computed: its rows are left as they are and the device error
    word is set.
    Returns out [tokens, heads, 128] (rows behind the last sequence are left as they are too; both
    kinds are undefined without ``out``), and with ``return_lse`` the base-2 log-sum-exp
    [tokens, heads] float32. Keys and values of a sequence have to be finite; rows of its last page
    behind its length are never used.
    """
    _on_gpu(q)
    if window is not None and window < 1:
        raise ValueError("window must be positive, or None")
    if longest is None:
        longest = q.shape[0]
    if out is None:
        out, lse = torch.ops.ab_attention.chunk_attention(q, cache.keys, cache.values, page_table, starts, lengths, longest,
                                                          window or 0, sinks, block, return_lse)
    else:
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
        torch.ops.ab_attention.chunk_attention_out(q, cache.keys, cache.values, page_table, starts, lengths, longest,
                                                   window or 0, sinks, block, out, lse)
    return (out, lse) if return_lse else out

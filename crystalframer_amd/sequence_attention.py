"""Attention between sequences: what reads an encoder's states from outside, and what attends along positions.

The encoder's own attention is over the atoms of one crystal (``attention.py``; reference:
models/indexed_lattice_multi_head_attention_cuda.py:737-996).  Here queries of one set of sequences read keys and values of another,
of other lengths (``cross_attention``: a crystal's atoms read by property queries, tokens or the atoms of another structure), or
sequences attend to themselves with a learned bias by relative position (``relative_attention``: the other attention of a layer that
reads such states).  Both are one launch forward (two where the keys are split) and two or three backward, for float32, bfloat16
and float16.  Also reachable as ``cuda_funcs.cross_attention``, ``cuda_funcs.relative_attention`` and ``cuda_funcs.position_buckets``.  The
checks, the library's calls and the autograd function are native (csrc/host_module.cpp).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

_native = None


def _call(query, key, value, table, buckets, query_starts, key_starts, query_sizes, key_sizes, key_mask, scale, causal, queries_last):
    global _native
    if _native is None:
        _native = _lib.load_host().sequence_attention
    if torch.autograd.forward_ad._current_level >= 0:
        raise RuntimeError("an attention has no forward-mode derivative")
    if scale is None:
        scale = 0.0                    # one over the root of the channels
    elif not scale > 0.0:
        raise ValueError(f"scale {scale} must be positive")
    return _native(query, key, value, table, buckets, query_starts, key_starts, query_sizes, key_sizes, key_mask, scale, causal, queries_last)


def cross_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, *, query_starts: Optional[torch.Tensor] = None,
                    key_starts: Optional[torch.Tensor] = None, query_sizes: Optional[torch.Tensor] = None,
                    key_sizes: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> torch.Tensor:
    """o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j of the query's own sequence.

    Packed: query (rows, heads, channels), key and value (rows, key heads, channels), the sequences of each behind one another;
    ``query_starts``, ``key_starts`` (batch + 1, int64, from 0 on, none below the one before) say where each begins and the last ends.  Rows
    behind that are 0 in the result and in all gradients.  Padded: (batch, positions, heads, channels), with ``query_sizes``,
    ``key_sizes`` (batch, int64) where not all positions are meant; the others are 0 in the result.  ``key_mask`` (key's leading dimensions, bool): keys with False are not
    there.  A query without keys gets 0.  What memory holds in the place of keys that are not there does not matter, NaN included.

    The heads may be a multiple of the key heads: head h reads key head h // (heads // key heads).  1 to 128 channels of a head;
    ``scale``: one over their root, up to 2.3e38, with a table from 2^-64 to 2^64.  One type, float32, bfloat16 or float16, for all and for
    the result; sums, maxima and the gradients' sums are in float32, probabilities and the scores' gradients are rounded to the type before
    their products.  Any strides; rows that do not begin at multiples of 16 bytes, do not fill them, or share their memory (one row expanded
    over positions) are laid out again first.  The values of starts and sizes are cut to the rows that are there.

    Float32 products are made of three bfloat16 parts, which hold 24 bits of numbers from 2^-110 to 3.38e38 in size (fewer below); what is
    beyond, infinities included, makes a NaN.  All gradients are there, with
    sums in a fixed order; a gradient of a gradient raises.  The graph keeps the inputs, the output, two numbers for each of its rows and,
    in 16 bits, what rounding took from the output."""
    return _call(query, key, value, None, None, query_starts, key_starts, query_sizes, key_sizes, key_mask, scale, False, False)


def relative_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, table: torch.Tensor, buckets: torch.Tensor, *,
                       causal: bool = False, queries_last: bool = False, query_starts: Optional[torch.Tensor] = None,
                       key_starts: Optional[torch.Tensor] = None, query_sizes: Optional[torch.Tensor] = None,
                       key_sizes: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None,
                       scale: Optional[float] = None) -> torch.Tensor:
    """``cross_attention`` with a learned bias by the bucket of the relative position,

        o_i = sum_j softmax_j(scale q_i . k_j + table[b(j - i - shift), head]) v_j.

    ``table`` (number of buckets, heads), of query's type or float32, gets a gradient.  ``buckets`` (2 reach + 1, int32): the bucket of
    each relative position from -reach to reach (``position_buckets`` makes one; positions beyond count as -reach and reach, reach up to
    1024; a number that is no row of ``table`` means no bias).  Finite entries of ``table`` beyond 65536 either way count as that; minus
    infinity takes a bucket's keys away, plus infinity and NaN make NaN of the rows that see such a key, and of no others.
    shift: 0, or with ``queries_last`` how many more keys than queries the sequence has (single tokens behind a cache, whose ``key_sizes``
    include them).  ``causal``: keys j <= i + shift only; one that no query
    of the sequence sees is not there, one that some see has to be finite for the others' sake (it is 0 times in their sums).

    The table's gradient from 16-bit tensors is as exact as the products of these are, in float32 as well."""
    if table is None or buckets is None:
        raise ValueError("table and buckets must not be None")
    return _call(query, key, value, table, buckets, query_starts, key_starts, query_sizes, key_sizes, key_mask, scale, causal, queries_last)


def position_buckets(num_buckets: int, max_distance: int, bidirectional: bool = True, device=None) -> torch.Tensor:
    """Buckets of the relative positions -max_distance ... max_distance (2 max_distance + 1, int32): near ones alone, far ones together.

    Of the n buckets of a direction the first e = n // 2 hold one distance each, and distance d >= e is in bucket
    min(n - 1, e + floor((n - e) log(d / e) / log(max_distance / e))), which is found by comparing powers in whole numbers.
    ``bidirectional``: n = num_buckets // 2, the upper half for keys behind the query; otherwise n = num_buckets, and these count as 0."""
    n = num_buckets // 2 if bidirectional else num_buckets
    e = n // 2
    if e < 1 or max_distance <= e or max_distance > _lib.ATTENTION_MAX_REACH:
        raise ValueError(f"{num_buckets} buckets up to distance {max_distance}: at least {4 if bidirectional else 2} buckets, a distance beyond "
                         f"those of one position ({e}) and up to {_lib.ATTENTION_MAX_REACH}")
    one = []
    t = 0
    for d in range(max_distance + 1):
        while d >= e and t + 1 < n - e and d ** (n - e) * e ** (t + 1) >= max_distance ** (t + 1) * e ** (n - e):
            t += 1
        one.append(d if d < e else e + t)
    ahead = [n + b for b in one[1:]] if bidirectional else [0] * max_distance
    return torch.tensor(one[:0:-1] + [one[0]] + ahead, dtype=torch.int32, device=device)

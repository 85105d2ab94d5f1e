"""Operators of the ordinary attention layers that stand between 2-simplicial ones: rotary positions, causal attention
over whole prompts, rows of a cache of keys and values, and attention of drafted tokens over it.

The kernels are the HIP library's (include/sa2.h), reached by the native host path (csrc/host/sa2_torch_layers.cpp), which
checks every argument, makes outputs and workspaces and holds the autograd formulas.  Like the rest of the package they
run on the GPU only, on the current stream of the tensors' device, without synchronising.

Rows are [batch, seq_len, heads, head_dim], or packed [rows, heads, head_dim] with ``cu_seqlens``: int32, on the GPU,
sequence s in rows cu_seqlens[s] .. cu_seqlens[s+1]-1, entries non-decreasing between 0 and the number of rows.
"""
import math

import torch

from . import _lib


def rotary_frequencies(rotary_dim, base=10000.0, *, scaling=None, factor=1.0, original_length=None, slow_turns=1.0,
                       fast_turns=32.0, device=None):
    """Radians per position of the rotary_dim / 2 pairs, float64: base ** (-2 j / rotary_dim), scaled for longer contexts
    by ``factor``:

    None      as they are
    "linear"  all divided by factor (positions squeezed)
    "base"    the base raised to base * factor ** (rotary_dim / (rotary_dim - 2)): the slowest pair is divided by
              factor, the fastest stays
    "parts"   pairs that make at most slow_turns turns over original_length positions are divided by factor, those that
              make fast_turns or more stay, between them the pair's number decides linearly ("NTK-by-parts" of the YaRN
              paper, Peng et al. 2023, with its ends of the ramp: whole pair numbers, 0 at least and rotary_dim - 1 at most)
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and at least 2, got %r" % (rotary_dim,))
    if not (base > 1 and factor > 0):
        raise ValueError("base must be above 1 and factor above 0, got %r and %r" % (base, factor))
    if scaling == "base":
        if rotary_dim == 2:
            raise ValueError('scaling="base" needs a rotary_dim above 2')
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    pairs = torch.arange(rotary_dim // 2, dtype=torch.float64)
    f = base ** (-2.0 * pairs / rotary_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        if not original_length or not 0 < slow_turns < fast_turns:
            raise ValueError('scaling="parts" needs original_length and 0 < slow_turns < fast_turns')
        # the pair, as a real number, that makes t turns over the original length; the last one may make more than slow_turns,
        # so that the ramp ends behind it
        pair = lambda t: rotary_dim * math.log(original_length / (2 * math.pi * t)) / (2 * math.log(base))
        first, last = max(0, math.floor(pair(fast_turns))), min(rotary_dim - 1, math.ceil(pair(slow_turns)))
        kept = 1 - ((pairs - first) / max(last - first, 1e-3)).clamp(0, 1)
        kept[pairs >= last] = 0
        f = f * kept + f / factor * (1 - kept)
    elif scaling not in (None, "base"):
        raise ValueError('unknown scaling %r (None, "linear", "base", "parts")' % (scaling,))
    return f.to(device)


def rotary_embedding(q, k, frequencies, positions=None, cu_seqlens=None, interleaved=False, amplitude=1.0):
    """(q', k'): the first 2 * len(frequencies) columns of every head turned by position * frequencies, the others copied;
    differentiable in q and k, to any order (the gradient is the rotation by the opposite angle).

    q, k         [batch, seq_len, heads, head_dim] or packed; k has heads of its own, or is None (then k' is None)
    frequencies  float64 vector (rotary_frequencies); the angles are formed in 64 bits, so positions may be far
    positions    int32 or int64, q's leading sizes; without them a row's place in its sequence (0 for rows outside of
                 cu_seqlens; packed rows without cu_seqlens are one sequence)
    interleaved  True: pair j is columns 2j and 2j + 1; False: columns j and j + len(frequencies)
    amplitude    factor on the turned columns"""
    return _lib.host().rotary(q, k, frequencies, positions, cu_seqlens, interleaved, amplitude)


def cache_append(k, v, k_cache, v_cache, lengths, page_table=None, rows=None, cu_seqlens=None):
    """Writes new rows of k and v behind the ``lengths`` rows that each sequence has in a cache, in place.

    k, v              [batch, seq_len, heads, head_dim], or packed with cu_seqlens
    k_cache, v_cache  [pages, page_size, heads, head_dim] with page_table, or [batch, capacity, heads, head_dim]
    lengths           int32 [batch]; new row a of a sequence goes to place lengths + a.  Not changed.
    page_table        int32 [batch, any]: place r of a sequence is row r % page_size of page page_table[r // page_size]
    rows              int32 [batch, any]: which of a sequence's seq_len rows to take, in this order (accepted nodes of a
                      draft); entries outside 0 .. seq_len-1 are left out, their places stay as they are

    Rows whose place lies beyond the capacity, or whose page is not one of the cache's, are left out.  k and v may be views
    of the cache itself: all rows are read before one is written.  Two rows of one call with the same place (a page that the
    table names twice) leave either or a mixture of both there: rows are moved in pieces."""
    _lib.host().cache_append(k, v, k_cache, v_cache, lengths, page_table, rows, cu_seqlens)


def causal_attention(q, k, v, cu_seqlens=None, scale=None, flags=_lib.FLAG_AUTO):
    """softmax(scale q k^T) v, query i of a sequence over its keys 0 .. i; differentiable in q, k and v (once: create_graph=True
    is refused).

    q        [batch, seq_len, heads, head_dim], or packed [rows, heads, head_dim] with cu_seqlens; head_dim up to 256
    k, v     as q, with heads that divide q's: query head h reads head h // (heads / key heads)
    scale    1 / sqrt(head_dim) if None
    flags    _lib.FLAG_FORCE_GENERIC runs the kernels with fp32 products whatever the type, gradients too

    Returns a tensor like q, zero in rows of no sequence.  bf16 and fp16 with a head_dim up to 128 that is a multiple of 8 and rows on
    the 16-byte grid run on the 16-bit matrix pipes (softmax weights rounded to the type, sums in fp32), everything else
    with fp32 products."""
    return _lib.host().causal(q, k, v, cu_seqlens, scale, int(flags))


def causal_attention_forward(q, k, v, cu_seqlens=None, scale=None, flags=_lib.FLAG_AUTO, keep_low=False):
    """(out, lse) without autograd: lse is log sum e^(scale q k), [batch, heads, seq_len] or packed [heads, rows], float32,
    -infinity in rows of no sequence.  flags: _lib.FLAG_FORCE_GENERIC runs the kernels with fp32 products.
    keep_low: (out, lse, out_low) with what rounding out to 16 bits left, for the backward (None for float32; not written in rows of
    no sequence)."""
    out, lse, out_low = _lib.host().causal_forward(q, k, v, cu_seqlens, scale, int(flags), bool(keep_low))
    return (out, lse, out_low) if keep_low else (out, lse)


def causal_attention_backward(q, k, v, out, lse, dout, cu_seqlens=None, scale=None, needs=(True, True, True),
                              flags=_lib.FLAG_AUTO, out_low=None):
    """(dq, dk, dv) in the inputs' type, None where ``needs`` is False.  ``out``, ``lse`` and ``out_low`` are what
    causal_attention_forward returned for the same inputs and arguments.  With out_low these are causal_attention's gradients, bit for
    bit; without it, in 16-bit types, dq and dk of short sequences are 1.5 to 2.3 times as far off as their own rounding.
    Deterministic."""
    if len(needs) != 3:
        raise ValueError("needs must have three entries (dq, dk, dv), got %d" % len(needs))
    mask = sum(1 << t for t, need in enumerate(needs) if need)
    return _lib.host().causal_backward(q, k, v, out, lse, dout, cu_seqlens, scale, mask, int(flags), out_low)


def tree_attention(q, k, v, parents, k_cache, v_cache, lengths, page_table=None, scale=None, flags=_lib.FLAG_AUTO):
    """Attention of drafted tokens over a cache: node i of a sequence attends to the ``lengths`` rows that the cache holds, to
    itself and to its ancestors in the draft.  One node is a decoding step.

    q                 [batch, nodes, heads, head_dim], 1 to 64 nodes
    k, v              [batch, nodes, key heads, head_dim]: the drafted tokens' own, not yet in the cache
    parents           int32 [batch, nodes]: the node that node i follows, smaller than i, or -1 for the last cached token; -2
                      (or any chain that does not end at -1) marks a place that is not used, whose output is zero.
                      None: a chain, each node behind the one before it
    k_cache, v_cache, lengths, page_table   as at cache_append, which brings the accepted nodes into the cache
    scale             1 / sqrt(head_dim) if None
    flags             _lib.FLAG_FORCE_GENERIC runs the kernels with fp32 products whatever the type

    No gradients.  Returns a tensor like q.  bf16 and fp16 with a head_dim up to 128 that is a multiple of 8 and rows on the 16-byte
    grid run on the 16-bit matrix pipes (softmax weights rounded to the type, sums in fp32), everything else with fp32 products."""
    return _lib.host().tree(q, k, v, parents, k_cache, v_cache, lengths, page_table, scale, int(flags))

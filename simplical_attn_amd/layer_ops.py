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
              make fast_turns or more stay, between them the pair's number decides linearly
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
        # the pair, as a real number, that makes t turns over the original length
        pair = lambda t: rotary_dim * math.log(original_length / (2 * math.pi * t)) / (2 * math.log(base))
        first, last = max(0, math.floor(pair(fast_turns))), min(rotary_dim // 2 - 1, math.ceil(pair(slow_turns)))
        kept = 1 - ((pairs - first) / max(last - first, 1e-3)).clamp(0, 1)
        f = f * kept + f / factor * (1 - kept)
    elif scaling not in (None, "base"):
        raise ValueError('unknown scaling %r (None, "linear", "base", "parts")' % (scaling,))
    return f.to(device)


def rotary_embedding(q, k, frequencies, positions=None, cu_seqlens=None, interleaved=False, amplitude=1.0):
    """(q', k'): the first 2 * len(frequencies) columns of every head turned by position * frequencies, the others copied;
    differentiable in q and k (the gradient is the rotation by the opposite angle).

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

    Rows whose place lies beyond the capacity, or whose page is not one of the cache's, are left out."""
    _lib.host().cache_append(k, v, k_cache, v_cache, lengths, page_table, rows, cu_seqlens)

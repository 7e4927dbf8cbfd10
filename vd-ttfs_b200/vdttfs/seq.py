"""Sequence operators: what a decoder next to a spiking encoder runs.

=====================  ==================================================  =========================
here                   what it computes                                    C ABI
=====================  ==================================================  =========================
quantize_rows          rows in 8 bits, a scale for each                    vdt_quantize_rows
int8_matmul            product of 8-bit rows and weights                   vdt_int8_matmul
int8_linear            the two together, for 16- or 32-bit rows            vdt_int8_linear
rope_table             cosines and sines, scaled for long contexts         vdt_rope_table
qk_norm_rope           norm of each head and rotation, queries and keys    vdt_qk_norm_rope
Cache8                 a paged cache of keys and values in 8 bits          vdt_cache8
cache_append           new keys and values into it                         vdt_cache_append
cache_load             sequences out of it, as values                      vdt_cache_load
cache_attention        attention over it, causal or not                    vdt_cache_attention
=====================  ==================================================  =========================

Inference only, like the rest of the package.  Tensors are CUDA tensors of the
current device; a call runs on ``stream`` (a raw handle) or torch's current
stream.  A ``stream`` of the caller's own is the current one for the length of
the call, with all that the call copies and allocates; the results' memory also
waits for the stream that was current.  Ordering the inputs before the call, and
keeping them until it is done, is the caller's.  Tensors that do not fit raise
ValueError, what the library refuses raises VdtError.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._lib import check, lib
lib()                       # the library itself, which the module below links
try:
    from . import _seq
except ModuleNotFoundError as e:
    raise RuntimeError("vdttfs/_seq.so is not built (make -C vd-ttfs_b200 seq)") from e

NORMS = {"none": 0, "rms": 1, "l2": 2}
SCALINGS = {"none": 0, "linear": 1, "base": 2, "parts": 3}


# -------------------------------------------------------- 8-bit product --
def quantize_rows(x, stream=None):
    """x [rows, cols] -> (codes int8 [rows, cols], scale [rows]): scale = largest
    magnitude / 127, codes = round(x / scale).  The codes' rows start on 16-byte
    boundaries, as int8_matmul wants them; weights [out, in] are quantised with
    this once, too (a scale for each output channel)."""
    return _seq.quantize_rows(x, stream)


def int8_matmul(a, a_scale, w, w_scale, bias=None, out_dtype=torch.bfloat16, out=None, stream=None):
    """a [rows, k] and w [n, k] int8, a_scale [rows], w_scale [n], bias [n] or
    None -> a_scale w_scale (a w^T) + bias [rows, n]."""
    return _seq.int8_matmul(a, a_scale, w, w_scale, bias, out_dtype, out, stream)


def int8_linear(x, w, w_scale, bias=None, out_dtype=None, out=None, stream=None):
    """x [rows, k] (float32, float16 or bfloat16), w [n, k] int8 and w_scale [n]
    from quantize_rows, bias [n] float32 or None: each row of x is rounded to 8
    bits under its own scale and multiplied.  Returns [rows, n], of x's type
    unless out_dtype or out says otherwise; out may be x, or lie over it."""
    return _seq.int8_linear(x, w, w_scale, bias, out_dtype, out, stream)


# ------------------------------------------------- head norms, rotation --
def rope_table(positions, rot, base=10000.0, scaling="none", factor=1.0, trained=0, fast=32.0, slow=1.0, device=None,
               stream=None):
    """[positions, rot] float32: cosines, then sines.  scaling: "none", "linear",
    "base" or "parts" (with the trained length, and the numbers of turns over it
    that bound the ramp), for contexts ``factor`` times as long as the trained one."""
    if scaling not in SCALINGS:
        raise ValueError(f"scaling: one of {sorted(SCALINGS)}, got {scaling!r}")
    before = torch.cuda.current_stream()
    if stream is None or stream == before.cuda_stream:
        on = before
    else:
        on = torch.cuda.ExternalStream(stream) if stream else torch.cuda.default_stream()
    with torch.cuda.stream(on):
        table = torch.empty((positions, rot), dtype=torch.float32, device=device or "cuda")
        check(lib().vdt_rope_table(positions, rot, base, SCALINGS[scaling], factor, trained, fast, slow, table.data_ptr(), on.cuda_stream),
              "vdt_rope_table")
    if on is not before and table.is_cuda:
        table.record_stream(before)
    return table


def qk_norm_rope(q, k, q_weight, k_weight, positions, table, interleaved=False, norm="rms", eps=1e-6, out=None, stream=None):
    """q [tokens, heads, dim], k [tokens, kv_heads, dim] (any strides between
    heads and tokens; k may be None): each head's norm ("rms", "l2" or "none")
    times its weight [dim] (or None), the first table.shape[1] values rotated
    by the table's row positions[token] (int32; table None: no rotation).
    Pairs are halves apart, or neighbours with ``interleaved``.  Returns (q, k),
    new tensors or the pair ``out``, which may be (q, k) themselves."""
    if norm not in NORMS:
        raise ValueError(f"norm: one of {sorted(NORMS)}, got {norm!r}")
    out_q, out_k = (None, None) if out is None else out
    return _seq.qk_norm_rope(q, k, q_weight, k_weight, positions, table, interleaved, NORMS[norm], eps, out_q, out_k, stream)


# ------------------------------------------------------------- the cache --
class Cache8(NamedTuple):
    """Keys [pages, heads, page, dim] and values [pages, heads, dim, page] in
    int8, and a float32 scale [pages, heads] for each.  Any four such tensors
    in a tuple serve."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, pages, heads, dim, page=64, device="cuda"):
        """Room for ``pages`` pages of ``page`` tokens.  Nothing needs to be zero."""
        return cls(torch.empty((pages, heads, page, dim), dtype=torch.int8, device=device),
                   torch.empty((pages, heads, dim, page), dtype=torch.int8, device=device),
                   torch.empty((pages, heads), dtype=torch.float32, device=device),
                   torch.empty((pages, heads), dtype=torch.float32, device=device))


def cache_append(cache, k, v, pages, held, starts, most, stream=None):
    """k, v [total, heads, dim]: rows starts[s]..starts[s + 1] become tokens
    held[s].. of sequence s, in the pages that row s of ``pages`` names; no
    sequence gets more than ``most`` of them.  held is not changed."""
    return _seq.cache_append(cache, k, v, pages, held, starts, most, stream)


def cache_load(cache, pages, kept, starts, total, most, dtype=torch.bfloat16, stream=None):
    """The sequences' kept[s] tokens as (k, v) [total, heads, dim], sequence s at
    rows starts[s]..starts[s + 1]; no sequence has more than ``most``.  One that has,
    or that does not fit its rows, gives NaN; rows of no token are not written."""
    return _seq.cache_load(cache, pages, kept, starts, total, most, dtype, stream)


def cache_attention(q, cache, pages, kept, starts, most, most_kept, causal=True, scale=None, out=None, stream=None):
    """q [total, heads, dim] (float16 or bfloat16), the queries of sequence s at
    rows starts[s]..starts[s + 1] (at most ``most``), over its kept[s] cached
    tokens (at most ``most_kept``).  causal: the queries are the last tokens of
    their sequence, in the cache already.  scale: 1 / sqrt(dim) unless given.
    A query that sees nothing gives zeros, a sequence beyond these bounds NaN; rows
    of no sequence are not written."""
    return _seq.cache_attention(q, cache, pages, kept, starts, most, most_kept, causal, scale, out, stream)


__all__ = ["quantize_rows", "int8_matmul", "int8_linear", "rope_table", "qk_norm_rope", "Cache8", "cache_append",
           "cache_load", "cache_attention", "NORMS", "SCALINGS"]

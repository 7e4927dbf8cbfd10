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
quantize_fp4           rows in 4-bit floating point, scales for blocks     vdt_quantize_fp4
fp4_values             the values that they stand for                      vdt_fp4_values
fp4_matmul             product of such rows and weights                    vdt_fp4_matmul
fp4_linear             the two together, for 16- or 32-bit rows            vdt_fp4_linear
add_rms_norm           the residual's addition and the norm of the sum     vdt_add_rms_norm
add_rms_norm_int8      the same in 8 bits, for int8_matmul                 vdt_add_rms_norm_int8
PagePool               the free pages of a cache                           (two buffers)
plan_pages             page tables, positions, slots from lengths          vdt_plan_pages
free_pages             finished sequences' pages back to the pool          vdt_free_pages
sample                 the next tokens from logits and random numbers      vdt_sample
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


# ------------------------------------- microscaled 4-bit floating point --
def quantize_fp4(x, stream=None):
    """x [rows, cols] -> (codes uint8 [rows, ceil(cols / 2)], scale uint8): every 32
    values of a row are rounded to 0, 1/2, 1, 3/2, 2, 3, 4, 6 or their negatives,
    ties to the even code, times the smallest power of two that no value passes
    6 of.  Two codes a byte, the even column in the low bits; the scales' bytes (the
    exponent + 127; 255: a block with an infinity or NaN) lie as the tensor cores
    read them, [rows / 128, cols / 128, 32, 16], columns in steps of 256, row r's four
    blocks at [r % 32, r % 128 // 32 * 4:].  Weights [out, in] are quantised
    with this once, too."""
    return _seq.quantize_fp4(x, stream)


def fp4_values(codes, scale, cols=None, dtype=torch.float32, stream=None):
    """The values [rows, cols] that quantize_fp4's results stand for (cols: two for
    each byte, or one less)."""
    return _seq.fp4_values(codes, scale, cols, dtype, stream)


def fp4_matmul(a, a_scale, w, w_scale, bias=None, out_dtype=torch.bfloat16, out=None, stream=None):
    """a [rows, k] and w [n, k], codes and scales from quantize_fp4, bias [n] float32
    or None -> a w^T + bias [rows, n], summed in 32 bits."""
    return _seq.fp4_matmul(a, a_scale, w, w_scale, bias, out_dtype, out, stream)


def fp4_linear(x, w, w_scale, bias=None, out_dtype=None, out=None, stream=None):
    """x [rows, k] (float32, float16 or bfloat16), w and w_scale from quantize_fp4,
    bias [n] float32 or None: x is rounded in blocks of 32 and multiplied.  Returns
    [rows, n], of x's type unless out_dtype or out says otherwise; out may be x,
    or lie over it."""
    return _seq.fp4_linear(x, w, w_scale, bias, out_dtype, out, stream)


# ------------------------------------------ residual's addition and norm --
def add_rms_norm(x, residual=None, weight=None, eps=1e-6, out=None, sum_out=None, stream=None):
    """x, residual [rows, cols] of one type (residual may be None) -> (y, t): t = x +
    residual, y = t / sqrt(mean(t^2) + eps) * weight (of the same type, or None).
    Without a residual t is x itself.  sum_out may be the residual or x, out x or the
    residual; they may not lie over each other."""
    return _seq.add_rms_norm(x, residual, weight, eps, out, sum_out, stream)


def add_rms_norm_int8(x, residual=None, weight=None, eps=1e-6, sum_out=None, stream=None):
    """The same with y in 8 bits, as int8_matmul takes it: (codes, scale, t).  The
    codes are those of t * weight, the norm is in the scale."""
    return _seq.add_rms_norm_int8(x, residual, weight, eps, sum_out, stream)


# ----------------------------------------------------------- page tables --
class PagePool(NamedTuple):
    """The free pages of a cache: ``ring`` int32 [pages] and ``span`` int32 [2], the
    first free one's place in it and their number; they go on round its end.  Any
    two such tensors in a tuple serve."""
    ring: torch.Tensor
    span: torch.Tensor

    @classmethod
    def full(cls, pages, device="cuda"):
        """All of ``pages`` pages free."""
        return cls(torch.arange(pages, dtype=torch.int32, device=device), torch.tensor([0, pages], dtype=torch.int32, device=device))


class PagePlan(NamedTuple):
    """What plan_pages gives: tokens in the cache after the step and first packed
    row of each sequence, position and slot of each row, the pool's span after."""
    kept: torch.Tensor
    starts: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    span: torch.Tensor


def plan_pages(pool, pages, held, new, page, total, out=None, stream=None):
    """A step's tokens, from the tokens held [seqs] and new [seqs] (int32): pages that
    the sequences begin are taken from the pool, sequence after sequence, and
    written into ``pages`` [seqs, width]; returns a PagePlan for ``total`` packed
    rows.  kept, starts and pages are what cache_append (with held) and cache_attention
    take, positions what qk_norm_rope takes; slots are page number * page + place.
    Rows past the last sequence's get -1, and so do slots of tokens without a page:
    those past the table's width, and those for which the pool has none (then
    span[1] is below zero, by as many pages; later steps do not ask for these again, so
    such a sequence is freed and begun anew).  ``out``: a PagePlan to write
    to, any of it None; its kept may be held, its span the pool's.  Nothing is
    copied to the host."""
    return PagePlan._make(_seq.plan_pages(pool, pages, held, new, page, total, stream, *(out or (None,) * 5)))


def free_pages(pool, pages, held, done, page, out=None, stream=None):
    """The pages of the sequences with done [seqs] (bool) go behind the pool's last:
    returns (held, span), 0 tokens held for these.  A page that stands in
    two rows goes back with each of them.  ``out``: the two to write
    to, which may be held and the pool's span."""
    return _seq.free_pages(pool, pages, held, done, page, stream, *(out or (None, None)))


# -------------------------------------------------------------- sampling --
def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, stream=None):
    """logits [rows, vocab] (float32, float16 or bfloat16) and a random number
    u [rows] (float32, in [0, 1)) for each row -> (tokens int32 [rows], logp float32
    [rows]).  Weights exp((x - max) / temperature); of the tokens by (value descending,
    index ascending) the first top_k are kept (<= 0: all), of these those before which
    less than top_p of their sum lies, of these those of at least min_p times the
    largest; the token is the first index at which the kept weights' sum passes
    u times the whole.  temperature 0: the lowest index of the largest.  Each parameter a
    number, or a tensor [rows] (float32; top_k int32).  logp: the logarithm of the
    probability that the token was drawn with.  A row that gives no token (a NaN in
    it, -inf alone, a parameter or u out of range) has -1 and NaN."""
    return _seq.sample(logits, u, temperature, top_k, top_p, min_p, stream)


__all__ = ["quantize_rows", "int8_matmul", "int8_linear", "rope_table", "qk_norm_rope", "Cache8", "cache_append",
           "cache_load", "cache_attention", "quantize_fp4", "fp4_values", "fp4_matmul", "fp4_linear", "add_rms_norm",
           "add_rms_norm_int8", "PagePool", "PagePlan", "plan_pages", "free_pages", "sample", "NORMS", "SCALINGS"]

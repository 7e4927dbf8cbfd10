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
stream.  With a ``stream`` of the caller's own, what the call allocates is
tied to that stream; ordering the inputs is the caller's.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple

import torch

from ._lib import Cache8Desc, check, lib

F32, F16, BF16 = 0, 1, 2
ROPE_HALF, ROPE_PAIRS = 0, 1
NORMS = {"none": 0, "rms": 1, "l2": 2}
SCALINGS = {"none": 0, "linear": 1, "base": 2, "parts": 3}
_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def _type(t, what):
    k = _TYPES.get(t.dtype if isinstance(t, torch.Tensor) else t)
    if k is None:
        raise ValueError(f"{what}: float32, float16 or bfloat16 is wanted, got {t.dtype if isinstance(t, torch.Tensor) else t}")
    return k


def _cuda(t, what, dtype=None, dims=None):
    if not t.is_cuda:
        raise ValueError(f"{what}: a CUDA tensor is wanted")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{what}: {dtype} is wanted, got {t.dtype}")
    if dims is not None and t.dim() != dims:
        raise ValueError(f"{what}: {dims} dimensions are wanted, got {tuple(t.shape)}")


def _flat(t, what, dtype, n):
    _cuda(t, what, dtype)
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what}: {n} contiguous values are wanted, got {tuple(t.shape)}")


def _run(stream, made):
    """The stream's handle; what this call allocated is tied to it."""
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    s = torch.cuda.ExternalStream(int(stream)) if int(stream) else torch.cuda.default_stream()
    for t in made:
        if t is not None:
            t.record_stream(s)
    return int(stream)


# -------------------------------------------------------- 8-bit product --
def _rows16(n, k, device):
    """[n, k] codes whose rows start 16 bytes apart or a multiple."""
    t = torch.empty((n, -(-k // 16) * 16), dtype=torch.int8, device=device)
    return t[:, :k]


def quantize_rows(x, stream=None):
    """x [rows, cols] -> (codes int8 [rows, cols], scale [rows]): scale = largest
    magnitude / 127, codes = round(x / scale).  The codes' rows start on 16-byte
    boundaries, as int8_matmul wants them; weights [out, in] are quantised with
    this once, too (a scale for each output channel)."""
    _cuda(x, "x", dims=2)
    kind = _type(x, "x")
    if x.shape[1] == 0:
        raise ValueError("x: no columns")
    if x.stride(1) != 1:
        x = x.contiguous()
    codes = _rows16(x.shape[0], x.shape[1], x.device)
    scale = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    s = _run(stream, (codes, scale, x))
    check(lib().vdt_quantize_rows(x.data_ptr(), kind, x.shape[0], x.shape[1], x.stride(0), codes.data_ptr(),
                                  codes.stride(0), scale.data_ptr(), s), "vdt_quantize_rows")
    return codes, scale


def _code_rows(t, what):
    _cuda(t, what, torch.int8, 2)
    if t.shape[1] == 0 or t.stride(1) != 1 or t.stride(0) % 16 or t.stride(0) < t.shape[1] or t.data_ptr() % 16:
        raise ValueError(f"{what}: rows that start on 16-byte boundaries are wanted (see quantize_rows), "
                         f"got shape {tuple(t.shape)}, strides {t.stride()}")
    if t.shape[0]:
        ends = t.storage_offset() + (t.shape[0] - 1) * t.stride(0) + -(-t.shape[1] // 16) * 16
        if ends > t.untyped_storage().nbytes():
            raise ValueError(f"{what}: the last row's storage must reach to the next multiple of 16 bytes")


def _product_out(x, w, w_scale, bias, out, out_dtype, rows):
    _code_rows(w, "w")
    n = w.shape[0]
    if n == 0 or x.shape[1] != w.shape[1]:
        raise ValueError(f"{tuple(x.shape)} and {tuple(w.shape)} do not multiply")
    _flat(w_scale, "w_scale", torch.float32, n)
    if bias is not None:
        _flat(bias, "bias", torch.float32, n)
    if out is None:
        return torch.empty((rows, n), dtype=out_dtype, device=x.device)
    _cuda(out, "out", dims=2)
    if tuple(out.shape) != (rows, n) or out.stride(1) != 1 or (rows > 1 and out.stride(0) < n):
        raise ValueError(f"out: [{rows}, {n}] with consecutive columns is wanted, got {tuple(out.shape)}, {out.stride()}")
    return out


def int8_matmul(a, a_scale, w, w_scale, bias=None, out_dtype=torch.bfloat16, out=None, stream=None):
    """a [rows, k] and w [n, k] int8, a_scale [rows], w_scale [n], bias [n] or
    None -> a_scale w_scale (a w^T) + bias [rows, n]."""
    _code_rows(a, "a")
    _flat(a_scale, "a_scale", torch.float32, a.shape[0])
    mine = out is None
    out = _product_out(a, w, w_scale, bias, out, out_dtype, a.shape[0])
    kind = _type(out, "out")
    s = _run(stream, (out,) if mine else ())
    check(lib().vdt_int8_matmul(a.data_ptr(), a.stride(0), a_scale.data_ptr(), w.data_ptr(), w.stride(0),
                                w_scale.data_ptr(), 0 if bias is None else bias.data_ptr(), a.shape[0], w.shape[0],
                                a.shape[1], kind, out.data_ptr(), max(out.stride(0), w.shape[0]), s), "vdt_int8_matmul")
    return out


def int8_linear(x, w, w_scale, bias=None, out_dtype=None, out=None, stream=None):
    """x [rows, k] (any of the three types), w [n, k] int8 and w_scale [n] from
    quantize_rows, bias [n] float32 or None: each row of x is rounded to 8 bits
    under its own scale and multiplied.  Returns [rows, n], of x's type unless
    out_dtype or out says otherwise."""
    _cuda(x, "x", dims=2)
    kind = _type(x, "x")
    rows, k = x.shape
    mine = out is None
    out = _product_out(x, w, w_scale, bias, out, out_dtype or x.dtype, rows)
    out_kind = _type(out, "out")
    if k and x.stride(1) != 1:
        x = x.contiguous()
    L = lib()
    need = L.vdt_int8_linear_scratch_bytes(rows, k)
    scratch = torch.empty(need, dtype=torch.uint8, device=x.device)
    s = _run(stream, (scratch, x, out if mine else None))
    check(L.vdt_int8_linear(x.data_ptr(), kind, x.stride(0), w.data_ptr(), w.stride(0), w_scale.data_ptr(),
                            0 if bias is None else bias.data_ptr(), rows, w.shape[0], k, out_kind, out.data_ptr(),
                            max(out.stride(0), w.shape[0]), scratch.data_ptr(), need, s), "vdt_int8_linear")
    return out


# ------------------------------------------------- head norms, rotation --
def rope_table(positions, rot, base=10000.0, scaling="none", factor=1.0, trained=0, fast=32.0, slow=1.0, device=None,
               stream=None):
    """[positions, rot] float32: cosines, then sines.  scaling: "none", "linear",
    "base" or "parts" (with the trained length, and the numbers of turns over it
    that bound the ramp), for contexts ``factor`` times as long as the trained one."""
    if scaling not in SCALINGS:
        raise ValueError(f"scaling: one of {sorted(SCALINGS)}, got {scaling!r}")
    table = torch.empty((positions, rot), dtype=torch.float32, device=device or "cuda")
    s = _run(stream, (table,))
    check(lib().vdt_rope_table(positions, rot, base, SCALINGS[scaling], factor, trained, fast, slow, table.data_ptr(), s),
          "vdt_rope_table")
    return table


def _heads(t, what, dim=None):
    _cuda(t, what, dims=3)
    if dim is not None and t.shape[2] != dim:
        raise ValueError(f"{what}: heads of {dim} are wanted, got {tuple(t.shape)}")
    if t.shape[2] != 1 and t.stride(2) != 1:
        raise ValueError(f"{what}: a head's values must be consecutive")


def qk_norm_rope(q, k, q_weight, k_weight, positions, table, interleaved=False, norm="rms", eps=1e-6, out=None, stream=None):
    """q [tokens, heads, dim], k [tokens, kv_heads, dim] (any strides between
    heads and tokens; k may be None): each head's norm ("rms", "l2" or "none")
    times its weight [dim] (or None), the first table.shape[1] values rotated
    by the table's row positions[token] (int32; table None: no rotation).
    Pairs are halves apart, or neighbours with ``interleaved``.  Returns (q, k),
    new tensors or the pair ``out``, which may be (q, k) themselves."""
    _heads(q, "q")
    tokens, heads, dim = q.shape
    kind = _type(q, "q")
    if k is not None:
        _heads(k, "k", dim)
        if k.shape[0] != tokens or k.dtype != q.dtype:
            raise ValueError(f"k: {tokens} tokens of {q.dtype} are wanted, got {tuple(k.shape)}, {k.dtype}")
    if norm not in NORMS:
        raise ValueError(f"norm: one of {sorted(NORMS)}, got {norm!r}")
    for w, what in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            _flat(w, what, q.dtype, dim)
    rot = n = 0
    if table is not None:
        _cuda(table, "table", torch.float32, 2)
        if not table.is_contiguous():
            raise ValueError("table: a contiguous one is wanted")
        n, rot = table.shape
        _flat(positions, "positions", torch.int32, tokens)
    made = ()
    if out is None:
        made = out = (torch.empty((tokens, heads, dim), dtype=q.dtype, device=q.device),
                      None if k is None else torch.empty((tokens, k.shape[1], dim), dtype=q.dtype, device=q.device))
    else:
        for o, i, what in zip(out, (q, k), ("q", "k")):
            if i is not None:
                _heads(o, f"out ({what})", dim)
                if o.shape != i.shape or o.dtype != q.dtype:
                    raise ValueError(f"out ({what}): {tuple(i.shape)} of {q.dtype} is wanted")
    s = _run(stream, made)
    ko, kv = out[1], k
    check(lib().vdt_qk_norm_rope(
        q.data_ptr(), q.stride(0), q.stride(1), 0 if kv is None else kv.data_ptr(), 0 if kv is None else kv.stride(0),
        0 if kv is None else kv.stride(1), 0 if q_weight is None else q_weight.data_ptr(),
        0 if k_weight is None else k_weight.data_ptr(), positions.data_ptr() if rot else 0, table.data_ptr() if rot else 0,
        n, rot, ROPE_PAIRS if interleaved else ROPE_HALF, NORMS[norm], eps, tokens, heads, 0 if kv is None else kv.shape[1],
        dim, kind, out[0].data_ptr(), out[0].stride(0), out[0].stride(1), 0 if kv is None else ko.data_ptr(),
        0 if kv is None else ko.stride(0), 0 if kv is None else ko.stride(1), s), "vdt_qk_norm_rope")
    return out


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


def _cache(cache):
    k, v, ks, vs = cache
    _cuda(k, "cache keys", torch.int8, 4)
    pages, heads, page, dim = k.shape
    if not k.is_contiguous():
        raise ValueError("cache keys: contiguous ones are wanted")
    _flat(v, "cache values", torch.int8, k.numel())
    if tuple(v.shape) != (pages, heads, dim, page):
        raise ValueError(f"cache values: {(pages, heads, dim, page)} is wanted, got {tuple(v.shape)}")
    _flat(ks, "cache key scales", torch.float32, pages * heads)
    _flat(vs, "cache value scales", torch.float32, pages * heads)
    return Cache8Desc(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, page, heads, dim)


def _table(pages, held, starts, what):
    _cuda(pages, "pages", torch.int32, 2)
    if not pages.is_contiguous():
        raise ValueError("pages: a contiguous table is wanted")
    n = pages.shape[0]
    _flat(held, what, torch.int32, n)
    _flat(starts, "starts", torch.int32, n + 1)
    return n, pages.shape[1]


def cache_append(cache, k, v, pages, held, starts, most, stream=None):
    """k, v [total, heads, dim]: rows starts[s]..starts[s + 1] become tokens
    held[s].. of sequence s, in the pages that row s of ``pages`` names; no
    sequence gets more than ``most`` of them.  held is not changed."""
    desc = _cache(cache)
    seqs, width = _table(pages, held, starts, "held")
    kind = _type(k, "k")
    for t, what in ((k, "k"), (v, "v")):
        _heads(t, what, desc.dim)
        if t.shape[:2] != (k.shape[0], desc.heads) or t.dtype != k.dtype:
            raise ValueError(f"{what}: [{k.shape[0]}, {desc.heads}, {desc.dim}] of {k.dtype} is wanted, got {tuple(t.shape)}, {t.dtype}")
    s = _run(stream, ())
    check(lib().vdt_cache_append(C.byref(desc), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                                 kind, pages.data_ptr(), width, held.data_ptr(), starts.data_ptr(), seqs, k.shape[0],
                                 min(most, k.shape[0]), s), "vdt_cache_append")


def cache_load(cache, pages, kept, starts, total, most, dtype=torch.bfloat16, stream=None):
    """The sequences' kept[s] tokens as (k, v) [total, heads, dim], sequence s at
    rows starts[s]..starts[s + 1]; no sequence has more than ``most``."""
    desc = _cache(cache)
    seqs, width = _table(pages, kept, starts, "kept")
    kind = _type(dtype, "dtype")
    k, v = (torch.empty((total, desc.heads, desc.dim), dtype=dtype, device=cache[0].device) for _ in range(2))
    s = _run(stream, (k, v))
    check(lib().vdt_cache_load(C.byref(desc), pages.data_ptr(), width, kept.data_ptr(), starts.data_ptr(), seqs, total,
                               min(most, total), kind, k.data_ptr(), v.data_ptr(), s), "vdt_cache_load")
    return k, v


def cache_attention(q, cache, pages, kept, starts, most, most_kept, causal=True, scale=None, out=None, stream=None):
    """q [total, heads, dim] (float16 or bfloat16), the queries of sequence s at
    rows starts[s]..starts[s + 1] (at most ``most``), over its kept[s] cached
    tokens (at most ``most_kept``).  causal: the queries are the last tokens of
    their sequence, in the cache already.  scale: 1 / sqrt(dim) unless given.
    A query that sees nothing gives zeros."""
    desc = _cache(cache)
    seqs, width = _table(pages, kept, starts, "kept")
    _heads(q, "q", desc.dim)
    total, heads, dim = q.shape
    kind = _type(q, "q")
    made = ()
    if out is None:
        out = torch.empty((total, heads, dim), dtype=q.dtype, device=q.device)
        made = (out,)
    else:
        _heads(out, "out", dim)
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError(f"out: {tuple(q.shape)} of {q.dtype} is wanted")
    L = lib()
    most = min(most, total)
    need = L.vdt_cache_attention_scratch_bytes(total, heads, desc.heads, dim, seqs, most, most_kept)
    scratch = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    s = _run(stream, made + (scratch,))
    check(L.vdt_cache_attention(C.byref(desc), q.data_ptr(), q.stride(0), q.stride(1), heads, kind, pages.data_ptr(), width,
                                kept.data_ptr(), starts.data_ptr(), seqs, total, most, most_kept, int(causal),
                                1.0 / math.sqrt(dim) if scale is None else scale, out.data_ptr(), out.stride(0), out.stride(1),
                                scratch.data_ptr() if need else 0, need, s), "vdt_cache_attention")
    return out


__all__ = ["quantize_rows", "int8_matmul", "int8_linear", "rope_table", "qk_norm_rope", "Cache8", "cache_append",
           "cache_load", "cache_attention", "NORMS", "SCALINGS"]

"""The sequence operators' measured cases, their plain forms in torch and their 64-bit definitions.

Four operators that a decoder next to the spiking networks runs, step after step:

* ``linear``  a product in 8-bit integers: each token's row is rounded to 8 bits under a scale of its own, multiplied with
  8-bit weights that have a scale for each output channel, and given a bias;
* ``rope``    the norm of every head of the queries and keys, and the position rotation of the first ``rot`` dimensions;
* ``append``  new keys and values into a paged cache held in 8 bits (a scale for each page and head), and the sequences read
  back as values, as a program does that moves them out of the cache;
* ``attend``  attention of packed queries over that cache, causal (the queries are a sequence's last tokens) or not (the
  cache holds an encoder's states).

``own`` false: elementary torch operations in 32 bits, rounded once at the end.  ``own`` true: vdttfs.seq.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_STEP = torch.tensor(1.0 / 127.0, dtype=torch.float32).item()   # scale = amax * _STEP, in 32 bits


def _seq():
    at = os.path.join(os.getcwd(), "vd-ttfs_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from vdttfs import seq
    return seq


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # one token's projection in a small decoder: nothing but latency
        dict(name="linear one token", op="linear", tokens=1, inner=1024, outer=1024, type="bf16", bias=True),
        # a decode step of a few dozen sequences through a 4096-wide layer: the weights' bytes
        dict(name="linear decode step", op="linear", tokens=24, inner=4096, outer=4096, type="f16", bias=False),
        # odd sizes everywhere, 32-bit activations as the spiking layers give them
        dict(name="linear odd sizes", op="linear", tokens=777, inner=1001, outer=1531, type="f32", bias=True),
        # a long prompt's up-projection: the tensor cores' rate
        dict(name="linear prompt", op="linear", tokens=8192, inner=4096, outer=8192, type="bf16", bias=False),
        # one token of a small decoder
        dict(name="rope one token", op="rope", tokens=1, heads=8, kv_heads=2, dim=64, rot=64, inter=False, type="bf16"),
        # prompts together, rotation on half of each head, neighbouring pairs
        dict(name="rope prompts", op="rope", tokens=16381, heads=32, kv_heads=8, dim=128, rot=64, inter=True, type="bf16"),
        # a decode step: one token to each sequence, most of them into a page that others are in already
        dict(name="append decode step", op="append", seqs=48, held=300, new=1, kv_heads=4, dim=64, page=16, type="f16"),
        # prompts of several lengths into fresh and begun pages
        dict(name="append prompts", op="append", seqs=6, held=100, new=4093, kv_heads=8, dim=128, page=64, type="bf16"),
        # the first tokens of one short sequence: nothing but latency
        dict(name="attend one short", op="attend", seqs=1, held=97, new=1, heads=8, kv_heads=2, dim=64, page=16, causal=True, type="bf16"),
        # a decode step of many sequences with long and short caches: the cache's bytes
        dict(name="attend decode step", op="attend", seqs=64, held=8191, new=1, heads=32, kv_heads=8, dim=128, page=64, causal=True, type="bf16"),
        # prompts behind a cached prefix: the tensor cores' rate
        dict(name="attend prompts", op="attend", seqs=3, held=4096, new=2049, heads=32, kv_heads=8, dim=128, page=32, causal=True, type="bf16"),
        # a decoder's queries over an encoder's states of other lengths, some of them empty
        dict(name="attend encoder", op="attend", seqs=16, held=1500, new=33, heads=16, kv_heads=16, dim=64, page=16, causal=False, type="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "rope", "append", "attend"])
    kind = rng.choice(["bf16", "f16"])
    if op == "linear":
        c = dict(op=op, tokens=_log(rng, 1, 8192), inner=_log(rng, 64, 8192), outer=_log(rng, 64, 8192),
                 type=rng.choice(["bf16", "f16", "f32"]), bias=rng.random() < 0.5)
        most = 8192 * 4096 * 8192
        c["tokens"] = max(1, min(c["tokens"], most // (c["inner"] * c["outer"])))
        return c
    dim = rng.choice([32, 64, 96, 128, 256])
    group = rng.choice([1, 2, 4, 7, 8])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    if op == "rope":
        rot = rng.choice([dim, dim, dim // 2])
        return dict(op=op, tokens=min(_log(rng, 1, 16384), 16381 * 40 * 128 // ((group + 1) * kv_heads * dim)), heads=group * kv_heads,
                    kv_heads=kv_heads, dim=dim, rot=rot, inter=rng.random() < 0.5, type=rng.choice(["bf16", "f16", "f32"]))
    page = rng.choice([16, 32, 64])
    if op == "append":
        c = dict(op=op, seqs=_log(rng, 1, 64), held=_log(rng, 1, 1000), new=_log(rng, 1, 4096), kv_heads=kv_heads, dim=dim, page=page, type=kind)
        most = 6 * (100 + 4093) * 8 * 128
        c["new"] = max(1, min(c["new"], most // (c["seqs"] * kv_heads * dim) - c["held"]))
        return c
    new = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
    c = dict(op=op, seqs=_log(rng, 1, 64), held=_log(rng, 1, 8192), new=new, heads=group * kv_heads, kv_heads=kv_heads, dim=dim, page=page,
             causal=rng.random() < 0.7, type=kind)
    # at most the decode step's cache and the prompts' products
    c["seqs"] = max(1, min(c["seqs"], 64 * 8192 * 8 * 128 // ((c["held"] + new) * kv_heads * dim),
                           3 * 2049 * 4096 * 32 * 128 // (new * (c["held"] + new) * c["heads"] * dim)))
    return c


def _spread(n, most, least):
    """n lengths between least and most, the first of them `most`, in no order."""
    return [most - (i * 7919 % n) * (most - least) // n for i in range(n)]


def _lengths(c):
    """(tokens held before the call, new tokens) of each sequence."""
    n = c["seqs"]
    new = [c["new"]] * n if c["new"] == 1 else _spread(n, c["new"], max(1, c["new"] // 4))
    if c["op"] == "attend" and not c["causal"]:
        return _spread(n, c["held"], 0), new            # an encoder's states; none for a sequence or so
    return _spread(n, c["held"], c["held"] // 8), new


def _cached(c):
    """Tokens in the cache at the time of attention, for each sequence."""
    held, new = _lengths(c)
    return [h + n for h, n in zip(held, new)] if c["op"] == "append" or c["causal"] else held


def work(c):
    e = _SIZE[c["type"]]
    if c["op"] == "linear":
        m, k, n = c["tokens"], c["inner"], c["outer"]
        return {"bytes": m * k * e + n * k + 4 * n + (4 * n if c["bias"] else 0) + m * n * e, "flops": 2 * m * k * n}
    if c["op"] == "rope":
        values = c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"]
        return {"bytes": 2 * values * e + c["tokens"] * (4 * c["rot"] + 4) + 2 * c["dim"] * e, "flops": 8 * values}
    row = c["kv_heads"] * c["dim"]
    held, new = _lengths(c)
    if c["op"] == "append":
        # new rows read, their codes written; every sequence's codes read, its values written
        return {"bytes": 2 * row * (sum(new) * (e + 1) + sum(_cached(c)) * (1 + e)), "flops": 2 * row * (4 * sum(new) + sum(_cached(c)))}
    pairs = sum(n * k - (n * (n - 1) // 2 if c["causal"] else 0) for n, k in zip(new, _cached(c)))
    return {"bytes": 2 * row * sum(_cached(c)) + 8 * c["kv_heads"] * sum(-(-k // c["page"]) for k in _cached(c)) + 2 * sum(new) * c["heads"] * c["dim"] * e,
            "flops": 4 * pairs * c["heads"] * c["dim"]}


# ------------------------------------------------------------------ inputs --
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = _TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    s = dict(case)
    if case["op"] == "linear":
        m, k, n = case["tokens"], case["inner"], case["outer"]
        x = normal(m, k)
        x[:, :: max(1, k // 7)] *= 8                       # a few outlying channels, as activations have
        # weights quantised once: rows of codes 16 bytes apart
        codes = torch.zeros(n, -(-k // 16) * 16, dtype=torch.int8, device="cuda")[:, :k]
        codes.copy_((normal(n, k) * 36).round().clamp(-127, 127))
        s.update(x=x.to(kind), codes=codes, scale=(torch.rand(n, generator=g, device="cuda") + 0.5) / (36 * math.sqrt(k)),
                 offset=normal(n) * 0.1 if case["bias"] else None)
        return s
    if case["op"] == "rope":
        t, h, hk, d, r = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "rot"))
        qkv = (normal(t, (h + 2 * hk) * d) * 2).to(kind)   # the fused projection's output
        most = 32768
        angle = torch.arange(most, dtype=torch.float64)[:, None] * 500000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
        table = torch.cat([angle.cos(), angle.sin()], 1).to(torch.float32).cuda()
        s.update(q=qkv[:, : h * d].view(t, h, d), k=qkv[:, h * d: (h + hk) * d].view(t, hk, d), table=table,
                 wq=(1 + 0.2 * normal(d)).to(kind), wk=(1 + 0.2 * normal(d)).to(kind),
                 at=torch.randint(0, most, (t,), generator=g, device="cuda", dtype=torch.int32))
        return s
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    held, new = _lengths(case)
    kept = _cached(case)
    width = max(1, max(-(-n // page) for n in kept))
    used = [-(-n // page) for n in kept]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[: sum(used)]   # pages are handed out in no order
    table = torch.zeros(case["seqs"], width, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None, :] < ints(used)[:, None]] = order
    codes = lambda *shape: (normal(*shape) * 32).round_().clamp_(-127, 127).to(torch.int8)  # noqa: E731
    scales = lambda: (torch.rand(pages, hk, generator=g, device="cuda") + 0.5) / 32  # noqa: E731
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s.update(cache=(codes(pages, hk, page, d), codes(pages, hk, d, page), scales(), scales()), pages=table,
             starts=ints(starts), total=starts[-1], most_new=max(new))
    if case["op"] == "append":
        kv = normal(starts[-1], 2 * hk * d).to(kind)
        ends = [0]
        for n in kept:
            ends.append(ends[-1] + n)
        s.update(k=kv[:, : hk * d].view(-1, hk, d), v=kv[:, hk * d:].view(-1, hk, d), held=ints(held), kept=ints(kept), ends=ints(ends),
                 total_kept=ends[-1], most_kept=max(kept))
        return s
    s.update(q=normal(starts[-1], case["heads"], d).to(kind), kept=ints(kept), most_kept=max(kept))
    return s


# ------------------------------------------------------------------ passes --
def run(s):
    if own:
        return _OWN[s["op"]](s)
    return _PLAIN[s["op"]](s)


def _own_linear(s):
    return _seq().int8_linear(s["x"], s["codes"], s["scale"], s["offset"])


def _own_rope(s):
    return _seq().qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["at"], s["table"], interleaved=s["inter"], eps=1e-6)


def _own_append(s):
    seq = _seq()
    seq.cache_append(s["cache"], s["k"], s["v"], s["pages"], s["held"], s["starts"], s["most_new"])
    k, v = seq.cache_load(s["cache"], s["pages"], s["kept"], s["ends"], s["total_kept"], s["most_kept"], _TYPES[s["type"]])
    return k, v, s["cache"][2], s["cache"][3]


def _own_attend(s):
    return _seq().cache_attention(s["q"], s["cache"], s["pages"], s["kept"], s["starts"], s["most_new"], s["most_kept"], causal=s["causal"])


def _quantize(x, scale):
    return (x / torch.where(scale > 0, scale, 1.0)).round().clamp(-127, 127)


def _plain_linear(s):
    x = s["x"].float()
    scale = x.abs().amax(1, keepdim=True) * _STEP
    y = _quantize(x, scale) @ s["codes"].float().T * scale * s["scale"]
    if s["offset"] is not None:
        y = y + s["offset"]
    return y.to(s["x"].dtype)


def _plain_rope(s):
    half = s["rot"] // 2
    rows = s["table"][s["at"].long()][:, None]
    cos, sin = rows[..., :half], rows[..., half:]

    def one(x, weight):
        x = x.float()
        y = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * weight.float()
        turned, rest = y[..., : s["rot"]], y[..., s["rot"]:]
        if s["inter"]:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = turned[..., :half], turned[..., half:]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([turned, rest], -1).to(s["q"].dtype)

    return one(s["q"], s["wq"]), one(s["k"], s["wk"])


def _owner(starts, total):
    """Each packed row's sequence, and its place in it."""
    row = torch.arange(total, device="cuda", dtype=torch.int32)
    of = torch.searchsorted(starts, row, right=True) - 1
    return of, row - starts[of]


def _plain_append(s):
    page = s["page"]
    of, at = _owner(s["starts"], s["total"])
    at = (s["held"][of] + at).long()
    slot, place = s["pages"][of, at // page].long(), at % page
    first = s["pages"].gather(1, (s["held"] // page).clamp(max=s["pages"].shape[1] - 1).long()[:, None])[:, 0].long()
    begun = (s["held"] % page > 0)[:, None]               # the page that the new tokens go on with
    for x, codes, scale in ((s["k"].float(), s["cache"][0], s["cache"][2]), (s["v"].float(), s["cache"][1].transpose(2, 3), s["cache"][3])):
        largest = torch.zeros_like(scale).index_reduce_(0, slot, x.abs().amax(2), "amax")
        was = scale[first]
        fresh = largest * _STEP
        touched = torch.zeros_like(scale, dtype=torch.bool).index_fill_(0, slot, True)
        now = torch.where(touched, fresh, scale)
        now[first] = torch.where(begun, torch.maximum(was, fresh[first]), now[first])
        ratio = torch.where(begun & (now[first] > 0), was / now[first], 1.0)
        codes[first] = (codes[first].float() * ratio[:, :, None, None]).round().to(torch.int8)
        scale.copy_(now)
        codes[slot, :, place] = _quantize(x, now[slot][..., None]).to(torch.int8)
    of, at = _owner(s["ends"], s["total_kept"])
    slot, place = s["pages"][of, at // page].long(), (at % page).long()
    k, v = (codes[slot, :, place].float() * scale[slot][..., None]
            for codes, scale in ((s["cache"][0], s["cache"][2]), (s["cache"][1].transpose(2, 3), s["cache"][3])))
    return k.to(_TYPES[s["type"]]), v.to(_TYPES[s["type"]]), s["cache"][2], s["cache"][3]


def _plain_attend(s):
    heads, kv_heads, d, page = s["heads"], s["kv_heads"], s["dim"], s["page"]
    kc, vc, ks, vs = s["cache"]
    slot = s["pages"].long()
    b, width = slot.shape
    keys = (kc[slot].float() * ks[slot][..., None, None]).transpose(1, 2).reshape(b, kv_heads, width * page, d)
    values = (vc[slot].float() * vs[slot][..., None, None]).permute(0, 2, 1, 4, 3).reshape(b, kv_heads, width * page, d)
    of, at = _owner(s["starts"], s["total"])
    q = torch.zeros(b, s["most_new"], heads, d, device="cuda")
    q[of, at.long()] = s["q"].float()
    q = q.transpose(1, 2).reshape(b, kv_heads, -1, d)      # the heads that share keys are rows of one product
    scores = (q @ keys.transpose(2, 3)).view(b, heads, s["most_new"], width * page) / math.sqrt(d)
    token = torch.arange(width * page, device="cuda")[None, None, :]
    last = s["kept"][:, None, None] - 1
    if s["causal"]:
        last = last - (s["starts"].diff()[:, None] - 1 - torch.arange(s["most_new"], device="cuda"))[:, :, None]
    seen = (token <= last)[:, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(top > -math.inf, top, 0.0)).exp()
    total = p.sum(-1, keepdim=True)
    out = (p.view(b, kv_heads, -1, width * page) @ values).view(b, heads, s["most_new"], d) / torch.where(total > 0, total, 1.0)
    return out.transpose(1, 2)[of, at.long()].to(s["q"].dtype)


_OWN = {"linear": _own_linear, "rope": _own_rope, "append": _own_append, "attend": _own_attend}
_PLAIN = {"linear": _plain_linear, "rope": _plain_rope, "append": _plain_append, "attend": _plain_attend}


# ------------------------------------------------- definitions in 64 bits --
def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "rope": _exact_rope, "append": _exact_append, "attend": _exact_attend}[case["op"]](s)


def _scale64(largest):
    """The scale as it is defined, a 32-bit number: the row's largest magnitude times 1/127."""
    return (largest.float() * _STEP).double()


def _codes64(x, scale):
    return torch.where(scale > 0, torch.clamp(torch.round(x / scale), -127, 127), 0.0)


def _exact_linear(s):
    x = s["x"].double()
    scale = _scale64(x.abs().max(1).values)[:, None]
    y = torch.einsum("mk,nk->mn", _codes64(x, scale), s["codes"].double()) * scale * s["scale"].double()[None]
    return y if s["offset"] is None else y + s["offset"].double()[None]


def _exact_rope(s):
    r = s["rot"]
    table = s["table"].double()[s["at"].long()]
    turn = torch.complex(table[:, : r // 2], table[:, r // 2:])[:, None]
    out = []
    for x, weight in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        y = x.double()
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + 1e-6) * weight.double()
        pairs = y[..., :r].unflatten(-1, (-1, 2)) if s["inter"] else y[..., :r].unflatten(-1, (2, -1)).transpose(-1, -2)
        pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        y[..., :r] = (pairs if s["inter"] else pairs.transpose(-1, -2)).flatten(-2)
        out.append(y)
    return tuple(out)


def _exact_append(s):
    page = s["page"]
    held, starts, kept, pages = (s[k].tolist() for k in ("held", "starts", "kept", "pages"))
    out = []
    for x, codes, scale in ((s["k"], s["cache"][0], s["cache"][2]), (s["v"], s["cache"][1].transpose(2, 3), s["cache"][3])):
        x, codes, scale, rows = x.double(), codes.double(), scale.double(), []
        for b, n in enumerate(kept):
            for j in range(-(-n // page)):
                at, lo, hi = pages[b][j], j * page, min(n, (j + 1) * page)
                old = max(0, min(page, held[b] - lo))              # tokens of the page that were there before
                if hi > held[b]:
                    first = starts[b] + max(lo, held[b]) - held[b]
                    new = x[first: starts[b] + hi - held[b]].transpose(0, 1)
                    to = _scale64(new.abs().amax((1, 2)))
                    if old:
                        to = torch.maximum(to, scale[at])
                        ratio = torch.where(to > 0, (scale[at] / to).float().double(), 1.0)
                        codes[at] = torch.round(codes[at] * ratio[:, None, None])
                    scale[at] = to
                    codes[at, :, old: hi - lo] = _codes64(new, to[:, None, None])
                rows.append((codes[at, :, : hi - lo] * scale[at][:, None, None]).transpose(0, 1))
        out.append((torch.cat(rows), scale))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_attend(s):
    page, group = s["page"], s["heads"] // s["kv_heads"]
    starts, kept = s["starts"].tolist(), s["kept"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(kept):
        if not n:
            continue
        at = s["pages"][b, : -(-n // page)].long()
        keys, values = (torch.cat(list((codes[at].double() * scale[at].double()[..., None, None]).unbind(0)), 1)[:, :n]
                        for codes, scale in ((s["cache"][0], s["cache"][2]), (s["cache"][1].transpose(2, 3), s["cache"][3])))
        q = s["q"][starts[b]: starts[b + 1]].double()
        sees = torch.full((q.shape[0],), n, device="cuda")
        if s["causal"]:
            sees = n - torch.arange(q.shape[0] - 1, -1, -1, device="cuda")
        hidden = torch.arange(n, device="cuda")[None] >= sees[:, None]
        for h in range(s["heads"]):
            scores = (q[:, h] @ keys[h // group].T / math.sqrt(s["dim"])).masked_fill(hidden, -math.inf)
            out[starts[b]: starts[b + 1], h] = torch.nan_to_num(torch.softmax(scores, -1)) @ values[h // group]
    return out

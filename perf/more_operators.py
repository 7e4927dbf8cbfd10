"""The step operators' measured cases, their plain forms in torch and their 64-bit definitions.

What a decoder's step runs around its products in 8 bits and its cached attention:

* ``fp4``     a product in microscaled 4-bit floating point: every 32 values of a token's row are rounded to 4 bits under a
  power of two of their own, multiplied with weights held that way, and given a bias;
* ``norm``    the residual's addition, the root-mean-square norm of the sum, and its result in 8 bits with a scale for each
  row (what the 8-bit product takes) or as values;
* ``plan``    page tables, first rows, positions and cache slots from the sequences' lengths, pages taken from a ring of free
  ones, and the pages of finished sequences put back;
* ``sample``  the next tokens from logits and given random numbers, with temperature, top-k, top-p and min-p, and the
  logarithms of the probabilities that they were drawn with.

``own`` false: elementary torch operations in 32 bits, rounded once at the end; the tokens' weights and their sums in 64
bits, since a token is chosen by comparing sums.  ``own`` true: vdttfs.seq.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_STEP = torch.tensor(1.0 / 127.0, dtype=torch.float32).item()   # scale = largest * _STEP, in 32 bits
_FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)                 # the magnitudes of codes 0 to 7; code + 8: negative
_EPS = 1e-6


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
        dict(name="fp4 one token", op="fp4", tokens=1, inner=1024, outer=1024, type="bf16", bias=True),
        # a decode step of a few dozen sequences through a wide layer: the weights' bytes
        dict(name="fp4 decode step", op="fp4", tokens=24, inner=4096, outer=8192, type="f16", bias=False),
        # odd sizes everywhere, 32-bit activations as the spiking layers give them
        dict(name="fp4 odd sizes", op="fp4", tokens=777, inner=1001, outer=1531, type="f32", bias=True),
        # a long prompt's up-projection: the tensor cores' rate
        dict(name="fp4 prompt", op="fp4", tokens=8192, inner=4096, outer=8192, type="bf16", bias=False),
        # one token between two layers of a small decoder
        dict(name="norm one token", op="norm", rows=1, cols=1024, type="bf16", residual=True, codes=True),
        # prompts together, into an 8-bit product
        dict(name="norm prompts", op="norm", rows=16381, cols=4096, type="bf16", residual=True, codes=True),
        # the last norm before the logits, odd sizes, values and no codes
        dict(name="norm odd sizes", op="norm", rows=777, cols=1001, type="f32", residual=False, codes=False),
        # a decode step: one token to each sequence, now and then a new page
        dict(name="plan decode step", op="plan", seqs=48, held=300, new=1, page=16),
        # prompts of several lengths into fresh and begun pages
        dict(name="plan prompts", op="plan", seqs=200, held=1000, new=4093, page=64),
        # one sequence's next token: nothing but latency
        dict(name="sample one", op="sample", rows=1, vocab=32768, type="bf16", kind="both"),
        # a decode step, every request with parameters of its own
        dict(name="sample step", op="sample", rows=64, vocab=131072, type="bf16", kind="mixed"),
        # many sequences, 32-bit logits, the nucleus alone: every token's weight counts
        dict(name="sample nucleus", op="sample", rows=250, vocab=100003, type="f32", kind="top_p"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["fp4", "norm", "plan", "sample"])
    kind = rng.choice(["bf16", "f16", "f32"])
    if op == "fp4":
        c = dict(op=op, tokens=_log(rng, 1, 8192), inner=_log(rng, 64, 8192), outer=_log(rng, 64, 8192), type=kind, bias=rng.random() < 0.5)
        c["tokens"] = max(1, min(c["tokens"], 8192 * 4096 * 8192 // (c["inner"] * c["outer"])))
        return c
    if op == "norm":
        c = dict(op=op, rows=_log(rng, 1, 16384), cols=_log(rng, 64, 16384), type=kind, residual=rng.random() < 0.7, codes=rng.random() < 0.7)
        c["rows"] = max(1, min(c["rows"], 16381 * 4096 * 2 // (c["cols"] * _SIZE[kind])))
        return c
    if op == "plan":
        c = dict(op=op, seqs=_log(rng, 1, 1000), held=_log(rng, 1, 8192), new=1 if rng.random() < 0.5 else _log(rng, 2, 4096),
                 page=rng.choice([16, 32, 64]))
        c["new"] = max(1, min(c["new"], 200 * 4093 // c["seqs"]))
        c["held"] = max(1, min(c["held"], 2000 * 1000 // c["seqs"]))
        return c
    c = dict(op=op, rows=_log(rng, 1, 250), vocab=_log(rng, 96, 131072), type=kind, kind=rng.choice(["mixed", "top_k", "top_p", "both", "min_p", "none"]))
    c["rows"] = max(1, min(c["rows"], 250 * 100003 // c["vocab"]))
    return c


def _spread(n, most, least):
    """n lengths between least and most, the first of them `most`, in no order."""
    return [most - (i * 7919 % n) * (most - least) // n for i in range(n)]


def _lengths(c):
    """(tokens held before the call, new tokens) of each sequence."""
    n = c["seqs"]
    return _spread(n, c["held"], 0), [1] * n if c["new"] == 1 else _spread(n, c["new"], max(1, c["new"] // 4))


def work(c):
    if c["op"] == "fp4":
        m, k, n, e = c["tokens"], c["inner"], c["outer"], _SIZE[c["type"]]
        return {"bytes": m * k * e + n * (k + 1) // 2 + n * -(-k // 32) + (4 * n if c["bias"] else 0) + m * n * e, "flops": 2 * m * k * n}
    if c["op"] == "norm":
        m, n, e = c["rows"], c["cols"], _SIZE[c["type"]]
        return {"bytes": m * n * (e * (3 if c["residual"] else 1) + (1 if c["codes"] else e)) + (4 * m if c["codes"] else 0) + n * e, "flops": 6 * m * n}
    if c["op"] == "plan":
        held, new = _lengths(c)
        pages = sum(-(-(h + n) // c["page"]) - -(-h // c["page"]) for h, n in zip(held, new))
        # lengths in and out, a position and a slot for each token, pages from the ring into the table
        return {"bytes": 16 * c["seqs"] + 12 * sum(new) + 8 * pages, "flops": 4 * sum(new)}
    return {"bytes": c["rows"] * (c["vocab"] * _SIZE[c["type"]] + 24), "flops": 4 * c["rows"] * c["vocab"]}


# ------------------------------------------------------------------ inputs --
def _block_exponent(largest):
    """The smallest whole number e, not below -127, with largest <= 6 * 2^e."""
    part, power = torch.frexp(largest)                     # largest = part * 2^power, part in [0.5, 1)
    e = torch.where(part > 0.75, power - 2, power - 3)
    return torch.where(largest > 0, e.clamp(min=-127), -127)


def _fp4_codes(y):
    """The nearest of the sixteen values, ties to the even code."""
    a = y.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    for i, (border, even) in enumerate([(0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)]):
        code += (a >= border) if even else (a > border)    # on the border: up where the code above is even
    return code + 8 * (y < 0).to(torch.uint8)


def _in_blocks(x):
    """Rows filled up with zeros to whole blocks: [rows, blocks, 32]."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).unflatten(1, (-1, 32))


def _scale_tiles(bytes_):
    """[rows, blocks] scale bytes as the tensor cores read them: [rows / 128, columns / 128, 32, 16], whole steps of 256
    columns, row r at [r % 32, r % 128 // 32 * 4 + block % 4]."""
    rows, blocks = bytes_.shape
    full = torch.zeros(-(-rows // 128) * 128, -(-blocks // 8) * 8, dtype=torch.uint8, device=bytes_.device)
    full[:rows, :blocks] = bytes_
    return full.view(-1, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(full.shape[0] // 128, -1, 32, 16)


def _scale_rows(tiles, rows, blocks):
    """The same read back: [rows, blocks]."""
    t, s = tiles.shape[:2]
    return tiles.view(t, s, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(t * 128, s * 4)[:rows, :blocks]


def _pack(w):
    """w [rows, columns] -> (codes [rows, columns / 2], rows 16 bytes apart, and their scales)."""
    b = _in_blocks(w)
    e = _block_exponent(b.abs().amax(2))
    codes = _fp4_codes(b * torch.exp2(-e.float())[..., None]).flatten(1)
    packed = torch.nn.functional.pad(codes[:, 0::2] | codes[:, 1::2] << 4, (0, -(b.shape[1] * 16) % 16)).contiguous()
    return packed[:, : -(-w.shape[1] // 2)], _scale_tiles((e + 127).to(torch.uint8))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    s = dict(case)
    if case["op"] == "fp4":
        kind, m, k, n = _TYPES[case["type"]], case["tokens"], case["inner"], case["outer"]
        x = normal(m, k)
        x[:, :: max(1, k // 7)] *= 8                       # a few outlying channels, as activations have
        codes, scale = _pack(normal(n, k) / math.sqrt(k))  # weights rounded once
        s.update(x=x.to(kind), codes=codes, scale=scale, offset=normal(n) * 0.1 if case["bias"] else None)
        return s
    if case["op"] == "norm":
        kind, m, n = _TYPES[case["type"]], case["rows"], case["cols"]
        x = normal(m, n)
        x[:, :: max(1, n // 5)] *= 12
        s.update(x=x.to(kind), stream=(normal(m, n) * 3).to(kind) if case["residual"] else None, weight=(1 + 0.2 * normal(n)).to(kind))
        return s
    if case["op"] == "plan":
        held, new = _lengths(case)
        page, seqs = case["page"], case["seqs"]
        used = [-(-h // page) for h in held]
        want = [-(-(h + n) // page) for h, n in zip(held, new)]
        pages = sum(want) + 7
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((seqs, max(want) + 1), -1, dtype=torch.int32, device="cuda")
        table[torch.arange(table.shape[1], device="cuda")[None, :] < ints(used)[:, None]] = order[: sum(used)]
        # the ring of free pages begins somewhere in its middle
        first, left = pages // 3, pages - sum(used)
        ring = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        ring[(first + torch.arange(left, device="cuda")) % pages] = order[sum(used):]
        s.update(pages=table, held=ints(held), new=ints(new), ring=ring, span=ints([first, left]), total=sum(new) + 5,
                 done=torch.rand(seqs, generator=g, device="cuda") < 0.03)
        return s
    kind, m, n = _TYPES[case["type"]], case["rows"], case["vocab"]
    # most of the vocabulary far below a few likely tokens, some rows flatter than others
    logits = normal(m, n) * (1.5 + torch.rand(m, 1, generator=g, device="cuda"))
    logits.scatter_add_(1, torch.randint(0, n, (m, 12), generator=g, device="cuda"), 4 + 6 * torch.rand(m, 12, generator=g, device="cuda"))
    some = lambda *values: torch.tensor(values, device="cuda")[torch.randint(0, len(values), (m,), generator=g, device="cuda")]  # noqa: E731
    s.update(logits=logits.to(kind), u=torch.rand(m, generator=g, device="cuda"), temperature=0.8, top_k=0, top_p=1.0, min_p=0.0)
    if case["kind"] == "mixed":
        s.update(temperature=some(0.0, 0.6, 0.8, 1.0, 1.3), top_k=some(0, 0, 20, 50, 1000).to(torch.int32), top_p=some(0.8, 0.95, 1.0),
                 min_p=some(0.0, 0.0, 0.02))
    elif case["kind"] in ("top_k", "both"):
        s.update(top_k=50, top_p=0.9 if case["kind"] == "both" else 1.0)
    elif case["kind"] == "top_p":
        s.update(top_p=0.92)
    elif case["kind"] == "min_p":
        s.update(min_p=0.05, temperature=1.2)
    return s


# ------------------------------------------------------------------ passes --
def run(s):
    if own:
        return _OWN[s["op"]](s)
    return _PLAIN[s["op"]](s)


def _own_fp4(s):
    return _seq().fp4_linear(s["x"], s["codes"], s["scale"], s["offset"])


def _own_norm(s):
    if not s["codes"]:
        y, stream = _seq().add_rms_norm(s["x"], s["stream"], s["weight"], eps=_EPS)
        return (y, stream) if s["residual"] else y
    codes, scale, stream = _seq().add_rms_norm_int8(s["x"], s["stream"], s["weight"], eps=_EPS)
    values = codes * scale[:, None]
    return (values, stream) if s["residual"] else values


def _own_plan(s):
    seq = _seq()
    plan = seq.plan_pages((s["ring"], s["span"]), s["pages"], s["held"], s["new"], s["page"], s["total"])
    held, span = seq.free_pages((s["ring"], plan.span), s["pages"], plan.kept, s["done"], s["page"])
    return plan.kept, plan.starts, plan.positions, plan.slots, plan.span, s["pages"], held, span, s["ring"]


def _own_sample(s):
    return _seq().sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])


def _plain_fp4(s):
    x = s["x"].float()
    b = _in_blocks(x)
    e = _block_exponent(b.abs().amax(2))
    value = torch.tensor(_FP4 + tuple(-v for v in _FP4), device="cuda")
    # 2^e in two steps: its reciprocal or itself may lie below the normal numbers
    half = (e // 2).float()
    up, down = torch.exp2(half)[..., None], torch.exp2(e - half)[..., None]
    a = (value[_fp4_codes(b / up / down).int()] * up * down).flatten(1)
    codes = torch.stack([s["codes"] & 15, s["codes"] >> 4], 2).flatten(1)
    w = value[torch.nn.functional.pad(codes, (0, a.shape[1] - codes.shape[1])).int()].unflatten(1, (-1, 32))
    w = (w * torch.exp2(_scale_rows(s["scale"], *w.shape[:2]).float() - 127)[..., None]).flatten(1)
    y = a @ w.T
    if s["offset"] is not None:
        y = y + s["offset"]
    return y.to(s["x"].dtype)


def _plain_norm(s):
    t = s["x"] if s["stream"] is None else (s["x"].float() + s["stream"].float()).to(s["x"].dtype)
    x = t.float()
    r = (x.square().mean(1, keepdim=True) + _EPS).rsqrt()
    z = x * s["weight"].float()
    if s["codes"]:
        scale = z.abs().amax(1, keepdim=True) * _STEP
        y = (z / torch.where(scale > 0, scale, 1.0)).round().clamp(-127, 127) * (scale * r)
    else:
        y = (z * r).to(s["x"].dtype)
    return (y, t) if s["residual"] else y


def _plain_plan(s):
    page, pages, ring, (first, left) = s["page"], s["pages"], s["ring"], (s["span"][0], s["span"][1])
    seqs, width = pages.shape
    size = ring.shape[0]
    held, new = s["held"].long(), s["new"].long()
    kept = held + new
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    # the pages that each sequence needs, in order, from the ring's beginning
    had, needs = (held + page - 1) // page, (kept + page - 1) // page
    before = (needs - had).cumsum(0) - (needs - had)
    column = torch.arange(width, device="cuda")[None]
    wanted = (column >= had[:, None]) & (column < needs[:, None])
    number = before[:, None] + column - had[:, None]
    taken = torch.where(number < left, ring[(first + number) % size], -1)
    pages.copy_(torch.where(wanted, taken, pages))
    took = (needs - had).sum()
    span = torch.stack([(first + torch.minimum(took, left)) % size, left - took]).int()
    row = torch.arange(s["total"], device="cuda")
    of = (torch.searchsorted(starts, row, right=True) - 1).clamp(max=seqs - 1)
    at = held[of] + row - starts[of]
    inside = row < starts[-1]
    place = pages[of, (at // page).clamp(max=width - 1)].long()
    positions = torch.where(inside, at, -1).int()
    slots = torch.where(inside & (place >= 0), place * page + at % page, -1)
    # the pages of those that are done, to the ring's end
    back = (s["done"][:, None] & (column < needs[:, None]) & (pages >= 0)).flatten().nonzero()[:, 0]
    ring[(span[0] + span[1] + torch.arange(back.shape[0], device="cuda")) % size] = pages.flatten()[back]
    last = torch.stack([span[0], span[1] + back.shape[0]]).int()
    return kept.int(), starts.int(), positions, slots, span, pages, torch.where(s["done"], 0, kept).int(), last, ring


def _column(value, rows, kind):
    return (value if torch.is_tensor(value) else torch.full((rows,), value, device="cuda")).to(torch.float32 if kind == torch.float64 else kind).to(kind)[:, None]


def _plain_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    t, p, least = (_column(s[k], rows, torch.float64) for k in ("temperature", "top_p", "min_p"))
    k = _column(s["top_k"], rows, torch.int64)
    ordered, index = torch.sort(x, dim=1, descending=True, stable=True)
    w = ((ordered - ordered[:, :1]) / torch.where(t > 0, t, 1.0)).exp()
    w = torch.where((k <= 0) | (torch.arange(vocab, device="cuda") < k), w, 0.0)
    sums = w.cumsum(1)
    w = torch.where((p >= 1) | (sums - w < p * sums[:, -1:]), w, 0.0)
    w = torch.where(w >= least.clamp(max=1.0), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, index, w)
    sums = w.cumsum(1)
    token = (sums <= s["u"].double()[:, None] * sums[:, -1:]).sum(1)
    share = w.gather(1, token.clamp(max=vocab - 1)[:, None])[:, 0] / sums[:, -1]
    return torch.where(t[:, 0] > 0, token, index[:, 0]).int(), torch.where(t[:, 0] > 0, share.log(), 0.0).float()


_OWN = {"fp4": _own_fp4, "norm": _own_norm, "plan": _own_plan, "sample": _own_sample}
_PLAIN = {"fp4": _plain_fp4, "norm": _plain_norm, "plan": _plain_plan, "sample": _plain_sample}


# ------------------------------------------------- definitions in 64 bits --
def exact(case, seed):
    s = prepare(case, seed)
    return {"fp4": _exact_fp4, "norm": _exact_norm, "plan": _exact_plan, "sample": _exact_sample}[case["op"]](s)


def _exact_fp4(s):
    x = s["x"].double()
    rows, cols = x.shape
    grid = torch.tensor(sorted(set(_FP4) | {-v for v in _FP4}), dtype=torch.float64, device="cuda")
    even = torch.tensor([_FP4.index(abs(v)) % 2 == 0 for v in grid.tolist()], device="cuda")
    a = torch.empty_like(x)
    for at in range(0, cols, 32):
        block = x[:, at: at + 32]
        largest = block.abs().max(1).values
        e = torch.ceil(torch.log2(torch.clamp(largest, min=2.0 ** -200) / 6)) - 1       # from below, up to the border
        for _ in range(2):
            e = torch.where(largest > 6 * 2.0 ** e, e + 1, e)
        unit = (2.0 ** e.clamp(min=-127))[:, None]
        y = block / unit
        low = (torch.searchsorted(grid, y.contiguous(), right=True) - 1).clamp(0, len(grid) - 1)
        high = (low + 1).clamp(max=len(grid) - 1)
        down, up = y - grid[low], grid[high] - y
        a[:, at: at + 32] = torch.where((down < up) | ((down == up) & even[low]), grid[low], grid[high]) * unit
    y = torch.zeros(rows, s["codes"].shape[0], dtype=torch.float64, device="cuda")
    value = torch.tensor(_FP4, dtype=torch.float64, device="cuda")
    n = torch.arange(s["codes"].shape[0], device="cuda")
    step = 4096
    for lo in range(0, cols, step):
        k = torch.arange(lo, min(cols, lo + step), device="cuda")
        code = (s["codes"][:, k // 2] >> (k % 2 * 4).to(torch.uint8)) & 15
        power = s["scale"][n[:, None] // 128, k // 128, n[:, None] % 32, n[:, None] % 128 // 32 * 4 + k // 32 % 4].double() - 127
        y += a[:, k] @ (value[(code & 7).long()] * torch.where(code >= 8, -1.0, 1.0).double() * 2.0 ** power).T
    return y if s["offset"] is None else y + s["offset"].double()[None]


def _exact_norm(s):
    t = s["x"].double()
    if s["residual"]:
        t = (t + s["stream"].double()).to(s["x"].dtype).double()       # the sum is held in its own type
    y = t * s["weight"].double()[None]
    root = torch.sqrt((t * t).sum(1, keepdim=True) / t.shape[1] + _EPS)
    if s["codes"]:
        unit = (y.abs().max(1, keepdim=True).values.float() * _STEP).double()
        # a 32-bit product, as the codes are defined
        y = torch.clamp(torch.round((y.float().double() / unit.clamp(min=1e-300)).float()), -127, 127).double() * unit
    return (y / root, t) if s["residual"] else y / root


def _exact_plan(s):
    page, size = s["page"], len(s["ring"])
    ring, table, held, new = s["ring"].tolist(), s["pages"].cpu().numpy().copy(), s["held"].tolist(), s["new"].tolist()
    done, (first, left) = s["done"].tolist(), s["span"].tolist()
    positions, slots = (np.full(s["total"], -1, t) for t in (np.int32, np.int64))
    starts, kept, took = [0], [], 0
    for i, (h, n) in enumerate(zip(held, new)):
        for j in range(-(-h // page), -(-(h + n) // page)):
            table[i, j] = ring[(first + took) % size]
            took += 1
        at = np.arange(h, h + n)
        positions[starts[-1]: starts[-1] + n] = at
        slots[starts[-1]: starts[-1] + n] = table[i, at // page].astype(np.int64) * page + at % page
        starts.append(starts[-1] + n)
        kept.append(h + n)
    span = [(first + took) % size, left - took]
    back = [int(p) for i in range(len(kept)) if done[i] for p in table[i, : -(-kept[i] // page)]]
    for i, p in enumerate(back):
        ring[(sum(span) + i) % size] = p
    whole = lambda v: torch.as_tensor(np.asarray(v), device="cuda")  # noqa: E731
    out = (kept, starts, positions, slots, span, table, [0 if d else n for d, n in zip(done, kept)], [span[0], span[1] + len(back)], ring)
    return tuple(whole(v) if i == 3 else whole(v).int() for i, v in enumerate(out))


def _exact_sample(s):
    x = s["logits"].double().cpu().numpy()
    u = s["u"].double().cpu().numpy()
    rows, vocab = x.shape
    each = {k: np.broadcast_to(np.float32(s[k]) if not torch.is_tensor(s[k]) else s[k].cpu().numpy(), (rows,)) for k in
            ("temperature", "top_k", "top_p", "min_p")}
    out, logs = [], []
    for r in range(rows):
        t, k, p, least = (float(each[n][r]) for n in ("temperature", "top_k", "top_p", "min_p"))
        order = np.argsort(-x[r], kind="stable")
        if t == 0:
            out.append(order[0])
            logs.append(0.0)
            continue
        if k > 0:
            order = order[: int(k)]
        w = np.exp((x[r][order].astype(np.longdouble) - x[r][order[0]]) / t)
        if p < 1:
            sums = np.cumsum(w)
            keep = max(1, int(np.searchsorted(sums, p * sums[-1], side="left")) + 1)     # the first sum at or above the share, too
            order, w = order[:keep], w[:keep]
        order, w = order[w >= min(least, 1.0)], w[w >= min(least, 1.0)]
        by_index = np.argsort(order)
        sums = np.cumsum(w[by_index])
        at = np.searchsorted(sums, u[r] * sums[-1], side="right")
        out.append(order[by_index][at])
        logs.append(float(np.log(w[by_index][at] / sums[-1])))
    return torch.tensor(np.array(out), dtype=torch.int32, device="cuda"), torch.tensor(logs, dtype=torch.float64, device="cuda")

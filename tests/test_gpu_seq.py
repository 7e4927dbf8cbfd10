"""The sequence operators against plain implementations in 64 bits.

Tolerances (u: half a unit in the last place of the output's type, 2^-24, 2^-11
or 2^-8): what is whole (codes, pages) is equal; a product's sum is exact, so
its output is off by the epilogue's three 32-bit operations and u; a norm and
rotation by the 32-bit sum of squares (at most dim / 32 + 5 additions deep) and
some ten operations; attention by the softmax weights' rounding to 16 bits
(2^-11, and 2^-25 for the smallest), the error of the scores, and u.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
STEP = np.float32(1.0) / np.float32(127.0)
KINDS = [torch.float32, torch.float16, torch.bfloat16]
INF = math.inf


@pytest.fixture(scope="module")
def S(dev):
    from vdttfs import seq
    return seq


def normal(seed, *shape, kind=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(kind)


def codes_of(x, scale):
    """The definition in IEEE 32-bit operations (on the CPU)."""
    q = torch.round(x / torch.where(scale > 0, scale, torch.ones(())))
    return torch.nan_to_num(q).clamp(-127, 127)


def quantized(x):
    x = x.float()
    scale = x.abs().amax(1) * torch.tensor(STEP)
    return codes_of(x, scale[:, None]), scale


# ---------------------------------------------------------- 8-bit product --
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 16), (2, 1000), (17, 4099), (1, 20000)])
def test_quantized_rows_are_the_definitions(S, kind, rows, cols):
    x = normal(rows * cols, rows, cols, kind=kind) * 3
    x[0, :] = 0 if rows > 1 else x[0, :]
    codes, scale = S.quantize_rows(x.cuda())
    want, want_scale = quantized(x)
    assert torch.equal(scale.cpu(), want_scale)
    assert torch.equal(codes.cpu().float(), want)


def test_quantized_rows_of_any_stride_and_alignment(S):
    x = normal(1, 9, 70, kind=torch.float16)
    for view in (x[:, 1:], x[1::2, 3:50], x.T, x[:, ::2]):
        codes, scale = S.quantize_rows(view.cuda() if view.is_contiguous() else x.cuda().as_strided(view.shape, view.stride(), view.storage_offset()))
        want, want_scale = quantized(view)
        assert torch.equal(scale.cpu(), want_scale) and torch.equal(codes.cpu().float(), want)


def test_rows_with_values_that_are_not_finite(S):
    x = normal(2, 4, 40)
    x[1, 3], x[2, 5], x[3, 0] = INF, math.nan, 1e-45
    codes, scale = S.quantize_rows(x.cuda())
    s = scale.cpu()
    assert math.isinf(s[1]) and math.isnan(s[2])
    assert torch.equal(codes[0].cpu().float(), quantized(x[:1])[0][0])
    w, ws = S.quantize_rows(normal(3, 11, 40).cuda())
    y = S.int8_linear(x.cuda(), w, ws)
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all()


def check_linear(S, rows, inner, outer, kind, bias, seed=0, **more):
    x = normal(seed, rows, inner, kind=kind)
    w, ws = S.quantize_rows(normal(seed + 1, outer, inner).cuda())
    b = normal(seed + 2, outer) if bias else None
    y = S.int8_linear(x.cuda(), w, ws, None if b is None else b.cuda(), **more)
    q, scale = quantized(x)
    product = (q.double() @ w.cpu().double().T) * scale.double()[:, None] * ws.cpu().double()
    want = product if b is None else product + b.double()
    size = product.abs() if b is None else product.abs() + b.double().abs()
    off = (y.cpu().double() - want).abs()
    assert y.dtype == more.get("out_dtype", kind)
    assert (off <= U[y.dtype] * want.abs() + 4 * 2.0 ** -24 * size + 1e-37).all(), off.max()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 127, 129, 300])
def test_linear_rows(S, kind, rows):
    check_linear(S, rows, 208, 72, kind, True, rows)


@pytest.mark.parametrize("rows", [3, 40, 200])
@pytest.mark.parametrize("inner", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 700, 2049])
def test_linear_inner(S, rows, inner):
    check_linear(S, rows, inner, 50, torch.bfloat16, False, inner)


@pytest.mark.parametrize("rows", [3, 40, 200])
@pytest.mark.parametrize("outer", [1, 2, 15, 17, 31, 32, 33, 63, 65, 127, 128, 129, 255, 257, 511, 1030])
def test_linear_outer(S, rows, outer):
    check_linear(S, rows, 144, outer, torch.float16, True, outer)


@pytest.mark.parametrize("rows,inner,outer", [(513, 1024, 1536), (1500, 640, 2500), (130, 4096, 260)])
def test_linear_larger(S, rows, inner, outer):
    for kind in KINDS:
        check_linear(S, rows, inner, outer, kind, True, rows)


@pytest.mark.parametrize("out_dtype", KINDS)
def test_linear_output_type(S, out_dtype):
    for rows in (5, 150):
        check_linear(S, rows, 96, 100, torch.float32, True, 5, out_dtype=out_dtype)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,inner", [(1, 16384), (1, 16385), (4, 4096), (4, 4097), (5, 64), (2, 37)])
def test_linear_is_its_two_steps(S, kind, rows, inner):
    """A few rows are rounded by the product's kernel, more by one of their own: the bits are those of the two calls."""
    x = normal(rows, rows, inner, kind=kind).cuda()
    w, ws = S.quantize_rows(normal(1, 33, inner).cuda())
    b = normal(2, 33).cuda()
    codes, scale = S.quantize_rows(x)
    for out in KINDS:
        assert torch.equal(S.int8_linear(x, w, ws, b, out_dtype=out), S.int8_matmul(codes, scale, w, ws, b, out_dtype=out))


def test_linear_extremes_are_exact(S):
    """All codes at +-127, a long inner dimension: the largest sums there are."""
    for rows, inner in ((2, 131072), (140, 16384)):
        a = torch.full((rows, inner), 127, dtype=torch.int8, device="cuda")
        w = torch.full((40, inner), -127, dtype=torch.int8, device="cuda")
        one = lambda n: torch.ones(n, device="cuda")  # noqa: E731
        y = S.int8_matmul(a, one(rows), w, one(40), out_dtype=torch.float32)
        assert (y.double() == float(np.float32(-127 * 127 * inner))).all()


def test_matmul_ignores_what_lies_behind_the_rows(S):
    """Between the inner size and the next multiple of 16 anything may stand."""
    for rows in (4, 200):
        full = torch.full((rows, 64), 77, dtype=torch.int8, device="cuda")
        wide = torch.full((90, 64), 55, dtype=torch.int8, device="cuda")
        full[:, :37] = 1
        wide[:, :37] = 2
        y = S.int8_matmul(full[:, :37], torch.ones(rows, device="cuda"), wide[:, :37], torch.ones(90, device="cuda"),
                          out_dtype=torch.float32)
        assert (y == 74).all()


def test_linear_writes_into_a_strided_output_and_no_further(S):
    for rows, cols in ((3, 50), (150, 200)):
        x = normal(4, rows, 80, kind=torch.bfloat16).cuda()
        w, ws = S.quantize_rows(normal(5, cols, 80).cuda())
        for pad in (0, 1, 8):
            for lead in (0, 1):
                big = torch.full((rows + 2, cols + pad + lead + 3), 7.0, dtype=torch.bfloat16, device="cuda")
                part = big[1: rows + 1, lead: lead + cols]
                S.int8_linear(x, w, ws, out=part)
                assert torch.equal(part, S.int8_linear(x, w, ws))
                part.fill_(7.0)
                assert (big == 7).all()


def test_linear_of_no_rows_and_of_strided_rows(S):
    w, ws = S.quantize_rows(normal(6, 30, 48).cuda())
    assert S.int8_linear(torch.empty(0, 48, device="cuda"), w, ws).shape == (0, 30)
    x = normal(7, 20, 100).cuda()
    for view in (x[:, 3:51], x[::2, :48], x.T[:, :].contiguous().T[:, :48]):
        assert torch.equal(S.int8_linear(view, w, ws), S.int8_linear(view.contiguous(), w, ws))


def test_linear_gives_the_same_bits_again_and_on_another_stream(S):
    for rows in (6, 333):
        x = normal(8, rows, 512, kind=torch.bfloat16).cuda()
        w, ws = S.quantize_rows(normal(9, 700, 512).cuda())
        first = S.int8_linear(x, w, ws)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        ys = [S.int8_linear(x, w, ws, stream=side.cuda_stream) for _ in range(5)]
        with torch.cuda.stream(side):
            ys.append(S.int8_linear(x, w, ws))
        side.synchronize()
        assert all(torch.equal(first, y) for y in ys)


# ---------------------------------------------------- head norms, rotation --
def rope_want(x, w, at, table, rot, inter, norm, eps):
    """The 64-bit values, and the sizes that their errors go by."""
    y = x.double()
    f = 1.0
    if norm == "rms":
        f = 1 / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
    if norm == "l2":
        f = 1 / torch.sqrt((y * y).sum(-1, keepdim=True) + eps)
    y = y * f * (1.0 if w is None else w.double())
    size = y.abs()
    if rot:
        rows = table.double()[at.long()][:, None]
        c, s = rows[..., : rot // 2], rows[..., rot // 2:]
        ia = torch.arange(0, rot, 2) if inter else torch.arange(rot // 2)
        ib = ia + 1 if inter else ia + rot // 2
        a, b = y[..., ia], y[..., ib]
        y, size = y.clone(), size.clone()
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
        size[..., ia] = (a * c).abs() + (b * s).abs()
        size[..., ib] = (b * c).abs() + (a * s).abs()
    return y, size


def check_rope(S, tokens, heads, kv, dim, rot, inter, norm="rms", kind=torch.bfloat16, weights=True, fused=True, seed=0, inplace=False):
    table = S.rope_table(500, rot) if rot else None
    qkv = normal(seed, tokens, (heads + 2 * kv) * dim, kind=kind)
    wq, wk = (normal(seed + i, dim, kind=kind) if weights else None for i in (1, 2))
    at = torch.randint(0, 500, (tokens,), dtype=torch.int32, generator=torch.Generator().manual_seed(seed))
    g = qkv.cuda()
    q, k = g[:, : heads * dim].view(tokens, heads, dim), g[:, heads * dim: (heads + kv) * dim].view(tokens, kv, dim)
    if not fused:
        q, k = q.contiguous(), k.contiguous()
    want = [rope_want(x.cpu(), w, at, None if table is None else table.cpu(), rot, inter, norm, 1e-5) for x, w in ((q, wq), (k, wk))]
    rest = g[:, (heads + kv) * dim:].clone()
    got = S.qk_norm_rope(q, k, None if wq is None else wq.cuda(), None if wk is None else wk.cuda(), at.cuda(), table,
                         interleaved=inter, norm=norm, eps=1e-5, out=(q, k) if inplace else None)
    for y, (w, size) in zip(got, want):
        off = (y.cpu().double() - w).abs()
        assert (off <= U[kind] * w.abs() + (dim / 64 + 24) * 2.0 ** -24 * size + 1e-37 + (2.0 ** -25 if kind == torch.float16 else 0)).all(), off.max()
    assert torch.equal(g[:, (heads + kv) * dim:], rest)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dim,rot", [(64, 64), (64, 32), (128, 128), (128, 64), (128, 32), (96, 96), (96, 48), (256, 256), (256, 64),
                                     (32, 16), (80, 80), (512, 128), (10, 6), (66, 64), (2, 2), (7, 4), (33, 0), (160, 160), (576, 64)])
def test_rope_sizes(S, kind, inter, dim, rot):
    check_rope(S, 5, 3, 2, dim, rot, inter, kind=kind)


@pytest.mark.parametrize("norm", ["none", "rms", "l2"])
@pytest.mark.parametrize("weights", [False, True])
def test_rope_norms(S, norm, weights):
    for dim, rot in ((128, 128), (30, 20)):
        check_rope(S, 9, 4, 1, dim, rot, False, norm=norm, weights=weights)


@pytest.mark.parametrize("tokens,heads,kv", [(1, 1, 1), (1, 8, 2), (2, 7, 1), (301, 5, 3), (64, 32, 8), (3, 1, 1), (1000, 2, 2)])
def test_rope_tokens_and_heads(S, tokens, heads, kv):
    check_rope(S, tokens, heads, kv, 64, 64, False)
    check_rope(S, tokens, heads, kv, 128, 64, True, fused=False)


def test_rope_in_place_leaves_the_values_alone(S):
    for dim, rot in ((128, 128), (48, 20)):
        check_rope(S, 33, 6, 2, dim, rot, False, inplace=True)


def test_rope_strides_and_alignment(S):
    """Heads outside, tokens inside; rows that start on odd values."""
    table = S.rope_table(100, 64)
    at = torch.arange(11, dtype=torch.int32, device="cuda")
    base = normal(5, 4, 11, 65, kind=torch.bfloat16).cuda()
    w = normal(6, 64, kind=torch.bfloat16).cuda()
    for view in (base[:, :, :64].transpose(0, 1), base[:, :, 1:].transpose(0, 1)):
        got, _ = S.qk_norm_rope(view, None, w, None, at, table)
        want, _ = S.qk_norm_rope(view.contiguous(), None, w, None, at, table)
        assert torch.equal(got, want)


def test_rope_of_keys_alone_zero_rows_and_no_tokens(S):
    table = S.rope_table(10, 32)
    zero = torch.zeros(3, 2, 32, device="cuda")
    at = torch.zeros(3, dtype=torch.int32, device="cuda")
    q, k = S.qk_norm_rope(zero, zero.clone(), None, None, at, table)
    assert (q == 0).all() and (k == 0).all()
    q, _ = S.qk_norm_rope(zero[:0], None, None, None, at[:0], table)
    assert q.shape == (0, 2, 32)


def test_rope_positions_outside_the_table_give_nan(S):
    table = S.rope_table(10, 32)
    for dim in (32, 34):
        x = normal(3, 4, 2, dim).cuda()
        at = torch.tensor([0, -1, 10, 9], dtype=torch.int32, device="cuda")
        q, _ = S.qk_norm_rope(x, None, None, None, at, table)
        assert torch.isnan(q[1:3]).all() and torch.isfinite(q[0]).all() and torch.isfinite(q[3]).all()


@pytest.mark.parametrize("scaling", ["none", "linear", "base", "parts"])
def test_rope_table_is_the_formula(S, scaling):
    n, rot, base, factor, trained, fast, slow = 9000, 64, 10000.0, 8.0, 1024, 32.0, 1.0
    got = S.rope_table(n, rot, base, scaling, factor, trained, fast, slow).cpu().double()
    i = torch.arange(rot // 2, dtype=torch.float64)
    b = base * factor ** (rot / (rot - 2)) if scaling == "base" else base
    f = b ** (-2 * i / rot)
    magnitude = 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        turns = lambda x: rot * math.log(trained / (x * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(turns(fast)), 0), min(math.ceil(turns(slow)), rot - 1)
        ramp = ((i - low) / (high - low)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        magnitude = 0.1 * math.log(factor) + 1
    angle = torch.arange(n, dtype=torch.float64)[:, None] * f
    want = torch.cat([angle.cos(), angle.sin()], 1) * magnitude
    # an angle up to 9000 from a frequency with a few 64-bit roundings, then one 32-bit rounding
    assert (got - want).abs().max() <= 2.0 ** -24 * magnitude + 1e-11


# ------------------------------------------------------------- the cache --
class Host:
    """The cache's definition on the CPU, page by page."""

    def __init__(self, cache):
        self.k, self.v, self.ks, self.vs = (t.cpu().clone() for t in cache)
        self.page = self.k.shape[2]

    def append(self, k, v, pages, held, starts):
        for b in range(len(held)):
            n = starts[b + 1] - starts[b]
            for j in range(held[b] // self.page, -(-(held[b] + n) // self.page)):
                lo, hi = max(held[b], j * self.page), min(held[b] + n, (j + 1) * self.page)
                if lo >= hi:
                    continue
                old, at = lo - j * self.page, pages[b][j]
                for x, codes, scale in ((k, self.k[at], self.ks[at]), (v, self.v[at].transpose(1, 2), self.vs[at])):
                    new = x[starts[b] + lo - held[b]: starts[b] + hi - held[b]].float().transpose(0, 1)     # [heads, n, dim]
                    to = new.abs().amax((1, 2)) * torch.tensor(STEP)
                    if old:
                        to = torch.maximum(to, scale)
                        ratio = torch.where(to > 0, scale / to, torch.ones(()))
                        codes[:, :old] = torch.round(codes[:, :old].float() * ratio[:, None, None]).to(torch.int8)
                    scale[:] = to
                    codes[:, old: old + hi - lo] = codes_of(new, to[:, None, None]).to(torch.int8)

    def values(self, at):
        """A page's keys and values as 64-bit [heads, page, dim]."""
        return (self.k[at].double() * self.ks[at].double()[:, None, None],
                self.v[at].transpose(1, 2).double() * self.vs[at].double()[:, None, None])


def make_cache(S, pages, heads, dim, page, seed=0):
    g = torch.Generator().manual_seed(seed)
    c = S.Cache8.empty(pages, heads, dim, page)
    for t in c[:2]:
        t.copy_((torch.randn(t.shape, generator=g) * 32).round().clamp(-127, 127))
    for t in c[2:]:
        t.copy_((torch.rand(t.shape, generator=g) + 0.5) / 32)
    return c


def make_table(counts, page, seed=0, spare=2, width=None):
    used = [-(-n // page) for n in counts]
    order = torch.randperm(sum(used) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max([1] + used) if width is None else width
    return [[order[sum(used[:b]) + j] if j < used[b] else -1 for j in range(width)] for b in range(len(used))], sum(used) + spare


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def sums(x):
    return [0] + np.cumsum(x).tolist()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("dim,heads", [(32, 3), (64, 1), (96, 2), (128, 8), (192, 1), (256, 2)])
def test_append_is_the_definition(S, kind, page, dim, heads):
    """Fresh and begun pages, pages that end inside, sequences that get nothing; in steps, so that pages are rounded anew."""
    steps = [[5, 0, page, 2 * page + 3, 1], [1, 1, 1, 1, 1], [page - 5, 2, page // 2, 3 * page, 0], [1, 0, 1, 1, 1]]
    final = [sum(s[b] for s in steps) for b in range(5)]
    table, pages = make_table(final, page)
    cache = make_cache(S, pages, heads, dim, page)
    host = Host(cache)
    held = [0] * 5
    for i, new in enumerate(steps):
        starts = sums(new)
        kv = normal(i, starts[-1], 2 * heads * dim, kind=kind) * (1 + i)       # later tokens are larger
        g = kv.cuda()
        view = lambda t, j: t[:, j * heads * dim: (j + 1) * heads * dim].view(-1, heads, dim)  # noqa: E731
        S.cache_append(cache, view(g, 0), view(g, 1), ints(table), ints(held), ints(starts), max(new))
        host.append(view(kv, 0), view(kv, 1), table, held, starts)
        held = [h + n for h, n in zip(held, new)]
    for got, want in zip(cache[2:], (host.ks, host.vs)):
        assert torch.equal(got.cpu(), want)
    starts = sums(held)
    for out in KINDS:
        k, v = S.cache_load(cache, ints(table), ints(held), ints(starts), starts[-1], max(held), out)
        for b, n in enumerate(held):
            for t in range(n):
                wk, wv = host.values(table[b][t // page])
                assert torch.equal(k[starts[b] + t].cpu(), wk[:, t % page].float().to(out))
                assert torch.equal(v[starts[b] + t].cpu(), wv[:, t % page].float().to(out))


def test_append_of_zeros_and_of_values_that_are_not_finite(S):
    cache = make_cache(S, 3, 2, 32, 16)
    table, starts = ints([[0], [1]]), ints([0, 2, 4])
    k = torch.zeros(4, 2, 32, device="cuda")
    v = torch.ones(4, 2, 32, device="cuda")
    v[0, 1, 3] = INF
    S.cache_append(cache, k, v, table, ints([0, 0]), starts, 2)
    ks, vs = S.cache_load(cache, table, ints([2, 2]), starts, 4, 2, torch.float32)
    assert (ks == 0).all() and (vs[2:] == 1).all() and (vs[:2, 0] == 1).all()
    assert torch.isnan(vs[:2, 1]).all()              # the page's scale of that head is not finite
    S.cache_append(cache, k[:1] + 1, v[2:3], table[1:], ints([2]), ints([0, 1]), 1)
    ks, vs = S.cache_load(cache, table[1:], ints([3]), ints([0, 3]), 3, 3, torch.float32)
    assert (ks[:2] == 0).all() and (ks[2] == 1).all() and (vs == 1).all()


def test_append_outside_the_table_or_the_cache_is_dropped(S):
    cache = make_cache(S, 4, 1, 32, 16)
    before = [t.clone() for t in cache]
    x = normal(1, 20, 1, 32).cuda()
    S.cache_append(cache, x, x, ints([[-1, 2], [9, 4]]), ints([0, 0]), ints([0, 10, 20]), 10)
    S.cache_append(cache, x, x, ints([[0]]), ints([16]), ints([0, 20]), 20)
    S.cache_append(cache, x, x, ints([[0, 1]]), ints([0]), ints([0, 20]), 19)      # more rows than it said
    S.cache_append(cache, x, x, ints([[0, 1]]), ints([-1]), ints([0, 20]), 20)
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    k, v = S.cache_load(cache, ints([[7]]), ints([3]), ints([0, 3]), 3, 3, torch.float32)
    assert torch.isnan(k).all() and torch.isnan(v).all()


# -------------------------------------------------------------- attention --
def check_attention(S, new, kept, heads, kv, dim, page, causal, kind=torch.bfloat16, seed=0, spread=1.0, most_kept=None, scale=None,
                    poison=False):
    table, pages = make_table(kept, page, seed)
    cache = make_cache(S, pages, kv, dim, page, seed)
    if spread != 1.0:                                     # scales that differ by powers between pages
        for t in cache[2:]:
            t.mul_(spread ** torch.randn(t.shape, generator=torch.Generator().manual_seed(seed)).cuda())
    host = Host(cache)
    if poison:                                            # pages that nobody has
        mine = {p for row in table for p in row if p >= 0}
        for p in set(range(pages)) - mine:
            cache.k_scale[p] = cache.v_scale[p] = math.nan
    starts = sums(new)
    q = normal(seed + 1, starts[-1], heads, dim, kind=kind)
    out = S.cache_attention(q.cuda(), cache, ints(table), ints(kept), ints(starts), max(new), max(kept) if most_kept is None else most_kept,
                            causal=causal, scale=scale).cpu().double()
    f, group = 1 / math.sqrt(dim) if scale is None else scale, heads // kv
    for b, n in enumerate(kept):
        if n:
            both = [host.values(table[b][j]) for j in range(-(-n // page))]
            keys, values = (torch.cat([x[i] for x in both], 1)[:, :n].repeat_interleave(group, 0) for i in (0, 1))
        for i in range(new[b]):
            got = out[starts[b] + i]
            m = n - new[b] + i + 1 if causal else n
            if m <= 0:
                assert (got == 0).all()
                continue
            x = q[starts[b] + i].double()
            k, v = keys[:, :m], values[:, :m]
            p = torch.softmax(torch.einsum("hd,htd->ht", x, k) * f, 1)
            want = torch.einsum("ht,htd->hd", p, v)
            # the scores' error: 32-bit sums of dim products and a few more roundings, and what 16 bits lose of a small q
            size = torch.einsum("hd,htd->ht", x.abs(), k.abs()).amax(1) * abs(f)
            d = (dim + 16) * 2.0 ** -23 * size + abs(f) * 2.0 ** -24 * x.abs().amax(1) * k.abs().sum(2).amax(1)
            d = d[:, None]
            tol = U[kind] * want.abs() + (2.0 ** -11 + 2 * d + 2.0 ** -18) * torch.einsum("ht,htd->hd", p, v.abs()) \
                + m * 2.0 ** -24 * v.abs().amax((1, 2))[:, None]
            off = (got - want).abs()
            assert (off <= tol).all(), (b, i, float((off / tol).max()))


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
def test_attention_sizes(S, page, dim):
    check_attention(S, [1, 1, 1], [97, 1, 300], 4, 2, dim, page, True)
    check_attention(S, [3, 5], [70, 5], 4, 2, dim, page, True, kind=torch.float16)
    check_attention(S, [40, 7], [170, 64], 4, 2, dim, page, True)
    check_attention(S, [130], [200], 2, 1, dim, page, False)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (7, 1), (8, 1), (16, 1), (17, 1), (14, 2), (40, 2), (6, 3)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_head_groups(S, heads, kv, causal):
    check_attention(S, [1, 1], [130, 31], heads, kv, 64, 16, causal)
    check_attention(S, [9, 1], [130, 31], heads, kv, 64, 32, causal)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 191, 255, 256, 257, 500])
def test_attention_lengths(S, n):
    for page in (16, 32, 64):
        check_attention(S, [1], [n], 2, 1, 64, page, True, seed=n)
    check_attention(S, [min(n, 150)], [n], 2, 1, 64, 32, True, seed=n)


@pytest.mark.parametrize("new", [1, 2, 16, 63, 64, 65, 127, 128, 129, 257, 300])
def test_attention_numbers_of_queries(S, new):
    check_attention(S, [new], [new + 37], 4, 1, 128, 64, True, seed=new)
    check_attention(S, [new], [50], 2, 2, 64, 16, False, seed=new)


def test_attention_long_and_split(S):
    check_attention(S, [1], [9000], 8, 1, 64, 16, True)
    check_attention(S, [1, 1], [6000, 1], 4, 1, 128, 64, True)
    check_attention(S, [4], [5001], 4, 1, 128, 32, True, kind=torch.float16)
    check_attention(S, [1, 2, 1], [0, 700, 3], 2, 1, 64, 16, False, most_kept=20000)


def test_attention_of_several_prompts(S):
    check_attention(S, [200, 33, 129, 1], [700, 33, 400, 250], 4, 2, 128, 32, True)
    check_attention(S, [200, 33, 129, 1], [700, 0, 400, 250], 4, 4, 64, 64, False, kind=torch.float16)


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_rows_that_see_nothing(S, dim):
    """Empty caches, more queries than tokens, sequences without queries."""
    for new, kept in (([3, 0, 2, 1], [0, 40, 1, 0]), ([20, 4], [7, 0]), ([300, 0, 1], [140, 0, 0])):
        for causal in (True, False):
            check_attention(S, new, kept, 4, 2, dim, 16, causal)


@pytest.mark.parametrize("new", [1, 150])
def test_attention_scales_far_apart(S, new):
    check_attention(S, [new], [400], 2, 1, 64, 16, True, spread=30.0, scale=0.02)
    check_attention(S, [new], [400], 2, 1, 128, 64, True, spread=1e4, scale=1e-4)


@pytest.mark.parametrize("new", [1, 150])
def test_attention_with_peaked_scores(S, new):
    check_attention(S, [new, new], [600, 300], 4, 2, 64, 32, True, scale=2.0)
    check_attention(S, [new], [300], 4, 2, 128, 32, False, scale=-0.5)


@pytest.mark.parametrize("new", [1, 150])
def test_attention_never_reads_pages_it_has_not(S, new):
    check_attention(S, [new, new], [333, 150], 4, 2, 64, 16, True, poison=True, most_kept=1000)


@pytest.mark.parametrize("new", [1, 40, 200])
def test_attention_broken_pages_reach_only_those_who_see_them(S, new):
    """A scale that is not a number on the last page: earlier causal rows are as they were."""
    heads, dim, page = 2, 64, 16
    kept = 208
    table, pages = make_table([kept], page)
    cache = make_cache(S, pages, 1, dim, page)
    q = normal(1, new, heads, dim, kind=torch.bfloat16).cuda()
    args = (ints(table), ints([kept]), ints([0, new]), new, kept)
    good = S.cache_attention(q, cache, *args)
    for broken, value in ((0, math.nan), (1, math.nan), (0, INF), (1, INF)):
        last = table[0][-1]
        c = S.Cache8(*(t.clone() for t in cache))
        c[2 + broken][last] = value
        got = S.cache_attention(q, c, *args)
        blind = max(0, new - page)
        assert torch.equal(got[:blind], good[:blind])
        assert torch.isnan(got[blind:]).all()
    wrong = ints([table[0][:-1] + [pages + 5]])
    got = S.cache_attention(q, cache, wrong, *args[1:])
    assert torch.equal(got[:blind], good[:blind]) and torch.isnan(got[blind:]).all()


@pytest.mark.parametrize("new", [1, 150])
def test_attention_lengths_beyond_the_bounds_give_nan(S, new):
    table, pages = make_table([160, 160], 16)
    cache = make_cache(S, pages, 1, 64, 16)
    q = normal(1, 2 * new, 1, 64, kind=torch.float16).cuda()
    for most in (160, 5000):
        out = S.cache_attention(q, cache, ints(table), ints([160, 161]), ints([0, new, 2 * new]), new, most)
        assert torch.isfinite(out[:new]).all() and torch.isnan(out[new:]).all()


@pytest.mark.parametrize("new", [2, 140])
def test_attention_strides(S, new):
    table, pages = make_table([200], 32)
    cache = make_cache(S, pages, 2, 64, 32)
    args = (cache, ints(table), ints([200]), ints([0, new]), new, 200)
    for base, view in ((normal(1, new, 4 * 64 + 5, kind=torch.float16).cuda(), lambda t: t.as_strided((new, 4, 64), (261, 64, 1), 1)),
                       (normal(2, 4, new, 64, kind=torch.float16).cuda(), lambda t: t.transpose(0, 1))):
        q = view(base)
        want = S.cache_attention(q.contiguous(), *args)
        assert torch.equal(S.cache_attention(q, *args), want)
        out = torch.zeros_like(base)
        S.cache_attention(q, *args, out=view(out))
        assert torch.equal(view(out), want)


def test_attention_on_another_stream_gives_the_same_bits(S):
    for new, kept in ((1, 3000), (200, 900)):
        table, pages = make_table([kept, kept], 64)
        cache = make_cache(S, pages, 2, 128, 64)
        q = normal(1, 2 * new, 8, 128, kind=torch.bfloat16).cuda()
        args = (q, cache, ints(table), ints([kept, kept]), ints([0, new, 2 * new]), new, kept)
        want = S.cache_attention(*args)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = [S.cache_attention(*args, stream=side.cuda_stream) for _ in range(4)]
        side.synchronize()
        assert all(torch.equal(g, want) for g in got)


# --------------------------------------------------------------- together --
def test_the_operators_replay_in_a_graph(S):
    """One decode step, captured: norms and rotation, append, attention, projection."""
    heads, kv, dim, page, seqs = 8, 2, 64, 16, 3
    table, pages = make_table([60] * seqs, page)
    cache = make_cache(S, pages, kv, dim, page)
    qkv = normal(1, seqs, (heads + 2 * kv) * dim, kind=torch.bfloat16).cuda()
    w, ws = S.quantize_rows(normal(2, 96, heads * dim).cuda())
    rope = S.rope_table(100, dim)
    pt, held, kept, starts, at = ints(table), ints([20, 31, 47]), ints([21, 32, 48]), ints([0, 1, 2, 3]), ints([20, 31, 47])

    def step():
        q, k = S.qk_norm_rope(qkv[:, : heads * dim].view(seqs, heads, dim), qkv[:, heads * dim: (heads + kv) * dim].view(seqs, kv, dim),
                              None, None, at, rope)
        S.cache_append(cache, k, qkv[:, (heads + kv) * dim:].view(seqs, kv, dim), pt, held, starts, 1)
        o = S.cache_attention(q, cache, pt, kept, starts, 1, 1000)
        return S.int8_linear(o.view(seqs, -1), w, ws)

    want = step()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


# --------------------------------------------------------------- refusals --
def test_tensors_that_do_not_fit_are_refused(S):
    """Before any launch, with ValueError (a tensor's shape, type or place) or TypeError (no tensor at all)."""
    x = torch.zeros(4, 32, device="cuda")
    w, ws = S.quantize_rows(torch.ones(8, 32, device="cuda"))
    cache = make_cache(S, 4, 2, 64, 16)
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda")
    one, starts = ints([1]), ints([0, 2])
    table = ints([[0]])
    rope = S.rope_table(8, 64)
    bad = [
        lambda: S.quantize_rows(x.cpu()), lambda: S.quantize_rows(x.int()), lambda: S.quantize_rows(x[0]), lambda: S.quantize_rows(x[:, :0]),
        lambda: S.int8_linear(x[:, :31], w, ws), lambda: S.int8_linear(x, w.float(), ws), lambda: S.int8_linear(x, w, ws[:7]),
        lambda: S.int8_linear(x, w, ws, ws.half()), lambda: S.int8_linear(x, w, ws, out=torch.empty(4, 7, device="cuda")),
        lambda: S.int8_linear(x, w, ws, out_dtype=torch.int32), lambda: S.int8_linear(x, w[:, 1:], ws),
        lambda: S.int8_linear(x[:, :20], torch.zeros(8, 20, dtype=torch.int8, device="cuda"), ws),       # rows 20 bytes apart
        lambda: S.int8_matmul(w[:, :20].contiguous(), ws, w[:, :20], ws),
        lambda: S.qk_norm_rope(q, q[:1], None, None, ints([0, 1]), rope), lambda: S.qk_norm_rope(q, q.float(), None, None, ints([0, 1]), rope),
        lambda: S.qk_norm_rope(q, None, q[0, 0, :63], None, ints([0, 1]), rope), lambda: S.qk_norm_rope(q, None, None, None, ints([0]), rope),
        lambda: S.qk_norm_rope(q, None, None, None, ints([0, 1]), rope, norm="layer"), lambda: S.qk_norm_rope(q.transpose(1, 2), None, None, None, None, None),
        lambda: S.rope_table(8, 64, scaling="more"),
        lambda: S.cache_append(cache, q[:, :2], q[:, :1], table, one, starts, 2), lambda: S.cache_append(cache, q, q, table, one, starts, 2),
        lambda: S.cache_append(cache, q[:, :2], q[:, :2], table, starts, starts, 2), lambda: S.cache_append(cache, q[:, :2], q[:, :2], table.long(), one, starts, 2),
        lambda: S.cache_load(cache, table, one, starts, -1, 1), lambda: S.cache_load(cache, table, one, starts, 2, 1, torch.int8),
        lambda: S.cache_attention(q[..., :32], cache, table, one, starts, 2, 16), lambda: S.cache_attention(q, cache, table, one, starts[:1], 2, 16),
        lambda: S.cache_attention(q, (cache[0], cache[0], cache[2], cache[3]), table, one, starts, 2, 16),
        lambda: S.cache_attention(q, cache, table, one, starts, 2, 16, out=q.bfloat16()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    for call in (lambda: S.quantize_rows(3), lambda: S.cache_attention(q, cache[:3], table, one, starts, 2, 16), lambda: S.int8_linear(x, w, ws, out_dtype=3)):
        with pytest.raises(TypeError):
            call()


def test_what_the_library_refuses_raises_its_error(S):
    from vdttfs._lib import VdtError
    cache = make_cache(S, 4, 2, 64, 16)
    q = torch.zeros(2, 4, 64, device="cuda")
    args = (ints([[0]]), ints([1]), ints([0, 2]), 2, 16)
    for call, status in ((lambda: S.cache_attention(q, cache, *args), 5), (lambda: S.cache_attention(q[:, :3].half(), cache, *args), 1),
                         (lambda: S.cache_attention(q.half(), cache, *args, scale=math.inf), 1), (lambda: S.rope_table(4, 3), 1)):
        with pytest.raises(VdtError) as e:
            call()
        assert e.value.status == status

"""The step operators against plain implementations in 64 bits.

Tolerances (u: half a unit in the last place of the output's type, 2^-24, 2^-11
or 2^-8): codes, scale bytes, tokens, pages, positions and slots are equal.  A
4-bit product's terms are exact; the tensor cores add 64 at a time to a 32-bit
sum, so it is off by at most inner / 64 + 2 steps of 2^-23 of the sum of the
terms' magnitudes, and u.  A norm: the 32-bit sum of squares (at most cols / 128 + 12
additions deep, each 2^-24), its root's half, and four more operations; and u.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
KINDS = [torch.float32, torch.float16, torch.bfloat16]
INF, NAN = math.inf, math.nan
FP4 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


@pytest.fixture(scope="module")
def S(dev):
    from vdttfs import seq
    return seq


def normal(seed, *shape, kind=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(kind)


# ----------------------------------------------- microscaled floating point --
def fp4_definition(x):
    """x on the CPU -> (codes [rows, cols], exponent bytes [rows, blocks]), by 64-bit comparisons."""
    x = x.double()
    rows, cols = x.shape
    blocks = -(-cols // 32)
    full = torch.nn.functional.pad(x, (0, blocks * 32 - cols)).view(rows, blocks, 32)
    most = full.abs().amax(2)
    broken = ~torch.isfinite(most) | torch.isnan(full).any(2)
    e = torch.full_like(most, -127)
    for k in range(-126, 128):                                   # the smallest e with most <= 6 * 2^e
        e = torch.where(most > 6 * 2.0 ** (k - 1), torch.full_like(e, k), e)
    y = torch.where(broken[..., None], torch.zeros(()).double(), full / 2.0 ** e[..., None])
    a, code = y.abs(), torch.zeros(full.shape, dtype=torch.int64)
    for i, border in enumerate([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]):
        code += ((a > border) | ((a == border) & (i % 2 == 1))).long()
    code = torch.where((y < 0) | ((y == 0) & torch.signbit(y)), code + 8, code)
    return code.view(rows, -1)[:, :cols], torch.where(broken, torch.full_like(e, 255), e + 127).long()


def unpacked(codes, scale, cols):
    """quantize_fp4's results -> the same two."""
    c = codes.cpu().long()
    c = torch.stack([c & 15, c >> 4], 2).flatten(1)[:, :cols]
    t, n = scale.shape[:2]
    s = scale.cpu().long().view(t, n, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(t * 128, n * 4)
    return c, s[: codes.shape[0], : -(-cols // 32)], s[: codes.shape[0], -(-cols // 32):]


def fp4_of(codes, bytes_):
    v = FP4[codes]
    return v * (2.0 ** (bytes_.double() - 127)).repeat_interleave(32, 1)[:, : v.shape[1]]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 31), (2, 32), (129, 33), (4, 64), (17, 1001), (130, 256), (2, 257), (1, 5000)])
def test_fp4_rows_are_the_definitions(S, kind, rows, cols):
    x = normal(rows * cols, rows, cols, kind=kind) * (1 + torch.arange(cols) % 7 * 3).to(kind)
    if rows > 2:
        x[1] = 0
    codes, scale = S.quantize_fp4(x.cuda())
    assert codes.shape == (rows, (cols + 1) // 2) and scale.shape == ((rows + 127) // 128, (cols + 255) // 256 * 2, 32, 16)
    got, bytes_, past = unpacked(codes, scale, cols)
    want, want_bytes = fp4_definition(x)
    assert torch.equal(bytes_, want_bytes) and not past.any()
    assert torch.equal(got % 8, want % 8) and ((got == want) | (want % 8 == 0)).all()
    if cols % 2:
        assert not (codes[:, -1] >> 4).any()
    value = fp4_of(want, want_bytes)
    for out in KINDS:
        assert torch.equal(S.fp4_values(codes, scale, cols, out).cpu().double(), value.to(out).double())


def test_fp4_ties_and_borders(S):
    """Every border between two codes, and every power of two that a block's largest value sits on, from both sides."""
    sides = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    near = torch.cat([sides, torch.nextafter(sides, torch.tensor(0.0)), torch.nextafter(sides, torch.tensor(9.0)), torch.tensor([6.0])])
    rows = []
    for e in (-126, -125, -20, -1, 0, 3, 100, 125):
        row = torch.zeros(64)
        row[: len(near)] = near * 2.0 ** e
        row[32: 32 + len(near)] = -near * 2.0 ** e
        row[63] = 6 * 2.0 ** e
        row[54:60] = 0
        row[22:32] = 0
        rows.append(row)
    for k in (-149, -140, -128, -127, -126, -124, 0, 50, 126, 127):
        for m in (1.0, 1.5, math.nextafter(1.5, 2), 1.5000001, 1.9999999):
            row = torch.zeros(64)
            row[[5, 40]] = (torch.tensor([1.0, -0.3], dtype=torch.float64) * m * 2.0 ** k).float()
            rows.append(row)
    x = torch.stack(rows)
    codes, scale = S.quantize_fp4(x.cuda())
    got, bytes_, _ = unpacked(codes, scale, 64)
    want, want_bytes = fp4_definition(x)
    assert torch.equal(bytes_, want_bytes)
    assert torch.equal(fp4_of(got, bytes_), fp4_of(want, want_bytes))


def test_fp4_rows_that_are_not_finite(S):
    x = normal(2, 6, 100)
    x[1, 3], x[2, 70], x[3, 99], x[4, 0] = INF, NAN, -INF, 1e-45
    codes, scale = S.quantize_fp4(x.cuda())
    got, bytes_, _ = unpacked(codes, scale, 100)
    want, want_bytes = fp4_definition(x)
    assert torch.equal(bytes_, want_bytes) and (bytes_ == 255).sum() == 3
    w, ws = S.quantize_fp4(normal(3, 40, 100).cuda())
    for rows in (x, x.repeat(40, 1)):
        y = S.fp4_linear(rows.cuda(), w, ws)[:6]
        assert torch.isnan(y[1:4]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[4:]).all()
        v = S.fp4_values(*S.quantize_fp4(rows.cuda()))[:6]
        assert torch.isnan(v[1, :32]).all() and torch.isfinite(v[1, 32:]).all() and torch.isnan(v[2, 64:96]).all() and torch.isnan(v[3, 96:]).all()


def check_fp4(S, rows, inner, outer, kind, bias, seed=0, **more):
    x = normal(seed, rows, inner, kind=kind)
    w, ws = S.quantize_fp4(normal(seed + 1, outer, inner).cuda())
    b = normal(seed + 2, outer) if bias else None
    y = S.fp4_linear(x.cuda(), w, ws, None if b is None else b.cuda(), **more)
    a, v = fp4_of(*fp4_definition(x)), S.fp4_values(w, ws, inner).cpu().double()
    want, size = a @ v.T, a.abs() @ v.abs().T
    if b is not None:
        want, size = want + b.double(), size + b.double().abs()
    off = (y.cpu().double() - want).abs()
    assert y.dtype == more.get("out_dtype", kind)
    assert (off <= U[y.dtype] * want.abs() + (inner / 64 + 2) * 2.0 ** -23 * size + 1e-37).all(), (off / size.clamp(min=1e-30)).max()
    return y


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 2, 7, 16, 17, 31, 32, 33, 64, 65, 127, 128, 129, 300])
def test_fp4_linear_rows(S, kind, rows):
    check_fp4(S, rows, 320, 72, kind, True, rows)


@pytest.mark.parametrize("rows", [3, 40, 200])
@pytest.mark.parametrize("inner", [1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 255, 256, 257, 511, 513, 700, 2049])
def test_fp4_linear_inner(S, rows, inner):
    check_fp4(S, rows, inner, 50, torch.bfloat16, False, inner)


@pytest.mark.parametrize("rows", [3, 40, 200])
@pytest.mark.parametrize("outer", [1, 2, 15, 17, 32, 33, 63, 65, 127, 128, 129, 191, 193, 255, 257, 511, 1030])
def test_fp4_linear_outer(S, rows, outer):
    check_fp4(S, rows, 144, outer, torch.float16, True, outer)


@pytest.mark.parametrize("rows,inner,outer", [(513, 1024, 1536), (1500, 640, 2500), (130, 4096, 260), (24, 4096, 1000), (5, 20000, 300), (700, 512, 6000)])
def test_fp4_linear_larger(S, rows, inner, outer):
    for kind in KINDS:
        check_fp4(S, rows, inner, outer, kind, True, rows)


@pytest.mark.parametrize("out_dtype", KINDS)
def test_fp4_linear_output_type(S, out_dtype):
    for rows in (5, 150):
        check_fp4(S, rows, 96, 100, torch.float32, True, 5, out_dtype=out_dtype)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,inner,outer", [(1, 4096, 33), (4, 1000, 700), (32, 260, 130), (33, 260, 130), (100, 999, 50)])
def test_fp4_linear_is_its_two_steps(S, kind, rows, inner, outer):
    x = normal(rows, rows, inner, kind=kind).cuda()
    w, ws = S.quantize_fp4(normal(1, outer, inner).cuda())
    b = normal(2, outer).cuda()
    codes, scale = S.quantize_fp4(x)
    for out in KINDS:
        assert torch.equal(S.fp4_linear(x, w, ws, b, out_dtype=out), S.fp4_matmul(codes, scale, w, ws, b, out_dtype=out))


def test_fp4_linear_of_any_stride_and_place(S):
    """Inputs off 16 bytes, every second row, a transposed one, outputs inside a wider buffer and over the input."""
    base = normal(1, 70, 90, kind=torch.bfloat16).cuda()
    w, ws = S.quantize_fp4(normal(2, 64, 64).cuda())
    for x in (base[:, 1:65], base[::2, 3:67], base.T[:, :64], base[:40, ::1][:, 26:]):
        want = S.fp4_linear(x.contiguous().clone(), w, ws)
        assert torch.equal(S.fp4_linear(x, w, ws), want)
        wide = torch.full((x.shape[0], 71), 7.0, dtype=torch.bfloat16, device="cuda")
        S.fp4_linear(x, w, ws, out=wide[:, 3:67])
        assert torch.equal(wide[:, 3:67], want) and (wide[:, :3] == 7).all() and (wide[:, 67:] == 7).all()
        y = x.contiguous().clone()
        assert torch.equal(S.fp4_linear(y, w, ws, out=y), want)


def test_fp4_scales_of_every_size(S):
    """Powers of two from the smallest to the largest on both sides: products that pass 32 bits are infinite or 0, the others exact."""
    x = torch.ones(40, 64) * 2.0 ** torch.linspace(-120, 120, 40).round()[:, None]
    w, ws = S.quantize_fp4((torch.ones(9, 64) * 2.0 ** torch.tensor([-120.0, -100, -30, -1, 0, 1, 30, 100, 120])[:, None]).cuda())
    for rows in (x, x.repeat(5, 1)):
        y = S.fp4_linear(rows.cuda(), w, ws).cpu()[:40]
        want = (x.double() @ S.fp4_values(w, ws).cpu().double().T)
        fine = (want < 3e38) & (want > 1.2e-38)
        assert torch.equal(y[fine].double(), want[fine]) and (y[want > 3.5e38] == INF).all() and (y[want < 1e-46] == 0).all()


# ------------------------------------------------ residual's addition, norm --
def check_norm(S, rows, cols, kind, residual, weight, seed=0, eps=1e-6):
    x = normal(seed, rows, cols, kind=kind) * 3
    t = normal(seed + 1, rows, cols, kind=kind) if residual else None
    w = (1 + 0.3 * normal(seed + 2, cols)).to(kind) if weight else None
    cuda = lambda v: None if v is None else v.cuda()  # noqa: E731
    total = x if t is None else (x.float() + t.float()).to(kind)
    z = total.float() * (1 if w is None else w.float())
    root = (total.double().square().mean(1, keepdim=True) + eps).sqrt()
    deep = (cols / 128 + 12) / 2 + 4                             # of the norm, in steps of 2^-24
    y, s = S.add_rms_norm(cuda(x), cuda(t), cuda(w), eps)
    assert torch.equal(s.cpu(), total) and y.dtype == kind
    want = z.double() / root
    assert ((y.cpu().double() - want).abs() <= (U[kind] + deep * 2.0 ** -24) * want.abs() + (2.0 ** -25 if kind == torch.float16 else 1e-37)).all()
    codes, scale, s = S.add_rms_norm_int8(cuda(x), cuda(t), cuda(w), eps)
    unit = z.abs().amax(1) * torch.tensor(np.float32(1) / np.float32(127))
    assert torch.equal(s.cpu(), total)
    assert torch.equal(codes.cpu().float(), torch.round(z / torch.where(unit > 0, unit, torch.ones(()))[:, None]))
    want = unit.double() / root[:, 0]
    assert ((scale.cpu().double() - want).abs() <= deep * 2.0 ** -24 * want).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (2, 1000), (17, 4099), (1, 20000), (1200, 520), (1190, 1030)])
def test_norm_sizes(S, kind, rows, cols):
    check_norm(S, rows, cols, kind, True, True, cols)
    check_norm(S, rows, cols, kind, False, cols % 2 == 0, cols)


def test_norm_of_any_stride_and_in_place(S):
    base, other = normal(1, 60, 90, kind=torch.float16).cuda(), normal(2, 60, 90, kind=torch.float16).cuda()
    w = normal(3, 64, kind=torch.float16).cuda()
    for cut in (lambda t: t[:, 1:65], lambda t: t[::2, 3:67], lambda t: t[:, 8:72], lambda t: t.T[:, :60].T[:, :64]):
        x, r = cut(base), cut(other)
        y, s = S.add_rms_norm(x.contiguous().clone(), r.contiguous().clone(), w)
        codes, scale, _ = S.add_rms_norm_int8(x.contiguous().clone(), r.contiguous().clone(), w)
        for a, b in zip(S.add_rms_norm(x, r, w) + S.add_rms_norm_int8(x, r, w), (y, s, codes, scale, s)):
            assert torch.equal(a, b)
        x2, r2 = x.contiguous().clone(), r.contiguous().clone()
        a, b = S.add_rms_norm(x2, r2, w, out=x2, sum_out=r2)
        assert a is x2 and b is r2 and torch.equal(a, y) and torch.equal(b, s)
        r2 = r.contiguous().clone()
        a, b, c = S.add_rms_norm_int8(x, r2, w, sum_out=r2)
        assert c is r2 and torch.equal(a, codes) and torch.equal(b, scale) and torch.equal(c, s)


def test_norm_of_zeros_and_what_is_not_finite(S):
    x = normal(4, 5, 200)
    x[1], x[2, 7], x[3, 9] = 0, INF, NAN
    y, t = S.add_rms_norm(x.cuda())
    codes, scale, _ = S.add_rms_norm_int8(x.cuda())
    assert (y[1] == 0).all() and (codes[1] == 0).all() and scale[1] == 0
    assert torch.isnan(y[2, 7]) and torch.isnan(y[3]).all() and not torch.isfinite(scale[2:4]).any()
    assert torch.isfinite(y[[0, 4]]).all() and torch.isfinite(scale[[0, 4]]).all()


def test_norm_feeds_the_8_bit_product(S):
    x, r, w = normal(1, 50, 256, kind=torch.bfloat16), normal(2, 50, 256, kind=torch.bfloat16), normal(3, 256, kind=torch.bfloat16)
    m, ms = S.quantize_rows(normal(4, 90, 256).cuda())
    codes, scale, _ = S.add_rms_norm_int8(x.cuda(), r.cuda(), w.cuda())
    y = S.int8_matmul(codes, scale, m, ms, out_dtype=torch.float32).cpu().double()
    want = codes.cpu().double() @ m.cpu().double().T * scale.cpu().double()[:, None] * ms.cpu().double()
    assert ((y - want).abs() <= 3 * 2.0 ** -24 * want.abs()).all()


# ------------------------------------------------------------- page tables --
def plan_definition(ring, span, pages, held, new, page, total):
    ring, table, (first, left) = list(ring), [list(r) for r in pages], span
    starts, kept, positions, slots, took = [0], [], [-1] * total, [-1] * total, 0
    width = len(table[0]) if table else 0
    for s, (h, n) in enumerate(zip(held, new)):
        h, n = max(h, 0), max(n, 0)
        for j in range(-(-h // page), min(-(-(h + n) // page), width)):
            table[s][j] = ring[(first + took) % len(ring)] if took < left else -1
            took += 1
        for i in range(n):
            row, at = starts[-1] + i, h + i
            if row < total:
                positions[row] = at
                number = table[s][at // page] if at // page < width else -1
                slots[row] = number * page + at % page if number >= 0 else -1
        starts.append(starts[-1] + n)
        kept.append(h + n)
    span = [(first + min(took, left)) % len(ring) if ring else 0, left - took]
    return kept, starts, positions, slots, span, table


def check_plan(S, seqs, most_held, most_new, page, seed, short=0, past=3, width=None, in_place=False):
    rng = np.random.default_rng(seed)
    held, new = rng.integers(0, most_held + 1, seqs), rng.integers(0, most_new + 1, seqs)
    if seqs > 4:
        new[rng.integers(0, seqs, max(1, seqs // 5))] = 0
    used, want = -(-held // page), -(-(held + new) // page)
    width = int(want.max()) if width is None else width
    count = int(want.sum()) + 5
    order = rng.permutation(count)
    pages = np.full((seqs, width), -1)
    at = 0
    for s in range(seqs):
        n = min(int(used[s]), width)
        pages[s, :n] = order[at: at + n]
        at += n
    free = order[at:]
    left = max(0, len(free) - 5 - short)
    first = int(rng.integers(0, count))
    ring = np.full(count, -7)
    ring[(first + np.arange(len(free))) % count] = free
    total = int(new.sum()) + past
    ints = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
    t_pages, t_held, t_ring, t_span, t_new = ints(pages), ints(held), ints(ring), ints([first, left]), ints(new)
    out = S.PagePlan(t_held, None, None, None, t_span) if in_place else None
    plan = S.plan_pages(S.PagePool(t_ring, t_span), t_pages, t_held, t_new, page, max(0, total), out)
    kept, starts, positions, slots, span, table = plan_definition(ring.tolist(), (first, left), pages.tolist(), held.tolist(), new.tolist(), page, max(0, total))
    assert plan.kept.tolist() == kept and plan.starts.tolist() == starts
    assert plan.positions.tolist() == positions and plan.slots.tolist() == slots
    assert plan.span.tolist() == span and t_pages.tolist() == table
    assert t_ring.tolist() == ring.tolist()
    return plan


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seqs,most_held,most_new,page", [(1, 0, 1, 16), (1, 50, 3000, 64), (3, 40, 5, 16), (48, 300, 1, 16), (255, 10, 30, 32),
                                                          (256, 0, 64, 64), (1024, 90, 7, 16), (1025, 90, 7, 16), (3000, 20, 3, 32), (5, 7, 40, 3)])
def test_plans(S, seqs, most_held, most_new, page, in_place):
    check_plan(S, seqs, most_held, most_new, page, seqs, in_place=in_place)


def test_plans_of_a_pool_or_a_table_that_is_short(S):
    for seqs in (20, 1500):
        check_plan(S, seqs, 50, 60, 16, 1, short=9)
        check_plan(S, seqs, 50, 60, 16, 2, short=10 ** 6)
        check_plan(S, seqs, 50, 60, 16, 3, width=2)
        check_plan(S, seqs, 50, 60, 16, 4, past=-40)             # fewer rows than tokens
        check_plan(S, seqs, 50, 0, 16, 5)


def test_plans_of_broken_lengths(S):
    """Negative and huge lengths, a ring's state out of range: no access outside, the other sequences as they are."""
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    big = 2 ** 31 - 1
    pages = torch.full((4, 3), -1, dtype=torch.int32, device="cuda")
    pool = S.PagePool.full(8)
    plan = S.plan_pages(pool, pages, ints(-5, 3, big, 0), ints(4, -2, 6, big), 16, 20)
    assert plan.kept.tolist() == [4, 3, big, big] and plan.starts.tolist() == [0, 4, 4, 10, big]
    assert plan.positions.tolist()[:4] == [0, 1, 2, 3] and plan.slots.tolist()[:4] == [0, 1, 2, 3]
    assert plan.slots.tolist()[4:10] == [-1] * 6 and plan.positions.tolist()[10:] == list(range(10))
    assert pages.tolist()[0] == [0, -1, -1] and pages.tolist()[3] == [1, 2, 3] and plan.span.tolist() == [4, 4]
    for span in (ints(-1, 5), ints(8, 5), ints(big, big), ints(2, -3)):
        pages.fill_(-1)
        plan = S.plan_pages((pool.ring, span), pages, ints(0, 0, 0, 0), ints(1, 1, 1, 1), 16, 4)
        assert plan.slots.tolist() == [-1] * 4 and plan.span.tolist()[1] == -4
    plan = S.plan_pages((pool.ring, ints(5, 100)), pages.fill_(-1), ints(0, 0, 0, 0), ints(33, 33, 33, 33), 16, 4)
    assert plan.span.tolist() == [5, -4] and pages.flatten().tolist() == [5, 6, 7, 0, 1, 2, 3, 4, -1, -1, -1, -1]


def test_plans_without_sequences_or_pages(S):
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    none = ints()
    plan = S.plan_pages(S.PagePool.full(3), torch.empty(0, 4, dtype=torch.int32, device="cuda"), none, none, 16, 2)
    assert plan.starts.tolist() == [0] and plan.positions.tolist() == [-1, -1] and plan.span.tolist() == [0, 3]
    plan = S.plan_pages((none, ints(0, 0)), torch.empty(2, 0, dtype=torch.int32, device="cuda"), ints(0, 4), ints(1, 1), 16, 2)
    assert plan.slots.tolist() == [-1, -1] and plan.positions.tolist() == [0, 4] and plan.span.tolist() == [0, 0]
    held, span = S.free_pages((none, ints(0, 0)), torch.empty(2, 0, dtype=torch.int32, device="cuda"), ints(3, 4), torch.tensor([True, False]).cuda(), 16)
    assert held.tolist() == [0, 4] and span.tolist() == [0, 0]


@pytest.mark.parametrize("seqs,in_place", [(1, False), (40, True), (1024, False), (2500, True)])
def test_free_pages(S, seqs, in_place):
    rng = np.random.default_rng(seqs)
    page, width = 16, 70
    held = rng.integers(0, page * width + 40, seqs)
    pages = rng.integers(-1, 10 ** 6, (seqs, width))
    pages[rng.random((seqs, width)) < 0.1] = -1
    done = rng.random(seqs) < 0.4
    back = [int(p) for s in range(seqs) if done[s] for p in pages[s, : -(-int(held[s]) // page)] if p >= 0]
    for size in (len(back) + 11, max(4, len(back) // 2)):
        first, left = size // 2, 3
        ring = rng.integers(0, 9, size)
        ints = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
        t_ring, t_span, t_held, t_done = ints(ring), ints([first, left]), ints(held), torch.tensor(done).cuda()
        got, span = S.free_pages((t_ring, t_span), ints(pages), t_held, t_done, page, out=(t_held, t_span) if in_place else None)
        for i, p in enumerate(back[: size - left]):
            ring[(first + left + i) % size] = p
        assert t_ring.tolist() == ring.tolist() and span.tolist() == [first, min(size, left + len(back))]
        assert got.tolist() == np.where(done, 0, held).tolist()


def test_pages_go_round(S):
    """Sequences that come, grow and end for a hundred steps: no page is ever in two places, none is lost."""
    rng = np.random.default_rng(7)
    seqs, width, page, count = 12, 6, 16, 40
    pool = S.PagePool.full(count)
    pages = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
    held = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    for _ in range(100):
        now = held.tolist()
        new = [int(rng.integers(0, 30)) if h == 0 else int(rng.integers(0, 2)) for h in now]
        new = [min(n, 60 - h) for n, h in zip(new, now)]
        plan = S.plan_pages(pool, pages, held, torch.tensor(new, dtype=torch.int32, device="cuda"), page, sum(new), S.PagePlan(held, None, None, None, pool.span))
        table, span, ring = pages.tolist(), pool.span.tolist(), pool.ring.tolist()
        used = [p for row, h in zip(table, held.tolist()) for p in row[: -(-h // page)]]
        free = [ring[(span[0] + i) % count] for i in range(span[1])]
        assert sorted(used + free) == list(range(count))
        assert len(set(plan.slots.tolist())) == sum(new)
        done = torch.tensor(rng.random(seqs) < 0.15).cuda()
        S.free_pages(pool, pages, held, done, page, out=(held, pool.span))


# ---------------------------------------------------------------- sampling --
def sample_definition(x, u, t, k, p, least):
    """One row of float64 logits -> (token, its probability's logarithm)."""
    if np.isnan(x).any() or not (x > -INF).any() or not (0 <= t < INF) or math.isnan(p) or math.isnan(least):
        return -1, NAN
    order = np.argsort(-x, kind="stable")
    if t == 0:
        return int(order[0]), 0.0
    if not 0 <= u < 1:
        return -1, NAN
    if 0 < k < len(x):
        order = order[:k]
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / t))
    if p < 1:
        before = np.cumsum(w) - w
        keep = before < max(p, 0.0) * w.sum()
        keep[0] = True
        order, w = order[keep], w[keep]
    keep = w >= min(least, 1.0)
    order, w = order[keep], w[keep]
    by = np.argsort(order)
    order, w = order[by], w[by]
    sums = np.cumsum(w)
    at = int(np.searchsorted(sums, u * sums[-1], side="right"))
    return int(order[at]), math.log(w[at] / sums[-1])


def check_sample(S, x, u, t, k, p, least):
    rows = x.shape[0]
    each = lambda v: v.cpu().tolist() if torch.is_tensor(v) else [float(np.float32(v)) if isinstance(v, float) else v] * rows  # noqa: E731
    tokens, logp = S.sample(x.cuda() if x.is_contiguous() else x, u.cuda(), *(v.cuda() if torch.is_tensor(v) else v for v in (t, k, p, least)))
    xs = x.cpu().double().numpy()
    for r, (a, b, c, d) in enumerate(zip(each(t), each(k), each(p), each(least))):
        token, log = sample_definition(xs[r], float(u[r]), a, b, c, d)
        assert int(tokens[r]) == token, (r, int(tokens[r]), token, a, b, c, d)
        got = float(logp[r])
        assert (math.isnan(log) and math.isnan(got)) or abs(got - log) <= 2.0 ** -24 * abs(log) + 2.0 ** -34


def uniform(seed, n):
    return torch.rand(n, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 2), (3, 31), (5, 1000), (4, 1025), (2, 32768), (3, 50001), (40, 5000), (160, 700), (2, 200000)])
def test_sample_sizes(S, kind, rows, vocab):
    x = (normal(vocab, rows, vocab) * 3).to(kind)
    u = uniform(rows, rows)
    for t, k, p, least in ((1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.3, 0, 0.999, 0.0), (1.0, 50, 0.8, 0.0), (1.0, 0, 1.0, 0.1),
                           (1.0, 3000, 0.95, 0.001), (0.0, 5, 0.5, 0.5)):
        check_sample(S, x, u, t, k, p, least)


@pytest.mark.parametrize("kind", KINDS)
def test_sample_draws_every_token(S, kind):
    """Many random numbers for the same logits, from 0 to the last below 1: every answer is the definition's."""
    x = torch.tensor([[0.0, 2.0, -1.0, 2.0, 1.5, -INF, 0.5]]).to(kind).repeat(200, 1)
    u = torch.cat([torch.linspace(0, 1, 198)[:-1], torch.tensor([1 - 2.0 ** -24, 2.0 ** -40, 1e-45])])
    for args in ((1.0, 0, 1.0, 0.0), (1.0, 3, 1.0, 0.0), (1.0, 0, 0.6, 0.0), (2.0, 1, 0.1, 0.0), (0.5, 0, 1.0, 1.0), (1.0, 2, 1.0, 0.0)):
        check_sample(S, x, u, *args)


def test_sample_ties(S):
    """Rows of a few values each: the kept ones end among equals, and the lowest indices of them stay."""
    for vocab in (900, 20000, 70000):
        x = torch.randint(0, 4, (6, vocab), generator=torch.Generator().manual_seed(vocab)).float()
        x[1] = 0.25
        x[2] = -3e38
        x[2, ::3] = -INF
        x[3, 17] = INF
        x[3, 100] = INF
        u = uniform(1, 6)
        for kind in KINDS:
            y = x.to(kind)
            for args in ((1.0, 0, 1.0, 0.0), (1.0, 5, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, vocab // 2, 0.7, 0.0), (0.3, vocab - 1, 1.0, 0.0), (1.0, 1100, 0.9999, 0.2),
                         (1.0, 0, 0.0, 0.0), (0.0, 0, 1.0, 0.0)):
                check_sample(S, y, u, *args)


@pytest.mark.parametrize("kind", KINDS)
def test_sample_of_masked_rows(S, kind):
    """Masks of the type's lowest value, of -inf and of both; rows in which they leave one token, or none but masked ones."""
    low = torch.finfo(kind).min
    x = (normal(9, 6, 5000) * 2).to(kind)
    x[0, 10:] = low
    x[1, 10:], x[1, :5] = -INF, low
    x[2], x[2, 1::2] = low, -INF
    x[3], x[3, 77] = low, 0.5
    x[4] = low
    x[5], x[5, 4000] = -INF, low
    u = uniform(4, 6)
    for t in (0.0, 1e-3, 1.0, 1e35):
        for k, p, least in ((0, 1.0, 0.0), (7, 1.0, 0.0), (0, 0.9, 0.0), (3000, 0.5, 0.1)):
            check_sample(S, x, u, t, k, p, least)


def test_sample_parameters_of_each_row(S):
    g = torch.Generator().manual_seed(3)
    rows, vocab = 60, 9000
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (rows,), generator=g)]  # noqa: E731
    x = torch.randn(rows, vocab, generator=g) * 4
    check_sample(S, x, uniform(5, rows), pick(0.0, 0.2, 1.0, 3.0, 50.0), pick(0, -1, 1, 7, 1024, 2000, 9000).int(), pick(0.0, 0.3, 0.95, 1.0, 2.0, -1.0),
                 pick(0.0, -1.0, 0.05, 1.0, 7.0))


def test_sample_extremes(S):
    """Temperatures and logits at the ends of their ranges."""
    x = normal(1, 8, 3000) * 2
    x[0] *= 1e-38
    x[1] *= 1e37
    x[2, 5] = 3.4e38
    x[3, :2990] = -INF
    x[4] = torch.where(x[4] > 0, 3.4e38, -3.4e38)
    x[5] = x[5] * 1e-6 + 80
    u = uniform(2, 8)
    for t in (1e-45, 1e-38, 1e-6, 1.0, 1e6, 3e38):
        for k, p in ((0, 1.0), (9, 1.0), (0, 0.7)):
            check_sample(S, x, u, t, k, p, 0.0)


def test_sample_rows_that_give_no_token(S):
    x = normal(1, 9, 500)
    x[1, 3], x[2] = NAN, -INF
    u = uniform(1, 9)
    u[3], u[4], u[5] = 1.0, -0.1, NAN
    t = torch.ones(9)
    t[6], t[7], t[8] = -1.0, NAN, INF
    for args in ((t, 0, 1.0, 0.0), (t, 10, 0.9, 0.1)):
        check_sample(S, x, u, *args)
    p = torch.ones(9)
    p[0] = NAN
    check_sample(S, x, u, 1.0, 0, p, 0.0)
    check_sample(S, x, u, 1.0, 0, 0.9, p)


def test_sample_of_several_ctas_a_row_again_and_again(S):
    """Rows that clusters of CTAs share, with parameters that send them different ways: the same tokens every time."""
    g = torch.Generator().manual_seed(8)
    rows, vocab = 64, 40000
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (rows,), generator=g)].cuda()  # noqa: E731
    x = (torch.randn(rows, vocab, generator=g) * 3).to(torch.bfloat16).cuda()
    args = (uniform(3, rows).cuda(), pick(0.0, 0.6, 1.0, 1.3), pick(0, 20, 1000, 3000).int(), pick(0.8, 0.95, 1.0), pick(0.0, 0.02))
    first = S.sample(x, *args)
    check_sample(S, x, *args)
    for _ in range(200):
        tokens, logp = S.sample(x, *args)
        assert torch.equal(tokens, first[0]) and torch.equal(logp, first[1])


def test_sample_of_strided_rows(S):
    x = normal(6, 20, 4111, kind=torch.bfloat16).cuda()
    u = uniform(6, 20)
    for view in (x[:, 1:4001], x[:, 8:], x[::2, 3:4099]):
        check_sample(S, view, u[: view.shape[0]], 0.8, 30, 0.9, 0.0)
        check_sample(S, view, u[: view.shape[0]], 0.8, 0, 0.9, 0.0)


def test_sample_frequencies(S):
    """65536 evenly spaced random numbers: each token comes as often as its probability says, to within one."""
    n = 1 << 16
    x = torch.tensor([[1.0, 0.0, 2.0, -1.0, 0.5, 3.0]]).cuda().repeat(n, 1)
    tokens, _ = S.sample(x, ((torch.arange(n) + 0.5) / n).cuda(), top_k=4)
    p = torch.softmax(torch.tensor([1.0, -INF, 2.0, -INF, 0.5, 3.0]).double(), 0)
    assert ((torch.bincount(tokens.long(), minlength=6).cpu() - p * n).abs() <= 1.0).all()


# --------------------------------------------------- streams, graphs, places --
def step_calls(S):
    """One call of each operator, on inputs of its own: name -> (call(stream), results)."""
    g = torch.Generator().manual_seed(11)
    x = torch.randn(40, 300, generator=g).to(torch.bfloat16).cuda()
    w, ws = S.quantize_fp4(torch.randn(200, 300, generator=g).cuda())
    c, cs = S.quantize_fp4(x)
    few, weight = x[:3].clone(), torch.ones(300, dtype=torch.bfloat16, device="cuda")
    logits, u = (torch.randn(9, 30000, generator=g) * 3).cuda(), torch.rand(9, generator=g).cuda()
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    pool, pages, held, new = S.PagePool.full(50), torch.full((3, 9), -1, dtype=torch.int32, device="cuda"), ints(0, 0, 0), ints(5, 100, 33)
    done = torch.tensor([True, False, True]).cuda()
    S.plan_pages(pool, pages, held, new, 16, 140)
    return {
        "quantize_fp4": lambda st: S.quantize_fp4(x, stream=st), "fp4_values": lambda st: (S.fp4_values(c, cs, stream=st),),
        "fp4_matmul": lambda st: (S.fp4_matmul(c, cs, w, ws, stream=st),), "fp4_linear": lambda st: (S.fp4_linear(x, w, ws, stream=st),),
        "fp4_linear few": lambda st: (S.fp4_linear(few, w, ws, stream=st),), "add_rms_norm": lambda st: S.add_rms_norm(x, x, weight, stream=st),
        "add_rms_norm_int8": lambda st: S.add_rms_norm_int8(x, x, weight, stream=st),
        "plan_pages": lambda st: tuple(S.plan_pages(pool, pages, held, new, 16, 140, stream=st)),
        "free_pages": lambda st: S.free_pages((pool.ring.clone(), pool.span), pages, new, done, 16, stream=st),
        "sample": lambda st: S.sample(logits, u, 0.8, 0, 0.9, stream=st), "sample k": lambda st: S.sample(logits, u, 0.8, 2000, 0.9, stream=st),
    }


# rows past the packed codes of quantised rows, and the padding rows of scale tiles, hold anything
def same(name, a, b):
    if name == "quantize_fp4":
        return all(torch.equal(p[:, :9] if i else p, q[:, :9] if i else q) for i, (p, q) in enumerate(zip(unpacked(*a, 300), unpacked(*b, 300))))
    return all(torch.equal(p, q) for p, q in zip(a, b))


def test_calls_on_a_stream_of_the_callers_own(S):
    side = torch.cuda.Stream()
    for name, call in step_calls(S).items():
        want = call(None)
        torch.cuda.synchronize()
        got = call(side.cuda_stream)
        side.synchronize()
        assert same(name, got, want), name
        assert torch.cuda.current_stream() == torch.cuda.default_stream()


def test_two_calls_at_once(S):
    """The same calls on two streams, many times over: nothing is shared between calls."""
    calls = step_calls(S)
    want = {name: call(None) for name, call in calls.items()}
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    for name, call in calls.items():
        if name == "plan_pages":
            continue                                         # its table is one
        got = []
        for _ in range(20):
            for s in sides:
                with torch.cuda.stream(s):
                    got.append(call(None))
        torch.cuda.synchronize()
        assert all(same(name, g, want[name]) for g in got), name


def test_calls_in_a_graph(S):
    calls = step_calls(S)
    want = {name: call(None) for name, call in calls.items()}
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = {name: call(None) for name, call in calls.items()}
        graphs.append((g, got))
    for _ in range(3):
        for g, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for _, got in graphs:
        for name in calls:
            assert same(name, got[name], want[name]), name


def test_a_step_in_place_in_a_graph(S):
    """Lengths and the pool's state advance with every replay."""
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    pool, pages, held, new = S.PagePool.full(40), torch.full((3, 9), -1, dtype=torch.int32, device="cuda"), ints(3, 15, 16), ints(1, 1, 1)
    S.plan_pages(pool, pages, ints(0, 0, 0), held, 16, 34, S.PagePlan(None, None, None, None, pool.span))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan = S.plan_pages(pool, pages, held, new, 16, 3, S.PagePlan(held, None, None, None, pool.span))
    state = (pool.ring.tolist(), tuple(pool.span.tolist()), pages.tolist(), held.tolist())
    for _ in range(40):
        g.replay()
        want = plan_definition(*state[:2], state[2], state[3], [1, 1, 1], 16, 3)
        assert [t.tolist() for t in plan] == list(want[:5]) and pages.tolist() == want[5] and held.tolist() == want[0]
        state = (pool.ring.tolist(), tuple(pool.span.tolist()), pages.tolist(), held.tolist())


def test_results_of_a_stream_go_on_on_the_current_one(S):
    """A result that is dropped while the current stream still reads it is not given out again before that is done."""
    side = torch.cuda.Stream()
    x = normal(1, 512, 2048, kind=torch.bfloat16).cuda()
    want, _ = S.add_rms_norm(x)
    for _ in range(20):
        y, _ = S.add_rms_norm(x, stream=side.cuda_stream)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda._sleep(200000)
        z = y.clone()
        del y
        S.add_rms_norm(-x, stream=side.cuda_stream)
        assert torch.equal(z, want)


def test_tensors_that_do_not_fit_are_refused(S):
    x = normal(1, 4, 64, kind=torch.bfloat16).cuda()
    w, ws = S.quantize_fp4(normal(2, 10, 64).cuda())
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    pool, pages, u = S.PagePool.full(4), torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.rand(4, device="cuda")
    held = ints(1, 2)
    for bad in (lambda: S.quantize_fp4(x.cpu()), lambda: S.quantize_fp4(x[0]), lambda: S.quantize_fp4(x.long()), lambda: S.fp4_linear(x[:, :60], w, ws),
                lambda: S.fp4_linear(x, w[:5], ws[:, :1]), lambda: S.fp4_linear(x, w, ws.flatten()[:512]), lambda: S.fp4_linear(x, w.view(torch.int8), ws),
                lambda: S.fp4_linear(x, w, ws, x[0]), lambda: S.fp4_linear(x, w, ws, out=x), lambda: S.fp4_matmul(x, ws, w, ws),
                lambda: S.fp4_linear(x, w[:, 1:], ws), lambda: S.fp4_values(w, ws, 40), lambda: S.add_rms_norm(x, x[:3]), lambda: S.add_rms_norm(x, x.float()),
                lambda: S.add_rms_norm(x, None, x[0].float()), lambda: S.add_rms_norm(x, sum_out=x), lambda: S.add_rms_norm(x, x, out=x[:, ::2]),
                lambda: S.add_rms_norm_int8(x, None, x[0, :5]), lambda: S.plan_pages(pool, pages.long(), held, held, 16, 2),
                lambda: S.plan_pages(pool, pages, held[:1], held, 16, 2), lambda: S.plan_pages(pool, pages, held, held, 0, 2),
                lambda: S.plan_pages(pool, pages, held, held, 16, -1), lambda: S.plan_pages(pool, pages, held, held, 16, 2, S.PagePlan(held[:1], *[None] * 4)),
                lambda: S.free_pages(pool, pages, held, held, 16), lambda: S.free_pages((pool.ring.view(2, 2), pool.span), pages, held, held.bool(), 16),
                lambda: S.sample(x, u[:3]), lambda: S.sample(x, u.double()), lambda: S.sample(x, u, u[:2]), lambda: S.sample(x, u, 1.0, u),
                lambda: S.sample(x.int(), u), lambda: S.sample(x[:, :0], u)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: S.quantize_fp4(3), lambda: S.plan_pages(pool.ring, pages, held, held, 16, 2), lambda: S.sample(x, u, "a"), lambda: S.sample(x, u, 1.0, 0.5),
                lambda: S.add_rms_norm(x, eps="b")):
        with pytest.raises(TypeError):
            bad()
    from vdttfs._lib import VdtError
    for bad in (lambda: S.sample(x, u, -1.0), lambda: S.sample(x, u, math.nan), lambda: S.add_rms_norm(x, eps=-1.0),
                lambda: S.sample(torch.zeros(1, 524289, device="cuda"), u[:1])):
        with pytest.raises(VdtError):
            bad()


def test_calls_of_nothing(S):
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    w, ws = S.quantize_fp4(normal(2, 10, 64).cuda())
    codes, scale = S.quantize_fp4(x)
    assert codes.shape == (0, 32) and S.fp4_values(codes, scale).shape == (0, 64) and S.fp4_linear(x, w, ws).shape == (0, 10)
    assert S.fp4_matmul(codes, scale, w, ws).shape == (0, 10)
    assert [t.shape[0] for t in S.add_rms_norm(x, x)] == [0, 0] and [t.shape[0] for t in S.add_rms_norm_int8(x, x)] == [0, 0, 0]
    assert [t.shape[0] for t in S.sample(x, torch.empty(0, device="cuda"))] == [0, 0]


def test_rows_further_apart_than_32_bits_count(S):
    far = 2 ** 31 + 64
    store = torch.zeros(far + 4096, dtype=torch.bfloat16, device="cuda")
    near = normal(5, 2, 1000, kind=torch.bfloat16).cuda()

    def view(t=None):
        v = store.as_strided((2, 1000), (far, 1))
        if t is not None:
            v.copy_(t)
        return v

    w, ws = S.quantize_fp4(normal(6, 1000, 1000).cuda())
    u = torch.tensor([0.3, 0.9], device="cuda")
    x = view(near)
    assert torch.equal(S.fp4_values(*S.quantize_fp4(x)), S.fp4_values(*S.quantize_fp4(near)))
    for a, b in zip(S.add_rms_norm(x, near) + S.add_rms_norm_int8(x, near) + S.sample(x, u, 1.0, 0, 0.9), S.add_rms_norm(near, near) + S.add_rms_norm_int8(near, near)
                    + S.sample(near, u, 1.0, 0, 0.9)):
        assert torch.equal(a, b)
    want = S.fp4_linear(near, w, ws)
    assert torch.equal(S.fp4_linear(x, w, ws), want)
    S.fp4_linear(near, w, ws, out=view())
    assert torch.equal(view(), want)
    codes, scale = S.quantize_fp4(near)
    S.fp4_matmul(codes, scale, w, ws, out=view(near))
    assert torch.equal(view(), want)
    S.add_rms_norm(near, near, out=view(), sum_out=near.clone())
    assert torch.equal(view(), S.add_rms_norm(near, near)[0])
    # many rows, the tiles' way
    wide = torch.zeros(200 * 2 ** 24, dtype=torch.bfloat16, device="cuda").as_strided((200, 256), (2 ** 24 + 32, 1))
    m, ms = S.quantize_fp4(normal(7, 256, 96).cuda())
    y = normal(8, 200, 96, kind=torch.bfloat16).cuda()
    S.fp4_linear(y, m, ms, out=wide)
    assert torch.equal(wide, S.fp4_linear(y, m, ms))

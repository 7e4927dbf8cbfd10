"""The step operators at the ends of their ranges.

Tolerances count roundings, u = 2^-24.  A norm's sum of squares: a thread adds the values of the vectors that it holds one
after another (at most 64), and what it reads beyond them a vector at a time, compensated (8 additions and 2); then 5
exchanges of a warp, at most 8 warps, one value behind the last whole vector.  So 80 u of the sum for any length, 40 u of
its root; 6 more for the mean, eps, root, reciprocal and products; and the output's own rounding.
"""
import math

import numpy as np
import pytest
import torch

from test_gpu_step import INF, KINDS, U, check_sample, normal, sample_definition, uniform

pytestmark = pytest.mark.gpu

u = 2.0 ** -24
NORM = 46 * u


@pytest.fixture(scope="module")
def S(dev):
    from vdttfs import seq
    return seq


# ------------------------------------------------------- norms of long rows --
def check_long(S, x, residual=None, weight=None):
    total = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    z = total.float() if weight is None else total.float() * weight.float()
    root = (total.double().square().mean(1, keepdim=True) + 1e-6).sqrt()
    y, s = S.add_rms_norm(x, residual, weight)
    assert torch.equal(s, total)
    want = z.double() / root
    assert ((y.double() - want).abs() <= (U[x.dtype] + NORM) * want.abs() + (2.0 ** -25 if x.dtype == torch.float16 else 1e-37)).all()
    codes, scale, _ = S.add_rms_norm_int8(x, residual, weight)
    unit = z.abs().amax(1) * torch.tensor(np.float32(1) / np.float32(127)).cuda()
    want = unit.double() / root[:, 0]
    assert ((scale.double() - want).abs() <= NORM * want).all(), ((scale.double() / want - 1).abs().max() / u).item()
    assert torch.equal(codes.float(), torch.round(z / unit[:, None]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cols", [16391, 1 << 20, (1 << 22) + 5])
def test_norm_of_long_rows(S, kind, cols):
    """Rows of one value, whose squares round the same way at every addition, and random ones; on 16 bytes and off them."""
    x = torch.stack([torch.full((cols + 1,), 1.1), torch.full((cols + 1,), 0.37), normal(cols, cols + 1)]).to(kind).cuda()
    check_long(S, x[:, :cols])
    check_long(S, x[:, 1:])
    check_long(S, x[:, :cols], x[:, 1:].flip(0), (1 + 0.3 * normal(1, cols)).to(kind).cuda())


def test_norm_of_a_row_of_16_million(S):
    check_long(S, torch.full((1, 1 << 24), 1.7, device="cuda"))


def test_norm_of_long_rows_that_pass_32_bits(S):
    """The squares' sum past 3.4e38 gives a factor of 0, wherever in the row it passes; an infinity or a NaN in what is
    read beyond the held vectors is seen."""
    x = torch.ones(5, 70000, device="cuda")
    x[0, :4] = 1.5e19
    x[1, 60000:60004] = 1.5e19
    x[2, 69999] = INF
    x[3, 65000] = math.nan
    y, _ = S.add_rms_norm(x)
    codes, scale, _ = S.add_rms_norm_int8(x)
    assert (y[:2] == 0).all() and (scale[:2] == 0).all()
    assert (y[2, :-1] == 0).all() and torch.isnan(y[2, -1]) and torch.isnan(y[3]).all() and not torch.isfinite(scale[2:4]).any()
    assert ((y[4].double() - 1 / math.sqrt(1 + 1e-6)).abs() <= NORM + u).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cols", [1000, 16384, 16391, 40003])
def test_norm_in_place_at_every_length(S, kind, cols):
    """Outputs over inputs, in rows that registers hold and in longer ones, which are read again."""
    x, r, w = normal(1, 5, cols, kind=kind).cuda(), normal(2, 5, cols, kind=kind).cuda(), (1 + 0.2 * normal(3, cols)).to(kind).cuda()
    y, t = S.add_rms_norm(x, r, w)
    codes, scale, _ = S.add_rms_norm_int8(x, r, w)
    alone = S.add_rms_norm(x, None, w)[0]
    for out, total in (("x", "r"), ("r", "x"), ("x", None), (None, "r"), (None, "x"), ("r", None)):
        a, b = x.clone(), r.clone()
        at = {"x": a, "r": b, None: None}
        got, s = S.add_rms_norm(a, b, w, out=at[out], sum_out=at[total])
        assert torch.equal(got, y) and torch.equal(s, t), (out, total)
        if out is None:
            a, b = x.clone(), r.clone()
            at = {"x": a, "r": b}
            for p, q in zip(S.add_rms_norm_int8(a, b, w, sum_out=at[total]), (codes, scale, t)):
                assert torch.equal(p, q), total
    a = x.clone()
    assert torch.equal(S.add_rms_norm(a, None, w, out=a)[0], alone)
    a = x.clone()
    assert torch.equal(S.add_rms_norm(a, a, w, sum_out=a)[0], S.add_rms_norm(x, x, w)[0])


# ----------------------------------------- every way through the 4-bit product --
def check_product(S, rows, inner, outer, kind, bias=True):
    """Against the 64-bit product of the values that codes and scales stand for; sums as in test_gpu_step.py: inner / 64 + 2
    steps of 2^-23 of the terms' magnitudes, and the output's rounding."""
    g = torch.Generator(device="cuda").manual_seed(rows + inner + outer)
    x = torch.randn(rows, inner, generator=g, device="cuda").to(kind)
    x *= (1 + torch.arange(rows, device="cuda") % 5).to(kind)[:, None]      # rows' and channels' scales differ, so that a wrong one shows
    m = torch.randn(outer, inner, generator=g, device="cuda") * 2.0 ** (torch.arange(outer, device="cuda") % 7)[:, None]
    b = torch.randn(outer, generator=g, device="cuda") if bias else None
    w, ws = S.quantize_fp4(m)
    codes, scale = S.quantize_fp4(x)
    a, v = S.fp4_values(codes, scale, inner).double(), S.fp4_values(w, ws, inner).double()
    want, size = a @ v.T, a.abs() @ v.abs().T
    if bias:
        want, size = want + b.double(), size + b.double().abs()
    room = (inner / 64 + 2) * 2.0 ** -23 * size + 1e-37
    # 16-bit floating point ends at 65504, and rounds what is 65520 and more, half a step of 32 past it, to infinity: the
    # sums of 4100 terms deviate by up to 5 x 64 x 4100^1/2 = 20490, and some of 33000 of them pass that
    past = 65520.0 if kind == torch.float16 else INF
    for y in (S.fp4_linear(x, w, ws, b), S.fp4_matmul(codes, scale, w, ws, b, out_dtype=kind)):
        assert y.dtype == kind
        over = torch.isinf(y)
        assert (want.abs() + room)[over].ge(past).all() and torch.equal(y[over].sign().double(), want[over].sign())
        assert (want.abs() - room)[~over].lt(past).all()
        off = torch.where(over, 0.0, (y.double() - want).abs()) - U[kind] * want.abs() - room
        assert (off <= 0).all(), (off.amax(1).argmax().item(), off.amax(0).argmax().item())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,inner,outer", [
    # tiles of 192 channels, which begin in the middle of a tile of scales and span two: one a CTA, two, three; 3, 6 and 2 steps
    (200, 700, 9601), (1000, 1300, 7001), (1000, 300, 10501),
    # of 128: one, two and three a CTA, the last past the ring's five stages
    (777, 1001, 1531), (1000, 1300, 4701), (51100, 300, 127),
    # of 64: three
    (51100, 300, 50),
    # of 256, whose sums fit once: two and three, six steps in four stages
    (1000, 1300, 9301), (1000, 1300, 13901)])
def test_fp4_tiles_of_every_width(S, kind, rows, inner, outer):
    check_product(S, rows, inner, outer, kind)
    if kind is torch.bfloat16:
        check_product(S, rows, inner, outer, kind, bias=False)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [33, 47, 63, 64])
def test_fp4_tokens_as_columns(S, kind, rows):
    """33 to 64 tokens as the products' columns: a long inner dimension, shared by a cluster."""
    check_product(S, rows, 2049, 50, kind)
    check_product(S, rows, 4100, 1001, kind, bias=False)


# ----------------------------------------------------- vocabularies of every size --
def equal_rows(x):
    """Rows in which one step of a histogram has every token, and one of two values."""
    x[0] = 0.25
    x[1] = -7.0
    x[1, ::2] = -7.5
    return x


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,vocab", [(2, 262144), (2, 262145), (3, 524287), (3, 524288)])
def test_sample_of_the_widest_vocabularies(S, kind, rows, vocab):
    """Up to 2^18 tokens weights have 44 bits, above it 43."""
    x = equal_rows((normal(vocab, rows + 2, vocab) * 3).to(kind))
    for t, k, p, least in ((1.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.0), (1.1, 0, 0.95, 0.0), (0.9, 5000, 0.9, 0.0), (1.0, vocab - 1, 0.5, 0.01), (0.0, 0, 1.0, 0.0)):
        check_sample(S, x, uniform(vocab, rows + 2), t, k, p, least)


def test_sample_of_a_full_part_a_cta(S):
    """So many rows that each has one CTA, and as many tokens as it counts: 2^17, from rows on 32 bytes and off them; one
    more, and two CTAs share a row."""
    rows = 150
    for vocab, off in ((1 << 17, 0), (1 << 17, 3), ((1 << 17) + 1, 0), ((1 << 17) + 1, 5)):
        store = (normal(vocab + off, rows, vocab + 8) * 2).cuda()
        x = store.flatten()[off: off + rows * vocab].view(rows, vocab)
        equal_rows(x)
        u = uniform(off, rows)
        some = [0, 1, *range(2, rows, 7)]
        host = x[some].cpu().double().numpy()
        for args in ((1.0, 0, 0.9, 0.0), (1.0, 2000, 0.8, 0.0), (1.0, 0, 1.0, 0.0)):
            tokens, logp = S.sample(x, u.cuda(), *args)
            for i, r in enumerate(some):
                token, log = sample_definition(host[i], float(u[r]), args[0], args[1], float(np.float32(args[2])), args[3])
                assert int(tokens[r]) == token and abs(float(logp[r]) - log) <= 2.0 ** -24 * abs(log) + 2.0 ** -34, (r, args)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,vocab", [(2, 40000), (2, 1200), (160, 3000)])
def test_sample_of_fewer_weights_than_top_k(S, kind, rows, vocab):
    """No token is the k-th with any weight: the histogram that was made for top_k serves for top_p, counted once."""
    x = torch.full((rows, vocab), -INF)
    x[:, 5::7] = -torch.arange(len(range(5, vocab, 7))) % 61 * 0.1
    x[:, 1::7] = -3000.0
    x = x.to(kind)
    for k in (1100, vocab // 2, vocab - 1):
        for p in (0.3, 0.9, 0.999):
            check_sample(S, x, uniform(k, rows), 1.0, k, p, 0.0)


def test_sample_tails_below_a_step(S):
    """Weights are rounded to multiples of 2^-44 of the largest (2^-43 above 2^18 tokens), so n of them are off by up to n
    halves of that; the polynomial by 2^-43 of each.  Here all but one token have 0.44 of such a step, and count
    nothing: the largest error there is but for the last bits."""
    for vocab, bits in ((1 << 17, 44), (1 << 18, 44), (1 << 19, 43)):
        x = torch.full((1, vocab), float(np.float32(-(bits + 1.2) * math.log(2))))
        x[0, 9] = 0
        for rows in (1, 160):
            tokens, logp = S.sample(x.cuda().repeat(rows, 1), torch.full((rows,), 0.5).cuda())
            _, want = sample_definition(x[0].double().numpy(), 0.5, 1.0, 0, 1.0, 0.0)
            assert (tokens == 9).all() and ((logp.cpu().double() - want).abs() <= vocab * 2.0 ** -(bits + 1) + 2.0 ** -42).all()
            assert abs(want) > 0.8 * vocab * 2.0 ** -(bits + 1)


# --------------------------------------------------------------- the C ABI, step by step --
def test_steps_of_the_c_abi(S):
    """Lengths and pages advance from step to step as a C caller has them: held into a plan, kept out of it, the next held
    from free_pages; no page is in two places, none is lost."""
    from vdttfs._lib import check, lib
    rng = np.random.default_rng(3)
    seqs, width, page, count = 9, 5, 16, 30
    ints = lambda v, n=torch.int32: torch.tensor(np.asarray(v), dtype=n, device="cuda")  # noqa: E731
    ring, span, pages = ints(np.arange(count)), ints([0, count]), torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
    held, kept, starts = ints([0] * seqs), ints([0] * seqs), ints([0] * (seqs + 1))
    need = lib().vdt_plan_pages_scratch_bytes(seqs)
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()  # noqa: E731
    lengths = [0] * seqs
    for _ in range(60):
        new = [min(int(rng.integers(0, 25)) if n == 0 else 1, width * page - n) for n in lengths]
        total = sum(new)
        fresh, positions, slots = ints(new), ints([0] * (total + 1)), ints([0] * (total + 1), torch.int64)
        check(lib().vdt_plan_pages(p(ring), count, p(span), p(pages), width, p(held), p(fresh), seqs, page, total, p(kept), p(starts), p(positions), p(slots),
                                   p(span), p(scratch), need, stream), "vdt_plan_pages")
        lengths = [a + b for a, b in zip(lengths, new)]
        assert held.tolist() == [a - b for a, b in zip(lengths, new)] and kept.tolist() == lengths
        first, left = span.tolist()
        if left < 0:
            break
        table, order = pages.tolist(), ring.tolist()
        used = [n for row, many in zip(table, lengths) for n in row[: -(-many // page)]]
        assert sorted(used + [order[(first + i) % count] for i in range(left)]) == list(range(count))
        assert positions.tolist()[:total] == [a - b + i for a, b in zip(lengths, new) for i in range(b)]
        done = rng.random(seqs) < (0.6 if left < 12 else 0.1)
        done_t = ints(done, torch.uint8)
        check(lib().vdt_free_pages(p(ring), count, p(span), p(pages), width, p(kept), p(done_t), seqs, page, p(held), p(span), stream), "vdt_free_pages")
        lengths = [0 if d else n for d, n in zip(done, lengths)]
        assert held.tolist() == lengths
    else:
        return
    raise AssertionError("the pool ran out")


@pytest.mark.parametrize("k", [1, 31, 32, 33, 63, 65])
def test_code_rows_of_the_c_abi(S, k):
    """Rows of ceil(k / 2) bytes, as far apart as the next multiple of 16; nearer ones are refused."""
    from vdttfs._lib import lib
    n, x = 7, normal(k, 7, k).cuda()
    stride, stream = ((k + 1) // 2 + 15) // 16 * 16, torch.cuda.current_stream().cuda_stream
    codes = torch.full((n, stride), 0xab, dtype=torch.uint8, device="cuda")
    scale = torch.empty(lib().vdt_fp4_scale_bytes(n, k), dtype=torch.uint8, device="cuda")
    go = lambda s: lib().vdt_quantize_fp4(x.data_ptr(), 0, n, k, k, codes.data_ptr(), s, scale.data_ptr(), stream)  # noqa: E731
    assert go(stride) == 0 and (stride == 16 or go(stride - 16) == 1)
    want, _ = S.quantize_fp4(x)
    assert torch.equal(codes[:, : want.shape[1]], want)


# ------------------------------------------------------------ results of one call --
def results(S):
    x = normal(1, 40, 300, kind=torch.bfloat16).cuda()
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    pool, pages, held, new = S.PagePool.full(50), torch.full((3, 9), -1, dtype=torch.int32, device="cuda"), ints(0, 0, 0), ints(5, 100, 33)
    plan = S.plan_pages(pool, pages, held, new, 16, 140)
    none = S.plan_pages(pool, torch.full((3, 9), -1, dtype=torch.int32, device="cuda"), held, ints(0, 0, 0), 16, 0)
    return {"quantize_fp4": S.quantize_fp4(x), "add_rms_norm": S.add_rms_norm(x, x), "add_rms_norm_int8": S.add_rms_norm_int8(x, x), "plan_pages": plan,
            "plan_pages of nothing": none, "free_pages": S.free_pages(pool, pages, new, torch.tensor([True, False, True]).cuda(), 16),
            "sample": S.sample(normal(2, 7, 900).cuda(), uniform(1, 7).cuda())}


def test_results_have_storage_of_their_own(S):
    """A result that is kept holds no other one in memory, and one that is used again at another size writes over none."""
    for name, out in results(S).items():
        places = [t.untyped_storage().data_ptr() for t in out if t.numel()]
        assert len(set(places)) == len(places), name
        for i, t in enumerate(out):
            others = [o.clone() for o in out]
            t.resize_(0).resize_(4 * others[i].numel() + 500).fill_(77)
            for j, o in enumerate(out):
                assert i == j or torch.equal(o, others[j]), (name, i, j)
            t.resize_(others[i].shape).copy_(others[i])


def test_a_kept_result_holds_its_own_bytes(S):
    plan = S.plan_pages(S.PagePool.full(4000), torch.full((3, 900), -1, dtype=torch.int32, device="cuda"), *(torch.zeros(3, dtype=torch.int32, device="cuda"),) * 2, 16, 50000)
    for t, most in ((plan.kept, 12), (plan.starts, 16), (plan.span, 8), (plan.positions, 200000)):
        assert t.untyped_storage().nbytes() == most
    assert plan.slots.untyped_storage().nbytes() <= 400000 + 4096


# ------------------------------------------------------------- what a page's owner is --
def test_a_lacking_page_is_not_asked_for_again(S):
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    pool, pages, held = S.PagePool.full(3), torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), ints(0, 0)
    plan = S.plan_pages(pool, pages, held, ints(32, 32), 16, 64)
    assert pages.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1]] and plan.span.tolist() == [0, -1]
    back, span = S.free_pages((pool.ring, plan.span), pages, plan.kept, torch.tensor([True, False]).cuda(), 16)
    assert back.tolist() == [0, 32] and span.tolist() == [0, 2]
    plan = S.plan_pages((pool.ring, span), pages, back, ints(0, 1), 16, 1)
    # sequence 1 goes on in its third page; tokens 16 to 31 stay without one
    assert pages.tolist()[1] == [2, -1, 0, -1] and plan.slots.tolist() == [0] and plan.span.tolist() == [1, 1]
    back, span = S.free_pages((pool.ring, plan.span), pages, plan.kept, torch.tensor([False, True]).cuda(), 16)
    assert back.tolist() == [0, 0] and span.tolist() == [1, 3] and sorted(pool.ring.tolist()) == [0, 1, 2]


def test_a_page_of_two_rows_is_taken_out_of_one(S):
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    pages, done = ints(4, 7, 4, 9).view(2, 2), torch.tensor([True, True]).cuda()
    ring, span = ints(-1, -1, -1, -1, -1), ints(0, 0)
    _, after = S.free_pages((ring, span), pages, ints(32, 32), done, 16)
    assert ring.tolist() == [4, 7, 4, 9, -1] and after.tolist() == [0, 4]
    pages[1, 0] = -1
    ring.fill_(-1)
    _, after = S.free_pages((ring, span), pages, ints(32, 32), done, 16)
    assert ring.tolist() == [4, 7, 9, -1, -1] and after.tolist() == [0, 3]


def test_a_plan_into_buffers_of_the_callers_own(S):
    """All results given, some of them, none: the same plan, and the given tensors are what comes back."""
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for seqs, total in ((3, 41), (3, 0), (1500, 1503)):
        new = torch.full((seqs,), total // seqs, dtype=torch.int32, device="cuda")
        held = torch.arange(seqs, dtype=torch.int32, device="cuda") % 40

        def go(out):
            return S.plan_pages(S.PagePool.full(9000), torch.full((seqs, 5), -1, dtype=torch.int32, device="cuda"), held, new, 16, total, out)

        want = go(None)
        room = [torch.empty_like(t) for t in want]
        for given in (range(5), (3,), (0, 2, 4), (1,)):
            out = S.PagePlan._make(room[i] if i in given else None for i in range(5))
            got = go(out)
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(got[i] is room[i] for i in given), (seqs, total, given)
    with pytest.raises(ValueError):
        S.plan_pages(S.PagePool.full(4), torch.zeros(2, 3, dtype=torch.int32, device="cuda"), ints(0, 0), ints(1, 1), 16, 2,
                     S.PagePlan(None, None, None, torch.empty(2, dtype=torch.int32, device="cuda"), None))

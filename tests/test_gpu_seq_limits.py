"""The sequence operators where their bounds lie: values of very different size in one cache, streams of the caller's own, results in place, lengths beyond the bounds.

Tolerances are derived as in test_gpu_seq.py; each test states what it adds.
"""
import math

import pytest
import torch

from test_gpu_seq import S, U, ints, make_cache, make_table, normal, sums  # noqa: F401

pytestmark = pytest.mark.gpu


# -------------------------------------------------------------- attention --
def cached(cache, row, n, page):
    """A sequence's keys, values and value scales in 64 bits: [heads, n, dim] twice, [heads, n]."""
    at = torch.tensor(row[: -(-n // page)], device="cuda")
    scale = [c[at].double().repeat_interleave(page, 0).T[:, :n] for c in cache[2:]]
    k = cache[0][at].double().transpose(0, 1).flatten(1, 2)[:, :n] * scale[0][..., None]
    v = cache[1][at].double().permute(1, 0, 3, 2).flatten(1, 2)[:, :n] * scale[1][..., None]
    return k, v, scale[1]


def strict(S, q, cache, table, kept, new, causal, scale, page):
    """Attention against 64 bits.  A weight (the probability with its page's value scale) is off by 2^-11 of itself or by
    2^-25 of the row's largest, and multiplies a code of up to 127; its exponent, of numbers up to 256, is rounded three
    times at 2^-17: 2^-15 of the weight; the rest is the scores' error and the output's rounding."""
    starts = sums(new)
    heads, dim = q.shape[1:]
    group = heads // cache[0].shape[1]
    out = S.cache_attention(q, cache, ints(table), ints(kept), ints(starts), max(new), max(kept), causal=causal, scale=scale).double()
    for b, n in enumerate(kept):
        k, v, vs = (x.repeat_interleave(group, 0) for x in cached(cache, table[b], n, page))
        x = q[starts[b]: starts[b + 1]].double().transpose(0, 1)
        s = x @ k.transpose(1, 2) * scale
        last = torch.arange(n - new[b] + 1, n + 1, device="cuda") if causal else torch.full((new[b],), n, device="cuda")
        s = s.masked_fill(torch.arange(n, device="cuda")[None] >= last[:, None], -math.inf)
        p = torch.softmax(s, -1)
        want = p @ v
        size = (x.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * abs(scale)
        d = (dim + 16) * 2.0 ** -23 * size + abs(scale) * 2.0 ** -24 * x.abs().amax(-1, keepdim=True) * k.abs().sum(2).amax(1)[:, None, None]
        tol = U[q.dtype] * want.abs() + (2.0 ** -11 + 2.0 ** -15 + 2 * d) * (p @ v.abs()) \
            + n * 127 * 2.0 ** -25 * (p * vs[:, None]).amax(-1, keepdim=True) + (2.0 ** -25 if q.dtype == torch.float16 else 0)
        off = (out[starts[b]: starts[b + 1]].transpose(0, 1) - want).abs()
        assert (off <= tol).all(), (b, float((off / tol).max()))


@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("power", [14, 20, 28])
@pytest.mark.parametrize("new,dim", [(5, 64), (16, 128), (40, 64), (150, 64), (150, 128), (300, 128), (40, 256)])
def test_attention_does_not_change_with_values_that_a_row_does_not_see(S, new, dim, power, page):
    """The last page's values grow by 2^power: the causal rows before it give the bits they gave."""
    kept = 256
    table, pages = make_table([kept], page)
    cache = make_cache(S, pages, 1, dim, page)
    q = normal(1, new, 1, dim, kind=torch.bfloat16).cuda()
    in_last = min(page, new // 2)                         # queries that see the last page
    args = (ints(table), ints([kept - page + in_last]), ints([0, new]), new, kept)
    blind = new - in_last
    before = S.cache_attention(q, cache, *args)
    cache.v_scale[table[0][-1]] *= 2.0 ** power
    after = S.cache_attention(q, cache, *args)
    assert torch.equal(after[:blind], before[:blind])
    assert not torch.equal(after[blind:], before[blind:])


@pytest.mark.parametrize("new", [1, 12, 40, 200])
@pytest.mark.parametrize("power", [10, 16, 24, 30])
def test_attention_keeps_its_bits_beside_large_values_of_no_weight(S, new, power):
    """One page has values 2^power times the others' and keys that give it next to no probability, first or last."""
    dim, page, kept = 64, 16, 240
    for where in (0, 7, 14):
        table, pages = make_table([kept], page)
        cache = make_cache(S, pages, 1, dim, page)
        q = normal(2, new, 2, dim).abs().add(0.5).to(torch.bfloat16).cuda()
        at = table[0][where]
        cache.k[at] = -100                                # against every query: scores some 40 to 120 below the others'
        cache.k_scale[at] = 1.0 / 32
        cache.v_scale[at] *= 2.0 ** power
        strict(S, q, cache, table, [kept], [new], False, 0.25, page)


@pytest.mark.parametrize("new", [1, 16, 33, 150])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (256, 64)])
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
def test_attention_value_scales_of_every_size(S, new, dim, page, kind):
    """Value scales from 2^-20 to 2^20 (f16: of their usual size and below), in every order, pages of zeros among them."""
    kept = [400, 333]
    table, pages = make_table(kept, page)
    for seed in range(3):
        cache = make_cache(S, pages, 2, dim, page, seed)
        g = torch.Generator().manual_seed(seed)
        most = 0 if kind == torch.float16 else 20
        cache.v_scale.mul_(2.0 ** (torch.rand(cache.v_scale.shape, generator=g) * (most + 20) - 20).cuda())
        zero = torch.randint(0, pages, (2,), generator=g).cuda()
        cache.v_scale[zero] = 0
        q = normal(seed, 2 * new, 4, dim, kind=kind).cuda()
        strict(S, q, cache, table, kept, [new, new], bool(seed % 2), 0.3 / math.sqrt(dim), page)


@pytest.mark.parametrize("new", [1, 150])
def test_attention_over_values_that_are_all_zero_then_not(S, new):
    """Pages of zeros with the largest scores: their weights count in the sum, and the values after them are whole."""
    dim, page, kept = 64, 16, 256
    table, pages = make_table([kept], page)
    cache = make_cache(S, pages, 1, dim, page)
    for j in range(4):
        cache.v_scale[table[0][j]] = 0
        cache.k[table[0][j]] = 60
    q = normal(3, new, 1, dim).abs().to(torch.float16).cuda()
    for power in (0, -30):
        cache.v_scale[table[0][9]] = 2.0 ** power
        strict(S, q, cache, table, [kept], [new], False, 0.02, page)


# ---------------------------------------------------------------- streams --
def calls(S):
    """Every call that copies or allocates."""
    x = normal(1, 96, 64, kind=torch.bfloat16).cuda()
    w, ws = S.quantize_rows(normal(2, 48, 96).cuda())
    codes, scale = S.quantize_rows(x.T)
    table, pages = make_table([200], 32)
    cache = make_cache(S, pages, 2, 64, 32)
    q = normal(3, 150, 4, 64, kind=torch.bfloat16).cuda()
    rope, at = S.rope_table(300, 64), torch.arange(150, dtype=torch.int32, device="cuda")
    pt, kept = ints(table), ints([200])
    packed, new = ints([0, 200]), ints([0, 150])
    return {
        "quantize_rows": lambda s: S.quantize_rows(x.T, stream=s),
        "quantize_rows of few": lambda s: S.quantize_rows(x[:, :3].T, stream=s),
        "int8_linear": lambda s: S.int8_linear(x.T, w, ws, stream=s),
        "int8_linear of few": lambda s: S.int8_linear(x[:, :3].T, w, ws, stream=s),
        "int8_matmul": lambda s: S.int8_matmul(codes, scale, w, ws, stream=s),
        "rope_table": lambda s: S.rope_table(300, 64, stream=s),
        "qk_norm_rope": lambda s: S.qk_norm_rope(q, q[:, :2], None, None, at, rope, stream=s),
        "cache_load": lambda s: S.cache_load(cache, pt, kept, packed, 200, 200, stream=s),
        "cache_attention": lambda s: S.cache_attention(q, cache, pt, kept, new, 150, 200, stream=s),
        "cache_attention of one": lambda s: S.cache_attention(q[:1], cache, pt, kept, ints([0, 1]), 1, 3000, stream=s),
    }


def flat(result):
    return [t.clone() for t in (result if isinstance(result, tuple) else (result,))]


def test_calls_on_a_stream_of_their_own_with_work_queued_on_the_current_one(S):
    """The inputs are there; the current stream is busy for some 20 ms, and behind that writes blocks that were let go:
    nothing of a call on another stream may wait there or lie in those blocks."""
    side = torch.cuda.Stream()
    for name, call in calls(S).items():
        want = flat(call(None))
        torch.cuda.synchronize()
        for handle in (side.cuda_stream, 0):
            current = torch.cuda.Stream() if handle == 0 else torch.cuda.current_stream()
            with torch.cuda.stream(current):
                torch.cuda._sleep(40_000_000)
                for n in (1 << 8, 1 << 12, 1 << 14, 1 << 16, 1 << 18, 1 << 20):
                    for _ in range(4):
                        torch.full((n,), -7, dtype=torch.int8, device="cuda")     # blocks whose last kernel is still queued
                got = call(handle)
            torch.cuda.synchronize()
            for g, t in zip(flat(got), want):
                assert torch.equal(g, t), (name, handle)


def test_a_result_of_another_stream_may_be_used_and_let_go_on_the_current_one(S):
    """Its block is not given out again to that stream while the current one reads it."""
    side = torch.cuda.Stream()
    w, ws = S.quantize_rows(normal(2, 700, 512).cuda())
    x = normal(1, 333, 512, kind=torch.bfloat16).cuda()
    want = S.int8_linear(x, w, ws)
    torch.cuda.synchronize()
    y = S.int8_linear(x, w, ws, stream=side.cuda_stream)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda._sleep(40_000_000)
    kept = y.clone()                                      # queued behind the sleep
    del y
    for _ in range(4):
        S.int8_linear(-x, w, ws, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(kept, want)


# ---------------------------------------------------------------- in place --
@pytest.mark.parametrize("kind", list(U))
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 12, 40, 200])
def test_linear_into_its_own_rows(S, kind, rows):
    """A few rows are read by every CTA of the product, whose outputs must not stand there yet."""
    for n in (64, 1024, 1000):
        x = normal(rows, rows, n, kind=kind).cuda()
        w, ws = S.quantize_rows(normal(1, n, n).cuda())
        want = S.int8_linear(x, w, ws)
        for _ in range(5):
            y = x.clone()
            assert S.int8_linear(y, w, ws, out=y) is not None and torch.equal(y, want)
        # an output that begins inside the rows, of the type of twice or half the size
        other = torch.float32 if kind != torch.float32 else torch.bfloat16
        room = torch.zeros(rows * n * 4 + 4096, dtype=torch.uint8, device="cuda")
        y = room[: rows * n * x.element_size()].view(kind).view(rows, n)
        y.copy_(x)
        out = room[2048: 2048 + rows * n * other.itemsize].view(other).view(rows, n)
        S.int8_linear(y, w, ws, out=out)
        assert torch.equal(out, S.int8_linear(x, w, ws, out_dtype=other))


# ------------------------------------------------- lengths beyond the bounds --
@pytest.mark.parametrize("new", [2, 40, 300])
@pytest.mark.parametrize("kept", [100, 3000])
def test_attention_of_runs_beyond_the_bounds_gives_nan(S, new, kept):
    """A run of more queries than was said, or one that ends outside the rows: NaN there, the other sequences as they are."""
    table, pages = make_table([kept] * 3, 64)
    cache = make_cache(S, pages, 2, 64, 64)
    q = normal(1, 3 * new, 4, 64, kind=torch.bfloat16).cuda()
    args = (ints(table), ints([kept] * 3))
    good = S.cache_attention(q, cache, *args, ints([0, new, 2 * new, 3 * new]), new, kept)
    for starts, most, broken in (([0, new, 2 * new + 1, 3 * new], new, slice(new, 2 * new + 1)),
                                 ([0, new - 1, 2 * new, 3 * new], new, slice(new - 1, 2 * new)),
                                 ([0, new, 2 * new, 3 * new + 1], new + 1, slice(2 * new, 3 * new)),
                                 ([-1, new, 2 * new, 3 * new], new + 1, slice(0, new))):
        out = torch.full_like(q, 7)
        S.cache_attention(q, cache, *args, ints(starts), most, kept, out=out)
        assert torch.isnan(out[broken]).all()
        whole = torch.ones(3 * new, dtype=torch.bool)
        whole[broken] = False
        assert torch.isfinite(out[whole.cuda()]).all()
        for b in range(3):                                # sequences of the lengths that `good` has
            if starts[b] == b * new and starts[b + 1] == (b + 1) * new and most == new:
                assert torch.equal(out[starts[b]: starts[b + 1]], good[starts[b]: starts[b + 1]])


def test_attention_leaves_rows_of_no_sequence(S):
    for new in (3, 50):
        table, pages = make_table([90], 16)
        cache = make_cache(S, pages, 1, 64, 16)
        q = normal(1, new + 4, 2, 64, kind=torch.float16).cuda()
        out = torch.full_like(q, 7)
        S.cache_attention(q, cache, ints(table), ints([90]), ints([1, new + 1]), new, 90, out=out)
        assert (out[0] == 7).all() and (out[new + 1:] == 7).all() and not (out[1: new + 1] == 7).all()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("kind,code", [(torch.float32, 0), (torch.float16, 1), (torch.bfloat16, 2)])
def test_load_of_lengths_beyond_the_bounds_gives_nan(S, kind, code, page):
    """More tokens than the run has rows or than was said, or a run that ends outside: NaN there, other sequences whole."""
    import ctypes as C
    from vdttfs import _lib
    heads, dim, n = 2, 64, 70
    table, pages = make_table([n] * 3, page)
    cache = make_cache(S, pages, heads, dim, page)
    pt = ints(table)
    desc = _lib.Cache8Desc(*(t.data_ptr() for t in cache), pages, page, heads, dim)
    good = S.cache_load(cache, pt, ints([n] * 3), ints(sums([n] * 3)), 3 * n, n, kind)

    def load(kept, starts, total, most):
        k, v = (torch.full((total, heads, dim), 7, dtype=kind, device="cuda") for _ in range(2))
        lengths, rows = ints(kept), ints(starts)
        assert _lib.lib().vdt_cache_load(C.byref(desc), pt.data_ptr(), pt.shape[1], lengths.data_ptr(), rows.data_ptr(), 3, total, most, code,
                                         k.data_ptr(), v.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        return k, v

    for out, want in zip(load([n] * 3, [0, n, 2 * n, 3 * n], 3 * n, n), good):
        assert torch.equal(out, want)
    for kept, starts, most, broken in (([n, n, n], [0, n, 2 * n - 1, 3 * n - 1], n, (1,)), ([n, n, n], [0, n, 2 * n, 3 * n], n - 1, (0, 1, 2)),
                                       ([5, n, 5], [0, n, 2 * n, 3 * n], 20, (1,)), ([n, n, n], [0, n, 2 * n, 3 * n + 1], n, (2,)),
                                       ([n, n, n], [-1, n, 2 * n, 3 * n], n, (0,))):
        for out, want in zip(load(kept, starts, 3 * n, most), good):
            for b in range(3):
                rows = out[max(starts[b], 0): starts[b + 1]]
                if b in broken:
                    assert torch.isnan(rows).all()
                else:
                    assert torch.equal(rows[: kept[b]], want[b * n: b * n + kept[b]]) and (rows[kept[b]:] == 7).all()


# ------------------------------------------------------------------- sizes --
def test_sizes_beyond_32_bits_are_refused(S):
    """2^32 + n would otherwise be taken for n."""
    long = (1 << 32) + 64
    a, w = (torch.empty(1, long, dtype=torch.int8, device="cuda") for _ in range(2))
    one = torch.ones(1, device="cuda")
    with pytest.raises(ValueError):
        S.int8_matmul(a, one, w, one)
    with pytest.raises(ValueError):
        S.int8_linear(a.view(torch.float16)[:, : long // 2].repeat(1, 2), w, one)
    del a, w
    x = torch.zeros(1, 1, 64, dtype=torch.float16, device="cuda")
    many = x.expand(1, (1 << 32) + 8, 64)                 # heads that share their memory
    with pytest.raises(ValueError):
        S.qk_norm_rope(many, None, None, None, None, None, out=(many, None))
    cache = make_cache(S, 2, 2, 64, 16)
    with pytest.raises(ValueError):
        S.cache_attention(many, cache, ints([[0]]), ints([4]), ints([0, 1]), 1, 16, out=many)


# --------------------------------------------------------------- refusals --
def test_a_table_without_positions_is_refused(S):
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="positions"):
        S.qk_norm_rope(q, None, None, None, None, S.rope_table(8, 64))


def test_flags_that_are_neither_true_nor_false_are_refused(S):
    class Neither:
        def __bool__(self):
            raise RuntimeError("neither")

    cache = make_cache(S, 2, 2, 64, 16)
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(TypeError, match="interleaved"):
        S.qk_norm_rope(q, None, None, None, None, None, interleaved=Neither())
    with pytest.raises(TypeError, match="causal"):
        S.cache_attention(q, cache, ints([[0]]), ints([4]), ints([0, 2]), 2, 16, causal=Neither())


SHIM = r"""
#define _GNU_SOURCE
#include <dlfcn.h>
#include <string.h>
static int fail;
void shim_fail(int n) { fail = n; }
static void* real(const char* name) { return dlsym(dlopen("libcudart.so.12", RTLD_LAZY | RTLD_NOLOAD), name); }
int cudaFuncGetAttributes(void* a, const void* f) {
    if (fail) return --fail, 999;
    return ((int (*)(void*, const void*))real("cudaFuncGetAttributes"))(a, f);
}
int cudaGetDriverEntryPointByVersion(const char* name, void** f, unsigned v, unsigned long long flags, int* q) {
    if (fail && !strcmp(name, "cuTensorMapEncodeTiled")) return --fail, 999;
    return ((int (*)(const char*, void**, unsigned, unsigned long long, int*))real("cudaGetDriverEntryPointByVersion"))(name, f, v, flags, q);
}
"""

FIRST_FAILS = """
import ctypes, sys
sys.path[:0] = [{tests!r}, {package!r}]
import torch
from vdttfs import seq as S, _lib
from test_gpu_seq import ints, make_cache, make_table, normal
shim = ctypes.CDLL({shim!r})
x, (w, ws) = normal(1, 40, 64).cuda(), S.quantize_rows(normal(2, 48, 64).cuda())
table, pages = make_table([300], 16)
cache = make_cache(S, pages, 1, 64, 16)
q = normal(3, 300, 1, 64, kind=torch.float16).cuda()
for call in (lambda: S.int8_linear(x, w, ws), lambda: S.cache_attention(q, cache, ints(table), ints([300]), ints([0, 300]), 300, 300)):
    shim.shim_fail(1)
    try:
        call()
        sys.exit("the first call was taken")
    except _lib.VdtError:
        pass
    assert torch.isfinite(call()).all()
torch.cuda.synchronize()
"""


def test_a_call_that_fails_in_the_runtime_is_not_kept(dev, tmp_path):
    """The runtime's answers that the launches go by are asked for again after a failure (made by a shim on the host)."""
    import os
    import shutil
    import subprocess
    import sys

    from conftest import ROOT
    cc = shutil.which("cc") or shutil.which("gcc")
    if not cc:
        pytest.skip("no C compiler")
    (tmp_path / "shim.c").write_text(SHIM)
    shim = str(tmp_path / "shim.so")
    subprocess.run([cc, "-shared", "-fPIC", "-o", shim, str(tmp_path / "shim.c"), "-ldl"], check=True)
    code = FIRST_FAILS.format(tests=os.path.join(ROOT, "tests"), package=os.path.join(ROOT, "vd-ttfs_b200"), shim=shim)
    done = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, LD_PRELOAD=shim), capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("new,kept", [(1, 90), (1, 9000), (12, 700), (40, 5000), (300, 900)])
def test_attention_into_its_own_queries(S, new, kept):
    table, pages = make_table([kept, kept], 64)
    cache = make_cache(S, pages, 2, 64, 64)
    q = normal(1, 2 * new, 4, 64, kind=torch.bfloat16).cuda()
    args = (cache, ints(table), ints([kept] * 2), ints([0, new, 2 * new]), new, kept)
    want = S.cache_attention(q, *args)
    for _ in range(3):
        x = q.clone()
        S.cache_attention(x, *args, out=x)
        assert torch.equal(x, want)

"""CPU: what the sequence operators refuse, before any device is touched."""
import ctypes as C

import pytest

from vdttfs import _lib

INVALID, UNSUPPORTED, CAPACITY = 1, 5, 6
P = 1 << 20            # a pointer that is never followed: every call here is refused first


def call(name, *args):
    return getattr(_lib.lib(), name)(*args)


def test_quantize_rows_refusals():
    ok = dict(x=P, type=0, rows=4, cols=8, stride=8, codes=P, cstride=16, scale=P)

    def go(**over):
        a = dict(ok, **over)
        return call("vdt_quantize_rows", a["x"], a["type"], a["rows"], a["cols"], a["stride"], a["codes"], a["cstride"], a["scale"], None)

    for over in (dict(x=None), dict(codes=None), dict(scale=None), dict(type=3), dict(type=-1), dict(rows=-1), dict(cols=0),
                 dict(stride=7), dict(cstride=7), dict(x=P + 2), dict(rows=1 << 30)):
        assert go(**over) == INVALID, over
    assert go(rows=0) == 0


def test_product_refusals():
    ok = dict(a=P, astride=32, asc=P, w=P, wstride=32, wsc=P, bias=None, rows=3, cols=5, inner=20, type=2, out=P, ostride=5)

    def go(**over):
        a = dict(ok, **over)
        return call("vdt_int8_matmul", a["a"], a["astride"], a["asc"], a["w"], a["wstride"], a["wsc"], a["bias"], a["rows"],
                    a["cols"], a["inner"], a["type"], a["out"], a["ostride"], None)

    for over in (dict(a=None), dict(asc=None), dict(w=None), dict(wsc=None), dict(out=None), dict(astride=20), dict(wstride=24),
                 dict(astride=16), dict(a=P + 8), dict(w=P + 4), dict(type=9), dict(rows=-1), dict(cols=0), dict(inner=0), dict(ostride=4),
                 dict(out=P + 1)):
        assert go(**over) == INVALID, over
    assert go(inner=131073, astride=1 << 18, wstride=1 << 18) == UNSUPPORTED
    assert go(rows=0) == 0


def test_linear_refusals():
    need = call("vdt_int8_linear_scratch_bytes", 3, 20)
    assert need >= 3 * 32 + 3 * 4 and call("vdt_int8_linear_scratch_bytes", 0, 20) == 0
    ok = dict(x=P, type=1, xstride=20, rows=3, scratch=P, size=need)

    def go(**over):
        a = dict(ok, **over)
        return call("vdt_int8_linear", a["x"], a["type"], a["xstride"], P, 32, P, None, a["rows"], 5, 20, 1, P, 5, a["scratch"], a["size"], None)

    for over in (dict(x=None), dict(type=7), dict(xstride=19), dict(scratch=None), dict(scratch=P + 16), dict(x=P + 1)):
        assert go(**over) == INVALID, over
    assert go(size=need - 1) == CAPACITY
    assert go(rows=0) == 0


def test_rope_refusals():
    ok = dict(q=P, k=P, at=P, table=P, n=10, rot=32, layout=0, norm=1, eps=1e-6, tokens=4, heads=2, kv=1, dim=64, type=2, qo=P, ko=P)

    def go(**over):
        a = dict(ok, **over)
        return call("vdt_qk_norm_rope", a["q"], 128, 64, a["k"], 64, 64, None, None, a["at"], a["table"], a["n"], a["rot"], a["layout"],
                    a["norm"], a["eps"], a["tokens"], a["heads"], a["kv"], a["dim"], a["type"], a["qo"], 128, 64, a["ko"], 64, 64, None)

    for over in (dict(q=None), dict(k=None), dict(qo=None), dict(ko=None), dict(at=None), dict(table=None), dict(n=0), dict(rot=31),
                 dict(rot=66), dict(rot=-2), dict(layout=2), dict(norm=3), dict(eps=-1.0), dict(tokens=-1), dict(heads=-1), dict(heads=2000),
                 dict(dim=0), dict(dim=10000), dict(type=4), dict(q=P + 1)):
        assert go(**over) == INVALID, over
    assert go(tokens=0) == 0 and go(heads=0, kv=0) == 0


def test_rope_table_refusals():
    ok = dict(n=8, rot=16, base=1e4, scaling=0, factor=1.0, trained=0, fast=32.0, slow=1.0, table=P)

    def go(**over):
        a = dict(ok, **over)
        return call("vdt_rope_table", a["n"], a["rot"], a["base"], a["scaling"], a["factor"], a["trained"], a["fast"], a["slow"], a["table"], None)

    for over in (dict(n=-1), dict(rot=0), dict(rot=15), dict(base=1.0), dict(base=float("inf")), dict(scaling=4), dict(scaling=1, factor=0.5),
                 dict(scaling=2, rot=2, factor=2.0), dict(scaling=3, factor=2.0), dict(scaling=3, factor=2.0, trained=100, fast=1.0),
                 dict(table=None), dict(table=P + 2)):
        assert go(**over) == INVALID, over
    assert go(n=0) == 0


def desc(**over):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, pages=4, page=16, heads=2, dim=64)
    d.update(over)
    return C.byref(_lib.Cache8Desc(*d.values()))


BAD_CACHE = [(dict(k=None), INVALID), (dict(v_scale=None), INVALID), (dict(pages=0), INVALID), (dict(heads=0), INVALID), (dict(k=P + 8), INVALID),
             (dict(page=48), UNSUPPORTED), (dict(page=128), UNSUPPORTED), (dict(dim=80), UNSUPPORTED), (dict(dim=512), UNSUPPORTED)]
BAD_ROWS = [dict(seqs=-1), dict(width=-1), dict(total=-1), dict(most=-1), dict(most=6), dict(table=None), dict(held=None), dict(starts=None),
            dict(total=1 << 30)]


def rows(over):
    d = dict(table=P, width=3, held=P, starts=P, seqs=2, total=5, most=3)
    d.update(over)
    return d


def append(cache, k=P, v=P, type=2, **over):
    r = rows(over)
    return call("vdt_cache_append", cache, k, 128, 64, v, 128, 64, type, r["table"], r["width"], r["held"], r["starts"], r["seqs"], r["total"], r["most"], None)


def load(cache, k=P, v=P, type=2, **over):
    r = rows(over)
    return call("vdt_cache_load", cache, r["table"], r["width"], r["held"], r["starts"], r["seqs"], r["total"], r["most"], type, k, v, None)


def attend(cache, q=P, out=P, type=2, heads=4, kept=100, scale=0.1, scratch=P, size=1 << 40, **over):
    r = rows(over)
    return call("vdt_cache_attention", cache, q, 256, 64, heads, type, r["table"], r["width"], r["held"], r["starts"], r["seqs"], r["total"],
                r["most"], kept, 1, scale, out, 256, 64, scratch, size, None)


@pytest.mark.parametrize("go", [append, load, attend])
def test_cache_refusals(go):
    assert go(None) == INVALID
    for over, status in BAD_CACHE:
        assert go(desc(**over)) == status, over
    for over in BAD_ROWS:
        assert go(desc(), **over) == INVALID, over
    assert go(desc(), seqs=70000) == UNSUPPORTED
    assert go(desc(), type=5) == INVALID
    assert go(desc(), total=0, most=0) == 0 and go(desc(), seqs=0) == 0
    first = {append: "k", load: "k", attend: "q"}[go]
    assert go(desc(), **{first: None}) == INVALID
    assert go(desc(), **{first: P + 1}) == INVALID


def test_attention_refusals():
    assert attend(desc(), type=0) == UNSUPPORTED
    for over in (dict(heads=3), dict(heads=0), dict(heads=4096), dict(kept=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(out=None),
                 dict(scratch=P + 4)):
        assert attend(desc(), **over) == INVALID, over
    need = call("vdt_cache_attention_scratch_bytes", 1, 4, 2, 64, 1, 1, 100000)
    assert need > 0
    assert attend(desc(), seqs=1, total=1, most=1, kept=100000, size=need - 1) == CAPACITY
    assert call("vdt_cache_attention_scratch_bytes", 1, 3, 2, 64, 1, 1, 100000) == 0
    assert call("vdt_cache_attention_scratch_bytes", 0, 4, 2, 64, 1, 1, 100000) == 0

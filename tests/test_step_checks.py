"""CPU: what the step operators refuse, before any device is touched."""
import math

from test_seq_checks import CAPACITY, INVALID, P, UNSUPPORTED, call


def refusals(go, invalid):
    for over in invalid:
        assert go(**over) == INVALID, over


def test_quantize_fp4_refusals():
    ok = dict(x=P, type=0, rows=4, cols=9, stride=9, codes=P, cstride=16, scale=P)

    def go(**over):
        a = dict(ok, **over)
        return call("vdt_quantize_fp4", a["x"], a["type"], a["rows"], a["cols"], a["stride"], a["codes"], a["cstride"], a["scale"], None)

    refusals(go, (dict(x=None), dict(codes=None), dict(scale=None), dict(type=3), dict(type=-1), dict(rows=-1), dict(cols=0), dict(stride=8),
                  dict(cstride=8), dict(cstride=24), dict(cols=40, stride=40), dict(x=P + 2), dict(codes=P + 8), dict(scale=P + 4), dict(rows=1 << 30)))
    assert go(cols=(1 << 30) + 1, stride=1 << 31, cstride=1 << 30) == UNSUPPORTED
    assert go(rows=0) == 0


def test_fp4_values_refusals():
    ok = dict(codes=P, cstride=16, scale=P, rows=3, cols=20, type=2, out=P, stride=20)

    def go(**over):
        a = dict(ok, **over)
        return call("vdt_fp4_values", a["codes"], a["cstride"], a["scale"], a["rows"], a["cols"], a["type"], a["out"], a["stride"], None)

    refusals(go, (dict(codes=None), dict(scale=None), dict(out=None), dict(cstride=9), dict(cols=0), dict(rows=-1), dict(type=5), dict(stride=19),
                  dict(out=P + 1), dict(codes=P + 1), dict(scale=P + 1)))
    assert go(rows=0) == 0


def test_fp4_product_refusals():
    ok = dict(a=P, astride=32, asc=P, w=P, wstride=32, wsc=P, bias=None, rows=3, cols=5, inner=40, type=2, out=P, ostride=5)

    def go(**over):
        a = dict(ok, **over)
        return call("vdt_fp4_matmul", a["a"], a["astride"], a["asc"], a["w"], a["wstride"], a["wsc"], a["bias"], a["rows"], a["cols"], a["inner"],
                    a["type"], a["out"], a["ostride"], None)

    refusals(go, (dict(a=None), dict(asc=None), dict(w=None), dict(wsc=None), dict(out=None), dict(astride=16), dict(wstride=40), dict(astride=24),
                  dict(a=P + 8), dict(w=P + 4), dict(asc=P + 8), dict(wsc=P + 8), dict(type=9), dict(rows=-1), dict(cols=0), dict(inner=0),
                  dict(ostride=4), dict(out=P + 1), dict(bias=P + 2)))
    assert go(cols=1 << 30, ostride=1 << 30) == UNSUPPORTED
    assert go(rows=0) == 0


def test_fp4_linear_refusals():
    need = call("vdt_fp4_linear_scratch_bytes", 3, 40)
    assert need >= 3 * 32 + 1024 and call("vdt_fp4_linear_scratch_bytes", 0, 40) == 0
    assert call("vdt_fp4_scale_bytes", 129, 257) == 2 * 4 * 512 and call("vdt_fp4_scale_bytes", 0, 5) == 0
    ok = dict(x=P, type=1, xstride=40, rows=3, scratch=P, size=need)

    def go(**over):
        a = dict(ok, **over)
        return call("vdt_fp4_linear", a["x"], a["type"], a["xstride"], P, 32, P, None, a["rows"], 5, 40, 1, P, 5, a["scratch"], a["size"], None)

    refusals(go, (dict(x=None), dict(type=7), dict(xstride=39), dict(scratch=None), dict(scratch=P + 16), dict(x=P + 1)))
    assert go(size=need - 1) == CAPACITY
    assert go(rows=0) == 0


def test_norm_refusals():
    ok = dict(x=P, xs=20, r=P, rs=20, w=P, rows=3, cols=20, eps=1e-6, type=2, sum=P, ss=20)

    def values(out=P, stride=20, **over):
        a = dict(ok, **over)
        return call("vdt_add_rms_norm", a["x"], a["xs"], a["r"], a["rs"], a["w"], a["rows"], a["cols"], a["eps"], a["type"], a["sum"], a["ss"], out, stride, None)

    def codes(out=P, stride=20, scale=P, **over):
        a = dict(ok, **over)
        return call("vdt_add_rms_norm_int8", a["x"], a["xs"], a["r"], a["rs"], a["w"], a["rows"], a["cols"], a["eps"], a["type"], a["sum"], a["ss"], out,
                    stride, scale, None)

    for go in (values, codes):
        refusals(go, (dict(x=None), dict(sum=None), dict(rows=-1), dict(rows=1 << 30), dict(cols=0), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf),
                      dict(type=4), dict(xs=19), dict(rs=19), dict(ss=19), dict(x=P + 1), dict(r=P + 1), dict(w=P + 1), dict(sum=P + 1), dict(out=None),
                      dict(stride=19)))
        assert go(rows=0) == 0
    refusals(values, (dict(out=P + 1),))
    refusals(codes, (dict(scale=None), dict(scale=P + 2)))


def test_norm_outputs_over_each_other_are_refused():
    def values(x=P, xs=20, r=2 * P, rs=20, rows=3, total=3 * P, ss=20, out=4 * P, stride=20):
        return call("vdt_add_rms_norm", x, xs, r, rs, None, rows, 20, 1e-6, 2, total, ss, out, stride, None)

    def codes(x=P, xs=20, r=2 * P, rs=20, rows=3, total=3 * P, ss=20):
        return call("vdt_add_rms_norm_int8", x, xs, r, rs, None, rows, 20, 1e-6, 2, total, ss, 4 * P, 20, 5 * P, None)

    for go in (values, codes):
        refusals(go, (dict(total=P, ss=24), dict(total=2 * P, rs=24), dict(x=2 * P, total=2 * P, xs=24)))
    refusals(values, (dict(out=3 * P), dict(out=3 * P, rows=1), dict(out=P, stride=24), dict(out=2 * P, stride=24), dict(r=None, out=P, stride=24)))


def plan(**over):
    a = dict(ring=P, n=8, span=P, pages=P, width=3, held=P, new=P, seqs=2, page=16, total=5, kept=P, starts=P, positions=P, slots=P, out=P, scratch=P,
             size=1 << 20)
    a.update(over)
    return call("vdt_plan_pages", a["ring"], a["n"], a["span"], a["pages"], a["width"], a["held"], a["new"], a["seqs"], a["page"], a["total"], a["kept"],
                a["starts"], a["positions"], a["slots"], a["out"], a["scratch"], a["size"], None)


def free(**over):
    a = dict(ring=P, n=8, span=P, pages=P, width=3, held=P, done=P, seqs=2, page=16, kept=P, out=P)
    a.update(over)
    return call("vdt_free_pages", a["ring"], a["n"], a["span"], a["pages"], a["width"], a["held"], a["done"], a["seqs"], a["page"], a["kept"], a["out"], None)


def test_page_table_refusals():
    for go in (plan, free):
        refusals(go, (dict(ring=None), dict(n=-1), dict(span=None), dict(pages=None), dict(width=-1), dict(held=None), dict(seqs=-1), dict(page=0),
                      dict(page=-16), dict(kept=None), dict(out=None), dict(ring=P + 2), dict(span=P + 2), dict(pages=P + 1), dict(held=P + 2),
                      dict(kept=P + 2), dict(out=P + 2)))
        assert go(seqs=65536) == UNSUPPORTED
    refusals(plan, (dict(new=None), dict(starts=None), dict(positions=None), dict(slots=None), dict(scratch=None), dict(total=-1), dict(total=1 << 30),
                    dict(new=P + 2), dict(starts=P + 2), dict(positions=P + 2), dict(slots=P + 4), dict(scratch=P + 8)))
    refusals(free, (dict(done=None),))
    need = call("vdt_plan_pages_scratch_bytes", 2)
    assert need > 0 and plan(size=need - 1) == CAPACITY and call("vdt_plan_pages_scratch_bytes", -1) == 0


def test_page_tables_past_32_bits_count_are_refused():
    for go in (plan, free):
        for over in (dict(width=(1 << 30) + 1), dict(n=(1 << 30) + 1), dict(width=(1 << 31) - 1), dict(n=(1 << 31) - 1)):
            assert go(**over) == UNSUPPORTED, over


def test_sample_refusals():
    ok = dict(x=P, type=0, rows=3, vocab=50, stride=50, u=P, ts=None, t=1.0, ks=None, k=0, ps=None, p=1.0, ms=None, m=0.0, tokens=P, logp=P)

    def go(**over):
        a = dict(ok, **over)
        return call("vdt_sample", a["x"], a["type"], a["rows"], a["vocab"], a["stride"], a["u"], a["ts"], a["t"], a["ks"], a["k"], a["ps"], a["p"], a["ms"],
                    a["m"], a["tokens"], a["logp"], None)

    refusals(go, (dict(x=None), dict(u=None), dict(tokens=None), dict(type=3), dict(rows=-1), dict(rows=1 << 27), dict(vocab=0), dict(stride=49),
                  dict(t=-0.5), dict(t=math.nan), dict(t=math.inf), dict(p=math.nan), dict(m=math.nan), dict(x=P + 2), dict(u=P + 2), dict(ts=P + 1),
                  dict(ks=P + 2), dict(ps=P + 2), dict(ms=P + 2), dict(tokens=P + 2), dict(logp=P + 2)))
    assert go(vocab=524289, stride=524289) == UNSUPPORTED
    assert go(rows=0) == 0

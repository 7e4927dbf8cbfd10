"""The step operators together, as examples/spike_batch.py runs them: every call of
theirs is checked on its own inputs against the 64-bit definitions, with the
tolerances of test_gpu_step.py; pages are in one place at a time."""
import os
import sys

import pytest
import torch

from conftest import ROOT
from test_gpu_step import FP4, U, fp4_definition, fp4_of, plan_definition, sample_definition

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(dev):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import spike_batch
    return spike_batch


class Checked:
    """vdttfs.seq with the step operators' results compared call by call."""

    def __init__(self, seq):
        self.seq, self.calls = seq, {}

    def __getattr__(self, name):
        return getattr(self.seq, name)

    def count(self, name):
        self.calls[name] = self.calls.get(name, 0) + 1

    def quantize_fp4(self, x):
        codes, scale = self.seq.quantize_fp4(x)
        assert torch.equal(self.seq.fp4_values(codes, scale, x.shape[1]).cpu().double(), fp4_of(*fp4_definition(x.cpu())))
        self.count("quantize_fp4")
        return codes, scale

    def fp4_linear(self, x, w, ws):
        y = self.seq.fp4_linear(x, w, ws)
        a, v = fp4_of(*fp4_definition(x.cpu())), self.seq.fp4_values(w, ws).cpu().double()
        a = torch.where(torch.isnan(x.cpu()).any(1, keepdim=True), torch.full((), float("nan"), dtype=torch.float64), a)
        want, size = a @ v.T, a.abs() @ v.abs().T
        off = (y.cpu().double() - want).abs()
        assert ((off <= U[y.dtype] * want.abs() + (x.shape[1] / 64 + 2) * 2.0 ** -23 * size + 1e-37) | torch.isnan(want)).all()
        assert torch.isnan(y.cpu()[torch.isnan(want)]).all()
        self.count("fp4_linear")
        return y

    def norm(self, x, t, w, total):
        want = x.float() if t is None else (x.float() + t.float()).to(x.dtype).float()
        assert torch.equal(torch.nan_to_num(total.float(), 7e30), torch.nan_to_num(want, 7e30))
        z = (want * w.float()).double()
        return z, (want.double().square().mean(1, keepdim=True) + 1e-6).sqrt(), (x.shape[1] / 128 + 12) / 2 + 4

    def add_rms_norm(self, x, t, w):
        y, total = self.seq.add_rms_norm(x, t, w)
        z, root, deep = self.norm(x, t, w, total)
        want = z / root
        fine = ~torch.isnan(want)
        assert ((y.double() - want).abs()[fine] <= (U[y.dtype] + deep * 2.0 ** -24) * want.abs()[fine] + 1e-37).all() and torch.isnan(y[~fine]).all()
        self.count("add_rms_norm")
        return y, total

    def add_rms_norm_int8(self, x, t, w):
        codes, scale, total = self.seq.add_rms_norm_int8(x, t, w)
        z, root, deep = self.norm(x, t, w, total)
        # a code is off by half a step at most, and by the scale's own error
        step = z.abs().amax(1, keepdim=True) / root / 127
        off = (codes.double() * scale.double()[:, None] - z / root).abs()
        assert ((off <= (0.5 + 128 * (deep + 2) * 2.0 ** -24) * step) | torch.isnan(step)).all()
        self.count("add_rms_norm_int8")
        return codes, scale, total

    def plan_pages(self, pool, pages, held, new, page, total):
        before, ring, span = pages.tolist(), pool[0].tolist(), tuple(pool[1].tolist())
        plan = self.seq.plan_pages(pool, pages, held, new, page, total)
        want = plan_definition(ring, span, before, held.tolist(), new.tolist(), page, total)
        assert [t.tolist() for t in plan] == list(want[:5]) and pages.tolist() == want[5]
        self.count("plan_pages")
        return plan

    def free_pages(self, pool, pages, held, done, page):
        ring, (first, left), h = pool[0].tolist(), pool[1].tolist(), held.tolist()
        left = max(left, 0)
        back = [p for i, row in enumerate(pages.tolist()) if done[i] for p in row[: -(-h[i] // page)] if p >= 0]
        got, span = self.seq.free_pages(pool, pages, held, done, page)
        for i, p in enumerate(back):
            ring[(first + left + i) % len(ring)] = p
        assert pool[0].tolist() == ring and span.tolist() == [first, left + len(back)]
        assert got.tolist() == [0 if d else n for d, n in zip(done.tolist(), h)]
        # every page once: free, or a running sequence's
        used = [p for row, n in zip(pages.tolist(), got.tolist()) for p in row[: -(-n // page)] if p >= 0]
        free = [ring[(first + i) % len(ring)] for i in range(left + len(back))]
        assert sorted(used + free) == list(range(len(ring)))
        self.count("free_pages")
        return got, span

    def sample(self, logits, u, temperature, top_k, top_p):
        tokens, logp = self.seq.sample(logits, u, temperature, top_k, top_p)
        x, p = logits.cpu().double().numpy(), float(torch.tensor(top_p))
        for r in range(len(x)):
            token, log = sample_definition(x[r], float(u[r]), float(temperature[r]), int(top_k[r]), p, 0.0)
            assert int(tokens[r]) == token
            assert abs(float(logp[r]) - log) <= 2.0 ** -22 * abs(log) + 2.0 ** -30 or token == -1
        self.count("sample")
        return tokens, logp


@pytest.mark.parametrize("seqs,steps", [(1, 12), (6, 40), (11, 30)])
def test_batches_of_the_example(example, seqs, steps):
    from vdttfs import seq
    assert len(FP4) == 16
    ops = Checked(seq)
    answers, batch = example.run(seqs, steps, ops)
    assert all(0 <= t < example.VOCAB for _, tokens in answers for t in tokens)
    assert ops.calls["sample"] == ops.calls["plan_pages"] == ops.calls["free_pages"] <= steps and ops.calls["fp4_linear"] >= 4
    if steps == 40:
        assert len(answers) > seqs                       # sequences ended, and others took their places


def test_batches_give_the_same_answers_again(example):
    a, b = (example.run(5, 25)[0] for _ in range(2))
    assert a == b

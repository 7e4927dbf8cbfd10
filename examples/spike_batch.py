"""Sequences that come and go behind a spiking encoder, on the step operators.

    python examples/spike_batch.py [--seqs 6] [--steps 40]

The decoder (random weights, two layers of 256, 4 heads of 64 over 2 cached
ones) answers prompts of different lengths in one batch.  A prompt's tokens are
the first-spike times of an encoded image row, the engine's own encoder; a
sequence that has drawn the end token, or has no more room, gives its pages back
and the next prompt takes its place.  Every step is the same few calls:

* plan_pages, free_pages     pages, first rows and positions of the step's tokens
* add_rms_norm_int8          each layer's first norm, straight into int8_matmul
* qk_norm_rope, cache_append, cache_attention
* add_rms_norm, fp4_linear   the second norm and the feed-forward in 4 bits
* sample                     the next tokens, each sequence with parameters of its own

Nothing is trained: the program shows how the calls fit together.
"""
import argparse
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vd-ttfs_b200"))

import torch

from vdttfs import engine as E, nets, seq, synth

WIDTH, HEADS, KV, DIM, LAYERS, HIDDEN, PAGE, MOST = 256, 4, 2, 64, 2, 640, 16, 96
VOCAB, END = 96, 0                     # tokens 1.. are spike times


def prompts(many, seed=0):
    """Token lists of different lengths: rows of encoded images, the pixels that fire."""
    net = nets.lenet5()
    image = torch.from_numpy(synth.images(1, many, net.in_h, net.in_w, net.in_c, 0.5, stream=seed)).cuda()
    times = E.encode_image(image.reshape(many, -1), net.encoder, net.tc_in, net.td_in, net.T, net.inf_time).cpu()
    out = []
    for i in range(many):
        fired = times[i][times[i] < net.inf_time].long()
        out.append((1 + fired[: 3 + (i * 17) % 41] % (VOCAB - 1)).tolist())
    return out


class Batch:
    """Random weights, quantised once; the caches and tables of ``seqs`` places in a batch."""

    def __init__(self, seqs, ops=seq, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.ops, self.seqs = ops, seqs

        def normal(*shape):
            return torch.randn(shape, generator=g, device="cuda")

        def norm():
            return (1 + 0.1 * normal(WIDTH)).to(torch.bfloat16)

        self.embedding = normal(VOCAB, WIDTH).to(torch.bfloat16)
        self.layers = [dict(n1=norm(), n2=norm(), qkv=seq.quantize_rows(normal((HEADS + 2 * KV) * DIM, WIDTH) / WIDTH ** 0.5),
                            o=seq.quantize_rows(normal(WIDTH, HEADS * DIM) / (HEADS * DIM) ** 0.5),
                            up=ops.quantize_fp4(normal(HIDDEN, WIDTH) / WIDTH ** 0.5), down=ops.quantize_fp4(normal(WIDTH, HIDDEN) / HIDDEN ** 0.5))
                       for _ in range(LAYERS)]
        self.last_norm, self.head = norm(), seq.quantize_rows(normal(VOCAB, WIDTH) / WIDTH ** 0.5)
        self.one = torch.ones(DIM, dtype=torch.bfloat16, device="cuda")
        self.rope = seq.rope_table(MOST, DIM)
        count = seqs * (MOST // PAGE) * 3 // 4             # not as many as all places could fill
        self.pool = seq.PagePool.full(count)
        self.caches = [seq.Cache8.empty(count, KV, DIM, PAGE) for _ in range(LAYERS)]
        self.pages = torch.full((seqs, MOST // PAGE), -1, dtype=torch.int32, device="cuda")
        self.held = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.temperature = torch.linspace(0.0, 1.2, seqs, device="cuda")
        self.top_k = (torch.arange(seqs, device="cuda", dtype=torch.int32) % 3) * 12

    def step(self, tokens, new, u):
        """tokens: the step's, sequence after sequence, new [seqs] of each -> the next of each, their
        probabilities' logarithms, and the logits."""
        ops, total = self.ops, tokens.shape[0]
        most, most_kept = int(max(new)), MOST
        plan = ops.plan_pages(self.pool, self.pages, self.held, torch.tensor(new, dtype=torch.int32, device="cuda"), PAGE, total)
        x, t = self.embedding[tokens], None
        for layer, cache in zip(self.layers, self.caches):
            codes, scale, t = ops.add_rms_norm_int8(x, t, layer["n1"])
            qkv = ops.int8_matmul(codes, scale, *layer["qkv"]).view(total, HEADS + 2 * KV, DIM)
            q, k = ops.qk_norm_rope(qkv[:, :HEADS], qkv[:, HEADS: HEADS + KV], self.one, self.one, plan.positions, self.rope)
            ops.cache_append(cache, k, qkv[:, HEADS + KV:], self.pages, self.held, plan.starts, most)
            a = ops.cache_attention(q, cache, self.pages, plan.kept, plan.starts, most, most_kept)
            y, t = ops.add_rms_norm(ops.int8_linear(a.view(total, -1), *layer["o"]), t, layer["n2"])
            x = ops.fp4_linear(torch.relu(ops.fp4_linear(y, *layer["up"])), *layer["down"])
        y, _ = ops.add_rms_norm(x, t, self.last_norm)
        rows = (plan.starts[1:] - 1).clamp(min=0).long()
        logits = ops.int8_linear(y[rows], *self.head, out_dtype=torch.float32)
        nxt, logp = ops.sample(logits, u, self.temperature, self.top_k, 0.95)
        self.held, self.pool = plan.kept, seq.PagePool(self.pool.ring, plan.span)
        return nxt, logp, logits

    def release(self, done):
        held, span = self.ops.free_pages(self.pool, self.pages, self.held, done, PAGE)
        self.held, self.pool = held, seq.PagePool(self.pool.ring, span)


def run(seqs=6, steps=40, ops=seq):
    """Answers, [(prompt, tokens)], in the order in which they ended or were cut off."""
    batch, waiting = Batch(seqs, ops), prompts(4 * seqs)
    g = torch.Generator(device="cuda").manual_seed(1)
    active, fresh, answers = [None] * seqs, [None] * seqs, []
    for _ in range(steps):
        # the first of those that wait into the places that are free, while pages for all of them are
        room = int(batch.pool.span[1]) - sum(1 for a in active if a)
        for i in range(seqs):
            if active[i] is None and waiting and room * PAGE >= len(waiting[0]) + PAGE:
                room -= -(-(len(waiting[0]) + 1) // PAGE) + 1
                active[i] = (waiting.pop(0), [])
                fresh[i] = active[i][0]
        new = [len(f) if f else 0 for f in fresh]
        if not any(new):
            break
        tokens = torch.tensor([t for f in fresh if f for t in f], device="cuda")
        nxt, _, _ = batch.step(tokens, new, torch.rand(seqs, generator=g, device="cuda"))
        held, done = batch.held.tolist(), []
        for i, t in enumerate(nxt.tolist()):
            fresh[i] = None
            # -1: the pool had no page for it, and it sees NaN
            done.append(active[i] is not None and new[i] > 0 and (t < 0 or t == END or held[i] + 1 >= MOST))
            if active[i] is not None and new[i] > 0:
                if t >= 0:
                    active[i][1].append(t)
                if done[i]:
                    answers.append(active[i])
                    active[i] = None
                else:
                    fresh[i] = [t]
        batch.release(torch.tensor(done, device="cuda"))
    return answers + [a for a in active if a], batch


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--seqs", type=int, default=6)
    ap.add_argument("--steps", type=int, default=40)
    a = ap.parse_args()
    answers, _ = run(a.seqs, a.steps)
    for prompt, tokens in answers:
        print(f"{len(prompt):3d} tokens in, {len(tokens):3d} out: {tokens[:16]}")


if __name__ == "__main__":
    main()

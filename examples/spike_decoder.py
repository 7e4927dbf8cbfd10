"""A small decoder behind a spiking encoder, on the sequence operators.

    python examples/spike_decoder.py [--steps 12] [--batch 4]

The encoder is the engine's VGG-16 (first-spike times, random weights): the map
of its tenth convolution, 4 x 4 pixels of 512 channels, gives 16 states an
image, the activation exp(-t / tau) of each first-spike time t (none: 0).  The
decoder (random weights, two layers of 512, 8 heads of 64 over 2 cached ones)
reads them by cross attention and answers with tokens one at a time:

* int8_linear        every projection, weights in 8 bits
* qk_norm_rope       norm of each head and rotation
* cache_append,
  cache_attention    the tokens so far (causal) and the encoder's states (not
                     causal), both in paged 8-bit caches
* engine.readout     the next token, the engine's own argmax

Nothing is trained: the program shows how the calls fit together.
"""
import argparse
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vd-ttfs_b200"))

import numpy as np
import torch

from vdttfs import engine as E, nets, seq, synth

WIDTH, HEADS, KV, DIM, LAYERS, VOCAB, PAGE = 512, 8, 2, 64, 2, 96, 16
STATE_LAYER = 9                        # VGG-16's tenth convolution: a 4 x 4 x 512 map


def encoder_states(images):
    """[batch, 32, 32, 3] pixels -> [batch, 16, 512] states: exp(-t / tau) of the layer's first-spike times."""
    net = nets.vgg16()
    model = E.Model(net, synth.kaiming_layers(net, 3), lut_source=E.LUT_HOST_LIBM)
    ctx = E.Context(model, images.shape[0])
    maps, _, _ = ctx.trace(images, pixels=True)
    t = maps[STATE_LAYER]
    fired = t < net.inf_time
    states = torch.where(fired, torch.exp(-(t - net.tfs) / net.T), torch.zeros((), device=t.device))
    ctx.close()
    model.close()
    return states.reshape(images.shape[0], -1, t.shape[-1])


class Decoder:
    """Random weights, quantised once; the caches of a batch of sequences."""

    def __init__(self, batch, most_tokens, most_states, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weights(n, k):
            return seq.quantize_rows(torch.randn(n, k, generator=g, device="cuda") / k ** 0.5)

        self.embedding = torch.randn(VOCAB, WIDTH, generator=g, device="cuda").to(torch.bfloat16)
        self.layers = [dict(qkv=weights((HEADS + 2 * KV) * DIM, WIDTH), o=weights(WIDTH, HEADS * DIM), q=weights(HEADS * DIM, WIDTH),
                            kv=weights(2 * KV * DIM, WIDTH), co=weights(WIDTH, HEADS * DIM), up=weights(4 * WIDTH, WIDTH),
                            down=weights(WIDTH, 4 * WIDTH)) for _ in range(LAYERS)]
        self.head = weights(VOCAB, WIDTH)
        self.one = torch.ones(DIM, dtype=torch.bfloat16, device="cuda")
        self.rope = seq.rope_table(most_tokens, DIM)
        self.batch, self.most_tokens, self.most_states = batch, most_tokens, most_states

        def caches(tokens):
            pages = -(-tokens // PAGE)
            table = torch.arange(batch * pages, dtype=torch.int32, device="cuda").view(batch, pages)
            return [seq.Cache8.empty(batch * pages, KV, DIM, PAGE) for _ in range(LAYERS)], table

        self.own, self.own_pages = caches(most_tokens)
        self.states, self.state_pages = caches(most_states)
        self.each = torch.arange(batch + 1, dtype=torch.int32, device="cuda")       # one token a sequence
        self.n_states = torch.full((batch,), most_states, dtype=torch.int32, device="cuda")

    def read(self, states):
        """The encoder's states [batch, n, width] into the layers' caches, once for an image."""
        b, n, _ = states.shape
        flat = states.reshape(b * n, -1)
        starts = self.each * n
        none = torch.zeros(b, dtype=torch.int32, device="cuda")
        for layer, cache in zip(self.layers, self.states):
            kv = seq.int8_linear(flat, *layer["kv"], out_dtype=torch.bfloat16).view(b * n, 2 * KV, DIM)
            k, _ = seq.qk_norm_rope(kv[:, :KV], None, self.one, None, None, None)
            seq.cache_append(cache, k, kv[:, KV:], self.state_pages, none, starts, n)

    def step(self, tokens, at):
        """One token of each sequence at place `at`: the logits of the next."""
        b = self.batch
        place = torch.full((b,), at, dtype=torch.int32, device="cuda")
        x = self.embedding[tokens.long()]
        for layer, own, states in zip(self.layers, self.own, self.states):
            qkv = seq.int8_linear(x, *layer["qkv"]).view(b, HEADS + 2 * KV, DIM)
            q, k = seq.qk_norm_rope(qkv[:, :HEADS], qkv[:, HEADS: HEADS + KV], self.one, self.one, place, self.rope)
            seq.cache_append(own, k, qkv[:, HEADS + KV:], self.own_pages, place, self.each, 1)
            a = seq.cache_attention(q, own, self.own_pages, place + 1, self.each, 1, self.most_tokens)
            x = x + seq.int8_linear(a.view(b, -1), *layer["o"])
            q, _ = seq.qk_norm_rope(seq.int8_linear(x, *layer["q"]).view(b, HEADS, DIM), None, self.one, None, None, None)
            a = seq.cache_attention(q, states, self.state_pages, self.n_states, self.each, 1, self.most_states, causal=False)
            x = x + seq.int8_linear(a.view(b, -1), *layer["co"])
            x = x + seq.int8_linear(torch.relu(seq.int8_linear(x, *layer["up"])), *layer["down"])
        return seq.int8_linear(x, *self.head, out_dtype=torch.float32)


def run(batch=4, steps=12):
    net = nets.vgg16()
    images = torch.from_numpy(synth.images(3, batch, net.in_h, net.in_w, net.in_c, 0.0, stream=7)).cuda()
    states = encoder_states(images)
    decoder = Decoder(batch, steps + 1, states.shape[1])
    decoder.read(states)
    tokens = torch.zeros(batch, dtype=torch.int32, device="cuda")
    out, logits = [], []
    for at in range(steps):
        y = decoder.step(tokens, at)
        tokens = E.readout(y, batch, VOCAB, nets.READ_ARGMAX)
        out.append(tokens)
        logits.append(y)
    return states, decoder, torch.stack(out, 1), torch.stack(logits, 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=12)
    ap.add_argument("--batch", type=int, default=4)
    a = ap.parse_args()
    states, _, tokens, _ = run(a.batch, a.steps)
    print(f"states {tuple(states.shape)}, {float((states > 0).float().mean()):.2f} of them fired")
    for i, row in enumerate(tokens.cpu().numpy()):
        print(f"image {i}: {np.array2string(row)}")


if __name__ == "__main__":
    main()

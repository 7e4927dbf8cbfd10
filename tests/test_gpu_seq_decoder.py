"""The example decoder (examples/spike_decoder.py) against its plain restatement.

The restatement has the same 8-bit weights, 32-bit activations and no caches: it
reads all keys and values at every step, unrounded.  What separates the two, for
each of the decoder's 2 x 9 stages: bf16 roundings (2^-9 of a value, rms), 8-bit
activations (a step is 1/127 of a row's largest value, some 3.5 rms, so an error
of 3.5 / 127 / sqrt(12) = 0.8% rms), 8-bit keys and values (the same over a page).
Independent, over 18 stages: sqrt(18) * 1.2% = 5%; twice that is allowed.
"""
import math
import os
import sys

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(dev):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import spike_decoder
    return spike_decoder


def plain_logits(S, states, decoder, tokens):
    """Logits of all places [batch, steps, vocab] for the tokens that the decoder went on with."""
    b, steps = tokens.shape
    real = lambda w: w[0].float() * w[1][:, None]  # noqa: E731
    first = torch.zeros(b, 1, dtype=tokens.dtype, device=tokens.device)
    x = decoder.embedding[torch.cat([first, tokens[:, :-1]], 1).long()].float()
    norm = lambda t: t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt()  # noqa: E731
    half = S.DIM // 2
    cos, sin = (decoder.rope[:steps, i * half: (i + 1) * half][:, None] for i in (0, 1))

    def turn(t):
        a, c = t[..., :half], t[..., half:]
        return torch.cat([a * cos - c * sin, c * cos + a * sin], -1)

    def attend(q, k, v, causal):
        k, v = (t.repeat_interleave(S.HEADS // S.KV, 2) for t in (k, v))
        s = torch.einsum("bqhd,bkhd->bhqk", q, k) / math.sqrt(S.DIM)
        if causal:
            s = s.masked_fill(torch.ones(steps, steps, device=s.device).triu(1).bool(), -math.inf)
        return torch.einsum("bhqk,bkhd->bqhd", s.softmax(-1), v).flatten(2)

    for layer in decoder.layers:
        qkv = (x @ real(layer["qkv"]).T).view(b, steps, -1, S.DIM)
        q, k, v = qkv.split([S.HEADS, S.KV, S.KV], 2)
        x = x + attend(turn(norm(q)), turn(norm(k)), v, True) @ real(layer["o"]).T
        kv = (states @ real(layer["kv"]).T).view(b, states.shape[1], -1, S.DIM)
        q = norm((x @ real(layer["q"]).T).view(b, steps, S.HEADS, S.DIM))
        x = x + attend(q, norm(kv[:, :, : S.KV]), kv[:, :, S.KV:], False) @ real(layer["co"]).T
        x = x + torch.relu(x @ real(layer["up"]).T) @ real(layer["down"]).T
    return x @ real(decoder.head).T


def test_example_decoder_matches_its_plain_restatement(example):
    states, decoder, tokens, logits = example.run(batch=3, steps=20)
    assert states.shape == (3, 16, 512) and 0 < float((states > 0).float().mean()) < 1
    assert (tokens == logits.argmax(-1)).all()
    want = plain_logits(example, states, decoder, tokens)
    assert float((logits - want).norm() / want.norm()) < 0.10


def test_example_decoder_gives_the_same_tokens_again(example):
    a, b = (example.run(batch=2, steps=6) for _ in range(2))
    assert torch.equal(a[3], b[3]) and torch.equal(a[2], b[2])

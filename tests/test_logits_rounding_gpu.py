"""Adjusted logits of ZG_BF16 are formed in 64 bits and rounded once: values
whose float32 rounding is a tie of bfloat16, on either side of it, against
the nearest bfloat16 of the 64-bit value, bit for bit."""
import math

import numpy as np
import pytest
import torch

import paged_reference as ref
from test_logits_gpu import device, random_rules
from zerogravity_amd import _lib as L
from zerogravity_amd import sampling

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def ctx():
    c = L.Context(0)
    yield c
    c.close()


def nearest(v):
    """float64 -> the nearest bfloat16 value (8 bits, ties to even; 2^-133 the
    least step, infinity from half a step past the largest), as float64."""
    _, e = np.frexp(v)
    step = np.maximum(e - 8, -133)
    y = np.ldexp(np.rint(np.ldexp(v, -step)), step)
    return np.where(np.abs(y) >= 2.0 ** 128, np.copysign(np.inf, y), y)


def adjust(ctx, x, bias):
    """Logits with a bias for every token, as written, and the ids."""
    rows, vocab = x.shape
    u = sampling.rules(bias_ids=torch.arange(vocab, dtype=torch.int32).repeat(rows, 1).cuda(),
                       bias_values=torch.from_numpy(bias).cuda(),
                       bias_lengths=torch.full((rows,), vocab, dtype=torch.int32, device="cuda"))
    greedy = torch.empty(rows, dtype=torch.int32, device="cuda")
    out = sampling.adjust(ctx, torch.from_numpy(x).to(BF16).cuda(), u, greedy=greedy)
    torch.cuda.synchronize()
    return out.double().cpu().numpy(), greedy.cpu().numpy().view(np.uint32)


def test_hand_computed_ties(ctx):
    top = 2.0 ** 127 * (2 - 2.0 ** -7)  # the largest bfloat16; infinity starts at 2^119 past it
    cases = [(256.0, 1 + 2.0 ** -20, 258.0), (256.0, 1 - 2.0 ** -20, 256.0), (256.0, 1.0, 256.0),
             (258.0, 1 - 2.0 ** -20, 258.0), (258.0, 1.0, 260.0), (-256.0, -1 - 2.0 ** -20, -258.0),
             (-258.0, -1 + 2.0 ** -20, -258.0), (top, 2.0 ** 119 * (1 - 2.0 ** -24), top), (top, 2.0 ** 119, math.inf),
             (0.0, 2.0 ** -134, 0.0), (2.0 ** -133, 2.0 ** -134, 2.0 ** -132), (1.0, -1.0, 0.0)]
    x, bias, want = (np.array(c, np.float64) for c in zip(*cases))
    got, _ = adjust(ctx, x.astype(np.float32)[None], bias.astype(np.float32)[None])
    assert got[0].tolist() == want.tolist()
    # the id goes by what is written: 258 twice
    assert adjust(ctx, np.float32([[256.0, 258.0]]), np.float32([[1 + 2.0 ** -20, 0.0]]))[1].tolist() == [0]


@pytest.mark.parametrize("rows,vocab", [(1, 60000), (40, 12301), (130, 8192)])
def test_values_beside_ties(ctx, rows, vocab):
    """A logit and a bias whose sum is a tie of bfloat16, or off it by 2^-22
    to 2^-36 of the step, which float32 drops or not: all slices and forms of
    the kernel."""
    g = np.random.default_rng(rows)
    x = nearest(np.ldexp(1 + g.random((rows, vocab)), g.integers(-20, 20, (rows, vocab))) *
                g.choice([-1.0, 1.0], (rows, vocab)))
    _, e = np.frexp(x)
    half = np.ldexp(1.0, e - 9)
    off = np.ldexp(g.integers(-3, 4, (rows, vocab)).astype(np.float64), e - 9 - g.integers(8, 23, (rows, vocab)))
    bias = (g.choice([-1.0, 1.0], (rows, vocab)) * (half + off)).astype(np.float32)
    v = x + bias.astype(np.float64)  # exact: both are within 24 bits, 2^31 steps apart at most
    twice = torch.from_numpy(v.astype(np.float32)).to(BF16).double().numpy()
    want = nearest(v)
    assert (twice != want).mean() > 0.01  # what the 64 bits are for
    got, ids = adjust(ctx, x.astype(np.float32), bias)
    assert np.array_equal(got, want) and np.array_equal(ids, ref.np_greedy(want))


def adjusted(x, u):
    """The rules in 64 bits, not rounded: history, biases and masks all there."""
    v, vocab = x.copy(), x.shape[1]
    for r in range(len(v)):
        tokens = u["history"][r].astype(np.int64)
        inside = (tokens >= 0) & (tokens < vocab)
        seen = np.unique(tokens[inside])
        rep = np.float64(u["repetition"][r])
        v[r, seen] = np.where(v[r, seen] > 0, v[r, seen] / rep, v[r, seen] * rep)
        start = u["prompt_lengths"][r]
        made, count = np.unique(tokens[start:][inside[start:]], return_counts=True)
        v[r, made] = v[r, made] - np.float64(u["frequency"][r]) * count - np.float64(u["presence"][r])
        ids = u["bias_ids"][r]
        sums, inside = np.zeros(vocab), (ids >= 0) & (ids < vocab)
        np.add.at(sums, ids[inside], u["bias_values"][r][inside].astype(np.float64))
        v[r, ids[inside]] += sums[ids[inside]]
        if u["mask_of"][r] >= 0:
            bits = np.unpackbits(u["masks"][u["mask_of"][r]].view(np.uint8), bitorder="little")[:vocab]
            v[r, bits == 0] = -np.inf
    return v


@pytest.mark.parametrize("rows,vocab,history,biases", [(50, 8191, 16000, 1100), (1100, 4000, 6000, 600)])
def test_most_of_a_vocabulary_is_rounded_once(ctx, rows, vocab, history, biases):
    """Drawn penalties and biases of most tokens; a few of the sums lie so near
    a tie that rounding to float32 first gives the other neighbour."""
    g = torch.Generator().manual_seed(rows)
    u = random_rules(g, rows, vocab, history, biases, 2)
    u["history_lengths"][:] = history
    u["bias_lengths"][:] = biases
    x = (3 * torch.randn(rows, vocab, generator=g)).to(BF16)
    held = {k: t.numpy() for k, t in u.items()}
    v = adjusted(x.double().numpy(), held)
    assert np.array_equal(v.astype(np.float32), ref.np_adjust(x.float().numpy(), held, vocab))
    want = nearest(v)
    assert (torch.from_numpy(v.astype(np.float32)).to(BF16).double().numpy() != want).any()
    greedy = torch.empty(rows, dtype=torch.int32, device="cuda")
    out = sampling.adjust(ctx, x.cuda(), sampling.rules(**device(u)), greedy=greedy)
    torch.cuda.synchronize()
    assert np.array_equal(out.double().cpu().numpy(), want)
    assert np.array_equal(greedy.cpu().numpy().view(np.uint32), ref.np_greedy(want))

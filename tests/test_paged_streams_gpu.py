"""Calls on another stream than the current one: their tensors may be dropped
as soon as the call returns, though that stream is far from through."""
import pytest
import torch

import paged_reference as ref
from test_paged_attn_gpu import Device
from zerogravity_amd import _lib as L
from zerogravity_amd import paged, sampling

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = L.Context(0)
    yield c
    c.close()


def behind(call, make):
    """call(tensors, stream) behind other work of a stream; the tensors are
    dropped at once and their memory, where it is given out again, filled."""
    busy = torch.randn(4096, 4096, device="cuda")
    torch.mm(busy, busy)
    stream = torch.cuda.Stream()
    tensors = make()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(40):
            torch.mm(busy, busy)
    call(tensors, stream)
    shapes = [(t.shape, t.dtype) for t in tensors]
    del tensors
    junk = [torch.full(s, 77, dtype=d, device="cuda") for s, d in shapes for _ in range(3)]
    assert not stream.query()  # the call has not run yet
    torch.cuda.synchronize()
    del junk


def test_attention(ctx):
    d = Device(ref.Batch(80, 40, 2, 4, 256, 16, 100, [50] * 40, torch.float32, torch.bfloat16))
    want = d.attend(ctx)
    got = []
    behind(lambda t, s: got.append(paged.attend(ctx, d.kv, d.rows, t[0], t[1], d.b.scale, stream=s)),
           lambda: [d.lengths.clone(), d.q.clone()])
    assert torch.equal(got[0], want)


def test_tables_and_caches(ctx):
    d = Device(ref.Batch(81, 40, 2, 4, 256, 16, 100, [50] * 40, torch.float32, torch.bfloat16))
    want = d.attend(ctx)
    got = []

    def call(t, s):
        kv, rows = paged.cache(t[0], t[1]), paged.rows(t[2], t[3], 100)
        got.append(paged.attend(ctx, kv, rows, d.lengths, d.q, d.b.scale, stream=s))

    behind(call, lambda: [d.keys.clone(), d.values.clone(), d.table.clone(), d.prefix.clone()])
    assert torch.equal(got[0], want)


def test_append(ctx):
    g = torch.Generator().manual_seed(4)
    k, v, q = (torch.randn(300, n, 64, generator=g).cuda() for n in (2, 2, 4))
    gamma = torch.randn(2, 64, generator=g).cuda()
    at = torch.arange(300, dtype=torch.int32, device="cuda")
    of = torch.zeros(300, dtype=torch.int32, device="cuda")
    table = torch.randperm(38, generator=g).int().view(1, -1).cuda()
    results = []

    def call(t, s):
        keys, values, out = torch.zeros(38, 8, 2, 64, device="cuda"), torch.zeros(38, 8, 2, 64, device="cuda"), torch.zeros_like(q)
        torch.cuda.current_stream().synchronize()
        results.append((keys, values, out))
        paged.append(ctx, paged.cache(keys, values), paged.rows(table), t[0], t[1], t[3], t[2], out, t[5][0], t[5][1],
                     rotate=32, theta_scale=0.8, token_rows=t[4], stream=s)

    call([k, v, q, at, of, gamma], None)
    behind(call, lambda: [t.clone() for t in (k, v, q, at, of, gamma)])
    assert all(torch.equal(a, b) for a, b in zip(*results)) and (results[0][0] != 0).any()


def test_logits(ctx):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(16, 5000, generator=g).cuda()
    history = torch.randint(0, 5000, (16, 300), generator=g).int().cuda()
    held = torch.full((16,), 300, dtype=torch.int32, device="cuda")
    rep = torch.full((16,), 1.5, device="cuda")
    masks = torch.randint(-2 ** 31, 2 ** 31, (16, 160), generator=g).int().cuda()
    results = []

    def call(t, s):
        out, greedy = torch.empty_like(x), torch.empty(16, dtype=torch.int32, device="cuda")
        results.append((out, greedy))
        u = sampling.rules(history=t[1], history_lengths=t[2], repetition=t[3], masks=t[4])
        sampling.adjust(ctx, t[0], u, out, greedy, stream=s)

    call([x, history, held, rep, masks], None)
    behind(call, lambda: [t.clone() for t in (x, history, held, rep, masks)])
    assert all(torch.equal(a, b) for a, b in zip(*results))

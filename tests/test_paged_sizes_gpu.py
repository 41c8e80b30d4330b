"""The largest and the smallest calls that the paged cache's and the readout's
entries take: rows, heads, pages and vocabularies at their limits."""
import numpy as np
import pytest
import torch

import paged_reference as ref
from test_logits_gpu import device, random_rules
from test_logits_rounding_gpu import nearest
from test_paged_append_gpu import close, expect
from test_paged_attn_gpu import Device, check, check_row
from zerogravity_amd import _lib as L
from zerogravity_amd import paged, sampling

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ctx():
    c = L.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("prefix", [0, 20, 100])
def test_4096_rows(ctx, prefix):
    """Over 20 tokens 16 queries at a time, over 100 128, one workgroup to a
    block: more blocks than there are CUs."""
    lengths = [(7 * r) % 40 if r % 9 else -1 for r in range(4096)]
    b = ref.Batch(71, 4096, 1, 16, 64, 8, prefix, lengths, F32, BF16)
    d = Device(b)
    out = d.attend(ctx, out=torch.full_like(d.q, 5.0))
    for r in [1, 2, 63, 64, 65, 2047, 2048, 4094, 4095]:
        if lengths[r] >= 0:
            check_row(b, out, r)
    unused = torch.tensor(lengths) < 0
    assert (out.cpu()[unused] == 5.0).all() and out.isfinite().all() and int(d.status) == 0


@pytest.mark.parametrize("io,cache", [(F32, BF16), (BF16, F32)])
def test_1024_kv_heads(ctx, io, cache):
    b = ref.Batch(72, 2, 1024, 1, 64, 4, 9, [7, 30], io, cache)
    d = Device(b)
    check(b, d.attend(ctx))
    # and a token appended to the second row, 1024 query heads beside it
    g = torch.Generator().manual_seed(1)
    k, v, q = (torch.randn(1, 1024, 64, generator=g).to(io) for _ in range(3))
    out = torch.empty(1, 1024, 64, dtype=io, device="cuda")
    paged.append(ctx, d.kv, d.rows, k.cuda(), v.cuda(), torch.tensor([9 + 29], dtype=torch.int32, device="cuda"), q.cuda(),
                 out, rotate=64, theta_scale=0.75, token_rows=torch.ones(1, dtype=torch.int32, device="cuda"),
                 status=d.status)
    torch.cuda.synchronize()
    at = torch.tensor([9 + 29])
    close(out, *expect(q.double(), None, 0, at, 64, 0.75, io))
    page = int(b.table[1, 29 // 4])
    close(d.keys[page, 29 % 4][None], *expect(k.double(), None, 0, at, 64, 0.75, cache))
    assert torch.equal(d.values[page, 29 % 4].cpu(), v[0].to(cache)) and int(d.status) == 0


def test_pages_of_65536_tokens(ctx):
    b = ref.Batch(73, 2, 1, 2, 64, 65536, 65537, [65535, 1], F32, BF16)
    check(b, Device(b).attend(ctx))


def test_one_of_everything(ctx):
    b = ref.Batch(74, 1, 1, 1, 64, 1, 0, [1], F32, F32)
    d = Device(b)
    out = d.attend(ctx)
    assert torch.equal(out.cpu()[0, 0], b.own[0][1][0, 0].float())  # one token has all the weight
    k = torch.full((1, 1, 64), 2.0, device="cuda")
    paged.append(ctx, d.kv, d.rows, k, -k, torch.zeros(1, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    page = int(b.table[0, 0])
    assert (d.keys[page] == 2.0).all() and (d.values[page] == -2.0).all()


def test_100000_tokens_appended(ctx):
    """A whole document in one call, its heads' stride past what a token needs."""
    n, g = 100000, torch.Generator().manual_seed(2)
    order = torch.randperm(n // 32, generator=g).int()
    keys = torch.zeros(n // 32, 32, 1, 64, dtype=BF16, device="cuda")
    values = torch.zeros_like(keys)
    wide = torch.randn(n, 2, 3, 64, generator=g).cuda()
    k, v = wide[:, 0, :1], wide[:, 1, :1]
    paged.append(ctx, paged.cache(keys, values), paged.rows(order.view(1, -1).cuda()), k, v,
                 torch.arange(n, dtype=torch.int32, device="cuda"), token_rows=torch.zeros(n, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    for got, sent in ((keys, k), (values, v)):
        assert torch.equal(got[order.long().cuda()].view(n, 1, 64), sent.to(BF16))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_65535_rows_of_logits(ctx, dtype):
    rows, vocab = 65535, 33
    g = torch.Generator().manual_seed(3)
    x = torch.randn(rows, vocab, generator=g).to(dtype)
    history = torch.randint(0, vocab, (rows, 2), generator=g).int()
    u = dict(history=history, history_lengths=torch.full((rows,), 2, dtype=torch.int32),
             frequency=torch.full((rows,), 0.5))
    want = x.double().scatter_add(1, history.long(), torch.full((rows, 2), -0.5, dtype=torch.float64))
    want = want.float() if dtype == F32 else torch.from_numpy(nearest(want.numpy())).float()
    greedy, out = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, vocab, dtype=dtype, device="cuda")
    sampling.adjust(ctx, x.cuda(), sampling.rules(**device(u)), out, greedy)
    torch.cuda.synchronize()
    assert torch.equal(out.float().cpu(), want)
    assert np.array_equal(greedy.cpu().numpy().view(np.uint32), ref.np_greedy(want.numpy()))


def test_a_vocabulary_of_millions(ctx):
    rows, vocab = 2, (1 << 22) + 5
    g = torch.Generator().manual_seed(4)
    u = random_rules(g, rows, vocab, 500, 20, 2)
    x = torch.randn(rows, vocab, generator=g)
    want = ref.np_adjust(x.numpy(), {k: t.numpy() for k, t in u.items()}, vocab)
    greedy, out = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, vocab, device="cuda")
    sampling.adjust(ctx, x.cuda(), sampling.rules(**device(u)), out, greedy)
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), want)
    assert np.array_equal(greedy.cpu().numpy().view(np.uint32), ref.np_greedy(want))


def test_the_same_row_many_times(ctx):
    """Rows that share their pages, as drafted tokens of one sequence do, and
    a table of one page for everybody."""
    b = ref.Batch(75, 6, 2, 4, 128, 16, 40, [90, 1, 1, 1, 1, 1], F32, BF16)
    b.table[:] = b.table[0].clone()
    b.lengths = [90, 89, 88, 17, 0, -1]
    b.own = [tuple(t[:max(n, 0)] for t in b.own[0]) for n in b.lengths]
    check(b, Device(b).attend(ctx))


def test_a_scale_of_zero_and_below(ctx):
    for scale in (0.0, -0.125):
        b = ref.Batch(76, 3, 2, 4, 128, 16, 33, [0, 50, 7], F32, BF16)
        b.scale = scale
        check(b, Device(b).attend(ctx))
        b = ref.Batch(77, 3, 2, 4, 128, 16, 33, [0, 50, 7], BF16, BF16)
        b.scale = scale
        check(b, Device(b).attend(ctx))

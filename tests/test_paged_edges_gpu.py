"""The paged cache's and the readout's kernels where their work is cut in
other ways: long pieces of a prefix, sixteen query heads to a kv head, full
lists of touched tokens, and calls that are captured or made at once."""
import threading

import numpy as np
import pytest
import torch

import paged_reference as ref
from test_logits_gpu import device, expect, random_rules, same
from test_paged_attn_gpu import TYPES, Device, check, check_row
from zerogravity_amd import _lib as L
from zerogravity_amd import paged, sampling

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ctx():
    c = L.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("bad_page", [False, True])
@pytest.mark.parametrize("io,cache,dim", [t + (64,) for t in TYPES] + [(F32, BF16, 256), (BF16, F32, 128)])
def test_long_pieces_of_a_prefix(ctx, io, cache, dim, bad_page):
    """16384 queries of a kv head: each workgroup goes through the whole
    prefix, 141 tiles of 32 or 282 of 16 tokens; a page past its first third
    is outside the pool."""
    lengths = [r % 5 for r in range(1024)]
    b = ref.Batch(dim, 1024, 2, 16, dim, 16, 4500, lengths, io, cache)
    if bad_page:
        b.prefix[170] = b.keys.shape[0] + 5
    d = Device(b)
    out = d.attend(ctx)
    assert int(d.status) == (1 if bad_page else 0)
    if bad_page:
        b.shared = tuple(torch.cat([t[:170 * 16], t[171 * 16:]]) for t in b.shared)
    for r in (0, 7, 500, 1023):
        check_row(b, out, r)
    assert out.isfinite().all()


@pytest.mark.parametrize("io,cache", TYPES)
def test_sixteen_query_heads_over_a_prefix(ctx, io, cache):
    lengths = [0, 5, 33, 200, -1, 64, 1, 90, 17]
    b = ref.Batch(31, 9, 2, 16, 256, 16, 301, lengths, io, cache)
    check(b, Device(b).attend(ctx))


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("prefix", [0, 20])
def test_sixteen_query_heads_of_many_rows(ctx, io, cache, prefix):
    lengths = [(41 * r) % 70 for r in range(70)]
    b = ref.Batch(34, 70, 1, 16, 256, 8, prefix, lengths, io, cache)
    check(b, Device(b).attend(ctx))


def test_scores_that_are_all_minus_infinity_give_zeros(ctx):
    b = ref.Batch(35, 3, 1, 1, 64, 16, 0, [20, 20, 1], F32, F32, junk=0.0)
    for r, n in ((0, 20), (2, 1)):
        i = torch.arange(n)
        b.keys[b.table[r].long()[i // 16], i % 16, 0] = -torch.inf * b.q[r, 0].sign()
    out = Device(b).attend(ctx)
    assert (out[0] == 0).all() and (out[2] == 0).all()
    check_row(b, out, 1)


@pytest.mark.parametrize("io,cache", [(F32, BF16), (BF16, F32)])
def test_captured_calls_over_a_prefix(ctx, io, cache):
    """Many queries over the prefix: replays follow lengths, tables and
    queries, with eager calls of the same batch between them."""
    b = ref.Batch(32, 16, 2, 4, 256, 16, 600, [100] * 16, io, cache, junk=0.0)
    d = Device(b)
    ws = torch.empty(paged.attend_workspace(d.kv, d.rows, 8), dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(d.q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attend(ctx, d.kv, d.rows, d.lengths, d.q, b.scale, out=out, workspace=ws)
    gen = torch.Generator().manual_seed(8)
    for step in range(4):
        d.lengths.copy_(torch.randint(0, 101, (16,), generator=gen))
        d.q.copy_(torch.randn(d.q.shape, generator=gen))
        d.table.copy_(d.table[torch.randperm(16, generator=gen).cuda()])
        graph.replay()
        torch.cuda.synchronize()
        eager = paged.attend(ctx, d.kv, d.rows, d.lengths, d.q, b.scale)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), step


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("rows,kv_heads,group,dim,prefix", [(65, 2, 16, 256, 1601), (65, 4, 5, 128, 2401),
                                                           (100, 8, 1, 64, 3601), (40, 1, 16, 256, 4999)])
def test_many_queries_over_a_prefix(ctx, io, cache, rows, kv_heads, group, dim, prefix):
    """So many that 128 of them go through a tile together, with long, empty
    and unused rows beside."""
    lengths = [(37 * r) % 90 if r % 7 else -1 if r % 2 else 0 for r in range(rows)]
    lengths[3], lengths[rows - 1] = 700, 1
    b = ref.Batch(rows + dim, rows, kv_heads, group, dim, 16, prefix, lengths, io, cache)
    d = Device(b)
    out = d.attend(ctx, out=torch.full_like(d.q, 77.0))
    check(b, out)
    assert int(d.status) == 0 and all((out[r] == 77.0).all() for r, n in enumerate(lengths) if n < 0)


@pytest.mark.parametrize("io,cache", [(F32, BF16), (BF16, F32)])
def test_captured_calls_of_many_queries(ctx, io, cache):
    b = ref.Batch(33, 40, 1, 16, 256, 16, 4999, [100] * 40, io, cache, junk=0.0)
    d = Device(b)
    ws = torch.empty(paged.attend_workspace(d.kv, d.rows, 16), dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(d.q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attend(ctx, d.kv, d.rows, d.lengths, d.q, b.scale, out=out, workspace=ws)
    gen = torch.Generator().manual_seed(9)
    for step in range(4):
        d.lengths.copy_(torch.randint(0, 101, (40,), generator=gen))
        d.q.copy_(torch.randn(d.q.shape, generator=gen))
        d.table.copy_(d.table[torch.randperm(40, generator=gen).cuda()])
        graph.replay()
        torch.cuda.synchronize()
        eager = paged.attend(ctx, d.kv, d.rows, d.lengths, d.q, b.scale)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), step


@pytest.mark.parametrize("rows,group,prefix", [(1, 4, 700), (4, 4, 700), (5, 4, 5000), (17, 16, 5000), (30, 16, 5000),
                                               (40, 16, 5000), (40, 16, 0), (40, 1, 31)])
@pytest.mark.parametrize("io,cache", TYPES)
def test_calls_stay_inside_their_workspace(ctx, io, cache, rows, group, prefix):
    """What the largest batch's workspace is sized for serves each of these, and
    nothing behind it changes."""
    b = ref.Batch(rows, rows, 2, group, 64, 16, prefix, [(29 * r) % 50 for r in range(rows)], io, cache, wide=4)
    d = Device(b)
    most = L.lib().zg_paged_attn_workspace_bytes(d.kv, L.PagedRows(4096, 40, 4, 4096, 5000), 2 * group)
    need = paged.attend_workspace(d.kv, d.rows, 2 * group)
    assert need <= most
    for n in (need, most):
        ws = torch.full((most + 65536,), 165, dtype=torch.uint8, device="cuda")
        check(b, d.attend(ctx, workspace=ws[:n]))
        assert (ws[n:] == 165).all()


def test_threads_share_a_context(ctx):
    """Two threads, each with its stream, its batch and its logits."""
    cases, want = [], []
    for i in range(2):
        d = Device(ref.Batch(40 + i, 9, 2, 4, 128, 16, 400 * i, [50 * (r + 1) for r in range(9)], F32, BF16))
        x = torch.randn(9, 20000, generator=torch.Generator().manual_seed(i)).cuda()
        u = sampling.rules(**device(random_rules(torch.Generator().manual_seed(i), 9, 20000, 300, 9, 3)))
        cases.append((d, x, u))
        want.append((d.attend(ctx), sampling.adjust(ctx, x, u, torch.empty_like(x))))
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        d, x, u = cases[i]
        stream = torch.cuda.Stream()
        for step in range(20):
            out = paged.attend(ctx, d.kv, d.rows, d.lengths, d.q, d.b.scale, stream=stream)
            with torch.cuda.stream(stream):
                logits = torch.empty_like(x)
            sampling.adjust(ctx, x, u, logits, stream=stream)
            stream.synchronize()
            if not torch.equal(out, want[i][0]) or not same(logits, want[i][1]):
                wrong.append((i, step))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not wrong and not any(t.is_alive() for t in threads)


@pytest.mark.parametrize("rows,vocab,history,biases,dtype", [
    (96, 4000, 9000, 700, F32), (50, 8191, 16000, 1100, BF16), (1, 1000, 6000, 900, F32), (1100, 4000, 6000, 600, F32),
    (1100, 4000, 6000, 600, BF16)])
def test_most_of_a_vocabulary_is_touched(ctx, rows, vocab, history, biases, dtype):
    """More tokens of a slice change than its list holds, more biases than a
    workgroup has threads, many of them for the same tokens."""
    g = torch.Generator().manual_seed(rows)
    u = random_rules(g, rows, vocab, history, biases, 2)
    u["history_lengths"][:] = history
    u["bias_lengths"][:] = biases
    x = (3 * torch.randn(rows, vocab, generator=g)).to(dtype)
    want, ids = expect(x, u, vocab)
    greedy, out = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, vocab, dtype=dtype, device="cuda")
    sampling.adjust(ctx, x.cuda(), sampling.rules(**device(u)), out, greedy)
    torch.cuda.synchronize()
    assert same(out.cpu(), want) and np.array_equal(greedy.cpu().numpy().view(np.uint32), ids)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(204, 20480), (205, 20480), (250, 17001), (256, 17001), (257, 17001)])
def test_slices_that_run_at_once(ctx, dtype, rows, vocab):
    """1020, 1025, 1250, 1280 and 1285 slices; in place on odd strides."""
    g = torch.Generator().manual_seed(vocab)
    u = random_rules(g, rows, vocab, 300, 20, 5)
    x = torch.randn(rows, vocab, generator=g).to(dtype)
    want, ids = expect(x, u, vocab)
    for pad in (0, 3):
        wide = torch.zeros(rows, vocab + pad, dtype=dtype, device="cuda")
        wide[:, :vocab] = x.cuda()
        greedy = torch.empty(rows, dtype=torch.int32, device="cuda")
        sampling.adjust(ctx, wide[:, :vocab], sampling.rules(**device(u)), greedy=greedy)
        torch.cuda.synchronize()
        assert same(wide[:, :vocab].cpu(), want) and np.array_equal(greedy.cpu().numpy().view(np.uint32), ids)
        assert (wide[:, vocab:] == 0).all()


def test_limits_are_refused(ctx):
    b = ref.Batch(50, 2, 2, 4, 128, 16, 20, [5, 6], F32, BF16)
    d = Device(b)
    with pytest.raises(L.ZgError) as e:
        paged.attend(ctx, d.kv, d.rows, d.lengths, d.q, 3e38)
    assert e.value.code == L.E_MALFORMED
    k = torch.zeros(2, 2, 128, device="cuda")
    at = torch.zeros(2, dtype=torch.int32, device="cuda")
    rc = L.lib().zg_paged_append_device(ctx.h, d.kv, d.rows, 1 << 24, 0, None, 0, 0, k.data_ptr(), 256, k.data_ptr(), 256,
                                        L.F32, None, None, 0.0, 0, 1.0, at.data_ptr(), at.data_ptr(), None, None, None)
    assert rc == L.E_LIMIT

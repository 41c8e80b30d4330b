"""zg_paged_attn_device against the softmax's definition in 64 bits, within
paged_reference.attend_bound."""
import math

import pytest
import torch

import paged_reference as ref
from zerogravity_amd import _lib as L
from zerogravity_amd import paged

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ctx():
    c = L.Context(0)
    yield c
    c.close()


class Device:
    """A Batch on the GPU."""

    def __init__(self, b):
        self.b = b
        self.keys, self.values, self.table, self.prefix = (t.cuda() for t in (b.keys, b.values, b.table, b.prefix))
        self.lengths = torch.tensor(b.lengths, dtype=torch.int32, device="cuda")
        self.q = b.q.cuda()
        self.kv = paged.cache(self.keys, self.values)
        self.rows = paged.rows(self.table, self.prefix, b.prefix_tokens)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def attend(self, ctx, **more):
        out = paged.attend(ctx, self.kv, self.rows, self.lengths, self.q, self.b.scale, status=self.status, **more)
        torch.cuda.synchronize()
        return out


def check_row(b, got, r, skip=()):
    want, mass, dots, tokens = b.reference(r, skip)
    bound = ref.attend_bound(want, mass, dots, tokens, want.shape[-1], b.q.dtype, b.keys.dtype)
    off = (got[r].double().cpu() - want).abs()
    assert (off <= bound).all(), (r, tokens, float((off / bound).max()))


def check(b, got):
    for r, n in enumerate(b.lengths):
        if n >= 0:
            check_row(b, got, r)


TYPES = [(F32, BF16), (BF16, BF16), (F32, F32), (BF16, F32)]


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("kv_heads,group,dim", [(2, 4, 256), (4, 5, 128), (1, 16, 64), (8, 1, 128), (1, 1, 256),
                                                (2, 8, 64), (3, 7, 256)])
def test_layouts_and_types(ctx, io, cache, kv_heads, group, dim):
    lengths = [0, 1, 15, 33, 64, 130]
    b = ref.Batch(dim + group, len(lengths), kv_heads, group, dim, 7, 45, lengths, io, cache)
    d = Device(b)
    check(b, d.attend(ctx))
    assert int(d.status) == 0


@pytest.mark.parametrize("page", [1, 2, 5, 16, 31, 32, 33, 100, 256, 4096])
def test_page_sizes(ctx, page):
    lengths = [3, 250, 31, 97]
    b = ref.Batch(page, 4, 2, 4, 256, page, 70, lengths, F32, BF16)
    check(b, Device(b).attend(ctx))


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 513])
def test_lengths_around_the_tiles(ctx, n):
    for prefix, own in ((n, 0), (0, n), (n, n)):
        b = ref.Batch(n, 2, 2, 4, 128, 16, prefix, [own, max(own - 1, 0)], F32, BF16)
        check(b, Device(b).attend(ctx))


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("rows", [2, 5, 17, 64, 65, 130])
def test_batches_over_a_prefix(ctx, io, cache, rows):
    """The rows of a kv head fill one tile of the prefix's products, part of
    one, or many; some rows are empty beside it and some not in use."""
    lengths = [(37 * r) % 90 if r % 7 else -1 if r % 2 else 0 for r in range(rows)]
    b = ref.Batch(rows, rows, 2, 4, 256, 16, 301, lengths, io, cache)
    d = Device(b)
    mark = torch.full_like(d.q, 77.0)
    out = d.attend(ctx, out=mark)
    check(b, out)
    for r, n in enumerate(lengths):
        assert n >= 0 or (out[r] == 77.0).all()


@pytest.mark.parametrize("io,cache", TYPES)
def test_long_contexts(ctx, io, cache):
    b = ref.Batch(5, 3, 1, 4, 128, 64, 5003, [9001, 0, 4], io, cache)
    check(b, Device(b).attend(ctx))
    b = ref.Batch(6, 1, 2, 4, 256, 16, 0, [12345], io, cache)
    check(b, Device(b).attend(ctx))


def test_many_short_rows(ctx):
    g = torch.Generator().manual_seed(2)
    lengths = [int(x) for x in torch.randint(0, 40, (1500,), generator=g)]
    b = ref.Batch(3, 1500, 1, 2, 64, 8, 0, lengths, F32, BF16)
    check(b, Device(b).attend(ctx))


def test_one_long_row_among_short_ones(ctx):
    lengths = [5] * 20 + [20000] + [0] * 10 + [64]
    b = ref.Batch(4, len(lengths), 2, 4, 64, 32, 0, lengths, BF16, BF16)
    check(b, Device(b).attend(ctx))


def test_rows_without_tokens_give_zeros(ctx):
    for io, cache in TYPES:
        b = ref.Batch(1, 3, 2, 4, 256, 16, 0, [0, 0, 0], io, cache)
        assert (Device(b).attend(ctx) == 0).all()


@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf, 3e38])
@pytest.mark.parametrize("cache", [F32, BF16])
def test_slots_past_a_length_do_not_matter(ctx, junk, cache):
    """Whole pages and the tail of the last one hold NaN or infinities; so
    may the table's entries past the row and the queries of unused rows."""
    lengths = [1, 17, 40, -1]
    b = ref.Batch(9, 4, 2, 4, 128, 16, 21, lengths, F32, cache, junk=junk, wide=6)
    b.table[1, 3:] = torch.tensor([2 ** 31 - 1, -2 ** 31, 7])
    b.q[3] = math.nan
    d = Device(b)
    check(b, d.attend(ctx))
    assert int(d.status) == 0


def test_infinite_and_nan_tokens_come_through(ctx):
    """What a row attends to it gets: a NaN key or an infinite score makes
    that row NaN, as the formula does, an infinite value an infinite sum; the
    other rows keep theirs."""
    b = ref.Batch(11, 4, 1, 4, 128, 16, 8, [30, 30, 30, 30], F32, F32, junk=0.0)
    page = b.table[:, 0].long()
    b.keys[page[0], 3, 0, 5] = math.nan
    b.keys[page[1], 3] = math.inf * b.q[1, 0].sign()  # query 0's score is +inf
    b.values[page[2], 3, 0, 9] = math.inf
    out = Device(b).attend(ctx).cpu()
    assert out[0].isnan().all() and out[1, 0].isnan().all()
    assert (out[2, :, 9] == math.inf).all() and out[2, :, :9].isfinite().all() and out[2, :, 10:].isfinite().all()
    check_row(b, out, 3)


def test_keys_that_score_minus_infinity_weigh_nothing(ctx):
    b = ref.Batch(12, 2, 1, 1, 64, 16, 0, [20, 20], F32, F32, junk=0.0)
    page = b.table[0, 0].long()
    b.keys[page, 2:9, 0] = -math.inf * b.q[0, 0].sign()
    got = Device(b).attend(ctx)
    check_row(b, got, 0, skip=range(2, 9))
    check_row(b, got, 1)


def test_steep_scores(ctx):
    """One token holds nearly all the weight, others are exp(-80) and less;
    and the maximum arrives last."""
    b = ref.Batch(13, 1, 1, 4, 128, 16, 100, [100], F32, BF16)
    b.scale = 4.0
    check(b, Device(b).attend(ctx))
    rising = torch.arange(200).view(-1, 1, 1) * 0.05 * b.q[0, 0].sign().double()
    for side, pages, n, at in ((0, b.prefix, 100, 0), (1, b.table[0], 100, 100)):
        i = torch.arange(n)
        keys = rising[at:at + n].to(BF16)
        b.keys[pages.long()[i // 16], i % 16] = keys
        if side:
            b.own[0] = (keys.double(), b.own[0][1])
        else:
            b.shared = (keys.double(), b.shared[1])
    b.scale = 1.0
    check(b, Device(b).attend(ctx))


@pytest.mark.parametrize("where", ["own", "prefix", "all"])
@pytest.mark.parametrize("page_id", [-1, 2 ** 31 - 1, "count"])
@pytest.mark.parametrize("io,cache", TYPES)
def test_pages_outside_the_pool_are_left_out(ctx, where, page_id, io, cache):
    b = ref.Batch(14, 2, 2, 4, 128, 16, 32, [50, 20], io, cache)
    bad = b.keys.shape[0] if page_id == "count" else page_id
    if where != "prefix":
        b.table[0, 1] = bad
    if where != "own":
        b.prefix[0] = bad
    if where == "all":
        b.table[0, :], b.prefix[:] = bad, bad
    d = Device(b)
    out = d.attend(ctx)
    assert int(d.status) == 1
    skip = range(16, 32) if where == "own" else ()
    if where != "own":
        first = 16 if where == "prefix" else 32
        b.shared = tuple(t[first:] for t in b.shared)
    if where == "all":
        assert (out[0] == 0).all()
    else:
        check_row(b, out, 0, skip)
    check_row(b, out, 1)


def test_lengths_past_the_table_are_cut(ctx):
    b = ref.Batch(15, 3, 2, 4, 128, 16, 5, [32, 20, 7], F32, BF16)
    d = Device(b)
    d.lengths = torch.tensor([2 ** 31 - 1, 20, 7], dtype=torch.int32, device="cuda")
    out = d.attend(ctx)
    assert int(d.status) == 2
    check(b, out)


def test_strides_interleaved_pools_and_in_place(ctx):
    b = ref.Batch(16, 5, 2, 4, 128, 16, 40, [3, 90, 0, 17, 64], F32, BF16)
    d = Device(b)
    plain = d.attend(ctx).cpu()
    check(b, plain)
    n = b.keys.shape[0]
    both = torch.full((n, 3, 16, 2, 128), math.nan, dtype=BF16, device="cuda")
    both[:, 0], both[:, 2] = d.keys, d.values
    d.kv = paged.cache(both[:, 0], both[:, 2])
    wide = torch.zeros(5, 11, 128, device="cuda")
    wide[:, :8] = d.q
    table = torch.full((5, 9), -1, dtype=torch.int32, device="cuda")
    table[:, :b.table.shape[1]] = d.table
    d.rows = paged.rows(table[:, :b.table.shape[1]], d.prefix, 40)
    keep = d.q
    d.q = wide[:, :8]
    out = torch.full((5, 13, 128), 5.0, device="cuda")
    got = d.attend(ctx, out=out[:, :8])
    assert torch.equal(got.cpu(), plain) and (out[:, 8:] == 5.0).all()
    d.q = keep
    got = d.attend(ctx, out=keep)
    assert torch.equal(got.cpu(), plain)


def test_the_same_bits_every_time(ctx):
    """Two calls, another stream, and a table with the pages elsewhere."""
    b = ref.Batch(17, 9, 2, 4, 256, 16, 600, [0, 1, 50, 300, 17, 1000, 3, 64, 2000], F32, BF16)
    d = Device(b)
    first = d.attend(ctx).cpu()
    check(b, first)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    assert torch.equal(first, d.attend(ctx, stream=stream).cpu())
    swap = torch.randperm(b.keys.shape[0], generator=torch.Generator().manual_seed(4))
    back = swap.argsort().int().cuda()
    d.keys, d.values = d.keys[swap.cuda()].contiguous(), d.values[swap.cuda()].contiguous()
    d.kv = paged.cache(d.keys, d.values)
    d.table = torch.where(d.table < 0, d.table, back[d.table.long().clamp(min=0)]).contiguous()
    d.rows = paged.rows(d.table, back[d.prefix.long()], 600)
    assert torch.equal(first, d.attend(ctx).cpu())


def test_captured_calls_follow_the_tables(ctx):
    """Two graphs over one cache, each with its workspace, replayed in turn
    with other lengths, tables and queries; eager work between them."""
    b = ref.Batch(18, 6, 2, 4, 128, 16, 77, [200] * 6, F32, BF16, junk=0.0)
    d = Device(b)
    need = paged.attend_workspace(d.kv, d.rows, 8)
    graphs = []
    for i in range(2):
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        out = torch.zeros_like(d.q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            paged.attend(ctx, d.kv, d.rows, d.lengths, d.q, b.scale * (1 + i), out=out, workspace=ws)
        graphs.append((g, out, ws))
    gen = torch.Generator().manual_seed(5)
    for step in range(4):
        d.lengths.copy_(torch.randint(0, 201, (6,), generator=gen))
        d.q.copy_(torch.randn(d.q.shape, generator=gen))
        d.table.copy_(d.table[torch.randperm(6, generator=gen).cuda()])
        for g, out, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i, (_, out, _) in enumerate(graphs):
            eager = paged.attend(ctx, d.kv, d.rows, d.lengths, d.q, b.scale * (1 + i))
            torch.cuda.synchronize()
            assert torch.equal(out, eager), (step, i)


def test_two_streams_at_once(ctx):
    cases = [Device(ref.Batch(19 + i, 16, 2, 4, 256, 16, 1000 * i, [100 * (r + 1) for r in range(16)], F32, BF16))
             for i in range(2)]
    want = [d.attend(ctx).cpu() for d in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for rep in range(5):
        for d, s in zip(cases, streams):
            outs.append(paged.attend(ctx, d.kv, d.rows, d.lengths, d.q, d.b.scale, stream=s))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o.cpu(), want[i % 2]), i


def test_offsets_past_32_bits(ctx):
    """Pages whose elements lie past 2^32 in the pool (and bytes past 2^33)."""
    page, heads, dim = 64, 8, 128
    per = page * heads * dim
    total = (1 << 32) // per + 40
    keys = torch.empty(total, page, heads, dim, dtype=BF16, device="cuda")
    values = torch.empty_like(keys)
    b = ref.Batch(21, 2, heads, 2, dim, page, 70, [100, 190], F32, BF16)
    n = b.keys.shape[0]
    keys[total - n:], values[total - n:] = b.keys.cuda(), b.values.cuda()
    d = Device(b)
    d.kv = paged.cache(keys, values)
    d.table = torch.where(d.table < 0, d.table, d.table + (total - n))
    d.rows = paged.rows(d.table, d.prefix + (total - n), 70)
    check(b, d.attend(ctx))
    # and an append there
    k = torch.randn(1, heads, dim, device="cuda")
    at = torch.tensor([70 + 100], dtype=torch.int32, device="cuda")
    paged.append(ctx, d.kv, d.rows, k, -k, at, token_rows=torch.zeros(1, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    where = int(d.table[0, 100 // page])
    assert torch.equal(keys[where, 100 % page], k[0].to(BF16)) and torch.equal(values[where, 100 % page], -k[0].to(BF16))
    del keys, values, d
    torch.cuda.empty_cache()


def test_refusals(ctx):
    b = ref.Batch(22, 2, 2, 4, 128, 16, 20, [5, 6], F32, BF16)
    d = Device(b)

    def code(**change):
        a = dict(kv=d.kv, r=d.rows, lengths=d.lengths, q=d.q, scale=0.1)
        a.update(change)
        with pytest.raises(L.ZgError) as e:
            paged.attend(ctx, **a)
        return e.value.code

    assert code(scale=math.nan) == code(scale=math.inf) == L.E_MALFORMED
    assert code(q=d.q[:1]) == code(q=d.q[:, :7].contiguous()) == code(q=d.q[..., :64]) == L.E_MALFORMED
    assert code(q=d.q.half()) == L.E_UNSUPPORTED
    assert code(lengths=d.lengths[:1]) == code(lengths=d.lengths.long()) == code(lengths=d.lengths.cpu()) == L.E_MALFORMED
    assert code(out=torch.empty(2, 8, 128, dtype=BF16, device="cuda")) == L.E_MALFORMED
    assert code(workspace=torch.empty(8, dtype=torch.uint8, device="cuda")) == L.E_MALFORMED
    assert code(r=paged.rows(d.table, d.prefix, 33)) == L.E_MALFORMED
    assert code(r=paged.rows(d.table, None, 20)) == L.E_MALFORMED
    assert code(q=torch.zeros(2, 34, 128, device="cuda")) == L.E_MALFORMED  # 17 query heads to a kv head
    odd = torch.zeros(2 * 8 * 128 + 4, device="cuda")[2:-2].view(2, 8, 128)
    assert code(q=odd) == L.E_MALFORMED  # 8-byte aligned
    assert code(q=torch.zeros(2, 1028, device="cuda")[:, :1024].unflatten(1, (8, 128))) == L.E_MALFORMED

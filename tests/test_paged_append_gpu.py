"""zg_paged_append_device against the operator's definition in 64 bits.

Bounds: a norm is a mean of squares summed in 32 bits (dim terms in a tree of
depth 10 at most, 12 U with the square and the division, half of it after the
root) and three more roundings, 10 U; a turned element is x c - o s with c
and s off by 4 U at most (argument within pi / 4 rounded once, 2 U of the
function) and three roundings: 17 U (|x| + |o|) altogether, plus what the
angle itself is off in 64 bits: position * frequency * (pair + 3) 2^-53.  The
store rounds once more."""
import math

import numpy as np
import pytest
import torch

import paged_reference as ref
from zerogravity_amd import _lib as L
from zerogravity_amd import paged

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
THETA = float(np.float32(1e7 ** (-2 / 64)))


@pytest.fixture(scope="module")
def ctx():
    c = L.Context(0)
    yield c
    c.close()


def expect(x, gamma, eps, positions, rotate, theta, out_type):
    """The 64-bit result of normed and turned heads and its bound."""
    y = ref.norm(x, gamma, eps) if gamma is not None else x
    z = ref.rotate(y, positions, rotate, theta)
    h = rotate // 2
    other = torch.cat([y[..., h:rotate], y[..., :h], torch.zeros_like(y[..., rotate:])], -1).abs()
    i = torch.arange(h, dtype=torch.float64)
    angle = positions.double()[:, None, None] * theta ** i * (i + 3) * 2.0 ** -53
    off = torch.cat([angle, angle, torch.zeros(angle.shape[0], 1, y.shape[-1] - rotate)], -1)
    return z, (17 * ref.U + off) * (y.abs() + other) + ref.half_step(out_type) * z.abs() + 1e-30


def close(got, want, bound):
    bad = (got.double().cpu() - want).abs() > bound
    assert not bad.any(), (int(bad.sum()), float(((got.double().cpu() - want).abs() / bound).max()))


@pytest.mark.parametrize("tokens,rows,heads,kv_heads,dim,rotate,page,prefix,first,io,cache,norm", [
    (1, 1, 8, 2, 256, 64, 16, 0, 2047, F32, BF16, True),
    (32, 32, 8, 2, 256, 64, 16, 100, 2048, F32, BF16, True),
    (33, 33, 8, 2, 256, 64, 1, 7, 0, BF16, BF16, True),
    (700, 3, 20, 4, 128, 128, 7, 5, 0, BF16, F32, False),
    (515, 2, 4, 4, 64, 32, 13, 0, 500000, F32, F32, True),
    (5, 2, 0, 1, 64, 8, 64, 0, 3, F32, BF16, True),
    (9, 9, 16, 1, 128, 0, 3, 2, 11, BF16, BF16, True),
    (40, 4, 3, 3, 256, 256, 5, 0, 1, F32, F32, False)])
def test_append_matches_the_definition(ctx, tokens, rows, heads, kv_heads, dim, rotate, page, prefix, first, io, cache,
                                       norm):
    g = torch.Generator().manual_seed(tokens + heads)
    of = torch.randint(0, rows, (tokens,), generator=g).int()
    own, held = torch.zeros(tokens, dtype=torch.int32), [first + r for r in range(rows)]
    for t in range(tokens):
        own[t] = held[of[t]]
        held[of[t]] += 1
    wide = max(held) // page + 1
    used = {(int(r), int(p) // page) for r, p in zip(of, own)}
    pages = len(used) + 2
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((rows, wide), -5, dtype=torch.int32)
    for (r, i), p in zip(sorted(used), order):
        table[r, i] = p
    both = torch.randn(pages, 2, page, kv_heads, dim, generator=g).to(cache)  # keys and values interleaved
    before = both.clone()
    proj = torch.randn(tokens, (2 * heads + 2 * kv_heads) * dim + 8, generator=g).to(io)  # [q | gate] heads, k, v
    qn, kn = (1 + 0.1 * torch.randn(2, dim, generator=g)) if norm else (None, None)
    positions = own + prefix
    theta = THETA if rotate == 64 else float(np.float32(10000.0 ** (-2.0 / max(rotate, 2))))
    d = [None if x is None else x.cuda() for x in (proj, table, both, positions, of, qn, kn)]
    dq = d[0][:, :2 * heads * dim].view(tokens, heads, 2 * dim)[..., :dim] if heads else None
    dk = d[0][:, 2 * heads * dim:(2 * heads + kv_heads) * dim].view(tokens, kv_heads, dim)
    dv = d[0][:, (2 * heads + kv_heads) * dim:(2 * heads + 2 * kv_heads) * dim].view(tokens, kv_heads, dim)
    out = torch.full((tokens, heads, dim), math.nan, dtype=io, device="cuda") if heads else None
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv = paged.cache(d[2][:, 0], d[2][:, 1])
    paged.append(ctx, kv, paged.rows(d[1], prefix_tokens=prefix), dk, dv, d[3], dq, out, d[5], d[6], 1e-6, rotate,
                 theta, d[4], status)
    torch.cuda.synchronize()
    assert int(status) == 0
    x = proj.double()
    if heads:
        want, bound = expect(x[:, :2 * heads * dim].view(tokens, heads, 2 * dim)[..., :dim], qn, 1e-6, positions,
                             rotate, theta, io)
        close(out, want, bound)
    want, bound = expect(x[:, 2 * heads * dim:(2 * heads + kv_heads) * dim].view(tokens, kv_heads, dim), kn, 1e-6,
                         positions, rotate, theta, cache)
    pg, slot = table[of.long(), (own // page).long()].long(), (own % page).long()
    got = d[2].cpu()
    close(got[pg, 0, slot], want, bound)
    v = proj[:, (2 * heads + kv_heads) * dim:(2 * heads + 2 * kv_heads) * dim].view(tokens, kv_heads, dim)
    assert torch.equal(got[pg, 1, slot], v.to(cache))  # a value is rounded, nothing else
    before[pg, 0, slot], before[pg, 1, slot] = got[pg, 0, slot], got[pg, 1, slot]
    assert torch.equal(got, before)  # every other slot as it was


def simple(ctx, **change):
    """Three tokens over two rows of two pages of four, and what they leave."""
    a = dict(positions=[0, 5, 7], token_rows=[0, 1, 1], table=[[0, 1], [2, 3]], prefix_tokens=0)
    a.update(change)
    n = len(a["positions"])
    keys = torch.zeros(4, 4, 1, 64, device="cuda")
    values = torch.zeros_like(keys)
    k = torch.ones(n, 1, 64, device="cuda") * torch.arange(1, n + 1, device="cuda").view(-1, 1, 1)
    q, out = torch.ones(n, 2, 64, device="cuda"), torch.full((n, 2, 64), -9.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ints = [None if a[x] is None else torch.tensor(a[x], dtype=torch.int32, device="cuda")
            for x in ("positions", "token_rows", "table")]
    paged.append(ctx, paged.cache(keys, values), paged.rows(ints[2], prefix_tokens=a["prefix_tokens"]), k, -k, ints[0],
                 q, out, token_rows=ints[1], status=status)
    torch.cuda.synchronize()
    assert torch.equal(keys, -values)
    return keys[:, :, 0, 0].cpu().tolist(), out[:, 0, 0].cpu().tolist(), int(status)


def test_places_that_are_not_there(ctx):
    empty = [[0.0] * 4 for _ in range(4)]

    def left(*at):
        want = [list(r) for r in empty]
        for page, slot, value in at:
            want[page][slot] = float(value)
        return want

    assert simple(ctx) == (left((0, 0, 1), (3, 1, 2), (3, 3, 3)), [1, 1, 1], 0)
    # a negative position: the token is not there at all
    assert simple(ctx, positions=[0, -1, 7]) == (left((0, 0, 1), (3, 3, 3)), [1, -9, 1], 0)
    # past the table, before the prefix, of no row: the query alone
    assert simple(ctx, positions=[0, 8, 7]) == (left((0, 0, 1), (3, 3, 3)), [1, 1, 1], 2)
    assert simple(ctx, positions=[0, 2 ** 31 - 1, 7]) == (left((0, 0, 1), (3, 3, 3)), [1, 1, 1], 2)
    assert simple(ctx, positions=[2, 3, 10], prefix_tokens=3) == (left((2, 0, 2), (3, 3, 3)), [1, 1, 1], 2)
    assert simple(ctx, token_rows=[0, 2, 1]) == (left((0, 0, 1), (3, 3, 3)), [1, 1, 1], 2)
    assert simple(ctx, token_rows=[0, -1, 1]) == (left((0, 0, 1), (3, 3, 3)), [1, 1, 1], 2)
    # pages outside the pool
    assert simple(ctx, table=[[0, 1], [2, 4]]) == (left((0, 0, 1)), [1, 1, 1], 1)
    assert simple(ctx, table=[[-1, 1], [2, 3]], positions=[0, 8, 7]) == (left((3, 3, 3)), [1, 1, 1], 3)
    # no rows given: token t is row t's
    assert simple(ctx, positions=[0, 5], token_rows=None) == (left((0, 0, 1), (3, 1, 2)), [1, 1], 0)


def test_far_positions_keep_their_angle(ctx):
    """Position 2^31 - 1: the angle in 64 bits is off by 2e9 * (i + 3) 2^-53."""
    p = torch.tensor([2 ** 31 - 1, 262143], dtype=torch.int32)
    keys = torch.zeros(1, 2, 1, 64, device="cuda")
    q = torch.randn(2, 1, 64, generator=torch.Generator().manual_seed(3))
    out = torch.empty(2, 1, 64, device="cuda")
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    k = torch.zeros(2, 1, 64, device="cuda")
    paged.append(ctx, paged.cache(keys, keys.clone()), paged.rows(table), k, k, p.cuda(), q.cuda(), out, rotate=64,
                 theta_scale=THETA)
    torch.cuda.synchronize()
    want, bound = expect(q.double(), None, 0, p, 64, THETA, F32)
    close(out, want, bound)


def test_queries_in_place_and_on_a_stream(ctx):
    g = torch.Generator().manual_seed(8)
    q, k = torch.randn(6, 4, 128, generator=g), torch.randn(6, 2, 128, generator=g)
    table = torch.arange(6, dtype=torch.int32).view(6, 1).cuda()
    p = torch.arange(6, dtype=torch.int32)
    stream = torch.cuda.Stream()
    results = []
    for place in (False, True):
        keys = torch.zeros(6, 8, 2, 128, dtype=BF16, device="cuda")
        dq, dk = q.cuda(), k.cuda()
        out = dq if place else torch.empty_like(dq)
        kv, rows, dp = paged.cache(keys, keys.clone()), paged.rows(table), p.cuda()
        stream.wait_stream(torch.cuda.current_stream())
        paged.append(ctx, kv, rows, dk, dk, dp, dq, out, rotate=64, theta_scale=THETA,
                     stream=stream if place else None)
        torch.cuda.synchronize()
        results.append((out.cpu(), keys.cpu()))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])


def test_a_captured_append_follows_its_positions(ctx):
    """Replays with other positions, tables and values, eager work between
    them; each equals the eager call's bits."""
    n, rows = 4, 4
    k, v = torch.zeros(n, 2, 64, device="cuda"), torch.zeros(n, 2, 64, device="cuda")
    q, out = torch.zeros(n, 4, 64, device="cuda"), torch.zeros(n, 4, 64, device="cuda")
    p = torch.zeros(n, dtype=torch.int32, device="cuda")
    table = torch.zeros(rows, 3, dtype=torch.int32, device="cuda")
    keys = torch.zeros(12, 4, 2, 64, dtype=BF16, device="cuda")
    values = torch.zeros_like(keys)
    kv, r = paged.cache(keys, values), paged.rows(table)

    def call():
        paged.append(ctx, kv, r, k, v, p, q, out, rotate=32, theta_scale=0.5)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    g = torch.Generator().manual_seed(1)
    for step in range(4):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g))
        p.copy_(torch.randint(-1, 12, (n,), generator=g))
        table.copy_(torch.randperm(12, generator=g).view(rows, 3))
        got = []
        for run in (graph.replay, call):
            keys.zero_(), values.zero_(), out.fill_(-3)
            run()
            torch.cuda.synchronize()
            got.append([t.cpu() for t in (keys, values, out)])
        assert all(torch.equal(a, b) for a, b in zip(*got)), step


def test_refusals(ctx):
    keys = torch.zeros(2, 4, 2, 64, device="cuda")
    kv = paged.cache(keys, keys.clone())
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    k, q = torch.zeros(2, 2, 64, device="cuda"), torch.zeros(2, 4, 64, device="cuda")
    p = torch.zeros(2, dtype=torch.int32, device="cuda")
    gamma = torch.ones(64, device="cuda")

    def code(fn=None, **change):
        a = dict(k=k, v=k, positions=p, q=q, q_out=torch.empty_like(q), rotate=64, theta_scale=0.9)
        a.update(change)
        with pytest.raises(L.ZgError) as e:
            paged.append(ctx, a.pop("kv", kv), a.pop("rows", paged.rows(table)), **a)
        return e.value.code

    assert code(rotate=4) == code(rotate=72) == L.E_MALFORMED
    assert code(theta_scale=0.0) == code(theta_scale=1.5) == code(theta_scale=math.nan) == L.E_MALFORMED
    assert code(k_norm=gamma, eps=0.0) == code(q_norm=gamma, eps=math.nan) == L.E_MALFORMED
    assert code(q_norm=gamma[:32]) == code(q_norm=gamma.double()) == L.E_MALFORMED
    assert code(positions=p.long()) == code(positions=p[:1]) == code(positions=p.cpu()) == L.E_MALFORMED
    assert code(k=k[:, :1], v=k[:, :1]) == code(v=k.bfloat16()) == code(k=k.transpose(0, 1)) == L.E_MALFORMED
    assert code(q_out=None) == code(q_out=q.bfloat16()) == L.E_MALFORMED
    assert code(k=k.half(), v=k.half(), q=q.half(), q_out=q.half()) == L.E_UNSUPPORTED
    # more tokens than rows, and none to say whose they are
    assert code(rows=paged.rows(table[:1])) == L.E_MALFORMED
    odd = torch.zeros(2 * 128 + 2, device="cuda")
    assert code(k=odd[2:].view(2, 2, 64)) == L.E_MALFORMED  # 8-byte aligned floats
    assert code(k=torch.zeros(2, 130, device="cuda")[:, :128].unflatten(1, (2, 64))) == L.E_MALFORMED
    gated = torch.zeros(2, 4, 128, device="cuda")[..., :64]
    rc = L.lib().zg_paged_append_device(ctx.h, kv, paged.rows(table), 2, 4, gated.data_ptr(), 512, 128, k.data_ptr(),
                                        128, k.data_ptr(), 128, L.F32, None, None, 0.0, 0, 1.0, p.data_ptr(), None,
                                        gated.data_ptr(), None, None)
    assert rc == L.E_MALFORMED and "in place" in ctx.error()

"""The paged operators together, as a decode loop uses them: a shared prompt
appended as the prefix, then per step one layer's projections, append,
attention, output projection, head and adjusted readout, every row on its own
continuation; against the same loop in 64 bits."""
import math

import numpy as np
import pytest
import torch

import paged_reference as ref
from zerogravity_amd import _lib as L
from zerogravity_amd import paged, sampling
from zerogravity_amd import regions as R

pytestmark = pytest.mark.gpu
HIDDEN, QH, KVH, D, VOCAB, ROWS, PREFIX, PAGE = 256, 4, 2, 64, 601, 3, 45, 8
WIDE = (QH + 2 * KVH) * D
THETA = float(np.float32(1e7 ** (-2 / 32)))


class Layer:
    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.kern = R.HipMatVecKernel(0)
        self.ctx = self.kern.ctx
        self.w = {n: torch.randn(o, i, generator=g) / math.sqrt(i)
                  for n, o, i in (("qkv", WIDE, HIDDEN), ("out", HIDDEN, QH * D), ("head", VOCAB, HIDDEN))}
        self.h = {n: self.kern.register(77, n, L.F32, w.shape[1], w.shape[0], w.numpy().view(np.uint8).reshape(-1))
                  for n, w in self.w.items()}
        self.embedding = torch.randn(VOCAB, HIDDEN, generator=g)
        self.qn, self.kn = 1 + 0.1 * torch.randn(2, D, generator=g)

    def gemv(self, name, x, y, st):
        self.ctx.check(L.lib().zg_gemv_device(self.ctx.h, self.h[name].h, x.data_ptr(), L.F32, x.shape[0], None, 0.0,
                                              y.data_ptr(), st))


def test_decode_loop_over_a_shared_prompt():
    m = Layer(1)
    g = torch.Generator().manual_seed(2)
    prompt = torch.randint(0, VOCAB, (PREFIX,), generator=g)
    steps = 14  # rows cross two pages of their own
    emb, qn, kn = (t.cuda() for t in (m.embedding, m.qn, m.kn))
    order = torch.randperm(40, generator=g).int()
    shared = order[:-(-PREFIX // PAGE)].cuda()
    table = order[10:10 + 3 * ROWS].view(ROWS, 3).cuda()
    pool = torch.full((40, 2, PAGE, KVH, D), math.nan, dtype=torch.bfloat16, device="cuda")
    kv = paged.cache(pool[:, 0], pool[:, 1])
    rows = paged.rows(table, shared, PREFIX)
    stream = torch.cuda.Stream()
    st = stream.cuda_stream
    tokens = torch.randint(0, VOCAB, (ROWS,), generator=g).int().cuda()
    first = tokens.cpu()
    history = torch.zeros(ROWS, PREFIX + 1 + steps, dtype=torch.int32, device="cuda")
    history[:, :PREFIX], history[:, PREFIX] = prompt.cuda(), tokens
    held = torch.full((ROWS,), PREFIX + 1, dtype=torch.int32, device="cuda")
    masks = torch.randint(-2 ** 31, 2 ** 31, (1, (VOCAB + 31) // 32), generator=g).int().cuda()
    u = sampling.rules(history=history, history_lengths=held, prompt_lengths=torch.full_like(held, PREFIX),
                       repetition=torch.tensor([1.0, 1.3, 1.1], device="cuda"),
                       frequency=torch.tensor([0.0, 0.4, 0.2], device="cuda"),
                       presence=torch.tensor([0.0, 0.0, 0.5], device="cuda"), masks=masks,
                       mask_of=torch.tensor([-1, 0, -1], dtype=torch.int32, device="cuda"))
    positions = torch.full((ROWS,), PREFIX, dtype=torch.int32, device="cuda")
    lengths = torch.ones(ROWS, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    proj = torch.zeros(ROWS, WIDE, device="cuda")
    q, out = (torch.zeros(ROWS, QH, D, device="cuda") for _ in range(2))
    mixed, logits, adjusted = (torch.zeros(ROWS, n, device="cuda") for n in (HIDDEN, VOCAB, VOCAB))
    ws = torch.empty(paged.attend_workspace(kv, rows, QH), dtype=torch.uint8, device="cuda")
    ls = torch.empty(L.lib().zg_logits_adjust_workspace_bytes(ROWS, VOCAB), dtype=torch.uint8, device="cuda")
    scale = 1 / math.sqrt(D)

    def parts(p):
        n = p.shape[0]
        return (p[:, :QH * D].view(n, QH, D), p[:, QH * D:(QH + KVH) * D].view(n, KVH, D),
                p[:, (QH + KVH) * D:].view(n, KVH, D))

    def step():
        x = emb[tokens.long()]
        m.gemv("qkv", x, proj, st)
        pq, pk, pv = parts(proj)
        paged.append(m.ctx, kv, rows, pk, pv, positions, pq, q, qn, kn, rotate=32, theta_scale=THETA, status=status)
        paged.attend(m.ctx, kv, rows, lengths, q, scale, out, ws, status)
        m.gemv("out", out.view(ROWS, QH * D), mixed, st)
        mixed.add_(x)
        m.gemv("head", mixed, logits, st)
        sampling.adjust(m.ctx, logits, u, adjusted, tokens, record=True, workspace=ls, status=status)
        positions.add_(1)
        lengths.add_(1)

    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        # the prompt's keys and values: one row of the prefix's pages
        x = emb[prompt.cuda()]
        whole = torch.empty(PREFIX, WIDE, device="cuda")
        for at in range(0, PREFIX, 4):
            m.gemv("qkv", x[at:at + 4], whole[at:at + 4], st)
        _, pk, pv = parts(whole)
        paged.append(m.ctx, kv, paged.rows(shared.view(1, -1)), pk, pv,
                     torch.arange(PREFIX, dtype=torch.int32, device="cuda"), k_norm=kn, rotate=32, theta_scale=THETA,
                     token_rows=torch.zeros(PREFIX, dtype=torch.int32, device="cuda"), status=status)
        start = [t.clone() for t in (tokens, history, held, positions, lengths)]
        got = []
        for _ in range(steps):
            step()
            got.append((tokens.cpu(), logits.cpu(), adjusted.cpu()))
        # the same loop from a captured step: the same bits
        for t, s in zip((tokens, history, held, positions, lengths), start):
            t.copy_(s)
        stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for i in range(steps):
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got[i], (tokens, logits, adjusted)):
            assert torch.equal(a, b.cpu()), i
    assert int(status) == 0
    assert held.cpu().tolist() == [PREFIX + 1 + steps] * ROWS
    assert history[:, PREFIX + 1:].cpu().t().tolist() == [t.tolist() for t, _, _ in got]

    # the loop in 64 bits, fed the device's tokens.  A projection of 256 terms
    # in 32 bits is off by 256 U of its terms' sum; the cache rounds keys and
    # values to bfloat16, half a step apart at most where the two round to
    # different sides, 2^-8 of a key or value each.  Scores are scale * sum
    # q.k over 64 normed pairs (|score| < 8), so a flipped rounding of every
    # element would move them by 2^-8 * 64 / 8: weights by e^(1/32); few flip.
    # Measured against logits of size sqrt(2): 2^-8 * 2 of their largest.
    w = {n: t.double() for n, t in m.w.items()}
    e = m.embedding.double()

    def token(x, at):
        tq, tk, tv = parts(x @ w["qkv"].t())
        at = torch.tensor(at)
        tq, tk = (ref.rotate(ref.norm(t, n, 1e-6), at, 32, THETA) for t, n in ((tq, m.qn), (tk, m.kn)))
        return tq, tk.float().bfloat16().double(), tv.float().bfloat16().double()

    _, shared_k, shared_v = token(e[prompt], list(range(PREFIX)))
    own = [(shared_k, shared_v)] * ROWS
    fed = first
    masks, mask_of = masks.cpu().numpy(), [-1, 0, -1]
    for i in range(steps):
        for r in range(ROWS):
            x = e[fed[r].long()].view(1, -1)
            tq, tk, tv = token(x, [PREFIX + i])
            own[r] = (torch.cat([own[r][0], tk]), torch.cat([own[r][1], tv]))
            o, _, _ = ref.softmax_rows(tq[0], *own[r], scale)
            want = ((o.view(1, -1) @ w["out"].t() + x) @ w["head"].t())[0]
            tol = 2 ** -7 * float(want.abs().max())
            assert float((got[i][1][r].double() - want).abs().max()) <= tol, (i, r)
            past = np.concatenate([prompt.numpy(), first[r:r + 1].numpy(),
                                   np.array([int(t[r]) for t, _, _ in got[:i]], np.int64)]).astype(np.int32)
            exact = ref.np_adjust(got[i][1][r:r + 1].numpy(), dict(
                history=past[None], history_lengths=[len(past)], prompt_lengths=[PREFIX],
                repetition=np.float32([[1.0, 1.3, 1.1][r]]), frequency=np.float32([[0.0, 0.4, 0.2][r]]),
                presence=np.float32([[0.0, 0.0, 0.5][r]]), masks=masks, mask_of=[mask_of[r]]), VOCAB)
            assert np.array_equal(exact[0], got[i][2][r].numpy()), (i, r)
            assert int(got[i][0][r]) == int(ref.np_greedy(exact)[0])
        fed = got[i][0]

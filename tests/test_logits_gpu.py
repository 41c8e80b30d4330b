"""zg_logits_adjust_device against the rules in 64 bits, rounded once: the
same bits, and the same ids."""
import math

import numpy as np
import pytest
import torch

import paged_reference as ref
from zerogravity_amd import _lib as L
from zerogravity_amd import sampling

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ctx():
    c = L.Context(0)
    yield c
    c.close()


def random_rules(g, rows, vocab, history, biases, mask_rows):
    def ints(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g).int()

    u = {}
    if history:
        # a third of the tokens from a handful of ids, a few outside the vocabulary
        few = ints(0, vocab, rows, history) % 7
        u["history"] = torch.where(torch.rand(rows, history, generator=g) < 0.3, few, ints(-2, vocab + 3, rows, history))
        u["history_lengths"] = ints(0, history + 1, rows)
        u["prompt_lengths"] = ints(0, history + 1, rows)
        u["repetition"], u["frequency"], u["presence"] = (0.7 + torch.rand(3, rows, generator=g))
    if biases:
        u["bias_ids"] = ints(-1, vocab + 1, rows, biases)
        u["bias_ids"][:, biases // 2] = u["bias_ids"][:, 0]  # one id twice
        u["bias_values"] = 5 * torch.randn(rows, biases, generator=g)
        u["bias_lengths"] = ints(0, biases + 1, rows)
        u["bias_lengths"][0] = biases
    if mask_rows:
        u["masks"] = torch.randint(-2 ** 31, 2 ** 31, (mask_rows, (vocab + 31) // 32 + 1), generator=g).int()
        u["mask_of"] = ints(-1, mask_rows, rows)
    return u


def expect(x, u, vocab):
    want = ref.np_adjust(x.float().numpy(), {k: v.numpy() for k, v in u.items()}, vocab)
    want = torch.from_numpy(want).to(x.dtype)
    return want, ref.np_greedy(want.float().numpy())


def same(a, b):
    a, b = a.float(), b.float()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


def device(u):
    return {k: v.cuda() for k, v in u.items()}


@pytest.mark.parametrize("rows,vocab,history,biases,mask_rows,dtype", [
    (1, 151936, 600, 5, 1, F32), (32, 151936, 2500, 40, 9, F32), (3, 151936, 9000, 300, 0, BF16),
    (5, 1, 4, 3, 1, F32), (4, 31, 9, 2, 2, BF16), (4, 33, 9, 2, 2, F32), (2, 4095, 70, 0, 2, F32),
    (2, 4096, 70, 9, 0, F32), (2, 4097, 0, 9, 2, BF16), (7, 12289, 500, 0, 0, F32), (3, 1003, 0, 0, 3, F32),
    (2, 777, 0, 0, 0, BF16), (65, 5000, 33, 7, 4, F32)])
def test_rules_match_the_definition(ctx, rows, vocab, history, biases, mask_rows, dtype):
    g = torch.Generator().manual_seed(vocab + rows)
    u = random_rules(g, rows, vocab, history, biases, mask_rows)
    x = (3 * torch.randn(rows, vocab, generator=g)).to(dtype)
    want, ids = expect(x, u, vocab)
    greedy = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    dx, out = x.cuda(), torch.empty(rows, vocab, dtype=dtype, device="cuda")
    sampling.adjust(ctx, dx, sampling.rules(**device(u)), out, greedy, status=status)
    torch.cuda.synchronize()
    assert same(out.cpu(), want) and torch.equal(dx.cpu(), x)
    assert np.array_equal(greedy.cpu().numpy().view(np.uint32), ids) and int(status) == 0
    # in place, padded rows on odd strides, no ids asked for
    wide = torch.full((rows, vocab + 3), 9.0, dtype=dtype, device="cuda")
    wide[:, :vocab] = dx
    sampling.adjust(ctx, wide[:, :vocab], sampling.rules(**device(u)))
    torch.cuda.synchronize()
    assert same(wide[:, :vocab].cpu(), want) and (wide[:, vocab:] == 9.0).all()


@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_that_start_anywhere(ctx, dtype, offset):
    g = torch.Generator().manual_seed(offset)
    rows, vocab = 3, 9001
    u = random_rules(g, rows, vocab, 100, 9, 3)
    x = torch.randn(rows, vocab, generator=g).to(dtype)
    want, ids = expect(x, u, vocab)
    a, b = (torch.zeros(rows * (vocab + 2) + offset, dtype=dtype, device="cuda")[offset:].view(rows, vocab + 2)[:, :vocab]
            for _ in range(2))
    a.copy_(x)
    greedy = torch.empty(rows, dtype=torch.int32, device="cuda")
    sampling.adjust(ctx, a, sampling.rules(**device(u)), b, greedy)
    torch.cuda.synchronize()
    assert same(b.cpu(), want) and np.array_equal(greedy.cpu().numpy().view(np.uint32), ids)


def run(ctx, x, dtype=F32, **u):
    x = torch.tensor(x, dtype=dtype)
    d = {k: torch.tensor(v, dtype=F32 if k in ("repetition", "frequency", "presence", "bias_values") else torch.int32,
                         device="cuda") for k, v in u.items()}
    out, greedy = x.cuda(), torch.full((x.shape[0],), -7, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    sampling.adjust(ctx, out, sampling.rules(**d), greedy=greedy, status=status)
    torch.cuda.synchronize()
    return out.cpu().tolist(), greedy.cpu().numpy().view(np.uint32).tolist(), int(status)


def test_hand_computed_rules(ctx):
    inf = math.inf
    # seen 0, 1, 3; generated 1 twice and 3 once
    assert run(ctx, [[2.0, -1.0, 1.0, 4.0]], history=[[0, 1, 1, 3]], history_lengths=[4], prompt_lengths=[1],
               repetition=[2.0], frequency=[0.25], presence=[0.5]) == ([[1.0, -3.0, 1.0, 1.25]], [3], 0)
    # no prompt lengths: all of it was generated
    assert run(ctx, [[2.0, -1.0]], history=[[0, 0]], history_lengths=[2], frequency=[1.0]) == ([[0.0, -1.0]], [0], 0)
    # the same id twice in the biases; lengths that cut them short
    assert run(ctx, [[0.0, 0.0, 0.0]], bias_ids=[[2, 1, 2, 0]], bias_values=[[1.0, 0.5, 2.0, 9.0]],
               bias_lengths=[3]) == ([[0.0, 0.5, 3.0]], [2], 0)
    # equal values: the lowest index, signed zeros among them
    assert run(ctx, [[-1.0, -0.0, 0.0, 0.0]])[1] == [1]
    # a mask over what is not a number, and a status for what it allows
    assert run(ctx, [[math.nan, inf, 1.0, -inf]], masks=[[0b1100]]) == ([[-inf, -inf, 1.0, -inf]], [2], 0)
    out, ids, status = run(ctx, [[math.nan, 2.0, inf]], masks=[[0b011], [0b110]], mask_of=[0])
    assert math.isnan(out[0][0]) and out[0][1:] == [2.0, -inf] and ids == [1] and status == 4
    assert run(ctx, [[0.0, 2.0, inf]], masks=[[0b011], [0b110]], mask_of=[1]) == ([[-inf, 2.0, inf]], [2], 4)
    # nothing allowed, or a mask that is not there
    assert run(ctx, [[1.0, 2.0]], masks=[[0]]) == ([[-inf, -inf]], [0xffffffff], 0)
    assert run(ctx, [[1.0, 2.0]], masks=[[3]], mask_of=[1]) == ([[-inf, -inf]], [0xffffffff], 0)
    assert run(ctx, [[math.nan, -inf]])[1:] == ([0xffffffff], 4)
    # a row that is left out
    assert run(ctx, [[1.0, 2.0], [3.0, 4.0]], history=[[1], [1]], history_lengths=[-1, 1],
               presence=[1.0, 2.0]) == ([[1.0, 2.0], [3.0, 2.0]], [0xfffffff9, 0], 0)
    # a history longer than its stride is cut
    assert run(ctx, [[1.0, 2.0]], history=[[1]], history_lengths=[2 ** 31 - 1], presence=[1.5]) == ([[1.0, 0.5]], [0], 0)
    # 16-bit logits are compared as they are written: 256.5 and 257 tie at 256
    assert run(ctx, [[254.0, 256.0]], BF16, bias_ids=[[0]], bias_values=[[2.5]], bias_lengths=[1]) == (
        [[256.0, 256.0]], [0], 0)


def test_recording_extends_the_history(ctx):
    vocab, cap = 5000, 6
    g = torch.Generator().manual_seed(6)
    history = torch.zeros(3, cap, dtype=torch.int32, device="cuda")
    lengths = torch.tensor([0, 5, 2], dtype=torch.int32, device="cuda")
    x = torch.randn(3, vocab, generator=g).cuda()
    x[2] = -math.inf  # nothing to take: nothing recorded
    u = sampling.rules(history=history, history_lengths=lengths, presence=torch.full((3,), 100.0, device="cuda"))
    greedy, out = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty_like(x)
    told = []
    for step in range(3):
        sampling.adjust(ctx, x, u, out, greedy, record=True)
        torch.cuda.synchronize()
        told.append(greedy.cpu().tolist())
    top = x[0].argsort(descending=True)[:3].cpu().tolist()
    assert [t[0] for t in told] == top  # a penalty of 100: each token once
    assert history[0].cpu().tolist() == top + [0, 0, 0] and lengths.cpu().tolist() == [3, 6, 2]
    assert history[1, 5] == told[0][1] and [t[2] for t in told] == [-1, -1, -1]


def test_captured_calls_read_their_rules_anew(ctx):
    rows, vocab = 4, 20000
    g = torch.Generator().manual_seed(7)
    u = device(random_rules(g, rows, vocab, 200, 20, 3))
    x, out = torch.zeros(rows, vocab, device="cuda"), torch.zeros(rows, vocab, device="cuda")
    greedy = torch.zeros(rows, dtype=torch.int32, device="cuda")
    ws = torch.empty(L.lib().zg_logits_adjust_workspace_bytes(rows, vocab), dtype=torch.uint8, device="cuda")
    r = sampling.rules(**u)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sampling.adjust(ctx, x, r, out, greedy, workspace=ws)
    for step in range(4):
        fresh = random_rules(g, rows, vocab, 200, 20, 3)
        logits = torch.randn(rows, vocab, generator=g)
        for k, v in fresh.items():
            u[k].copy_(v)
        x.copy_(logits)
        graph.replay()
        torch.cuda.synchronize()
        want, ids = expect(logits, fresh, vocab)
        assert same(out.cpu(), want) and np.array_equal(greedy.cpu().numpy().view(np.uint32), ids), step


def test_refusals(ctx):
    x = torch.zeros(2, 40, device="cuda")
    i = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device="cuda")  # noqa: E731
    f = lambda *shape: torch.ones(*shape, device="cuda")  # noqa: E731

    def code(logits=x, more=None, **u):
        with pytest.raises(L.ZgError) as e:
            sampling.adjust(ctx, logits, sampling.rules(**u), **(more or {}))
        return e.value.code

    assert code(history=i(2, 3)) == code(history_lengths=i(2)) == code(presence=f(2)) == L.E_MALFORMED
    assert code(history=i(1, 3), history_lengths=i(2)) == code(history=i(2, 0), history_lengths=i(2)) == L.E_MALFORMED
    assert code(bias_ids=i(2, 3), bias_values=f(2, 3)) == code(masks=i(2, 1)) == code(masks=i(1, 2)) == L.E_MALFORMED
    assert code(logits=x.half()) == L.E_UNSUPPORTED
    assert code(bias_ids=i(2, 70000), bias_values=f(2, 70000), bias_lengths=i(2)) == L.E_LIMIT
    assert code(more=dict(record=True)) == code(more=dict(record=True, greedy=i(2))) == L.E_MALFORMED
    assert code(more=dict(out=f(2, 39))) == code(more=dict(greedy=i(3))) == L.E_MALFORMED
    assert code(more=dict(greedy=i(2), workspace=torch.empty(1, dtype=torch.uint8, device="cuda"))) == L.E_MALFORMED

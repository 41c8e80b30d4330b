"""Adjusted logits on both sides of each choice of threads: rounds of
workgroups that 256 threads spare or do not, and histories too long for them."""
import numpy as np
import pytest
import torch

import paged_reference as ref
from test_logits_gpu import device, random_rules
from test_logits_rounding_gpu import adjusted, nearest
from zerogravity_amd import _lib as L
from zerogravity_amd import sampling

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ctx():
    c = L.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab,history", [
    (342, 8193, 900), (205, 20477, 9216), (205, 20477, 9217),  # 1026, 1025 slices: one round
    (683, 8193, 30), (512, 16385, 30), (410, 20001, 6144), (410, 20001, 6145), (853, 8193, 30), (854, 8193, 30),
    (1025, 8193, 20), (1280, 8193, 4608), (1281, 8193, 20)])  # 2049 to 2562 and 3075 to 3843 slices
def test_rounds_of_workgroups(ctx, dtype, rows, vocab, history):
    g = torch.Generator().manual_seed(rows + history)
    held = min(history, 300)
    u = random_rules(g, rows, vocab, held, 5, 3)
    u["history_lengths"][:], u["bias_lengths"][:] = held, 5
    x = torch.randn(rows, vocab, generator=g).to(dtype)
    v = adjusted(x.double().numpy(), {k: t.numpy() for k, t in u.items()})
    want = (nearest(v) if dtype == BF16 else v).astype(np.float32)
    if history > held:  # room for more tokens than a row holds
        u["history"] = torch.cat([u["history"], torch.full((rows, history - held), vocab // 2, dtype=torch.int32)], 1)
    greedy, out = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, vocab, dtype=dtype, device="cuda")
    sampling.adjust(ctx, x.cuda(), sampling.rules(**device(u)), out, greedy)
    torch.cuda.synchronize()
    assert np.array_equal(out.float().cpu().numpy(), want)
    assert np.array_equal(greedy.cpu().numpy().view(np.uint32), ref.np_greedy(want))

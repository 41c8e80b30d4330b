"""The paged cache and the readout beside the framework's own decode step: a
session's logits adjusted on the device and fed back to it, and a contiguous
cache moved into pages."""
import math

import numpy as np
import pytest
import torch

import paged_reference as ref
from zerogravity_amd import _lib as L
from zerogravity_amd import gguf, paged, qwen35, sampling
from zerogravity_amd import regions as R

pytestmark = pytest.mark.gpu


def test_a_session_decodes_by_adjusted_logits():
    """Steps of the session, the rules and the id of each in turn on one
    stream, nothing waiting in between; then the rules again from the logits
    that the steps left."""
    g = dict(hidden=256, layers=4, ffn=512, vocab=1000, gdn_heads=2, gdn_dim=128, q_heads=2, kv_heads=1, head_dim=256,
             full_attention_interval=4, max_context=64, eps=1e-6)
    kern = R.HipMatVecKernel(0)
    model = qwen35.QwenModelHip(g, qwen35.synthetic_tensors(g, gguf.Q8_0, seed=5), kernel=kern)
    rows, steps = 3, 10
    s = model.session(max_batch=rows, max_context=32, kv_dtype=L.F32)
    stream = torch.cuda.Stream()
    first = [3, 141, 592]
    tokens = torch.tensor(first, dtype=torch.int32, device="cuda")
    logits, adjusted = torch.empty(2, rows, 1000, device="cuda")
    plain = torch.empty(rows, dtype=torch.int32, device="cuda")
    history = torch.zeros(rows, 1 + steps, dtype=torch.int32, device="cuda")
    history[:, 0] = tokens
    held = torch.ones(rows, dtype=torch.int32, device="cuda")
    knobs = dict(repetition=np.float32([1.0, 1.5, 1.2]), frequency=np.float32([0.0, 1.0, 0.3]),
                 presence=np.float32([0.0, 100.0, 0.2]))
    u = sampling.rules(history=history, history_lengths=held, **{k: torch.from_numpy(v).cuda() for k, v in knobs.items()})
    kept = torch.empty(steps, 2, rows, 1000, device="cuda")
    ids = torch.empty(steps, rows, dtype=torch.int32, device="cuda")
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for i in range(steps):
            kern.ctx.check(L.lib().zg_decode_step_device(s.h, rows, tokens.data_ptr(), logits.data_ptr(), plain.data_ptr(),
                                                         stream.cuda_stream))
            sampling.adjust(kern.ctx, logits, u, adjusted, tokens, record=True)
            kept[i, 0], kept[i, 1], ids[i] = logits, adjusted, tokens
        kern.ctx.check(L.lib().zg_session_check(s.h, stream.cuda_stream))
    torch.cuda.synchronize()
    assert s.positions() == [steps] * rows
    kept, ids = kept.cpu().numpy(), ids.cpu().numpy()
    past = np.array(first, np.int32)[:, None]
    again = model.session(max_batch=rows, max_context=32, kv_dtype=L.F32)
    for i in range(steps):
        assert np.array_equal(again.step(past[:, -1].astype(np.uint32))[0].view(np.uint32), kept[i, 0].view(np.uint32)), i
        want = ref.np_adjust(kept[i, 0], dict(history=past, history_lengths=[past.shape[1]] * rows, **knobs), 1000)
        assert np.array_equal(want, kept[i, 1]) and np.array_equal(ref.np_greedy(want).astype(np.int32), ids[i]), i
        past = np.concatenate([past, ids[i][:, None]], 1)
    assert np.array_equal(history.cpu().numpy(), past) and held.cpu().tolist() == [1 + steps] * rows
    assert len(set(past[1])) == 1 + steps  # a penalty of 100: no token twice
    model.close()
    kern.ctx.close()


@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float32])
def test_a_contiguous_cache_moved_into_pages(cache):
    """One step of zg_attn_decode_device, its cache copied into pages, then the
    same layer by append and attend and the gate by torch.  The two rotations
    part: that one multiplies its angle up in 32 bits, off by (i + 1) U of it
    or, over all pairs, 2 U of the position at most, which turns a pair by as
    much and moves a score by that times sum |q||k|; the rest is within the
    attention's own bound."""
    ctx = L.Context(0)
    nq, nkv, d, page, room = 8, 2, 256, 16, 512
    positions, theta = [0, 17, 300, 511], math.pow(1e7, -2.0 / 64.0)
    rows = len(positions)
    g = torch.Generator().manual_seed(9)
    stride = (2 * nq + 2 * nkv) * d
    proj = torch.randn(rows, stride, generator=g)
    qn, kn = 1 + 0.1 * torch.randn(2, d, generator=g)
    keys, values = torch.randn(2, rows, room, nkv, d, generator=g).to(cache)
    c = [t.cuda() for t in (proj, qn, kn, keys, values)]
    at = torch.tensor(positions, dtype=torch.int32, device="cuda")
    kind = L.BF16 if cache == torch.bfloat16 else L.F32
    ws = torch.empty(L.lib().zg_attn_decode_workspace_bytes(rows, nq, room), dtype=torch.uint8, device="cuda")
    out = torch.empty(rows, nq * d, device="cuda")
    torch.cuda.synchronize()
    ctx.check(L.lib().zg_attn_decode_device(ctx.h, rows, nq, nkv, c[0].data_ptr(), stride, c[1].data_ptr(), c[2].data_ptr(),
                                            1e-6, theta, at.data_ptr(), c[3].data_ptr(), c[4].data_ptr(), room, kind,
                                            ws.data_ptr(), out.data_ptr(), None))
    torch.cuda.synchronize()
    # pages of the contiguous cache, dealt at random
    order = torch.randperm(rows * room // page, generator=g)
    pool = torch.empty(rows * room // page, 2, page, nkv, d, dtype=cache, device="cuda")
    pool[order.cuda(), 0], pool[order.cuda(), 1] = (t.view(-1, page, nkv, d) for t in c[3:])
    kv, table = paged.cache(pool[:, 0], pool[:, 1]), paged.rows(order.int().view(rows, -1).cuda())
    heads = c[0][:, :2 * nq * d].view(rows, nq, 2 * d)
    k, v = (c[0][:, 2 * nq * d:].view(rows, 2, nkv, d)[:, i] for i in range(2))
    q = torch.empty(rows, nq, d, device="cuda")
    moved = pool.clone()
    paged.append(ctx, kv, table, k, v, at, heads[..., :d], q, c[1], c[2], rotate=64, theta_scale=theta)
    torch.cuda.synchronize()
    # what the append stores is what the step stored, but for the angle: keys
    # of size 4 a step of the cache's type apart, or their turn
    off = (pool.float() - moved.float()).abs()
    assert (off[:, 1] == 0).all() and off[:, 0].max() <= 4 * torch.finfo(cache).eps + 2 * ref.U * 512 * 8
    pool.copy_(moved)
    got = paged.attend(ctx, kv, table, at + 1, q, 1 / 16) * torch.sigmoid(heads[..., d:])
    torch.cuda.synchronize()
    held = [t.cpu().double() for t in c[3:]]
    gate = torch.sigmoid(proj[:, :2 * nq * d].view(rows, nq, 2 * d)[..., d:].double())
    for r, p in enumerate(positions):
        want, mass, dots = ref.softmax_rows(q[r].cpu().double(), held[0][r, :p + 1], held[1][r, :p + 1], 1 / 16)
        bound = ref.attend_bound(want, mass, dots, p + 1, d, torch.float32, cache) + 2 * (2 * ref.U * p) * dots * mass
        assert ((got[r].cpu().double() - want * gate[r]).abs() <= bound * gate[r] + 4 * ref.U * want.abs()).all(), r
        # the step's own sums are off by as much again
        assert ((out[r].view(nq, d).cpu().double() - want * gate[r]).abs() <= 2 * bound * gate[r] + 8 * ref.U * want.abs()).all(), r
    ctx.close()

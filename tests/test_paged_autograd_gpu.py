"""Tensors that require gradients: never written to behind autograd's back;
read as values."""
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


def refused(call):
    with pytest.raises(L.ZgError) as e:
        call()
    assert e.value.code == L.E_MALFORMED and "no_grad" in str(e.value)


def test_outputs_that_require_a_gradient_are_refused(ctx):
    d = Device(ref.Batch(60, 2, 2, 4, 64, 16, 0, [5, 6], torch.float32, torch.float32))
    plain = d.attend(ctx)
    for leaf in (True, False):
        out = torch.zeros_like(plain).requires_grad_()
        out = out if leaf else out * 2
        refused(lambda: d.attend(ctx, out=out))
        with torch.no_grad():
            assert torch.equal(d.attend(ctx, out=out), plain)
        x = torch.zeros(2, 40, device="cuda").requires_grad_()
        x = x if leaf else x + 1
        refused(lambda: sampling.adjust(ctx, x, sampling.rules()))
        refused(lambda: sampling.adjust(ctx, x.detach(), sampling.rules(), out=x))
        with torch.no_grad():
            sampling.adjust(ctx, x, sampling.rules())
    # inputs are read as values
    d.q.requires_grad_()
    assert torch.equal(d.attend(ctx), plain) and not d.attend(ctx).requires_grad


@pytest.mark.parametrize("which", ["keys", "values", "q_out"])
def test_caches_that_require_a_gradient_are_refused(ctx, which):
    t = dict(keys=torch.zeros(2, 4, 1, 64, device="cuda"), values=torch.zeros(2, 4, 1, 64, device="cuda"),
             q_out=torch.zeros(2, 2, 64, device="cuda"))
    t[which].requires_grad_()
    k, q = torch.ones(2, 1, 64, device="cuda"), torch.ones(2, 2, 64, device="cuda")
    rows = paged.rows(torch.tensor([[0], [1]], dtype=torch.int32, device="cuda"))
    at = torch.zeros(2, dtype=torch.int32, device="cuda")

    def call():
        paged.append(ctx, paged.cache(t["keys"], t["values"]), rows, k, k, at, q, t["q_out"])

    refused(call)
    torch.cuda.synchronize()
    assert all((x == 0).all() for x in t.values())
    with torch.no_grad():
        call()
    torch.cuda.synchronize()
    assert all((x[..., 0] == 1).any() for x in t.values())

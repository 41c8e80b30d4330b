"""Tensors of the wrong number of dimensions are refused by the paged forms,
before anything asks for a dimension that is not there."""
from types import SimpleNamespace

import pytest
import torch

from test_paged_cpu import pool
from zerogravity_amd import _lib as L
from zerogravity_amd import paged

HERE = SimpleNamespace(device=0)


def code(call):
    with pytest.raises(L.ZgError) as e:
        call()
    return e.value.code


@pytest.mark.parametrize("shape", [(), (2,), (2, 512), (1, 2, 2, 256)])
def test_dimensions_of_activations(shape):
    kv, r = pool(), paged.rows(torch.zeros(2, 2, dtype=torch.int32))
    good, bad, at = torch.zeros(2, 2, 256), torch.zeros(shape), torch.zeros(2, dtype=torch.int32)
    assert code(lambda: paged.append(HERE, kv, r, bad, bad, at)) == L.E_MALFORMED
    assert code(lambda: paged.append(HERE, kv, r, good, bad, at)) == L.E_MALFORMED
    assert code(lambda: paged.append(HERE, kv, r, good, good, at, bad, bad)) == L.E_MALFORMED
    assert code(lambda: paged.attend(HERE, kv, r, at, bad, 1.0)) == L.E_MALFORMED

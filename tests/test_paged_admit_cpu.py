"""Host arrays of another type than int32 in the scheduler's check: taken as
they are, never wrapped or cut to something that fits."""
import numpy as np
import pytest
import torch

from test_paged_cpu import pool, refused
from zerogravity_amd import _lib as L
from zerogravity_amd import paged


@pytest.mark.parametrize("wide", [2 ** 32, 2 ** 32 + 1, -2 ** 32 + 3, 2 ** 63 - 1, -2 ** 31 - 1])
def test_numbers_past_32_bits_do_not_wrap_into_the_pool(wide):
    refused(L.E_MALFORMED, table=np.array([[0, 1], [wide, -1]], np.int64))
    refused(L.E_MALFORMED, prefix=np.array([5, wide], np.int64))
    refused(L.E_MALFORMED, lengths=np.array([20, wide], np.int64))


@pytest.mark.parametrize("kind", [np.float32, np.float64, bool])
def test_numbers_that_are_not_whole_are_refused(kind):
    refused(L.E_MALFORMED, table=np.array([[0.5, 1], [1, 1]], kind))
    refused(L.E_MALFORMED, prefix=np.array([0.5, 1], kind))
    refused(L.E_MALFORMED, lengths=np.array([0.5, 1], kind))


def test_other_whole_numbers_are_taken():
    for kind in (np.int64, np.uint16, np.int8):
        paged.admit(pool(), np.array([[0, 1], [2, 7]], kind), np.array([20, 3], kind), 8, np.array([5, 6], kind), 30)
    paged.admit(pool(), [[0, 1]], [20], 8, [], 0)
    paged.admit(pool(), torch.tensor([[0, 1]]), torch.tensor([20]), 8)
    paged.admit(pool(), np.array([[0, 1], [2, 3]], np.int32)[:, ::-1], np.array([20, -1], np.int32), 8)

"""Host side of the paged cache and of the logits readout: the scheduler's
check of page tables, refusals before any device work, workspace sizes."""
import numpy as np
import pytest
import torch

from zerogravity_amd import _lib as L
from zerogravity_amd import paged, sampling


def pool(pages=8, page=16, heads=2, dim=256, dtype=torch.bfloat16):
    t = torch.zeros(pages, page, heads, dim, dtype=dtype)
    return paged.cache(t, t.clone())


def refused(code, kv=None, **change):
    args = dict(table=np.array([[0, 1], [2, -1]], np.int32), lengths=np.array([20, 3], np.int32), q_heads=8,
                prefix=np.array([5, 6], np.int32), prefix_tokens=30)
    args.update(change)
    with pytest.raises(L.ZgError) as e:
        paged.admit(kv or pool(), **args)
    assert e.value.code == code, e.value
    return str(e.value)


def test_tables_that_fit_are_admitted():
    paged.admit(pool(), np.array([[0, 1], [2, -1], [9, 9]], np.int32), np.array([32, 0, -1], np.int32), 8)
    paged.admit(pool(), np.array([[7]], np.int32), np.array([16], np.int32), 32, np.array([0, 1], np.int32), 17)


def test_pages_outside_the_pool_are_refused():
    assert "row 0: page 1 is 8" in refused(L.E_MALFORMED, table=np.array([[0, 8], [2, -1]], np.int32))
    assert "row 1: page 0 is -1" in refused(L.E_MALFORMED, table=np.array([[0, 1], [-1, -1]], np.int32))
    assert "prefix page 1 is -7" in refused(L.E_MALFORMED, prefix=np.array([5, -7], np.int32))
    # an entry that no token needs may hold anything
    paged.admit(pool(), np.array([[0, 900]], np.int32), np.array([16], np.int32), 8)


def test_lengths_past_a_table_are_refused():
    assert "past its 2 pages" in refused(L.E_MALFORMED, lengths=np.array([33, 1], np.int32))
    refused(L.E_MALFORMED, prefix_tokens=33)
    refused(L.E_MALFORMED, prefix=None)


@pytest.mark.parametrize("field,value,code", [
    ("keys", None, L.E_MALFORMED), ("values", None, L.E_MALFORMED), ("pages", 0, L.E_MALFORMED),
    ("page_tokens", 0, L.E_MALFORMED), ("kv_heads", 0, L.E_MALFORMED), ("head_dim", 96, L.E_UNSUPPORTED),
    ("head_dim", 512, L.E_UNSUPPORTED), ("dtype", L.F16, L.E_UNSUPPORTED), ("dtype", -1, L.E_UNSUPPORTED),
    ("page_stride", 16 * 2 * 256 - 64, L.E_MALFORMED), ("page_stride", 16 * 2 * 256 + 8, L.E_MALFORMED),
    ("pages", 1 << 31, L.E_LIMIT), ("page_tokens", 65537, L.E_LIMIT), ("page_stride", 1 << 38, L.E_LIMIT),
    ("kv_heads", 1025, L.E_LIMIT), ("kv_heads", 3, L.E_MALFORMED)])
def test_malformed_pools_are_refused(field, value, code):
    kv = pool()
    setattr(kv, field, value)
    refused(code, kv)
    r = L.PagedRows(4096, 2, 2, None, 0)
    assert L.lib().zg_paged_attn_workspace_bytes(kv, r, 8) == 0


def test_misaligned_pools_are_refused():
    kv = pool()
    kv.keys += 8
    refused(L.E_MALFORMED, kv)


@pytest.mark.parametrize("q_heads,code", [(0, L.E_MALFORMED), (7, L.E_MALFORMED), (34, L.E_UNSUPPORTED)])
def test_head_counts_are_checked(q_heads, code):
    refused(code, q_heads=q_heads)


@pytest.mark.parametrize("rows,stride,prefix_tokens,code", [
    (0, 2, 0, L.E_MALFORMED), (1, 0, 0, L.E_MALFORMED), (4097, 2, 0, L.E_LIMIT), (1, (1 << 26) + 1, 0, L.E_LIMIT),
    (1, 2, (1 << 30) + 1, L.E_LIMIT), (1, 2, 5, L.E_MALFORMED)])
def test_malformed_tables_are_refused(rows, stride, prefix_tokens, code):
    r = L.PagedRows(4096, rows, stride, None, prefix_tokens)
    msg = __import__("ctypes").create_string_buffer(64)
    assert L.lib().zg_paged_admit(pool(), r, 4096, 8, msg, 64) == code
    assert msg.value
    assert L.lib().zg_paged_attn_workspace_bytes(pool(), r, 8) == 0


def test_null_arguments_are_refused_without_a_device():
    lib = L.lib()
    assert lib.zg_paged_admit(None, None, None, 8, None, 0) == L.E_MALFORMED
    assert lib.zg_paged_append_device(*[None] * 3, 1, 0, None, 0, 0, None, 0, None, 0, 0, None, None, 1e-6, 0, 1.0,
                                      None, None, None, None, None) == L.E_MALFORMED
    assert lib.zg_paged_attn_device(*[None] * 4, 8, None, 0, 0, 1.0, None, None, 0, None, None) == L.E_MALFORMED
    assert lib.zg_logits_adjust_device(None, 1, 1, None, 1, 0, None, None, 1, None, 0, None, None, None) == L.E_MALFORMED


def test_workspace_sizes():
    lib = L.lib()
    assert lib.zg_logits_adjust_workspace_bytes(0, 5) == 0
    assert lib.zg_logits_adjust_workspace_bytes(65536, 5) == 0
    assert lib.zg_logits_adjust_workspace_bytes(1, (1 << 30) + 1) == 0
    assert lib.zg_logits_adjust_workspace_bytes(3, 151936) > 0
    for rows in (1, 33, 4096):
        for prefix in (0, 1, 1 << 20):
            for heads, q in ((2, 8), (1, 16), (8, 8)):
                kv = pool(heads=heads)
                n = lib.zg_paged_attn_workspace_bytes(kv, L.PagedRows(4096, rows, 64, 4096, prefix), q)
                assert 0 < n < 1 << 32


def test_python_forms_refuse_what_is_not_the_pools():
    t = torch.zeros(4, 16, 2, 256, dtype=torch.bfloat16)
    for bad in (t.float(), t[:3], t.transpose(0, 1)):
        with pytest.raises(L.ZgError):
            paged.cache(t, bad)
    with pytest.raises(L.ZgError):
        paged.cache(t.half(), t.half())
    with pytest.raises(L.ZgError):
        paged.cache(t[:, :, :, :128], t[:, :, :, :128])
    with pytest.raises(L.ZgError):
        paged.rows(torch.zeros(2, 2, dtype=torch.int64))
    with pytest.raises(L.ZgError):
        paged.rows(torch.zeros(2, 4, dtype=torch.int32)[:, ::2])
    both = torch.zeros(4, 2, 16, 2, 256)  # keys and values of a page next to each other
    kv = paged.cache(both[:, 0], both[:, 1])
    assert kv.page_stride == 2 * 16 * 2 * 256 and kv.dtype == L.F32
    with pytest.raises(L.ZgError):
        sampling.rules(history=torch.zeros(2, 3))
    with pytest.raises(L.ZgError):
        sampling.rules(repetition=torch.zeros(2, dtype=torch.float64))
    with pytest.raises(L.ZgError):
        sampling.rules(bias_ids=torch.zeros(2, 3, dtype=torch.int32), bias_values=torch.zeros(2, 4))


def test_table_views_end_inside_their_storage():
    """A row of the table counts as long as the row stride, the last row too."""
    wide = torch.zeros(5, 9, dtype=torch.int32)
    assert paged.rows(wide[:, :4]).stride == paged.rows(wide).stride == 9
    assert paged.rows(wide[3:4, 5:]).stride == 4  # one row is as long as the view
    paged.rows(wide[:4, 5:])
    with pytest.raises(L.ZgError):
        paged.rows(wide[:, 5:])
    with pytest.raises(L.ZgError):
        paged.rows(wide[1:, 1:])


def test_streams_of_another_device_are_refused():
    from types import SimpleNamespace

    from zerogravity_amd import _torch
    ctx = SimpleNamespace(device=0)
    here = SimpleNamespace(device=torch.device("cuda", 0))
    assert _torch.stream_of(ctx, here) is here
    with pytest.raises(L.ZgError):
        _torch.stream_of(ctx, SimpleNamespace(device=torch.device("cuda", 1)))


def test_workspace_of_a_larger_batch_serves_smaller_ones():
    rng = np.random.default_rng(3)
    lib = L.lib()
    for heads, q, dim, dtype in ((2, 8, 256, torch.bfloat16), (4, 20, 128, torch.float32), (8, 8, 64, torch.bfloat16)):
        kv = pool(heads=heads, dim=dim, dtype=dtype)

        def need(rows, stride, prefix):
            return lib.zg_paged_attn_workspace_bytes(kv, L.PagedRows(4096, rows, stride, 4096, prefix), q)

        for rows, stride, prefix in rng.integers(1, (200, 3000, 70000), (100, 3)):
            most = need(rows, stride, prefix)
            for part in rng.random((20, 3)):
                assert need(max(1, int(rows * part[0])), max(1, int(stride * part[1])), int(prefix * part[2])) <= most

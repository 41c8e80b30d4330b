"""A KV cache in pages: appending with the position rotation, and attention
over a prefix that the batch shares and each row's own pages.

Thin forms of zg_paged_append_device and zg_paged_attn_device
(include/zg_hip.h) over torch tensors on the context's device.  The pool is
two tensors [pages, page_tokens, kv_heads, head_dim], bfloat16 or float32
(slices of one interleaved pool will do); a row's tokens lie in the pages its
row of the table lists.  Calls go to torch's current stream, or to the torch
stream `stream`, and return without waiting; what that stream has to wait for
before it reads the tensors is the caller's to say.  No gradient passes through
them: what they write may not require one.
"""
import numpy as np

from . import _lib as L
from ._torch import device_array, dtype_code, launching, malformed, on_device, room, stream_of, written


def cache(keys, values):
    """The zg_paged_kv of a pool's two tensors."""
    if keys.dim() != 4 or keys.shape != values.shape or keys.dtype != values.dtype or keys.stride() != values.stride():
        malformed("paged cache: keys and values [pages, page_tokens, kv_heads, head_dim] of one type and stride")
    pages, page_tokens, heads, dim = keys.shape
    if keys.stride()[1:] != (heads * dim, dim, 1) or keys.device != values.device:
        malformed("paged cache: a page's slots, heads and elements are contiguous")
    kv = L.PagedKv(keys.data_ptr(), values.data_ptr(), pages, page_tokens,
                   keys.stride(0) if pages > 1 else page_tokens * heads * dim, heads, dim,
                   dtype_code(keys, "paged cache"))
    kv.tensors = (keys, values)  # the pool lives as long as its description
    return kv


def rows(table, prefix=None, prefix_tokens=0):
    """The zg_paged_rows of a table [rows, stride] (int32; a view's rows may lie
    further apart, and then count as that long) and of the shared prefix's
    pages."""
    if table.dim() != 2 or str(table.dtype) != "torch.int32" or (table.shape[1] > 1 and table.stride(1) != 1):
        malformed("page table: int32 [rows, pages]")
    if prefix is not None and (prefix.dim() != 1 or prefix.dtype != table.dtype or not prefix.is_contiguous() or
                               prefix.device != table.device):
        malformed("prefix pages: int32 [pages]")
    stride = table.stride(0) if table.shape[0] > 1 else table.shape[1]
    # a length may ask for entries up to the row stride: the last row's are
    # there too
    if table.storage_offset() + table.shape[0] * stride > table.untyped_storage().nbytes() // 4:
        malformed("page table: the last row's stride ends past the tensor's storage")
    r = L.PagedRows(table.data_ptr(), table.shape[0], stride,
                    prefix.data_ptr() if prefix is not None and prefix.numel() else None, prefix_tokens)
    r.tensors = (table, prefix)
    return r


def host_ints(a, what):
    """A host array as int32; what that would cut off or wrap is refused."""
    a = np.asarray(a)
    if a.dtype != np.int32 and a.size and (a.dtype.kind not in "iu" or a.min() < -2 ** 31 or a.max() >= 2 ** 31):
        malformed(f"{what}: whole numbers of 32 bits")
    return np.ascontiguousarray(a, np.int32)


def admit(kv, table, lengths, q_heads, prefix=None, prefix_tokens=0):
    """Whether a batch's page tables, still in host memory (numpy int32, or
    what int32 holds without a change), fit the pool; ZgError with the reason
    if they do not."""
    import ctypes as C
    table, lengths = host_ints(table, "page table"), host_ints(lengths, "lengths")
    shared = None if prefix is None else host_ints(prefix, "prefix pages")
    if table.ndim != 2 or lengths.shape != table.shape[:1]:
        malformed("page table [rows, pages] and lengths [rows]")
    if prefix_tokens > (0 if shared is None else shared.size) * max(1, kv.page_tokens):
        malformed("prefix pages: fewer than its tokens need")
    r = L.PagedRows(table.ctypes.data, table.shape[0], table.shape[1],
                    shared.ctypes.data if shared is not None and shared.size else None, prefix_tokens)
    why = C.create_string_buffer(256)
    rc = L.lib().zg_paged_admit(kv, r, lengths.ctypes.data, q_heads, why, len(why))
    if rc != L.COMPLETED:
        raise L.ZgError(rc, why.value.decode())


def append(ctx, kv, r, k, v, positions, q=None, q_out=None, q_norm=None, k_norm=None, eps=1e-6, rotate=0,
           theta_scale=1.0, token_rows=None, status=None, stream=None):
    """zg_paged_append_device: k, v [tokens, kv_heads, head_dim] and q
    [tokens, q_heads, head_dim], of any token stride; q_out like q,
    contiguous."""
    import torch
    if k.dim() != 3 or (q is not None and q.dim() != 3):
        malformed("paged append: q, k and v [tokens, heads, head_dim]")
    tokens = k.shape[0]
    if k.shape[1:] != (kv.kv_heads, kv.head_dim) or v.shape != k.shape or v.dtype != k.dtype:
        malformed("paged append: k and v [tokens, kv_heads, head_dim]")
    for t, name in ((k, "k"), (v, "v")):
        if t.stride()[1:] != (kv.head_dim, 1):
            malformed(f"paged append: {name}'s heads are contiguous")
    q_heads = 0
    if q is not None:
        q_heads = q.shape[1]
        if (q.shape != (tokens, q_heads, kv.head_dim) or q.dtype != k.dtype or q.stride(2) != 1 or
                q_out is None or q_out.shape != q.shape or q_out.dtype != q.dtype or not q_out.is_contiguous()):
            malformed("paged append: q and q_out [tokens, q_heads, head_dim]")
    for t, name in zip(kv.tensors + (q_out,), ("keys", "values", "q_out")):
        written(t, name)
    strides = [t.stride(0) if tokens > 1 else t.shape[1] * t.stride(1) for t in (k, v)]
    q_stride = 0 if q is None else q.stride(0) if tokens > 1 else q_heads * q.stride(1)
    args = (device_array(ctx, q_norm, "q_norm", torch.float32, kv.head_dim),
            device_array(ctx, k_norm, "k_norm", torch.float32, kv.head_dim), eps, rotate, theta_scale,
            device_array(ctx, positions, "positions", torch.int32, tokens),
            device_array(ctx, token_rows, "token_rows", torch.int32, tokens), on_device(ctx, q_out, "q_out"),
            device_array(ctx, status, "status", torch.int32, 1))
    for t, name in zip(kv.tensors + r.tensors, ("keys", "values", "page table", "prefix pages")):
        on_device(ctx, t, name)
    tensors = kv.tensors + r.tensors + (k, v, positions, q, q_out, q_norm, k_norm, token_rows, status)
    with launching(ctx, stream, tensors) as st:
        ctx.check(L.lib().zg_paged_append_device(
            ctx.h, kv, r, tokens, q_heads, on_device(ctx, q, "q"), q_stride, 0 if q is None else q.stride(1),
            on_device(ctx, k, "k"), strides[0], on_device(ctx, v, "v"), strides[1], dtype_code(k, "paged append"),
            *args, st))


def attend_workspace(kv, r, q_heads):
    """Bytes of attend's workspace; ZgError where it refuses the arguments."""
    n = L.lib().zg_paged_attn_workspace_bytes(kv, r, q_heads)
    if not n:
        malformed("paged attention is not offered for this cache, table or head count")
    return n


def attend(ctx, kv, r, lengths, q, scale, out=None, workspace=None, status=None, stream=None):
    """zg_paged_attn_device: q and out [rows, q_heads, head_dim], of any row
    stride; returns out.  Without a workspace (uint8) one is made for the
    call."""
    import torch
    if q.dim() != 3 or q.shape[0] != r.rows or q.shape[2] != kv.head_dim or q.stride()[1:] != (kv.head_dim, 1):
        malformed("paged attention: q [rows, q_heads, head_dim] with contiguous heads")
    if out is None:
        with torch.cuda.stream(stream_of(ctx, stream)):
            out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    written(out, "out")
    if out.shape != q.shape or out.dtype != q.dtype or out.stride()[1:] != q.stride()[1:]:
        malformed("paged attention: out like q")
    if r.prefix_tokens > (0 if r.tensors[1] is None else r.tensors[1].numel()) * kv.page_tokens:
        malformed("prefix pages: fewer than its tokens need")
    workspace = room(ctx, stream, workspace, attend_workspace(kv, r, q.shape[1]))
    strides = [t.stride(0) if r.rows > 1 else q.shape[1] * kv.head_dim for t in (q, out)]
    for t, name in zip(kv.tensors + r.tensors, ("keys", "values", "page table", "prefix pages")):
        on_device(ctx, t, name)
    tensors = kv.tensors + r.tensors + (lengths, q, workspace, out, status)
    with launching(ctx, stream, tensors) as st:
        ctx.check(L.lib().zg_paged_attn_device(
            ctx.h, kv, r, device_array(ctx, lengths, "lengths", torch.int32, r.rows), q.shape[1],
            on_device(ctx, q, "q"), strides[0], dtype_code(q, "paged attention"), scale,
            on_device(ctx, workspace, "workspace"), on_device(ctx, out, "out"), strides[1],
            device_array(ctx, status, "status", torch.int32, 1), st))
    return out

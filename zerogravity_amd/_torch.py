"""Torch tensors as arguments of the device entry points."""
import contextlib

from . import _lib as L

_SIDE = {}  # device -> the stream that stands in for torch's default one


def malformed(why):
    raise L.ZgError(L.E_MALFORMED, why)


def dtype_code(t, what):
    import torch
    code = {torch.float32: L.F32, torch.bfloat16: L.BF16}.get(t.dtype)
    if code is None:
        raise L.ZgError(L.E_UNSUPPORTED, f"{what}: float32 or bfloat16")
    return code


def device_array(ctx, t, what, dtype, *shape):
    """The pointer of a contiguous tensor of this type and shape (None: any
    extent) on the context's device; None stays None."""
    if t is None:
        return None
    if t.dtype != dtype or t.dim() != len(shape) or any(n is not None and n != m for n, m in zip(shape, t.shape)):
        malformed(f"{what}: {dtype} of shape {shape}, not {t.dtype} of {tuple(t.shape)}")
    if not t.is_contiguous():
        malformed(f"{what}: contiguous")
    return on_device(ctx, t, what)


def on_device(ctx, t, what):
    if t is None:
        return None
    if not t.is_cuda or (ctx is not None and t.device.index != ctx.device):
        malformed(f"{what}: on the context's device")
    return t.data_ptr()


def written(t, what):
    """A tensor that a call writes to: autograd does not see that."""
    import torch
    if t is not None and t.requires_grad and torch.is_grad_enabled():
        malformed(f"{what}: written without autograd's knowledge; detach it, or call under torch.no_grad()")


def stream_of(ctx, stream):
    """The torch stream of one call: the one given, else the current one."""
    import torch
    if stream is None:
        return torch.cuda.current_stream(ctx.device)
    if stream.device.index != ctx.device:
        malformed("stream: of the context's device")
    return stream


def room(ctx, stream, workspace, need):
    """A call's workspace: the caller's, or one that torch's allocator ties to
    the call's stream."""
    import torch
    if workspace is None:
        with torch.cuda.stream(stream_of(ctx, stream)):
            return torch.empty(max(need, 16), dtype=torch.uint8, device=f"cuda:{ctx.device}")
    if workspace.numel() * workspace.element_size() < need or not workspace.is_contiguous():
        malformed(f"a workspace of {need} bytes")
    return workspace


@contextlib.contextmanager
def launching(ctx, stream, tensors):
    """The handle of the call's stream.  On another stream than the current
    one the memory of the call's tensors is kept until it is through, whatever
    becomes of them.  The library takes a null handle for its context's own
    stream, which does not wait for torch's default stream; a call on the
    default stream therefore runs on a stream that waits for it and that it
    waits for."""
    import torch
    stream = stream_of(ctx, stream)
    if stream != torch.cuda.current_stream(ctx.device):
        for t in tensors:
            if t is not None and t.is_cuda:  # what is not is refused
                t.record_stream(stream)
    if stream.cuda_stream:
        yield stream.cuda_stream
        return
    if ctx.device not in _SIDE:
        _SIDE[ctx.device] = torch.cuda.Stream(ctx.device)
    side = _SIDE[ctx.device]
    side.wait_stream(stream)
    yield side.cuda_stream
    stream.wait_stream(side)

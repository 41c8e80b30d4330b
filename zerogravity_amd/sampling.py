"""Logits before the readout: penalties for repeated tokens, biases, a
grammar's mask, and the highest token left.

A thin form of zg_logits_adjust_device (include/zg_hip.h) over torch tensors
on the context's device.  Calls go to torch's current stream, or to the torch
stream `stream`, and return without waiting; what that stream has to wait for
before it reads the tensors is the caller's to say.  No gradient passes through
them: what they write may not require one.
"""
from . import _lib as L
from ._torch import device_array, dtype_code, launching, malformed, on_device, room, written


def rules(history=None, history_lengths=None, prompt_lengths=None, repetition=None, frequency=None, presence=None,
          bias_ids=None, bias_values=None, bias_lengths=None, masks=None, mask_of=None):
    """The zg_logit_rules of a batch's tensors; None: that rule is off.  Ids,
    lengths, masks (32 tokens a word) and mask_of are int32, the rest
    float32; bias_values and bias_lengths count with bias_ids only, mask_of
    with masks only."""
    import torch
    if bias_ids is None:
        bias_values = bias_lengths = None
    if masks is None:
        mask_of = None
    ints = dict(history=history, history_lengths=history_lengths, prompt_lengths=prompt_lengths, bias_ids=bias_ids,
                bias_lengths=bias_lengths, masks=masks, mask_of=mask_of)
    floats = dict(repetition=repetition, frequency=frequency, presence=presence, bias_values=bias_values)
    shaped = {"history": 2, "bias_ids": 2, "bias_values": 2, "masks": 2}
    for name, t in {**ints, **floats}.items():
        if t is not None and (t.dim() != shaped.get(name, 1) or not t.is_contiguous() or
                              t.dtype != (torch.int32 if name in ints else torch.float32)):
            malformed(f"{name}: contiguous, {'int32' if name in ints else 'float32'}, {shaped.get(name, 1)} dimensions")
    if (bias_ids is not None and bias_values is not None) and bias_ids.shape != bias_values.shape:
        malformed("bias_values: like bias_ids")

    def p(t):
        return None if t is None else t.data_ptr()

    def wide(t):
        return 0 if t is None else t.shape[1]

    u = L.LogitRules(p(history), wide(history), p(history_lengths), p(prompt_lengths), p(repetition), p(frequency),
                     p(presence), p(bias_ids), p(bias_values), wide(bias_ids), p(bias_lengths), p(masks),
                     0 if masks is None else masks.shape[0], wide(masks), p(mask_of))
    u.tensors = {**ints, **floats}
    return u


def adjust(ctx, logits, u, out=None, greedy=None, record=False, workspace=None, status=None, stream=None):
    """zg_logits_adjust_device: logits and out [rows, vocab], of any row
    stride (out None: in place); greedy [rows] int32 or None.  Returns out.
    Without a workspace (uint8) one is made for the call."""
    import torch
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        malformed("logits [rows, vocab]")
    out = logits if out is None else out
    written(out, "out")
    if out.shape != logits.shape or out.dtype != logits.dtype or (out.shape[1] > 1 and out.stride(1) != 1):
        malformed("out: like logits")
    n, vocab = logits.shape
    for name, t in u.tensors.items():
        on_device(ctx, t, name)
        if t is not None and name != "masks" and t.shape[0] != n:
            malformed(f"{name}: one entry for each of {n} rows")
    need = L.lib().zg_logits_adjust_workspace_bytes(n, vocab)
    workspace = None if greedy is None else room(ctx, stream, workspace, need)
    strides = [t.stride(0) if n > 1 else vocab for t in (logits, out)]
    tensors = (*u.tensors.values(), logits, out, greedy, workspace, status)
    with launching(ctx, stream, tensors) as st:
        ctx.check(L.lib().zg_logits_adjust_device(
            ctx.h, n, vocab, on_device(ctx, logits, "logits"), strides[0], dtype_code(logits, "logits"), u,
            on_device(ctx, out, "out"), strides[1], device_array(ctx, greedy, "greedy", torch.int32, n), int(record),
            on_device(ctx, workspace, "workspace"), device_array(ctx, status, "status", torch.int32, 1), st))
    return out

"""Prefill of packed prompts for linear attention with a decay per head.

Per sequence and v-head h (q/k head h // (HV / H)), k-last state S [128, 128]:

    S_t = exp(log_decay_t) S_{t-1} + v_t k_t^T        output_t = scale * S_t q_t

``run(q, k, v, state, log_decay, cu_seqlens, scale) -> (output, new_state)``
    q, k [T, H, 128] bf16; v, output [T, HV, 128] bf16; state (or None: zero) and
    new_state [N, HV, 128, 128] fp32; log_decay [HV] or [T, HV] fp32 (natural
    logarithm, <= 0; -inf forgets the state); cu_seqlens [N + 1] int32 or int64,
    read on the device only; scale float or 0-d tensor, None / 0 -> 1/sqrt(128).

A sequence without tokens keeps its state (zero where ``state`` is None).
Tokens outside [cu_seqlens[0], cu_seqlens[N]) get a zero output and are not read
into any state.  Inputs are never modified; ``run_into(..., output, new_state)``
is the destination-passing form and accepts ``new_state is state``.  The work
is queued on the current stream of the inputs' device without a host
synchronisation (unless ``scale`` is a device tensor, which is read with
``.item()``); the workspace comes from torch's caching allocator.  No gradients.
The chunked products take 64 tokens at a time: a value of v that is not finite
spoils the outputs of its whole chunk, earlier tokens' among them.
"""
from __future__ import annotations

import torch

from . import _common as C
from ._lib import check, lib


def _inputs(q, k, v, state, log_decay, cu_seqlens):
    dev = C.cuda_device_of(q)
    bf = torch.bfloat16
    q, k, v = C.require16(q, "q", bf, dev), C.require16(k, "k", bf, dev), C.require16(v, "v", bf, dev)
    if q.dim() != 3:
        raise ValueError(f"q must be [T, H, K], got {tuple(q.shape)}")
    T = q.shape[0]
    H, HV, K, V = C.require_heads(q, k, v, (T,))
    g, per_token = C.require_log_decay(log_decay, (T,), HV, dev)
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise TypeError("cu_seqlens must be an int32 or int64 tensor")
    if cu_seqlens.device != dev:
        raise ValueError(f"cu_seqlens is on {cu_seqlens.device}, expected {dev}")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens must be a 1-d tensor of N + 1 offsets")
    N = cu_seqlens.numel() - 1
    if state is not None:
        state = C.require16(state, "state", torch.float32, dev, 32)
        if tuple(state.shape) != (N, HV, V, K):
            raise ValueError(f"state must be {(N, HV, V, K)}, got {tuple(state.shape)}")
    return dev, (q, k, v, state, g, cu_seqlens.contiguous()), per_token, (T, N, H, HV, K, V)


def _run_checked(dev, tensors, per_token, dims, scale, output, new_state):
    q, k, v, state, g, cu = tensors
    T, N, H, HV, K, V = dims
    with C.on_device(dev):
        nbytes = lib().gdn_decay_prefill_workspace_bytes(N, T, HV)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        st = lib().gdn_decay_prefill_fwd(
            C.ptr(q), C.ptr(k), C.ptr(v), C.ptr(state), C.ptr(g), per_token, C.ptr(cu),
            int(cu.dtype == torch.int64), N, T, C.normalize_scale(scale, K), H, HV, K, V, C.ptr(output),
            C.ptr(new_state), C.ptr(ws), nbytes, C.stream_handle(dev))
    check("gdn_decay_prefill_fwd", st)
    return output, new_state


def run_into(q, k, v, state, log_decay, cu_seqlens, scale, output, new_state):
    """Destination-passing form of ``run`` (``new_state`` may be ``state``)."""
    dev, tensors, per_token, dims = _inputs(q, k, v, state, log_decay, cu_seqlens)
    T, N, H, HV, K, V = dims
    C.require_out(output, "output", torch.bfloat16, (T, HV, V), dev)
    C.require_out(new_state, "new_state", torch.float32, (N, HV, V, K), dev)
    return _run_checked(dev, tensors, per_token, dims, scale, output, new_state)


def run(q, k, v, state, log_decay, cu_seqlens, scale):
    """See the module docstring."""
    dev, tensors, per_token, dims = _inputs(q, k, v, state, log_decay, cu_seqlens)
    T, N, H, HV, K, V = dims
    output = torch.empty((T, HV, V), dtype=torch.bfloat16, device=dev)
    new_state = torch.empty((N, HV, V, K), dtype=torch.float32, device=dev)
    return _run_checked(dev, tensors, per_token, dims, scale, output, new_state)

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
spoils the outputs of its whole chunk, earlier tokens' among them.  Other values
that are not finite reach what the formula lets them reach, but may arrive as NaN
where it has an infinity.

The states are advanced in fp32.  For the outputs the state before a chunk and the
decayed scores are rounded to bf16, so an output is off by up to 2^-8 of
scale * (|S| |q| + sum |decayed score| |v|) beside its own rounding (all of it
together about 0.0023 of the outputs' norm, 0.0017 from their own rounding).
``output`` must not overlap an input, nor ``new_state`` any but ``state``.
"""
from __future__ import annotations

import torch

from . import _common as C
from ._lib import check, lib


_BF16, _F32 = torch.bfloat16, torch.float32
_MIN_SEGMENT = 256  # calls of up to this many tokens need no workspace


def _inputs(q, k, v, state, log_decay, cu_seqlens):
    dev = C.cuda_device_of(q)
    ready = C.ready
    if not ready(q, _BF16, dev):
        q = C.require16(q, "q", _BF16, dev)
    if not ready(k, _BF16, dev):
        k = C.require16(k, "k", _BF16, dev)
    if not ready(v, _BF16, dev):
        v = C.require16(v, "v", _BF16, dev)
    qs, vs = q.shape, v.shape
    if len(qs) != 3:
        raise ValueError(f"q must be [T, H, K], got {tuple(qs)}")
    T, H, K = qs
    if k.shape != qs or len(vs) != 3 or vs[0] != T or H < 1 or vs[1] < 1:
        C.require_heads(q, k, v, (T,))
    _, HV, V = vs
    if ready(log_decay, _F32, dev) and log_decay.shape == (T, HV):
        g, per_token = log_decay, 1
    else:
        g, per_token = C.require_log_decay(log_decay, (T,), HV, dev)
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise TypeError("cu_seqlens must be an int32 or int64 tensor")
    if cu_seqlens.device != dev:
        raise ValueError(f"cu_seqlens is on {cu_seqlens.device}, expected {dev}")
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must be a 1-d tensor of N + 1 offsets")
    N = cu_seqlens.shape[0] - 1
    if state is not None:
        if not ready(state, _F32, dev):
            state = C.require16(state, "state", _F32, dev, 32)
        if state.shape != (N, HV, V, K):
            raise ValueError(f"state must be {(N, HV, V, K)}, got {tuple(state.shape)}")
    return dev, q, k, v, state, g, per_token, cu_seqlens.contiguous(), T, N, H, HV, K, V


def _launch(inputs, scale, output, new_state):
    dev, q, k, v, state, g, per_token, cu, T, N, H, HV, K, V = inputs
    if dev.index != C.current_device():
        with torch.cuda.device(dev):
            return _launch(inputs, scale, output, new_state)
    L = lib()
    nbytes = L.gdn_decay_prefill_workspace_bytes(N, T, HV) if T > _MIN_SEGMENT else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    st = L.gdn_decay_prefill_fwd(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if state is None else state.data_ptr(), g.data_ptr(), per_token,
        cu.data_ptr(), cu.dtype is torch.int64, N, T, C.normalize_scale(scale, K), H, HV, K, V, output.data_ptr(),
        new_state.data_ptr(), 0 if ws is None else ws.data_ptr(), nbytes, C.stream_handle(dev))
    if st:
        check("gdn_decay_prefill_fwd", st)


def run_into(q, k, v, state, log_decay, cu_seqlens, scale, output, new_state):
    """Destination-passing form of ``run`` (``new_state`` may be ``state``)."""
    inputs = _inputs(q, k, v, state, log_decay, cu_seqlens)
    dev, _, _, _, _, _, _, _, T, N, H, HV, K, V = inputs
    C.require_out(output, "output", _BF16, (T, HV, V), dev)
    C.require_out(new_state, "new_state", _F32, (N, HV, V, K), dev)
    _launch(inputs, scale, output, new_state)
    return output, new_state


def run(q, k, v, state, log_decay, cu_seqlens, scale):
    """See the module docstring."""
    inputs = _inputs(q, k, v, state, log_decay, cu_seqlens)
    dev, _, _, v, state, _, _, _, T, N, H, HV, K, V = inputs
    output = torch.empty_like(v)
    new_state = torch.empty((N, HV, V, K), dtype=_F32, device=dev)
    _launch(inputs, scale, output, new_state)
    return output, new_state

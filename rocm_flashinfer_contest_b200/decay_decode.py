"""Single-token linear attention with a decay per head, over states or a pool.

Per entry and v-head h (q/k head h // (HV / H)), k-last state S [128, 128]:

    S' = exp(log_decay) S + v k^T            output = scale * S' q

``run(q, k, v, state, log_decay, scale) -> (output, new_state)``
    state [B, HV, 128, 128] fp32 or None (zero); new_state is a fresh tensor and
    no input is modified.  ``run_into(..., output, new_state)`` is the
    destination-passing form; ``new_state`` may be ``state``.

``run_pool(q, k, v, initial_state, initial_state_indices, log_decay, scale=None,
output=None, output_state_indices=None) -> (output, initial_state)``
    The serving form: entry i advances slot ``initial_state_indices[i]`` of the
    pool [slots, HV, 128, 128] (fp32, or bf16: advanced in fp32 and rounded once
    when stored) in place, or writes slot ``output_state_indices[i]``.  An index
    outside the pool is padding (-1): zero output, no state touched; an output
    index outside it skips the write.  No slot may be written by one entry and
    read or written by another.

q, k [B, 1, H, 128] bf16; v, output [B, 1, HV, 128] bf16; log_decay [HV] or
[B, 1, HV] fp32 (natural logarithm, <= 0; -inf forgets the state); scale float
or 0-d tensor, None / 0 -> 1/sqrt(128); indices [B] int32 or int64.  One kernel
launch on the current stream of the inputs' device, no host synchronisation
(unless ``scale`` is a device tensor, which is read with ``.item()``), no
gradients.
"""
from __future__ import annotations

import torch

from . import _common as C
from ._lib import check, lib


def _inputs(q, k, v, log_decay):
    dev = C.cuda_device_of(q)
    bf = torch.bfloat16
    q, k, v = C.require16(q, "q", bf, dev), C.require16(k, "k", bf, dev), C.require16(v, "v", bf, dev)
    if q.dim() != 4 or q.shape[1] != 1:
        raise ValueError(f"q must be [B, 1, H, K], got {tuple(q.shape)}")
    B = q.shape[0]
    H, HV, K, V = C.require_heads(q, k, v, (B, 1))
    g, per_token = C.require_log_decay(log_decay, (B, 1), HV, dev)
    return dev, (q, k, v, g), per_token, (B, H, HV, K, V)


def _launch(dev, tensors, per_token, dims, scale, pool_in, pool_out, idx, out_idx, output):
    q, k, v, g = tensors
    B, H, HV, K, V = dims
    with C.on_device(dev):
        st = lib().gdn_decay_decode_fwd(
            C.ptr(q), C.ptr(k), C.ptr(v), C.ptr(pool_in), C.ptr(pool_out), int(pool_out.dtype == torch.bfloat16),
            C.ptr(idx), C.ptr(out_idx), int(idx is not None and idx.dtype == torch.int64), C.ptr(g), per_token,
            C.normalize_scale(scale, K), B, H, HV, K, V, pool_out.shape[0], C.ptr(output), C.stream_handle(dev))
    check("gdn_decay_decode_fwd", st)


def _run_checked(dev, tensors, per_token, dims, state, scale, output, new_state):
    B, H, HV, K, V = dims
    if state is not None:
        state = C.require16(state, "state", torch.float32, dev)
        if tuple(state.shape) != (B, HV, V, K):
            raise ValueError(f"state must be {(B, HV, V, K)}, got {tuple(state.shape)}")
    _launch(dev, tensors, per_token, dims, scale, state, new_state, None, None, output)
    return output, new_state


def run_into(q, k, v, state, log_decay, scale, output, new_state):
    """Destination-passing form of ``run`` (``new_state`` may be ``state``)."""
    dev, tensors, per_token, dims = _inputs(q, k, v, log_decay)
    B, H, HV, K, V = dims
    C.require_out(output, "output", torch.bfloat16, (B, 1, HV, V), dev)
    C.require_out(new_state, "new_state", torch.float32, (B, HV, V, K), dev)
    return _run_checked(dev, tensors, per_token, dims, state, scale, output, new_state)


def run(q, k, v, state, log_decay, scale):
    """See the module docstring."""
    dev, tensors, per_token, dims = _inputs(q, k, v, log_decay)
    B, H, HV, K, V = dims
    output = torch.empty((B, 1, HV, V), dtype=torch.bfloat16, device=dev)
    new_state = torch.empty((B, HV, V, K), dtype=torch.float32, device=dev)
    return _run_checked(dev, tensors, per_token, dims, state, scale, output, new_state)


def run_pool(q, k, v, initial_state, initial_state_indices, log_decay, scale=None, output=None,
             output_state_indices=None):
    """See the module docstring."""
    dev, tensors, per_token, dims = _inputs(q, k, v, log_decay)
    B, H, HV, K, V = dims
    pool = C.require_pool(initial_state, HV, V, K, dev)
    idx = C.require_indices(initial_state_indices, B, dev, "initial_state_indices")
    out_idx = None if output_state_indices is None else \
        C.require_indices(output_state_indices, B, dev, "output_state_indices", like=idx)
    if output is None:
        output = torch.empty((B, 1, HV, V), dtype=torch.bfloat16, device=dev)
    else:
        C.require_out(output, "output", torch.bfloat16, (B, 1, HV, V), dev)
    _launch(dev, tensors, per_token, dims, scale, pool, pool, idx, out_idx, output)
    return output, initial_state

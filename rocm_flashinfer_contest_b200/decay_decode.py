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
gradients.  ``output`` must not overlap an input.
"""
from __future__ import annotations

import torch

from . import _common as C
from ._lib import check, lib


_BF16, _F32 = torch.bfloat16, torch.float32


def _inputs(q, k, v, log_decay):
    dev = C.cuda_device_of(q)
    ready = C.ready
    if not ready(q, _BF16, dev):
        q = C.require16(q, "q", _BF16, dev)
    if not ready(k, _BF16, dev):
        k = C.require16(k, "k", _BF16, dev)
    if not ready(v, _BF16, dev):
        v = C.require16(v, "v", _BF16, dev)
    qs, vs = q.shape, v.shape
    if len(qs) != 4 or qs[1] != 1:
        raise ValueError(f"q must be [B, 1, H, K], got {tuple(qs)}")
    B, _, H, K = qs
    if k.shape != qs or len(vs) != 4 or vs[:2] != qs[:2] or H < 1 or vs[2] < 1:
        C.require_heads(q, k, v, (B, 1))
    _, _, HV, V = vs
    if ready(log_decay, _F32, dev) and log_decay.shape == (HV,):
        return dev, q, k, v, log_decay, 0, B, H, HV, K, V
    g, per_token = C.require_log_decay(log_decay, (B, 1), HV, dev)
    return dev, q, k, v, g, per_token, B, H, HV, K, V


def _launch(inputs, scale, pool_in, pool_out, idx, out_idx, output):
    dev, q, k, v, g, per_token, B, H, HV, K, V = inputs
    if dev.index != C.current_device():
        with torch.cuda.device(dev):
            return _launch(inputs, scale, pool_in, pool_out, idx, out_idx, output)
    st = lib().gdn_decay_decode_fwd(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if pool_in is None else pool_in.data_ptr(), pool_out.data_ptr(),
        pool_out.dtype is _BF16, 0 if idx is None else idx.data_ptr(), 0 if out_idx is None else out_idx.data_ptr(),
        idx is not None and idx.dtype is torch.int64, g.data_ptr(), per_token, C.normalize_scale(scale, K),
        B, H, HV, K, V, pool_out.shape[0], output.data_ptr(), C.stream_handle(dev))
    if st:
        check("gdn_decay_decode_fwd", st)


def _state(state, inputs):
    dev, _, _, _, _, _, B, _, HV, K, V = inputs
    if state is not None:
        state = C.require16(state, "state", _F32, dev)
        if tuple(state.shape) != (B, HV, V, K):
            raise ValueError(f"state must be {(B, HV, V, K)}, got {tuple(state.shape)}")
    return state


def run_into(q, k, v, state, log_decay, scale, output, new_state):
    """Destination-passing form of ``run`` (``new_state`` may be ``state``)."""
    inputs = _inputs(q, k, v, log_decay)
    dev, _, _, _, _, _, B, H, HV, K, V = inputs
    C.require_out(output, "output", _BF16, (B, 1, HV, V), dev)
    C.require_out(new_state, "new_state", _F32, (B, HV, V, K), dev)
    _launch(inputs, scale, _state(state, inputs), new_state, None, None, output)
    return output, new_state


def run(q, k, v, state, log_decay, scale):
    """See the module docstring."""
    inputs = _inputs(q, k, v, log_decay)
    dev, q, k, v, _, _, B, H, HV, K, V = inputs
    output = torch.empty_like(v)
    new_state = torch.empty((B, HV, V, K), dtype=_F32, device=dev)
    _launch(inputs, scale, _state(state, inputs), new_state, None, None, output)
    return output, new_state


def run_pool(q, k, v, initial_state, initial_state_indices, log_decay, scale=None, output=None,
             output_state_indices=None):
    """See the module docstring."""
    inputs = _inputs(q, k, v, log_decay)
    dev, q, k, v, _, _, B, H, HV, K, V = inputs
    C.require_pool(initial_state, HV, V, K, dev)
    idx, out_idx = C.require_index_pair(initial_state_indices, output_state_indices, B, dev,
                                        ("initial_state_indices", "output_state_indices"))
    if output is None:
        output = torch.empty_like(v)
    else:
        C.require_out(output, "output", _BF16, (B, 1, HV, V), dev)
    _launch(inputs, scale, initial_state, initial_state, idx, out_idx, output)
    return output, initial_state

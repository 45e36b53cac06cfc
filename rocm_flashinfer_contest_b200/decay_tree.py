"""Trees of drafted tokens for linear attention with a decay per head.

Speculative decoding drafts several continuations of each sequence at once.
``run`` scores all nodes of each entry's tree against the entry's pooled state
without changing it; ``commit`` then advances the state over the accepted path.

``run(q, k, v, initial_state, initial_state_indices, parents, log_decay,
scale=None, output=None) -> output``
    Node t of entry i continues from node ``parents[i, t]`` (before it, in
    [0, t)) or, for -1, from pool slot ``initial_state_indices[i]``:
    output[i, t] = scale * S q_t with S the state after the path down to node t,
    advanced at each node as S' = exp(log_decay) S + v k^T.  A chain of tokens is
    ``parents[i, t] = t - 1``.  A parent below -1 or not before its node marks
    padding, which extends to whatever hangs below it: zero output, and its q, k
    and v are not used.  An index outside the pool: the entry's outputs are zero.
    Entries may share a slot.

``commit(k, v, initial_state, initial_state_indices, parents, accepted,
log_decay, output_state_indices=None) -> initial_state``
    Advances each entry's slot in place over the path down to node
    ``accepted[i]`` (or writes slot ``output_state_indices[i]``).  -1, or a node
    that does not exist or is padding, accepts nothing.  No slot may be written
    by one entry and read or written by another.

q, k [B, T, H, 128] bf16; v, output [B, T, HV, 128] bf16; T <= 64; pool
[slots, HV, 128, 128] fp32 or bf16; indices [B] int32 or int64; parents [B, T]
and accepted [B] int32; log_decay [HV] or [B, T, HV] fp32; scale float or 0-d
tensor, None / 0 -> 1/sqrt(128).  One kernel launch each on the current stream
of the inputs' device, no host synchronisation (unless ``scale`` is a device
tensor, which is read with ``.item()``), no gradients.  ``output`` must not overlap
an input.  A value of v that is not finite, at a node that is not padding, spoils
the outputs of its entry's tree; other values that are not finite reach what the
formula lets them reach, but may arrive in ``output`` as NaN where it has an infinity.
"""
from __future__ import annotations

import torch

from . import _common as C
from ._lib import check, lib

MAX_NODES = 64  # GDN_DECAY_TREE_MAX (include/gdn_decay_b200.h)


_BF16, _F32 = torch.bfloat16, torch.float32


def _inputs(q, k, v, initial_state, initial_state_indices, parents, log_decay, output_state_indices=None):
    dev = C.cuda_device_of(k)
    ready = C.ready
    if q is not None and not ready(q, _BF16, dev):
        q = C.require16(q, "q", _BF16, dev)
    if not ready(k, _BF16, dev):
        k = C.require16(k, "k", _BF16, dev)
    if not ready(v, _BF16, dev):
        v = C.require16(v, "v", _BF16, dev)
    ks, vs = k.shape, v.shape
    if len(ks) != 4:
        raise ValueError(f"k must be [B, T, H, K], got {tuple(ks)}")
    B, T, H, K = ks
    if (q is not None and q.shape != ks) or len(vs) != 4 or vs[:2] != ks[:2] or H < 1 or vs[2] < 1:
        C.require_heads(q, k, v, (B, T))
    _, _, HV, V = vs
    if T > MAX_NODES:
        raise ValueError(f"a tree has at most {MAX_NODES} nodes, got {T}")
    if ready(log_decay, _F32, dev) and log_decay.shape == (HV,):
        g, per_token = log_decay, 0
    else:
        g, per_token = C.require_log_decay(log_decay, (B, T), HV, dev)
    C.require_pool(initial_state, HV, V, K, dev)
    idx, out_idx = C.require_index_pair(initial_state_indices, output_state_indices, B, dev,
                                        ("initial_state_indices", "output_state_indices"))
    if not ready(parents, torch.int32, dev):
        parents = C.require(parents, "parents", torch.int32, dev)
    if parents.shape != (B, T):
        raise ValueError(f"parents must be {(B, T)}, got {tuple(parents.shape)}")
    return (dev, q, k, v, initial_state, idx, parents, g, per_token, B, T, H, HV, K, V), out_idx


def run(q, k, v, initial_state, initial_state_indices, parents, log_decay, scale=None, output=None):
    """See the module docstring."""
    if q is None:
        raise TypeError("q must be a torch.Tensor, got NoneType")
    inputs, _ = _inputs(q, k, v, initial_state, initial_state_indices, parents, log_decay)
    if output is None:
        output = torch.empty_like(inputs[3])
    else:
        C.require_out(output, "output", _BF16, inputs[3].shape, inputs[0])
    return _run(inputs, scale, output)


def _run(inputs, scale, output):
    dev, q, k, v, pool, idx, parents, g, per_token, B, T, H, HV, K, V = inputs
    if dev.index != C.current_device():
        with torch.cuda.device(dev):
            return _run(inputs, scale, output)
    st = lib().gdn_decay_verify_fwd(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), pool.data_ptr(), pool.dtype is _BF16, idx.data_ptr(),
        idx.dtype is torch.int64, parents.data_ptr(), g.data_ptr(), per_token, C.normalize_scale(scale, K),
        B, T, H, HV, K, V, pool.shape[0], output.data_ptr(), C.stream_handle(dev))
    if st:
        check("gdn_decay_verify_fwd", st)
    return output


def commit(k, v, initial_state, initial_state_indices, parents, accepted, log_decay, output_state_indices=None):
    """See the module docstring."""
    inputs, out_idx = _inputs(None, k, v, initial_state, initial_state_indices, parents, log_decay,
                              output_state_indices)
    dev, B = inputs[0], inputs[9]
    if not C.ready(accepted, torch.int32, dev):
        accepted = C.require(accepted, "accepted", torch.int32, dev)
    if accepted.shape != (B,):
        raise ValueError(f"accepted must be {(B,)}, got {tuple(accepted.shape)}")
    _commit(inputs, accepted, out_idx)
    return initial_state


def _commit(inputs, accepted, out_idx):
    dev, _, k, v, pool, idx, parents, g, per_token, B, T, H, HV, K, V = inputs
    if dev.index != C.current_device():
        with torch.cuda.device(dev):
            return _commit(inputs, accepted, out_idx)
    st = lib().gdn_decay_commit(
        k.data_ptr(), v.data_ptr(), pool.data_ptr(), pool.dtype is _BF16, idx.data_ptr(),
        0 if out_idx is None else out_idx.data_ptr(), idx.dtype is torch.int64, parents.data_ptr(),
        accepted.data_ptr(), g.data_ptr(), per_token, B, T, H, HV, K, V, pool.shape[0], C.stream_handle(dev))
    if st:
        check("gdn_decay_commit", st)

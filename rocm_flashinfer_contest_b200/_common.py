"""Argument handling shared by the decode and prefill ``run`` shims."""
from __future__ import annotations

import math

import torch


def normalize_scale(scale, K: int) -> float:
    """The reference's scale rule (solutions/gdn_decode/main.py:118-123,
    solutions/gdn_prefill/main.py:32-37): a tensor is read with ``.item()``,
    ``None`` or 0 means 1/sqrt(K)."""
    if isinstance(scale, torch.Tensor):
        scale = float(scale.item())
    elif scale is None:
        scale = 0.0
    else:
        scale = float(scale)
    if scale == 0.0:
        scale = 1.0 / math.sqrt(K)
    return scale


def require(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return t if t.is_contiguous() else t.contiguous()


def cuda_device_of(q: torch.Tensor) -> torch.device:
    if not isinstance(q, torch.Tensor) or q.device.type != "cuda":
        raise RuntimeError(
            "the GDN kernels run on CUDA devices only (sm_100a); got "
            f"{getattr(q, 'device', type(q).__name__)} — there is no CPU path")
    return q.device


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_handle(device: torch.device) -> int:
    """The device's current CUDA stream as a raw handle (torch's internal
    accessor, ~0.1 us, when it exists; the public one builds a Stream object
    on every call, ~2 us)."""
    if _raw_stream is not None:
        return _raw_stream(device.index if device.index is not None else torch.cuda.current_device())
    return torch.cuda.current_stream(device).cuda_stream


def ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


# ---- the decay operators and the state cache ----

# A call's host time is a good part of a small step, so the checks ask ready()
# first: one short test that nearly always passes, before the functions that say
# what is wrong or copy what can be copied.

_Tensor = torch.Tensor
current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def ready(t, dtype: torch.dtype, device: torch.device) -> bool:
    """Whether a kernel can take ``t`` as it is: its type and device, contiguous,
    on a 32-byte boundary."""
    return isinstance(t, _Tensor) and t.dtype is dtype and t.device == device and t.is_contiguous() \
        and not t.data_ptr() & 31


def require16(t, name: str, dtype: torch.dtype, device: torch.device, align: int = 16) -> torch.Tensor:
    """``require`` for a read-only operand of a kernel that loads ``align`` bytes
    at a time: a view that starts off such a boundary is copied."""
    t = require(t, name, dtype, device)
    return t if t.data_ptr() % align == 0 else t.clone()


def require_out(t, name: str, dtype: torch.dtype, shape, device: torch.device) -> torch.Tensor:
    """A tensor the kernel writes (or updates in place): taken as it is or refused."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be a contiguous {dtype} {tuple(shape)} tensor on {device}, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t


def require_log_decay(g, lead, HV: int, device: torch.device):
    """``log_decay`` as ([HV] or [*lead, HV]) fp32 -> (tensor, 1 if per token)."""
    g = require(g, "log_decay", torch.float32, device)
    if tuple(g.shape) == (HV,):
        return g, 0
    if tuple(g.shape) == (*lead, HV):
        return g, 1
    raise ValueError(f"log_decay must be {(HV,)} or {(*lead, HV)}, got {tuple(g.shape)}")


def require_heads(q, k, v, lead):
    """Head counts and sizes of q, k [*lead, H, K] and v [*lead, HV, V] -> (H, HV, K, V)."""
    n = len(lead)
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t is not None and (t.dim() != n + 2 or tuple(t.shape[:n]) != tuple(lead)):
            raise ValueError(f"{name} must be {tuple(lead)} + (heads, size), got {tuple(t.shape)}")
    H, K = k.shape[n:]
    if q is not None and tuple(q.shape) != tuple(k.shape):
        raise ValueError(f"q and k must have one shape, got {tuple(q.shape)} and {tuple(k.shape)}")
    HV, V = v.shape[n:]
    if H < 1 or HV < 1:
        raise ValueError("at least one q/k head and one v head are needed")
    return H, HV, K, V


def require_pool(pool, HV: int, V: int, K: int, device: torch.device, name: str = "initial_state"):
    """A pool of states [slots, HV, V, K], fp32 or bf16, contiguous (it is updated in place)."""
    if not isinstance(pool, torch.Tensor) or pool.dtype not in (torch.float32, torch.bfloat16) \
            or pool.device != device:
        raise TypeError(f"{name} must be an fp32 or bf16 tensor on {device}")
    if pool.dim() != 4 or tuple(pool.shape[1:]) != (HV, V, K) or not pool.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [slots, {HV}, {V}, {K}] tensor, got {tuple(pool.shape)}")
    return pool


def require_indices(idx, B: int, device: torch.device, name: str):
    """[B] int32/int64 indices on the device."""
    if not isinstance(idx, torch.Tensor) or idx.dtype not in (torch.int32, torch.int64) \
            or idx.device != device or tuple(idx.shape) != (B,):
        raise ValueError(f"{name} must be an int32/int64 [{B}] tensor on {device}")
    return idx.contiguous()


def require_index_pair(a, b, B: int, device: torch.device, names):
    """Two index tensors (``b`` may be None) as one type: the kernels take one.  Where
    they differ int32 becomes int64, never the other way: 2^32 narrowed would be
    slot 0."""
    a = require_indices(a, B, device, names[0])
    if b is not None:
        b = require_indices(b, B, device, names[1])
        if a.dtype != b.dtype:
            a, b = a.to(torch.int64), b.to(torch.int64)
    return a, b

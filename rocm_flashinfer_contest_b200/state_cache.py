"""Pool slots parked in 8 bits and read back (preempted requests, prefix states).

A cache of C slots beside a pool [slots, ...] of fp32 or bf16 states (those of
the gated delta rule or of the decay operators) is two tensors: ``codes``
[C, ...], int8 or float8_e4m3fn, one code for each value, and ``exponents``
[C, ..., last / 32] uint8, one power-of-two scale for 32 values: a quarter of
an fp32 pool's bytes.  ``empty`` allocates them.

``store(pool, slots, codes, exponents, cache_slots)``
    Writes pool slot ``slots[i]`` to cache slot ``cache_slots[i]``.  Per group of
    32 values 2^e is the smallest power of two (e >= -127) with max|x| <= 127 * 2^e
    (int8) or 448 * 2^e (e4m3); code = x / 2^e rounded to nearest-even, exponent
    byte e + 127.  A value is off by at most 2^(e-1) (int8), or by 2^-4 of itself
    or 2^(e-10) (e4m3).  A group with a value that is not finite reads back as NaN
    (byte 255).

``load(codes, exponents, cache_slots, pool, slots) -> pool``
    Reads them back: pool value = code * 2^e.

slots and cache_slots: [B] int32 or int64, on the device.  A pair
with either index outside its tensor (-1) is padding and skipped; otherwise no
two pairs may write the same slot.  One kernel launch each on the current stream of the
pool's device, no host synchronisation.
"""
from __future__ import annotations

import math

import torch

from . import _common as C
from ._lib import check, lib

GROUP = 32  # GDN_STATE_CACHE_GROUP (include/gdn_decay_b200.h)
_CODES = (torch.int8, torch.float8_e4m3fn)


def empty(num_slots: int, state_shape, dtype=torch.int8, device="cuda"):
    """``(codes, exponents)`` of ``num_slots`` slots for states of ``state_shape``
    (last size a multiple of 32), uninitialised."""
    shape = tuple(state_shape)
    if dtype not in _CODES:
        raise TypeError(f"codes are int8 or float8_e4m3fn, got {dtype}")
    if not shape or shape[-1] % GROUP != 0:
        raise ValueError(f"the last size must be a multiple of {GROUP}, got {shape}")
    codes = torch.empty((num_slots, *shape), dtype=dtype, device=device)
    return codes, torch.empty((num_slots, *shape[:-1], shape[-1] // GROUP), dtype=torch.uint8, device=device)


def _check(pool, slots, codes, exponents, cache_slots):
    dev = C.cuda_device_of(pool)
    if pool.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"pool must be fp32 or bf16, got {pool.dtype}")
    if not isinstance(codes, torch.Tensor) or codes.dtype not in _CODES:
        raise TypeError("codes must be an int8 or float8_e4m3fn tensor")
    shape, cshape = pool.shape, codes.shape
    if len(shape) < 2 or shape[-1] % GROUP != 0 or not pool.is_contiguous():
        raise ValueError(f"pool must be contiguous [slots, ..., a multiple of {GROUP}], got {tuple(shape)}")
    if cshape[1:] != shape[1:] or not codes.is_contiguous() or codes.device != dev:
        raise ValueError(f"codes must be contiguous [slots, {', '.join(map(str, shape[1:]))}] on {dev}, "
                         f"got {tuple(cshape)} on {codes.device}")
    want = (cshape[0], *shape[1:-1], shape[-1] // GROUP)
    if not (isinstance(exponents, torch.Tensor) and exponents.dtype is torch.uint8 and exponents.shape == want
            and exponents.is_contiguous() and exponents.device == dev):
        C.require_out(exponents, "exponents", torch.uint8, want, dev)
    if not isinstance(slots, torch.Tensor) or slots.dim() != 1:
        raise ValueError("slots must be a 1-d int32/int64 tensor")
    B = slots.shape[0]
    if max(B, shape[0], cshape[0]) >= 2 ** 31:
        raise ValueError("fewer than 2^31 pairs and slots are needed")
    slots, cache_slots = C.require_index_pair(slots, cache_slots, B, dev, ("slots", "cache_slots"))
    return dev, pool, slots, codes, exponents, cache_slots, B, math.prod(shape[1:])


def store(pool, slots, codes, exponents, cache_slots):
    """See the module docstring; returns ``(codes, exponents)``."""
    _store(_check(pool, slots, codes, exponents, cache_slots))
    return codes, exponents


def _store(args):
    dev, pool, slots, codes, exponents, cache_slots, B, elems = args
    if not elems:
        return
    if dev.index != C.current_device():
        with torch.cuda.device(dev):
            return _store(args)
    st = lib().gdn_state_cache_store(
        pool.data_ptr(), pool.dtype is torch.bfloat16, slots.data_ptr(), cache_slots.data_ptr(),
        slots.dtype is torch.int64, codes.data_ptr(), codes.dtype is torch.float8_e4m3fn,
        exponents.data_ptr(), B, elems, pool.shape[0], codes.shape[0], C.stream_handle(dev))
    if st:
        check("gdn_state_cache_store", st)


def load(codes, exponents, cache_slots, pool, slots):
    """See the module docstring; returns ``pool``."""
    _load(_check(pool, slots, codes, exponents, cache_slots))
    return pool


def _load(args):
    dev, pool, slots, codes, exponents, cache_slots, B, elems = args
    if not elems:
        return
    if dev.index != C.current_device():
        with torch.cuda.device(dev):
            return _load(args)
    st = lib().gdn_state_cache_load(
        codes.data_ptr(), codes.dtype is torch.float8_e4m3fn, exponents.data_ptr(), cache_slots.data_ptr(),
        slots.data_ptr(), slots.dtype is torch.int64, pool.data_ptr(), pool.dtype is torch.bfloat16,
        B, elems, pool.shape[0], codes.shape[0], C.stream_handle(dev))
    if st:
        check("gdn_state_cache_load", st)

"""Sizes at the ends of the decay operators' ranges, by status code at the C ABI and by call."""
import ctypes

import pytest
import torch

from rocm_flashinfer_contest_b200 import _lib
from test_decay_abi import COMMIT, LOAD, PREFILL, STORE, call

INV, UNS, OK = _lib.GDN_ERR_INVALID, _lib.GDN_ERR_UNSUPPORTED, _lib.GDN_OK


@pytest.mark.parametrize("N,T,HV", [(2 ** 31 - 1, 256, 1), (2 ** 31 - 1, 2 ** 31 - 1, 1), (2 ** 31 - 2, 512, 1),
                                    (2 ** 31 - 1, 0, 2 ** 31 - 1), (2 ** 26, 1, 1)])
def test_prefill_refuses_more_sequences_than_a_grid_has(N, T, HV):
    """The number of segments, T / 256 + N, does not fit 32 bits here; it was taken for a negative, small one."""
    assert call("gdn_decay_prefill_fwd", PREFILL, dict(N=N, T=T, H=1, HV=HV, ws=64, wsb=2 ** 40)) == UNS


def test_pools_without_slots_are_padding():
    """Nothing is launched where no slot could be written and there is no output."""
    assert call("gdn_decay_commit", COMMIT, dict(pool=None, slots=0)) == OK
    assert call("gdn_decay_commit", COMMIT, dict(pool=None)) == INV
    for fn, args in (("gdn_state_cache_store", STORE), ("gdn_state_cache_load", LOAD)):
        n = ctypes.c_longlong(64)
        assert call(fn, args, dict(n=n, pool=None, slots=0)) == OK
        assert call(fn, args, dict(n=n, codes=None, exps=None, cslots=0)) == OK
        assert call(fn, args, dict(n=n, pool=None)) == INV
        assert call(fn, args, dict(n=n, exps=None, slots=0)) == INV
        assert call(fn, args, dict(n=n, codes=None, slots=0)) == INV


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
def test_calls_over_a_pool_without_slots(bf16):
    from rocm_flashinfer_contest_b200 import decay_decode, decay_tree, state_cache
    bf = dict(dtype=torch.bfloat16, device="cuda")
    q, v = torch.ones(3, 5, 1, 128, **bf), torch.ones(3, 5, 2, 128, **bf)
    g = torch.zeros(2, device="cuda")
    pool = torch.empty(0, 2, 128, 128, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    idx = torch.tensor([-1, 0, 7], dtype=torch.int32, device="cuda")
    parents = torch.full((3, 5), -1, dtype=torch.int32, device="cuda")
    out = torch.full_like(v, 3.0)
    assert decay_tree.run(q, q, v, pool, idx, parents, g, output=out) is out and (out == 0).all()
    assert decay_tree.commit(q, v, pool, idx, parents, idx, g) is pool
    one = torch.full((3, 1, 2, 128), 3.0, **bf)
    o, p = decay_decode.run_pool(q[:, :1].contiguous(), q[:, :1].contiguous(), v[:, :1].contiguous(), pool, idx, g,
                                 output=one)
    assert p is pool and (o == 0).all()
    full = torch.ones(4, 2, 128, 128, dtype=pool.dtype, device="cuda")
    none, some = state_cache.empty(0, (2, 128, 128)), state_cache.empty(4, (2, 128, 128))
    some[0].fill_(3), some[1].fill_(9)
    for cache, where in ((none, full), (some, pool), (none, pool)):
        state_cache.store(where, idx, *cache, idx)
        state_cache.load(*cache, idx, where, idx)
    assert (full == 1).all() and (some[0] == 3).all() and (some[1] == 9).all()

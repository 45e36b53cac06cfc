"""Refusals of the decay operators and the state cache, by status code at the C
ABI and by exception in Python; none of them needs a GPU or launches anything."""
import ctypes

import pytest
import torch

from rocm_flashinfer_contest_b200 import _lib, decay_decode, decay_prefill, decay_tree, state_cache

INV, UNS, ALI, OK = _lib.GDN_ERR_INVALID, _lib.GDN_ERR_UNSUPPORTED, _lib.GDN_ERR_ALIGN, _lib.GDN_OK


def call(fn, defaults, over):
    d = dict(defaults)
    d.update(over)
    return getattr(_lib.lib(), fn)(*d.values())


PREFILL = dict(q=32, k=32, v=32, state=None, g=32, per=0, cu=32, cu64=0, N=1, T=64, scale=0.0, H=1, HV=2, K=128, V=128,
               out=32, new=64, ws=None, wsb=0, stream=None)


@pytest.mark.parametrize("over,code", [
    (dict(K=64), UNS), (dict(V=256), UNS), (dict(H=3, HV=4), UNS), (dict(H=0), INV), (dict(HV=0), INV),
    (dict(N=-1), INV), (dict(T=-1), INV), (dict(per=2), INV), (dict(cu64=2), INV), (dict(q=None), INV),
    (dict(g=None), INV), (dict(cu=None), INV), (dict(new=None), INV), (dict(out=None), INV),
    (dict(q=40), ALI), (dict(out=40), ALI), (dict(state=48), ALI), (dict(new=48), ALI), (dict(g=34), ALI),
    (dict(cu=36, cu64=1), ALI), (dict(N=2 ** 26, T=0), UNS),
    (dict(T=4096), INV),                                   # needs a workspace
    (dict(T=4096, ws=64, wsb=1024), INV),                  # too small
    (dict(T=4096, ws=48, wsb=1 << 30), ALI),
    (dict(state=64, new=96), INV), (dict(state=64 + 65536 * 2 - 32, new=64), INV),   # the states overlap
    (dict(N=0, T=0), OK), (dict(N=0, T=0, g=None, q=None, k=None, v=None, out=None), OK),
])
def test_prefill_refuses(over, code):
    assert call("gdn_decay_prefill_fwd", PREFILL, over) == code


def test_prefill_workspace_bytes():
    f = _lib.lib().gdn_decay_prefill_workspace_bytes
    assert f(0, 100, 4) == 0 and f(1, 0, 4) == 0 and f(1, 256, 4) == 0 and f(3, 100, 0) == 0
    # 8,192 tokens of 32 v-heads: 5 segments of 1,664 tokens, at most 2 * 8192 / 1664 = 9 slots
    assert f(1, 8192, 32) == 9 * 32 * (128 * 128 + 1) * 4
    assert f(7, 8192, 100) == 0                            # whole sequences: no segments
    assert f(1, 2 ** 31 - 1, 1) > 0


DECODE = dict(q=16, k=16, v=16, pin=4096, pout=4096, bf16=0, idx=16, oidx=None, i64=0, g=16, per=0, scale=0.0, B=1, H=1,
              HV=2, K=128, V=128, slots=4, out=16, stream=None)


@pytest.mark.parametrize("over,code", [
    (dict(K=64), UNS), (dict(H=2, HV=3), UNS), (dict(B=-1), INV), (dict(slots=-1), INV), (dict(bf16=2), INV),
    (dict(i64=-1), INV), (dict(per=3), INV), (dict(q=None), INV), (dict(pout=None), INV), (dict(g=None), INV),
    (dict(out=None), INV), (dict(q=24), ALI), (dict(pin=4100, pout=4100), ALI), (dict(idx=18), ALI),
    (dict(oidx=20, i64=1), ALI), (dict(pout=4096 + 1024), INV),                     # the pools overlap
    (dict(B=2 ** 27), UNS), (dict(B=0), OK),
])
def test_decode_refuses(over, code):
    assert call("gdn_decay_decode_fwd", DECODE, over) == code


VERIFY = dict(q=16, k=16, v=16, pool=16, bf16=0, idx=16, i64=0, par=16, g=16, per=0, scale=0.0, B=1, T=4, H=1, HV=2, K=128,
              V=128, slots=4, out=16, stream=None)
COMMIT = dict(k=16, v=16, pool=16, bf16=0, idx=16, oidx=None, i64=0, par=16, acc=16, g=16, per=0, B=1, T=4, H=1, HV=2,
              K=128, V=128, slots=4, stream=None)


@pytest.mark.parametrize("over,code", [
    (dict(T=65), UNS), (dict(T=-1), INV), (dict(K=32), UNS), (dict(H=3), UNS), (dict(pool=None), INV),
    (dict(idx=None), INV), (dict(par=None), INV), (dict(g=None), INV), (dict(k=None), INV), (dict(pool=24), ALI),
    (dict(par=18), ALI), (dict(k=8), ALI), (dict(bf16=-1), INV), (dict(B=0), OK),
])
def test_tree_refuses(over, code):
    assert call("gdn_decay_verify_fwd", VERIFY, over) == code
    assert call("gdn_decay_commit", COMMIT, over) == code


def test_tree_refuses_more():
    assert call("gdn_decay_verify_fwd", VERIFY, dict(out=None)) == INV
    assert call("gdn_decay_verify_fwd", VERIFY, dict(T=0)) == OK
    assert call("gdn_decay_commit", COMMIT, dict(acc=None)) == INV
    assert call("gdn_decay_commit", COMMIT, dict(acc=18)) == ALI


STORE = dict(pool=16, bf16=0, s=16, c=16, i64=0, codes=16, e4m3=0, exps=1, B=1, n=64, slots=2, cslots=2, stream=None)
LOAD = dict(codes=16, e4m3=0, exps=1, c=16, s=16, i64=0, pool=16, bf16=0, B=1, n=64, slots=2, cslots=2, stream=None)


@pytest.mark.parametrize("over,code", [
    (dict(n=33), UNS), (dict(n=0), INV), (dict(B=-1), INV), (dict(bf16=2), INV), (dict(e4m3=2), INV), (dict(i64=2), INV),
    (dict(pool=None), INV), (dict(codes=None), INV), (dict(exps=None), INV), (dict(s=None), INV), (dict(c=None), INV),
    (dict(pool=8), ALI), (dict(codes=4), ALI), (dict(s=20, i64=1), ALI), (dict(slots=-1), INV), (dict(cslots=-1), INV),
    (dict(n=2 ** 40, B=2 ** 30), UNS), (dict(B=0), OK),
])
def test_state_cache_refuses(over, code):
    over = {k: ctypes.c_longlong(v) if k == "n" else v for k, v in over.items()}
    assert call("gdn_state_cache_store", STORE, over) == code
    assert call("gdn_state_cache_load", LOAD, over) == code


def test_python_needs_cuda():
    x = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16)
    g, s, i = torch.zeros(1), torch.zeros(1, 1, 128, 128), torch.zeros(1, dtype=torch.int32)
    for f in (lambda: decay_decode.run(x, x, x, None, g, None),
              lambda: decay_decode.run_pool(x, x, x, s, i, g),
              lambda: decay_prefill.run(x[0], x[0], x[0], None, g, i, None),
              lambda: decay_tree.run(x, x, x, s, i, i[None], g),
              lambda: decay_tree.commit(x, x, s, i, i[None], i, g),
              lambda: state_cache.store(s, i, s.to(torch.int8), i, i),
              lambda: state_cache.load(s.to(torch.int8), i, i, s, i)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            f()


def test_state_cache_empty():
    codes, exps = state_cache.empty(3, (4, 128, 128), torch.float8_e4m3fn, device="cpu")
    assert codes.shape == (3, 4, 128, 128) and exps.shape == (3, 4, 128, 4) and exps.dtype == torch.uint8
    with pytest.raises(TypeError):
        state_cache.empty(3, (4, 128), torch.float16, device="cpu")
    with pytest.raises(ValueError):
        state_cache.empty(3, (4, 100), device="cpu")


@pytest.mark.gpu
def test_python_refuses_on_the_gpu():
    bf = dict(dtype=torch.bfloat16, device="cuda")
    q, v = torch.zeros(2, 1, 1, 128, **bf), torch.zeros(2, 1, 2, 128, **bf)
    g, pool = torch.zeros(2, device="cuda"), torch.zeros(4, 2, 128, 128, device="cuda")
    idx = torch.zeros(2, dtype=torch.int32, device="cuda")
    d = decay_decode.run_pool
    for bad in (lambda: d(q.float(), q, v, pool, idx, g), lambda: d(q, q, v, pool.half(), idx, g),
                lambda: d("q", q, v, pool, idx, g), lambda: d(q, None, v, pool, idx, g)):
        with pytest.raises((TypeError, RuntimeError)):
            bad()
    for bad in (lambda: d(q, q[:1], v, pool, idx, g), lambda: d(q[..., :64], q, v, pool, idx, g),
                lambda: d(q, q, v, pool[:, :1], idx, g), lambda: d(q, q, v, pool.transpose(2, 3), idx, g),
                lambda: d(q, q, v, pool, idx[:1], g), lambda: d(q, q, v, pool, idx.float(), g),
                lambda: d(q, q, v, pool, idx, torch.zeros(3, device="cuda")),
                lambda: d(q, q, v, pool, idx, g, None, v[:1]),
                lambda: d(q, q, v, pool, idx.cpu(), g),
                lambda: decay_decode.run(q, q, v, pool, g, None)):
        with pytest.raises(ValueError):
            bad()
    p = torch.zeros(2, 65, dtype=torch.int32, device="cuda")
    big = torch.zeros(2, 65, 1, 128, **bf)
    with pytest.raises(ValueError, match="64 nodes"):
        decay_tree.run(big, big, big, pool[:, :1].contiguous(), idx, p, g[:1])
    with pytest.raises(ValueError):
        decay_tree.run(q, q, v, pool, idx, p, g)
    with pytest.raises(_lib.GDNError):
        decay_decode.run(q[..., :64].contiguous(), q[..., :64].contiguous(), v[..., :64].contiguous(), None, g, None)
    cu = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (lambda: decay_prefill.run(q[:, 0], q[:, 0], v[:, 0], pool, g, cu, None),
                lambda: decay_prefill.run(q, q, v, None, g, cu, None),
                lambda: decay_prefill.run(q[:, 0], q[:, 0], v[:, 0], None, g, cu.cpu(), None)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        decay_prefill.run(q[:, 0], q[:, 0], v[:, 0], None, g, cu.float(), None)
    codes, exps = state_cache.empty(4, (2, 128, 128))
    for bad in (lambda: state_cache.store(pool, idx, codes[:, :1], exps, idx),
                lambda: state_cache.store(pool, idx, codes, exps[:2], idx),
                lambda: state_cache.store(pool.transpose(2, 3), idx, codes, exps, idx),
                lambda: state_cache.store(pool, idx, codes, exps, idx[:1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        state_cache.load(codes.to(torch.int16), exps, idx, pool, idx)
    many = idx[:1].expand(2 ** 31)
    with pytest.raises(ValueError, match="2\\^31"):
        state_cache.load(codes, exps, many, pool, many)

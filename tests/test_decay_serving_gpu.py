"""States of both recurrences parked in one 8-bit cache and continued from what was
read back, a server's steps with a slot parked between them, and each operator's
first call of a process inside a graph capture."""
import os
import subprocess
import sys

import pytest
import torch

from decay_reference import U_BF16, U_F32, close, decays, heads, step
from oracle import oracle
from parity import assert_output_close, assert_state_close
from test_decay_gpu import SCALE, _status, gates, prefill_case, rnd  # noqa: F401
from test_state_cache_gpu import reference

pytestmark = pytest.mark.gpu
FORMATS = [torch.int8, torch.float8_e4m3fn]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("pdt", [torch.float32, torch.bfloat16])
def test_both_recurrences_continue_from_one_cache(fmt, pdt):
    from rocm_flashinfer_contest_b200 import decay_decode, decay_prefill, gdn_decode, gdn_mtp, inputs, state_cache
    dev, HV = torch.device("cuda"), 4
    args = inputs.decode_inputs(2, 2, HV, seed=5)
    _, delta = gdn_decode.run(*inputs.to_device(args, dev))
    q, k, v, _, g, cu = prefill_case([70, 9], 2, HV, "token", 6, state=False)
    _, decay = decay_prefill.run(q, k, v, None, g, torch.tensor(cu, device=dev), None)
    # one pool and one cache: slots 0, 1 are the delta rule's, 2, 3 the decay's
    pool = torch.cat([delta, decay]).to(pdt)
    want = torch.stack([reference(x.float(), fmt)[0] for x in pool])                 # [4, HV, 128, 128] in 64 bits
    assert torch.equal(want, want.to(pdt).double())                                   # (a code fits either pool's type)
    codes, exps = state_cache.empty(6, (HV, 128, 128), fmt)
    slots, where = torch.arange(4, device=dev), torch.tensor([5, 2, 0, 3], device=dev)
    state_cache.store(pool, slots, codes, exps, where)
    pool.fill_(float("nan"))
    state_cache.load(codes, exps, where, pool, slots)
    assert torch.equal(pool.cpu().double(), want)

    # the delta rule goes on
    nxt = inputs.mtp_inputs(2, 1, 4, 2, HV, seed=7, indices=[0, 1], idx_dtype=torch.int64)
    dn = inputs.to_device(nxt, dev)
    out = torch.empty(2, 1, HV, 128, dtype=torch.bfloat16, device=dev)
    gdn_mtp.run_into(*dn[:3], pool, *dn[4:10], out, pool)
    nxt[3] = want.to(pdt)
    ro, rs = oracle.mtp(*inputs.to_cpu(nxt[:10]))
    assert_output_close(out.cpu(), ro)
    if pdt == torch.float32:
        assert_state_close(pool[:2].cpu(), rs[:2])
    # and so does the decay
    gen = torch.Generator(device="cuda").manual_seed(8)
    q, k, v = rnd(gen, 2, 1, 2, 128), rnd(gen, 2, 1, 2, 128, s=0.2), rnd(gen, 2, 1, HV, 128)
    g = gates(gen, (2, 1), HV, "token")
    o, _ = decay_decode.run_pool(q, k, v, pool, slots[2:], g, SCALE)
    ro, om, rs, rm = step(want[2:], heads(q.cpu(), HV)[:, 0], heads(k.cpu(), HV)[:, 0], v.cpu().double()[:, 0],
                          decays(g.cpu(), (2, 1), HV).exp()[:, 0], SCALE)
    close(o[:, 0], ro, U_BF16 * ro.abs() + 32 * U_F32 * om + 1e-30, "output")
    close(pool[2:], rs, 4 * U_F32 * rm + (U_BF16 * rs.abs() if pdt == torch.bfloat16 else 0) + 1e-30, "state")


@pytest.mark.parametrize("fmt", FORMATS)
def test_prompt_parked_resumed_tree_decode(fmt):
    """A prompt, its state parked and another's step meanwhile, resumed into another slot, a tree, its path, a token:
    each step's output is that of the values the cache held."""
    from rocm_flashinfer_contest_b200 import decay_decode, decay_prefill, decay_tree, state_cache
    H, HV, T = 2, 4, 6
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v, _, g, cu = prefill_case([333], H, HV, "token", 3, state=False)
    _, s = decay_prefill.run(q, k, v, None, g, torch.tensor(cu, device="cuda"), None)
    pool = torch.zeros(3, HV, 128, 128, device="cuda")
    pool[1:2] = s
    codes, exps = state_cache.empty(2, (HV, 128, 128), fmt)
    i = lambda x: torch.tensor([x], device="cuda", dtype=torch.int32)  # noqa: E731
    state_cache.store(pool, i(1), codes, exps, i(1))
    one = lambda *lead: (rnd(gen, *lead, H, 128), rnd(gen, *lead, H, 128, s=0.2), rnd(gen, *lead, HV, 128))  # noqa: E731
    decay_decode.run_pool(*one(1, 1), pool, i(1), gates(gen, (1, 1), HV, "token"))       # the slot is another's now
    state_cache.load(codes, exps, i(1), pool, i(2))
    S = reference(s[0], fmt)[0][None]                                                     # what the cache holds
    assert torch.equal(pool[2:].cpu().double(), S)
    tq, tk, tv = one(1, T)
    tg = gates(gen, (1, T), HV, "token")
    parents = torch.tensor([[-1, 0, 0, 2, 1, 3]], device="cuda", dtype=torch.int32)
    ov = decay_tree.run(tq, tk, tv, pool, i(2), parents, tg)
    decay_tree.commit(tk, tv, pool, i(2), parents, i(5), tg)
    dq, dk, dv = one(1, 1)
    dg = gates(gen, (1, 1), HV, "token")
    od, _ = decay_decode.run_pool(dq, dk, dv, pool, i(2), dg)
    Sm = S.abs()
    a = decays(tg.cpu(), (1, T), HV).exp()
    for t in (0, 2, 3, 5):
        ro, om, S, _ = step(S, heads(tq.cpu(), HV)[:, t], heads(tk.cpu(), HV)[:, t], tv.cpu().double()[:, t], a[:, t], SCALE)
        kv = tv.cpu().double()[:, t][..., :, None] * heads(tk.cpu(), HV)[:, t][..., None, :]
        Sm = a[:, t][..., None, None] * Sm + kv.abs()
        om = SCALE * (Sm * heads(tq.cpu(), HV)[:, t].abs()[..., None, :]).sum(-1)
        close(ov[:, t], ro, U_BF16 * ro.abs() + 2.0 ** -14 * om + 1e-30, "tree")
    ro, om, S, rm = step(S, heads(dq.cpu(), HV)[:, 0], heads(dk.cpu(), HV)[:, 0], dv.cpu().double()[:, 0],
                         decays(dg.cpu(), (1, 1), HV).exp()[:, 0], SCALE)
    ad = decays(dg.cpu(), (1, 1), HV).exp()[:, 0]
    Sm = ad[..., None, None] * Sm + (dv.cpu().double()[:, 0][..., :, None] * heads(dk.cpu(), HV)[:, 0][..., None, :]).abs()
    om = SCALE * (Sm * heads(dq.cpu(), HV)[:, 0].abs()[..., None, :]).sum(-1)
    close(od[:, 0], ro, U_BF16 * ro.abs() + 2.0 ** -16 * om + 1e-30, "token")
    # four nodes committed as in test_decay_gpu.py, (4 * 4 + 8) * 2 roundings, and the token's four
    close(pool[2:], S, (24 * 2 + 4) * U_F32 * Sm + 1e-30, "state")


FIRST = """
import sys, torch
sys.path[:0] = [{root!r}, {tests!r}]
from test_decay_gpu import pool_case, prefill_case, tree_parents
from rocm_flashinfer_contest_b200 import decay_decode, decay_prefill, decay_tree, state_cache
case = {case!r}
if case == "prefill":
    q, k, v, st, g, cu = prefill_case([900, 70, 0, 333], 1, 2, "token", 1)
    cu = torch.tensor(cu, device="cuda")
    run = lambda: decay_prefill.run(q, k, v, st, g, cu, None)
else:
    gen, pool, idx, q, k, v, g = pool_case(5, 1 if case == "decode" else 9, 2, 4, "token", 2, case.endswith("bf16"), 7)
    start, parents, acc = pool.clone(), tree_parents(gen, 5, v.shape[1], "mixed"), torch.full((5,), 3, dtype=torch.int32, device="cuda")
    codes, exps = state_cache.empty(7, pool.shape[1:])
    if case == "decode":
        run = lambda: (decay_decode.run_pool(q, k, v, pool, idx, g, None)[0], pool)
    elif case.startswith("verify"):
        run = lambda: (decay_tree.run(q, k, v, pool, idx, parents, g, None),)
    elif case == "commit":
        run = lambda: (decay_tree.commit(k, v, pool, idx, parents, acc, g),)
    else:
        run = lambda: (state_cache.store(pool, idx, codes, exps, idx)[0], state_cache.load(codes, exps, idx, pool, idx))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
if case != "prefill":
    pool.copy_(start)
graph.replay()
torch.cuda.synchronize()
got = [x.clone() for x in got]
if case != "prefill":
    pool.copy_(start)
want = run()
torch.cuda.synchronize()
pairs = list(zip(got, want))
if case == "cache":
    pairs = [(a[idx], b[idx]) for a, b in pairs]
assert all(torch.equal(a, b) for a, b in pairs)
from rocm_flashinfer_contest_b200._lib import lib
assert lib().gdn_device_status(0) == 0
print("same")
"""


@pytest.mark.parametrize("case", ["prefill", "decode", "verify", "verify_bf16", "commit", "cache"])
def test_first_call_of_a_process_inside_a_capture(case):
    here = os.path.dirname(os.path.abspath(__file__))
    code = FIRST.format(root=os.path.dirname(here), tests=here, case=case)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stdout + r.stderr

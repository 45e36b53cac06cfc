"""Runs one GDN workload a few times so a profiler can wrap it.

The B200 counterpart of the reference's tools/profile_kernel.py:30-94 (which
drives one solution's run() on one workload under rocprofv3): inputs are
built once, outside the profiled loop, then the kernel is launched
``--warmup`` + ``--iters`` times.  Use with ncu, e.g.

    ncu --set full --clock-control none -k regex:gdn_decode -s 2 -c 1 \\
        python -m rocm_flashinfer_contest_b200.profile_case decode --B 64
"""
from __future__ import annotations

import argparse

import torch

from . import decay_decode, decay_prefill, decay_tree, gdn_decode, gdn_mtp, gdn_prefill, inputs, state_cache


def _decay_case(a, dev):
    """The decay operators and the state cache on random inputs, gates of each token and v-head."""
    gen = torch.Generator(device=dev).manual_seed(0)

    def rnd(*shape, dtype=torch.bfloat16, s=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * s).to(dtype)

    def gates(*lead):
        return -torch.nn.functional.softplus(rnd(*lead, a.HV, dtype=torch.float32)) * 0.1

    if a.op == "decay-prefill":
        lens = torch.full((a.seqs,), a.T // a.seqs, dtype=torch.int64)
        lens[-1] += a.T - int(lens.sum())
        cu = torch.nn.functional.pad(lens.cumsum(0), (1, 0)).to(dev)
        q, k, v = rnd(a.T, a.H, 128), rnd(a.T, a.H, 128, s=0.1), rnd(a.T, a.HV, 128)
        state = None if a.no_state else rnd(a.seqs, a.HV, 128, 128, dtype=torch.float32)
        out, ns = torch.empty_like(v), torch.empty(a.seqs, a.HV, 128, 128, device=dev)
        g = gates(a.T)
        return lambda: decay_prefill.run_into(q, k, v, state, g, cu, None, out, ns)
    pool = rnd(a.B, a.HV, 128, 128, dtype=torch.bfloat16 if a.bf16_state else torch.float32)
    idx = torch.arange(a.B, dtype=torch.int32, device=dev)
    if a.op.startswith("cache"):
        codes, exps = state_cache.empty(a.B, (a.HV, 128, 128), device=dev)
        state_cache.store(pool, idx, codes, exps, idx)
        if a.op == "cache-store":
            return lambda: state_cache.store(pool, idx, codes, exps, idx)
        return lambda: state_cache.load(codes, exps, idx, pool, idx)
    T = 1 if a.op == "decay-decode" else a.steps
    q, k, v, g = rnd(a.B, T, a.H, 128), rnd(a.B, T, a.H, 128, s=0.1), rnd(a.B, T, a.HV, 128), gates(a.B, T)
    if a.op == "decay-decode":
        return lambda: decay_decode.run_pool(q, k, v, pool, idx, g)
    parents = torch.arange(-1, T - 1, dtype=torch.int32, device=dev).expand(a.B, T).contiguous()
    if a.op == "decay-verify":
        return lambda: decay_tree.run(q, k, v, pool, idx, parents, g)
    accepted = torch.full((a.B,), T // 4, dtype=torch.int32, device=dev)
    return lambda: decay_tree.commit(k, v, pool, idx, parents, accepted, g)


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("op", choices=["decode", "prefill", "mtp", "decay-decode", "decay-prefill", "decay-verify",
                                   "decay-commit", "cache-store", "cache-load"])
    ap.add_argument("--B", type=int, default=64)
    ap.add_argument("--T", type=int, default=8192)
    ap.add_argument("--seqs", type=int, default=1)
    ap.add_argument("--H", type=int, default=16)
    ap.add_argument("--HV", type=int, default=32)
    ap.add_argument("--warmup", type=int, default=2)
    ap.add_argument("--iters", type=int, default=1)
    ap.add_argument("--no-state", action="store_true")
    ap.add_argument("--steps", type=int, default=4, help="mtp: tokens per batch entry; decay-verify / decay-commit: nodes (a chain)")
    ap.add_argument("--no-snapshots", action="store_true", help="mtp: no intermediate states")
    ap.add_argument("--bf16-state", action="store_true", help="mtp (no snapshots), decay and cache ops: bf16 state pool")
    a = ap.parse_args(argv)
    dev = torch.device("cuda:0")
    if a.op == "decode":
        args = inputs.decode_inputs(a.B, a.H, a.HV, seed=0, device=dev, with_state=not a.no_state)
        out = torch.empty((a.B, 1, a.HV, 128), dtype=torch.bfloat16, device=dev)
        ns = args[3] if args[3] is not None else torch.empty((a.B, a.HV, 128, 128), device=dev)
        fn = lambda: gdn_decode.run_into(*args, output=out, new_state=ns)  # noqa: E731
    elif a.op == "mtp":
        args = inputs.mtp_inputs(a.B, a.steps, 2 * a.B, a.H, a.HV, seed=0, device=dev,
                                 intermediate=not (a.no_snapshots or a.bf16_state))
        if a.bf16_state:
            args[3] = args[3].to(torch.bfloat16)
        out = torch.empty((a.B, a.steps, a.HV, 128), dtype=torch.bfloat16, device=dev)
        fn = lambda: gdn_mtp.run_into(*args[:10], out, args[3],  # noqa: E731
                                      intermediate_states_buffer=args[10])
    elif a.op.startswith(("decay", "cache")):
        fn = _decay_case(a, dev)
    else:
        lens = [a.T // a.seqs] * a.seqs
        lens[-1] += a.T - sum(lens)
        args = inputs.prefill_inputs(lens, a.H, a.HV, seed=0, device=dev, with_state=not a.no_state)
        out = torch.empty((a.T, a.HV, 128), dtype=torch.bfloat16, device=dev)
        ns = torch.empty((a.seqs, a.HV, 128, 128), device=dev)
        fn = lambda: gdn_prefill.run_into(*args, output=out, new_state=ns)  # noqa: E731
    torch.cuda.synchronize()
    for _ in range(a.warmup + a.iters):
        fn()
    torch.cuda.synchronize()
    print(f"profile_case {a.op}: {a.warmup} + {a.iters} launches done")


if __name__ == "__main__":
    main()

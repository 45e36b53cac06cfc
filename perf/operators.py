"""Operators of linear attention with a per-head decay, as they are measured.

The recurrence, for v-head h (q/k head h // (HV / H)) and its k-last state
S [V, K] (V = K = 128):

    S_t = exp(g_t) S_{t-1} + v_t k_t^T          o_t = scale * S_t q_t

with a log decay g that is one number per v-head ([HV]) or one per token and
v-head.  Four operators are built on it:

* ``prefill``: packed prompts of any lengths (chunked form);
* ``decode``: one token per entry over a pool of states (recurrent form);
* ``verify`` / ``commit``: a tree of drafted tokens over the pooled states, and
  the accepted path's update of them;
* ``park`` / ``resume``: pool slots written to an 8-bit cache (int8 or e4m3
  codes, one power-of-two scale for 32 values) and read back.

``run`` computes them in plain torch where ``own`` is false and calls the
package where it is true; ``exact`` follows the definitions in 64 bits.
"""
import math
import random

import torch

own = False

D = 128       # head size: K == V
GROUP = 32    # values that share one scale of the 8-bit cache


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one long prompt, gates that depend on the token
        dict(name="prefill_long", op="prefill", n=1, T=8192, H=16, HV=32, per_token=True, state=False, cut=0),
        # a batch of ragged prompts continued from their states, fixed decays
        dict(name="prefill_ragged", op="prefill", n=13, T=16309, H=4, HV=8, per_token=False, state=True, cut=1),
        # a serving step of many short prompts
        dict(name="prefill_many_short", op="prefill", n=61, T=5003, H=16, HV=32, per_token=True, state=True, cut=2),
        # one short prompt, where latency counts
        dict(name="prefill_short", op="prefill", n=1, T=37, H=4, HV=8, per_token=False, state=False, cut=3),
        # single-token decode of one request
        dict(name="decode_one", op="decode", B=1, H=4, HV=8, pool=5, bf16=False, per_token=False),
        # a decode batch, fp32 states
        dict(name="decode_batch", op="decode", B=64, H=16, HV=32, pool=80, bf16=False, per_token=True),
        # a large decode batch, bf16 states, an odd number of entries
        dict(name="decode_large_bf16", op="decode", B=221, H=16, HV=32, pool=256, bf16=True, per_token=True),
        # a small drafted tree of few requests
        dict(name="verify_small", op="verify", B=3, T=7, H=4, HV=8, pool=8, bf16=False, per_token=True),
        # a wide drafted tree of a batch
        dict(name="verify_batch", op="verify", B=64, T=32, H=16, HV=32, pool=80, bf16=False, per_token=True),
        # the accepted paths of that batch folded into the states
        dict(name="commit_batch", op="commit", B=64, T=32, H=16, HV=32, pool=80, bf16=False, per_token=True),
        # the states of a batch of preempted requests parked in 8 bits and resumed
        dict(name="park_resume_int8", op="park", B=48, HV=32, pool=64, bf16=False, fmt="int8"),
        # a few prefix states read back from the 8-bit cache
        dict(name="resume_e4m3", op="resume", B=5, HV=8, pool=9, bf16=False, fmt="e4m3"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "decode", "verify", "commit", "park", "resume"])
    H, HV = rng.choice([(4, 8), (16, 32), (8, 8), (2, 16), (5, 15)])
    flags = dict(per_token=rng.random() < 0.6)
    if op == "prefill":
        T = _log_int(rng, 1, 8192 * 32 // max(HV, 32))
        return dict(op=op, n=min(_log_int(rng, 1, 48), 2 * T), T=T, H=H, HV=HV, state=rng.random() < 0.5,
                    cut=rng.randrange(1 << 20), **flags)
    bf16 = rng.random() < 0.4
    B = _log_int(rng, 1, min(160, (6000 if bf16 else 3000) // HV))
    if op in ("park", "verify", "commit"):
        B = min(B, 64)
    c = dict(op=op, B=B, HV=HV, pool=B + rng.randrange(1, 9), bf16=bf16)
    if op in ("park", "resume"):
        c["fmt"] = rng.choice(["int8", "e4m3"])
        return c
    c.update(H=H, **flags)
    if op in ("verify", "commit"):
        c["T"] = _log_int(rng, 1, 64)
    return c


def lengths(case):
    """The prompts' lengths: random cuts of T tokens (a length may be zero)."""
    r = random.Random(1000 + case["cut"])
    cuts = sorted(r.randint(0, case["T"]) for _ in range(case["n"] - 1))
    edges = [0] + cuts + [case["T"]]
    return [b - a for a, b in zip(edges, edges[1:])]


# ---------------------------------------------------------------- inputs

def _log_decay(gen, dev, shape, HV, per_token):
    """Fixed decays: 1 - 2^-x, x spread over 2 to 8 for the heads.  By token: minus
    a positive gate, from about a thousandth to a few units."""
    if not per_token:
        return torch.log1p(-torch.exp2(-torch.linspace(2, 8, HV, device=dev))).float()
    rate = torch.linspace(-5, 1, HV, device=dev).exp()
    x = torch.randn(*shape, HV, generator=gen, device=dev)
    return (-rate * torch.nn.functional.softplus(x)).float()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))

    def randn(*shape, dtype=torch.bfloat16, s=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * s).to(dtype)

    op, HV = case["op"], case["HV"]
    st = {"case": case, "op": op, "scale": 1.0 / math.sqrt(D)}
    if op == "prefill":
        T, H, n = case["T"], case["H"], case["n"]
        st["lens"] = lengths(case)
        edges = [0]
        for x in st["lens"]:
            edges.append(edges[-1] + x)
        st["cu"] = torch.tensor(edges, dtype=torch.int32, device=dev)
        st.update(q=randn(T, H, D), k=randn(T, H, D, s=0.2), v=randn(T, HV, D),
                  g=_log_decay(gen, dev, (T,), HV, case["per_token"]),
                  state=randn(n, HV, D, D, dtype=torch.float32, s=0.5) if case["state"] else None)
        return st
    B, P = case["B"], case["pool"]
    slots = torch.randperm(P, generator=gen, device=dev)[:B].to(torch.int32)
    live = torch.arange(B, device=dev)
    if B > 8:
        slots[B // 2] = -1      # a padded batch entry
        live = torch.cat([live[:B // 2], live[B // 2 + 1:]])
    st["slots"], st["live"] = slots, live
    st["pool"] = randn(P, HV, D, D, dtype=torch.bfloat16 if case["bf16"] else torch.float32, s=0.5)
    if op in ("park", "resume"):
        st["cache_slots"] = torch.randperm(P, generator=gen, device=dev)[:B].to(torch.int32)
        st["fmt"] = torch.int8 if case["fmt"] == "int8" else torch.float8_e4m3fn
        # the cache as a serving program allocates it: codes, and biased exponents of the scales
        st["codes"] = torch.zeros(P, HV, D, D, dtype=torch.int8, device=dev).view(st["fmt"])
        st["exps"] = torch.zeros(P, HV, D, D // GROUP, dtype=torch.uint8, device=dev)
        if op == "resume":
            c = torch.randint(-127, 128, (P, HV, D, D), generator=gen, device=dev)
            if case["fmt"] == "e4m3":   # every finite code: magnitudes below 0x7f
                c = torch.where(c < 0, -c + 127, c.clamp(max=126)).clamp(max=254)
                st["codes"] = c.to(torch.uint8).view(torch.float8_e4m3fn)
            else:
                st["codes"] = c.to(torch.int8)
            st["exps"] = torch.randint(110, 125, (P, HV, D, D // GROUP), generator=gen, device=dev).to(torch.uint8)
        return st
    T, H = case.get("T", 1), case["H"]
    st.update(q=randn(B, T, H, D), k=randn(B, T, H, D, s=0.2), v=randn(B, T, HV, D),
              g=_log_decay(gen, dev, (B, T), HV, case["per_token"]))
    if op in ("verify", "commit"):
        # node t hangs below one of the six nodes before it, or below the cached state (-1);
        # an entry's tokens past its own count are padding (-2)
        t = torch.arange(T, device=dev)
        back = (torch.rand(B, T, generator=gen, device=dev) * torch.clamp(t + 1, max=6)).long()
        count = torch.randint(max(1, T // 2), T + 1, (B, 1), generator=gen, device=dev)
        st["parents"] = torch.where(t < count, t - 1 - back, -2).to(torch.int32)
        st["accepted"] = (torch.rand(B, 1, generator=gen, device=dev) * (count + 1)).long().squeeze(1).sub(1).to(torch.int32)
    return st


# ---------------------------------------------------------------- plain forms

def _heads(x, HV):
    return x.float().repeat_interleave(HV // x.shape[-2], -2)


def _plain_prefill(s):
    """Chunks of 64 tokens: the products inside a chunk under the decayed causal mask, every
    chunk's own contribution to the state, and the states at the chunk starts as one
    triangular product over the chunks."""
    q, k, v, g, lens = s["q"], s["k"], s["v"], s["g"], s["lens"]
    T, HV = v.shape[:2]
    dev, N, C = q.device, len(lens), 64
    nc = max(1, -(-max(lens) // C))
    cu = s["cu"].long()
    tok = torch.arange(T, device=dev)
    n = torch.searchsorted(cu[1:], tok, right=True)
    at = n * nc * C + tok - cu[n]

    def pad(x):
        y = torch.zeros(N * nc * C, *x.shape[1:], dtype=x.dtype, device=dev)
        return y.index_copy(0, at, x).view(N, nc, C, *x.shape[1:])

    g = pad((g if g.dim() == 2 else g.expand(T, HV)).double()).permute(0, 3, 1, 2)
    q, k, v = (pad(x).permute(0, 3, 1, 2, 4) for x in (_heads(q, HV), _heads(k, HV), v.float()))
    cum = g.cumsum(-1)
    tot = cum[..., -1]
    live = torch.ones(C, C, dtype=torch.bool, device=dev).tril()
    dec = (cum[..., :, None] - cum[..., None, :]).masked_fill(~live, -math.inf).exp().float()
    out = ((q @ k.transpose(-1, -2)) * dec) @ v
    own_part = v.transpose(-1, -2) @ (k * (tot[..., None] - cum).exp().float()[..., None])
    upto = torch.nn.functional.pad(tot.cumsum(-1), (1, 0))                 # [N, HV, nc + 1]
    before = torch.arange(nc + 1, device=dev)[:, None] > torch.arange(nc, device=dev)
    w = (upto[..., :, None] - upto[..., None, 1:]).masked_fill(~before, -math.inf).exp().float()
    states = (w @ own_part.reshape(N, HV, nc, D * D)).view(N, HV, nc + 1, D, D)
    if s["state"] is not None:
        states = states + upto.exp().float()[..., None, None] * s["state"][:, :, None]
    out = out + cum.exp().float()[..., None] * (q @ states[:, :, :nc].transpose(-1, -2))
    out = (out * s["scale"]).to(torch.bfloat16).permute(0, 2, 3, 1, 4).reshape(N * nc * C, HV, D)[at]
    return out, states[:, :, nc].contiguous()


def _pool_rows(s):
    valid = s["slots"] >= 0
    return valid, s["slots"].long().clamp(min=0)


def _put(s, slots, new):
    """pool[slot] = new for the entries that are not padding."""
    s["pool"][slots[s["live"]]] = new[s["live"]].to(s["pool"].dtype)
    return s["pool"]


def _plain_decode(s):
    valid, slots = _pool_rows(s)
    HV = s["v"].shape[2]
    q, k, v = _heads(s["q"], HV)[:, 0], _heads(s["k"], HV)[:, 0], s["v"].float()[:, 0]
    g = s["g"][:, 0] if s["g"].dim() == 3 else s["g"].expand(v.shape[0], HV)
    new = g.exp()[..., None, None] * s["pool"][slots].float() + v[..., :, None] * k[..., None, :]
    out = s["scale"] * (new * q[..., None, :]).sum(-1)
    out = torch.where(valid[:, None, None], out, 0.0).to(torch.bfloat16)[:, None]
    return out, _put(s, slots, new)


def _tree(parents):
    """Which nodes lie on each node's path from the cached state (itself among them)."""
    B, T = parents.shape
    t = torch.arange(T, device=parents.device)
    inner = (parents >= 0) & (parents < t)
    step = ((parents[..., None] == t) & inner[..., None]).float()
    path = torch.eye(T, device=parents.device) + step
    hops = 1
    while hops < T:                                                        # paths of up to 2, 4, 8, ... hops
        step = step @ step
        path = path + path @ step
        hops *= 2
    path = path > 0
    reached = (path & (parents == -1)[:, None, :]).any(-1)                 # the path starts at the cached state
    return path & reached[..., None], reached


def _plain_verify(s):
    valid, slots = _pool_rows(s)
    HV = s["v"].shape[2]
    path, reached = _tree(s["parents"])
    q, k, v = (x.permute(0, 2, 1, 3) for x in (_heads(s["q"], HV), _heads(s["k"], HV), s["v"].float()))
    g = (s["g"] if s["g"].dim() == 3 else s["g"].expand(*s["parents"].shape, HV)).double().transpose(1, 2)
    cum = (path.double()[:, None] @ g[..., None])[..., 0]                  # [B, HV, T]
    dec = (cum[..., :, None] - cum[..., None, :]).masked_fill(~path[:, None], -math.inf).exp().float()
    out = ((q @ k.transpose(-1, -2)) * dec) @ v
    out = out + cum.exp().float()[..., None] * (q @ s["pool"][slots].float().transpose(-1, -2))
    live = (reached & valid[:, None])[:, None, :, None]
    return torch.where(live, out * s["scale"], 0.0).to(torch.bfloat16).transpose(1, 2).contiguous()


def _plain_commit(s):
    valid, slots = _pool_rows(s)
    HV, T = s["v"].shape[2], s["v"].shape[1]
    path, reached = _tree(s["parents"])
    last = s["accepted"].long()
    ok = valid & (last >= 0) & reached.gather(1, last.clamp(min=0)[:, None])[:, 0]
    on = path[torch.arange(last.numel(), device=last.device), last.clamp(min=0)]    # [B, T]
    k, v = (x.permute(0, 2, 1, 3) for x in (_heads(s["k"], HV), s["v"].float()))
    g = (s["g"] if s["g"].dim() == 3 else s["g"].expand(*on.shape, HV)).double().transpose(1, 2)
    g = g.masked_fill(~on[:, None], 0.0)
    after = g.flip(-1).cumsum(-1).flip(-1) - g                             # decays behind each node
    w = after.masked_fill(~on[:, None], -math.inf).exp().float()
    old = s["pool"][slots].float()
    new = v.transpose(-1, -2) @ (k * w[..., None]) + g.sum(-1).exp().float()[..., None, None] * old
    return _put(s, slots, torch.where(ok[:, None, None, None], new, old))


def _plain_store(s):
    """The smallest power of two 2^e with max |x| <= top * 2^e, and x / 2^e rounded to the code's type."""
    _, slots = _pool_rows(s)
    x = s["pool"][slots].float()
    x = x.view(*x.shape[:-1], D // GROUP, GROUP)
    top = x.abs().amax(-1, keepdim=True)
    m, p = torch.frexp(top)
    lim, bits = (127 / 128, 7) if s["fmt"] == torch.int8 else (448 / 512, 9)
    e = torch.where(top > 0, p - bits + (m > lim), -127).clamp(min=-127)
    y = torch.ldexp(x, -e)
    y = (y.round() if s["fmt"] == torch.int8 else y).to(s["fmt"])
    where, live = s["cache_slots"].long()[s["live"]], s["live"]
    s["codes"].view(torch.uint8)[where] = y.flatten(-2).view(torch.uint8)[live]
    s["exps"][where] = (e + 127).squeeze(-1).to(torch.uint8)[live]


def _plain_load(s):
    _, slots = _pool_rows(s)
    cs = s["cache_slots"].long()
    y = s["codes"].view(torch.uint8)[cs].view(s["fmt"]).float()
    e = s["exps"][cs].to(torch.int32) - 127
    x = torch.ldexp(y.view(*y.shape[:-1], D // GROUP, GROUP), e[..., None]).flatten(-2)
    return _put(s, slots, x)


# ---------------------------------------------------------------- one pass

def run(s):
    op = s["op"]
    if own:
        from rocm_flashinfer_contest_b200 import decay_decode, decay_prefill, decay_tree, state_cache
        if op == "prefill":
            return decay_prefill.run(s["q"], s["k"], s["v"], s["state"], s["g"], s["cu"], s["scale"])
        if op == "decode":
            return decay_decode.run_pool(s["q"], s["k"], s["v"], s["pool"], s["slots"], s["g"], s["scale"])
        if op == "verify":
            return decay_tree.run(s["q"], s["k"], s["v"], s["pool"], s["slots"], s["parents"], s["g"], s["scale"])
        if op == "commit":
            return decay_tree.commit(s["k"], s["v"], s["pool"], s["slots"], s["parents"], s["accepted"], s["g"])
        if op == "park":
            state_cache.store(s["pool"], s["slots"], s["codes"], s["exps"], s["cache_slots"])
        return state_cache.load(s["codes"], s["exps"], s["cache_slots"], s["pool"], s["slots"])
    if op == "prefill":
        return _plain_prefill(s)
    if op == "decode":
        return _plain_decode(s)
    if op == "verify":
        return _plain_verify(s)
    if op == "commit":
        return _plain_commit(s)
    if op == "park":
        _plain_store(s)
    return _plain_load(s)


# ---------------------------------------------------------------- bytes and operations

def work(case):
    """Every input element once, every output element once; the recurrence's 4 V K operations for each
    token and v-head (two multiply-adds a state element), none for the conversions."""
    HV, op = case["HV"], case["op"]
    head = D * D
    if op == "prefill":
        T, H, n = case["T"], case["H"], case["n"]
        b = T * (2 * H * D * 2 + 2 * HV * D * 2) + (T if case["per_token"] else 1) * HV * 4
        return {"bytes": b + n * HV * head * 4 * (2 if case["state"] else 1), "flops": 4 * T * HV * head}
    B, el = case["B"], 2 if case["bf16"] else 4
    live = B - (1 if B > 8 else 0)
    states = live * HV * head
    eight = states * (1 + 1 / GROUP)
    if op == "park":
        return {"bytes": 2 * (states * el + eight), "flops": 2 * states}
    if op == "resume":
        return {"bytes": states * el + eight, "flops": states}
    T, H = case.get("T", 1), case["H"]
    gates = (B * T if case["per_token"] else 1) * HV * 4
    if op == "decode":
        return {"bytes": 2 * states * el + live * (2 * H + 2 * HV) * D * 2 + gates, "flops": 4 * states}
    if op == "verify":
        return {"bytes": states * el + live * T * (2 * H + 2 * HV) * D * 2 + gates, "flops": 2 * T * states}
    # commit: only the accepted paths are needed; a quarter of the nodes stands for them
    return {"bytes": 2 * states * el + live * max(1, T // 4) * (H + HV) * D * 2 + gates // 4, "flops": 2 * states * max(1, T // 4)}


# ---------------------------------------------------------------- 64 bits

def _each(x, HV):
    idx = torch.arange(HV, device=x.device) // (HV // x.shape[-2])
    return x.double().index_select(-2, idx)


def exact(case, seed):
    s = prepare(case, seed)
    op, HV = s["op"], case["HV"]
    if op == "prefill":
        # the recurrence, token by token, over all prompts that still have one
        lens = torch.tensor(s["lens"], device="cuda")
        cu = s["cu"].long()
        S = torch.zeros(len(s["lens"]), HV, D, D, dtype=torch.float64, device="cuda")
        if s["state"] is not None:
            S += s["state"]
        q, k, v = _each(s["q"], HV), _each(s["k"], HV), s["v"].double()
        out = torch.zeros_like(v)
        fixed = s["g"].dim() == 1
        order = sorted(range(len(s["lens"])), key=lambda i: -s["lens"][i])
        by_len = torch.tensor(order, device="cuda")
        R = S[by_len]
        for t in range(max(s["lens"])):
            m = sum(1 for x in s["lens"] if x > t)
            rows = cu[by_len[:m]] + t
            a = (s["g"].double().expand(m, HV) if fixed else s["g"][rows].double()).exp()
            R[:m] = R[:m] * a[..., None, None] + v[rows][..., :, None] * k[rows][..., None, :]
            out[rows] = torch.matmul(R[:m], q[rows][..., None])[..., 0] * s["scale"]
        S[by_len] = R
        del lens
        return out, S
    pool = s["pool"].double()
    slots = s["slots"].tolist()
    if op in ("park", "resume"):
        cs = s["cache_slots"].tolist()
        for i, (a, c) in enumerate(zip(slots, cs)):
            if a < 0:
                continue
            if op == "park":
                x = pool[a].view(HV, D, D // GROUP, GROUP)
                top = x.abs().amax(-1, keepdim=True)
                lim = 127.0 if case["fmt"] == "int8" else 448.0
                e = torch.floor(torch.log2(top.clamp(min=2.0 ** -140))) - 12
                for _ in range(16):                       # raise 2^e until the largest value fits
                    e = torch.where(top > lim * torch.exp2(e), e + 1, e)
                e = e.clamp(min=-127)
                y = x / torch.exp2(e)
                if case["fmt"] == "int8":
                    y = torch.round(y)
                else:                                     # three fraction bits, exponents from -6
                    unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                    y = torch.round(y / unit) * unit
                pool[a] = (y * torch.exp2(e)).view(HV, D, D)
            else:
                y = s["codes"][c].double()
                e = s["exps"][c].double() - 127
                pool[a] = (y.view(HV, D, D // GROUP, GROUP) * torch.exp2(e)[..., None]).view(HV, D, D)
        return pool
    B, T = case["B"], case.get("T", 1)
    live = [i for i in range(B) if slots[i] >= 0]
    q, k, v = _each(s["q"], HV), _each(s["k"], HV), s["v"].double()
    a = (s["g"].double() if s["g"].dim() == 3 else s["g"].double().expand(B, T, HV)).exp()
    out = torch.zeros(B, T, HV, D, dtype=torch.float64, device="cuda")
    if op == "decode":
        for i in live:
            S = pool[slots[i]] * a[i, 0][:, None, None] + v[i, 0][:, :, None] * k[i, 0][:, None, :]
            out[i, 0] = torch.matmul(S, q[i, 0][:, :, None])[..., 0] * s["scale"]
            pool[slots[i]] = S
        return out, pool
    parents, accepted = s["parents"].tolist(), s["accepted"].tolist()
    for i in live:
        S0, nodes = pool[slots[i]].clone(), {}
        path = []
        if op == "commit":                                 # only the accepted path's nodes matter
            t = accepted[i]
            while t >= 0 and parents[i][t] != -2:
                path.append(t)
                t = parents[i][t]
        for t in range(T) if op == "verify" else reversed(path):
            par = parents[i][t]
            if par != -1 and par not in nodes:
                continue
            S = S0 if par == -1 else nodes[par]
            nodes[t] = S * a[i, t][:, None, None] + v[i, t][:, :, None] * k[i, t][:, None, :]
            out[i, t] = torch.matmul(nodes[t], q[i, t][:, :, None])[..., 0] * s["scale"]
        if op == "commit" and path:
            pool[slots[i]] = nodes[path[0]]
    return out if op == "verify" else pool

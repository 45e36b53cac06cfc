"""64-bit references of the decay operators, and how far an exact kernel's
roundings can be from them.

Each reference also returns the sum of the magnitudes that its result is made
of, so that a tolerance counts roundings: u = 2^-8 for one to bf16 (half its
step), 2^-24 for one to fp32.
"""
from __future__ import annotations

import torch

U_BF16 = 2.0 ** -8
U_F32 = 2.0 ** -24
CHUNK = 64


def heads(x, HV):
    """[..., H, K] -> [..., HV, K] in 64 bits: v-head h reads q/k head h // (HV / H)."""
    return x.double().repeat_interleave(HV // x.shape[-2], -2)


def decays(g, lead, HV):
    """exp(log_decay) per token and v-head in 64 bits; below -104 it counts as -104."""
    g = g.double().clamp(min=-104.0)
    return g.expand(*lead, HV) if g.dim() == 1 else g


def prefill(q, k, v, state, g, cu, scale):
    """(output, its magnitudes, new_state, its magnitudes), chunk by chunk: the
    magnitudes of an output are those of the two products a chunk form rounds an
    operand of, scale * (e^c |S| |q| + |P| |v|)."""
    q, k, v, g = (x.cpu() for x in (q, k, v, g))
    T, HV = v.shape[:2]
    qh, kh, vh, gg = heads(q, HV), heads(k, HV), v.double(), decays(g, (T,), HV)
    N = len(cu) - 1
    out, mag = torch.zeros(T, HV, 128, dtype=torch.float64), torch.zeros(T, HV, 128, dtype=torch.float64)
    S = torch.zeros(N, HV, 128, 128, dtype=torch.float64) if state is None else state.cpu().double()
    Sm = S.abs()
    for n in range(N):
        for a in range(cu[n], cu[n + 1], CHUNK):
            b = min(a + CHUNK, cu[n + 1])
            qq, kk, vv = (x[a:b].transpose(0, 1) for x in (qh, kh, vh))      # [HV, L, 128]
            c = gg[a:b].cumsum(0).T                                          # [HV, L]
            live = torch.ones(b - a, b - a, dtype=torch.bool).tril()
            D = (c[:, :, None] - c[:, None, :]).masked_fill(~live, -torch.inf).exp()
            P = (qq @ kk.transpose(1, 2)) * D
            e = c.exp()[:, :, None]
            out[a:b] = (scale * (e * (qq @ S[n].transpose(1, 2)) + P @ vv)).transpose(0, 1)
            mag[a:b] = (abs(scale) * (e * (qq.abs() @ S[n].abs().transpose(1, 2)) + P.abs() @ vv.abs())).transpose(0, 1)
            w = (c[:, -1:] - c).exp()[:, :, None]
            tot = c[:, -1].exp()[:, None, None]
            S[n] = tot * S[n] + vv.transpose(1, 2) @ (kk * w)
            Sm[n] = tot * Sm[n] + vv.abs().transpose(1, 2) @ (kk.abs() * w)
    return out, mag, S, Sm


def step(S, q, k, v, a, scale):
    """One token over states [B, HV, 128, 128]: (o, its magnitudes, new states, theirs)."""
    kv = v[..., :, None] * k[..., None, :]
    new = a[..., None, None] * S + kv
    o = scale * (new * q[..., None, :]).sum(-1)
    om = abs(scale) * (new.abs() * q[..., None, :].abs()).sum(-1)
    return o, om, new, a[..., None, None] * S.abs() + kv.abs()


def paths(parents):
    """For each node of one tree the nodes from the cached state down to it, or None
    for padding."""
    res = []
    for t, p in enumerate(parents):
        up = [] if p == -1 else res[p] if 0 <= p < t else None
        res.append(None if up is None else up + [t])
    return res


def close(got, want, tol, what):
    got, want, tol = got.detach().cpu().double(), want.cpu().double(), tol.cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    err = (got - want).abs()
    bad = err > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol.clamp(min=1e-300)).max()):.3g} times the tolerance"

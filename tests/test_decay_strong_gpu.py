"""Trees and prompts behind gates that forget (each counts as -104): a path's sum of
log decays is in the thousands there, and the decay between two of its nodes, a
difference of two such sums, still has to be that of the gates between them.

Tolerances as in test_decay_gpu.py (u = 2^-8 to bf16, 2^-24 to fp32).  A tree's
weights e^{c_t - c_j} come from sums in two parts, the first exact and the second
below 2^-5: their difference d is off by a rounding or two of itself, |d| 2^-23 at
most, and a weight that fp32 holds has |d| <= 104, so 2^-16.3 relative; S and P in two bf16 terms,
2^-16; 32 fp32 roundings of the magnitudes.
"""
import pytest
import torch

from decay_reference import U_BF16, U_F32, close
from test_decay_gpu import SCALE, _status, check_prefill, gates, pool_case, prefill_case, tree_parents, verify_reference  # noqa: F401

pytestmark = pytest.mark.gpu

SLACK = 2.0 ** -16 + 2.0 ** -16 + 32 * U_F32


@pytest.mark.parametrize("T,tree", [(64, "chain"), (64, "mixed"), (33, "chain"), (16, "chain")])
@pytest.mark.parametrize("bf16", [False, True])
def test_tree_behind_strong_gates(T, tree, bf16):
    from rocm_flashinfer_contest_b200 import decay_tree
    gen, pool, idx, q, k, v, g = pool_case(2, T, 1, 2, "strong", T, bf16, 3)
    parents = tree_parents(gen, 2, T, tree)
    g[0, : T - 5] = float("-inf")                       # the last five nodes' own gates stay
    g[0, T - 5:] = gates(gen, (5,), 2, "token")
    ro, rm = verify_reference(pool, idx, parents, q, k, v, g, SCALE)
    o = decay_tree.run(q, k, v, pool, idx, parents, g, SCALE)
    close(o, ro, U_BF16 * ro.abs() + SLACK * rm + 1e-30, "output")


@pytest.mark.parametrize("T", [64, 40])
@pytest.mark.parametrize("gate", [-2.0 ** -12, -2.0 ** -9, -0.1])
def test_difference_of_two_nodes_behind_strong_gates(T, gate):
    """The last two nodes of a chain have one key and opposite values: the output is what the gate between them takes."""
    from rocm_flashinfer_contest_b200 import decay_tree
    gen, pool, idx, q, k, v, _ = pool_case(1, T, 1, 2, "token", T, False, 2)
    parents = torch.arange(-1, T - 1, device="cuda", dtype=torch.int32)[None].contiguous()
    g = torch.full((1, T, 2), float("-inf"), device="cuda")
    g[0, T - 1] = gate
    g[0, T - 3] = -103.37
    k[0, T - 1] = k[0, T - 2]
    v[0, T - 1] = -v[0, T - 2]
    ro, rm = verify_reference(pool, idx, parents, q, k, v, g, SCALE)
    o = decay_tree.run(q, k, v, pool, idx, parents, g, SCALE)
    close(o, ro, U_BF16 * ro.abs() + SLACK * rm + 1e-30, "output")


@pytest.mark.parametrize("lens", [[64], [130], [900]])
def test_prompt_behind_strong_gates(lens):
    from rocm_flashinfer_contest_b200 import decay_prefill
    q, k, v, st, g, cu = case = prefill_case(lens, 1, 2, "token", seed=lens[0])
    for a in range(0, lens[0], 64):
        g[a:a + 58] = float("-inf")
    g[::7, 1] = -77.7
    o, s = decay_prefill.run(q, k, v, st, g, torch.tensor(cu, device="cuda"), SCALE)
    check_prefill(o, s, case)


def test_prompt_weights_behind_strong_gates():
    """The decay between tokens 61 and 62 of 64, behind gates of -60 to -104, over 1,024 heads: a weight's rounding
    to bf16 is at most u either way and differs from head to head, so its mean over the heads has a deviation of u / 3^0.5
    / 32 at most; five of them.  (The output's own rounding differs from element to element, 128 for a head.)"""
    from rocm_flashinfer_contest_b200 import decay_prefill
    N, HV = 8, 1024
    gen = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(torch.bfloat16)  # noqa: E731
    q, k, v = rnd(N, 64, HV, 128), rnd(N, 64, HV, 128), torch.zeros(N, 64, HV, 128, dtype=torch.bfloat16, device="cuda")
    v[:, 61] = 1 + torch.rand(N, HV, 128, generator=gen, device="cuda").to(torch.bfloat16)
    g = (-104 + 44 * torch.rand(N, 64, 1, generator=gen, device="cuda")).expand(N, 64, HV).contiguous()
    g[:, 62] = -0.1
    o, _ = decay_prefill.run(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), None, g.flatten(0, 1),
                             torch.arange(0, 64 * N + 1, 64, device="cuda"), SCALE)
    P = SCALE * (q[:, 62].double() * k[:, 61].double()).sum(-1) * g[:, 62].double().exp()
    ratio = o.view(N, 64, HV, 128)[:, 62].double() / (P[..., None] * v[:, 61].double())
    off = (ratio.mean(-1) - 1).mean(-1).abs()
    assert (off < 5 * U_BF16 / 3 ** 0.5 / 32).all(), off.tolist()

"""The decay operators' persistent CTAs on their second and later items, against the
64-bit references: more work than CTAs, padding between live entries, sequences
beyond the first 32, states that start from the workspace next to others.

Tolerances as in test_decay_gpu.py and test_decay_strong_gpu.py.
"""
import pytest
import torch

from decay_reference import U_BF16, close
from test_decay_gpu import SCALE, _status, check_prefill, pool_case, prefill_case, tree_parents, verify_reference  # noqa: F401
from test_decay_strong_gpu import SLACK

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,H,HV,bf16,kind", [
    (40, 9, 8, 16, False, "token"), (40, 9, 8, 16, True, "token"),     # 640 items: 296 CTAs, up to three each
    (40, 32, 8, 16, True, "token"), (56, 3, 4, 16, False, "head"),
    (24, 48, 4, 16, False, "token"),                                   # 384 items on 148 CTAs, one an SM
    (24, 64, 4, 16, True, "strong"),
    (11, 17, 5, 60, False, "token"),
])
def test_verify_takes_turns(B, T, H, HV, bf16, kind):
    from rocm_flashinfer_contest_b200 import decay_tree
    gen, pool, idx, q, k, v, g = pool_case(B, T, H, HV, kind, B + T, bf16, B + 2)
    parents = tree_parents(gen, B, T, "mixed")
    parents[:, 0] = -1                                    # (so that most trees have nodes in use)
    # a CTA's items are 148 or 296 apart, so B / 3 or so entries: live after padding, padding after live, and two
    # paddings in a row on some CTA, whichever it is
    per = 296 / HV
    dead = {1, int(per) + 2, int(per) + 3, int(2 * per) + 3, int(per / 2), int(per / 2) + 1, int(per * 1.5), B - 1}
    dead = sorted(b for b in dead if b < B)
    idx[dead] = -1
    o = decay_tree.run(q, k, v, pool, idx, parents, g, SCALE)
    assert (o[dead] == 0).all()
    ro, rm = verify_reference(pool, idx, parents, q, k, v, g, SCALE)
    close(o, ro, U_BF16 * ro.abs() + SLACK * rm + 1e-30, "output")
    few = torch.full((B, T, HV, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    only = torch.full_like(idx, -1)
    only[[0, B - 2]] = idx[[0, B - 2]]                    # all padding but the first turn's and the last turn's entry
    decay_tree.run(q, k, v, pool, only, parents, g, SCALE, output=few)
    live = [b for b in (0, B - 2) if b not in dead]
    rest = [b for b in range(B) if b not in (0, B - 2)]
    assert torch.equal(few[live], o[live]) and (few[rest] == 0).all()


@pytest.mark.parametrize("lens,H,HV,kind", [
    ([7 * i % 83 for i in range(90)], 4, 8, "token"),                            # 720 items: one look after the other
    ([13 * i % 131 for i in range(140)], 2, 4, "strong"),
    ([11 * i % 90 + 1 for i in range(40)] + [1500, 3, 1800, 60, 1025] + [5 * i % 70 for i in range(25)], 4, 8, "token"),
    ([0] * 45 + [700, 1, 0, 900] + [64] * 30 + [640], 16, 16, "head"),           # the first pass of two segments each
    ([90] * 33 + [2000] + [90] * 33 + [777], 1, 5, "token"),
])
@pytest.mark.parametrize("state", [True, False])
def test_prefill_takes_turns(lens, H, HV, kind, state):
    from rocm_flashinfer_contest_b200 import decay_prefill
    q, k, v, st, g, cu = case = prefill_case(lens, H, HV, kind, seed=len(lens) + HV, state=state)
    o, s = decay_prefill.run(q, k, v, st, g, torch.tensor(cu, device="cuda"), SCALE)
    check_prefill(o, s, case)


@pytest.mark.parametrize("lens,H,HV,kind", [
    ([120_001, 1, 30_000], 1, 2, "token"),          # a hundred segments, one joined to the other
    ([65_537], 1, 1, "strong"),
    ([i % 4 for i in range(2500)], 1, 1, "head"),   # more sequences than CTAs, by far
])
def test_prefill_of_long_and_of_many(lens, H, HV, kind):
    from rocm_flashinfer_contest_b200 import decay_prefill
    q, k, v, st, g, cu = case = prefill_case(lens, H, HV, kind, seed=len(lens), state=True)
    o, s = decay_prefill.run(q, k, v, st, g, torch.tensor(cu, device="cuda"), SCALE)
    check_prefill(o, s, case)


@pytest.mark.parametrize("B,T,HV,bf16", [(900, 2, 1, False), (700, 1, 2, True), (350, 35, 1, False)])
def test_verify_takes_many_turns(B, T, HV, bf16):
    from rocm_flashinfer_contest_b200 import decay_tree
    gen, pool, idx, q, k, v, g = pool_case(B, T, 1, HV, "token", B, bf16, B)
    parents = tree_parents(gen, B, T, "mixed")
    idx[torch.rand(B, generator=gen, device="cuda") < 0.4] = -1
    ro, rm = verify_reference(pool, idx, parents, q, k, v, g, SCALE)
    o = decay_tree.run(q, k, v, pool, idx, parents, g, SCALE)
    close(o, ro, U_BF16 * ro.abs() + SLACK * rm + 1e-30, "output")

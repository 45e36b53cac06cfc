"""Values that are not finite spoil what the formulas let them reach, as infinity or
NaN, and nothing else (a value of v also its whole chunk or tree, as documented):
everything beside is bit for bit what it is without them."""
import pytest
import torch

from test_decay_gpu import SCALE, _status, pool_case, prefill_case  # noqa: F401

pytestmark = pytest.mark.gpu
BAD = [float("inf"), float("-inf"), float("nan")]


def check(got, clean, spoiled, what, also=None):
    """Not finite where `spoiled`, as `clean` elsewhere (`also`: places that may be either)."""
    assert not torch.isfinite(got[spoiled]).any(), what
    rest = ~spoiled if also is None else ~(spoiled | also)
    assert torch.equal(got[rest], clean[rest]), what


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("where", ["q", "k", "v", "state"])
def test_prefill(bad, where):
    from rocm_flashinfer_contest_b200 import decay_prefill
    q, k, v, st, g, cu = prefill_case([100, 300, 70], 2, 4, "token", 17)     # (the second in two segments)
    cu_t = torch.tensor(cu, device="cuda")
    run = lambda: decay_prefill.run(q, k, v, st, g, cu_t, SCALE)  # noqa: E731
    o, s = run()
    so, ss, also = torch.zeros_like(o, dtype=torch.bool), torch.zeros_like(s, dtype=torch.bool), None
    t, end = 100 + 70, 400                 # token 70 of the second: in its second chunk
    if where == "q":
        q[t, 1, 5] = bad
        so[t, 2:] = True                   # v-heads 2 and 3 read q/k head 1
    elif where == "k":
        k[t, 1, 5] = bad
        so[t:end, 2:] = True
        ss[1, 2:, :, 5] = True
    elif where == "v":
        v[t, 3, 9] = bad
        so[t:end, 3, 9] = True
        ss[1, 3, 9] = True
        also = torch.zeros_like(so)
        also[164:t, 3, 9] = True           # earlier tokens of its chunk
    else:
        st[1, 3, 9, 5] = bad
        so[100:end, 3, 9] = True
        ss[1, 3, 9, 5] = True
    got_o, got_s = run()
    check(got_o, o, so, "output", also)
    check(got_s, s, ss, "new_state")


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("token", [0, 1, 64, 70, 71, 127, 299])
def test_prefill_gates(bad, token):
    """A gate that is not finite (nor -inf, which forgets) reaches its token and what follows, not the token before."""
    from rocm_flashinfer_contest_b200 import decay_prefill
    q, k, v, st, g, cu = prefill_case([100, 300, 70], 2, 4, "token", 17)
    cu_t = torch.tensor(cu, device="cuda")
    o, s = decay_prefill.run(q, k, v, st, g, cu_t, SCALE)
    g[100 + token, 2] = bad
    so, ss = torch.zeros_like(o, dtype=torch.bool), torch.zeros_like(s, dtype=torch.bool)
    so[100 + token:400, 2] = True
    ss[1, 2] = True
    got_o, got_s = decay_prefill.run(q, k, v, st, g, cu_t, SCALE)
    check(got_o, o, so, "output")
    check(got_s, s, ss, "new_state")


@pytest.mark.parametrize("node", [0, 2, 12, 19])
def test_tree_gates(node):
    from rocm_flashinfer_contest_b200 import decay_tree
    gen, pool, idx, q, k, v, g = pool_case(2, 20, 2, 4, "token", 19, False, 3)
    parents = torch.tensor([[-1, *range(9), 2, *range(10, 19)]] * 2, dtype=torch.int32, device="cuda")
    o = decay_tree.run(q, k, v, pool, idx, parents, g, SCALE)
    g[0, node, 2] = float("nan")
    so = torch.zeros_like(o, dtype=torch.bool)
    so[0, node:, 2] = True
    if node == 0:
        so[0, :, 2] = True
    check(decay_tree.run(q, k, v, pool, idx, parents, g, SCALE), o, so, "output")


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("where", ["q", "k", "v", "pool"])
def test_tree(bad, bf16, where):
    from rocm_flashinfer_contest_b200 import decay_tree
    gen, pool, idx, q, k, v, g = pool_case(2, 20, 2, 4, "token", 19, bf16, 3)
    # nodes 0..9 a chain, 10..19 another one that hangs below node 2
    parents = torch.tensor([[-1, *range(9), 2, *range(10, 19)]] * 2, dtype=torch.int32, device="cuda")
    accepted = torch.tensor([19, 9], dtype=torch.int32, device="cuda")
    before = pool.clone()

    def run():
        pool.copy_(start)
        o = decay_tree.run(q, k, v, pool, idx, parents, g, SCALE)
        return o, decay_tree.commit(k, v, pool, idx, parents, accepted, g).clone()

    start = before
    o, p = run()
    so, sp, also = torch.zeros_like(o, dtype=torch.bool), torch.zeros_like(p, dtype=torch.bool), None
    slot = int(idx[0])
    if where == "q":
        q[0, 12, 1, 5] = bad
        so[0, 12, 2:] = True
    elif where == "k":
        k[0, 12, 1, 5] = bad
        so[0, 12:, 2:] = True              # the nodes below it
        sp[slot, 2:, :, 5] = True
    elif where == "v":
        v[0, 12, 3, 9] = bad
        so[0, 12:, 3, 9] = True
        sp[slot, 3, 9] = True
        also = torch.zeros_like(so)
        also[0, :, 3, 9] = True
    else:
        start = before.clone()
        start[slot, 3, 9, 5] = bad
        so[0, :, 3, 9] = True
        sp[slot, 3, 9, 5] = True
    got_o, got_p = run()
    check(got_o, o, so, "output", also)
    check(got_p, p, sp, "state")


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("bf16", [False, True])
def test_decode_gives_what_the_formula_gives(bad, bf16):
    from rocm_flashinfer_contest_b200 import decay_decode
    _, pool, idx, q, k, v, g = pool_case(3, 1, 2, 4, "token", 23, bf16, 5)
    clean = pool.clone()
    o, _ = decay_decode.run_pool(q, k, v, clean, idx, g, SCALE)
    slot = int(idx[1])
    pool[slot, 3, 9, 5] = bad
    got, _ = decay_decode.run_pool(q, k, v, pool, idx, g, SCALE)
    so, sp = torch.zeros_like(o, dtype=torch.bool), torch.zeros_like(pool, dtype=torch.bool)
    so[1, 0, 3, 9], sp[slot, 3, 9, 5] = True, True
    check(got, o, so, "output")
    check(pool, clean, sp, "state")
    if bad == bad:
        assert float(pool[slot, 3, 9, 5]) == bad
        assert float(got[1, 0, 3, 9]) == bad * (1 if float(q[1, 0, 1, 5]) > 0 else -1)

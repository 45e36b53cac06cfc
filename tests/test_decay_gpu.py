"""Decay operators on the GPU against 64-bit references: prefill, pooled decode,
drafted trees and their commit, one after the other as a server runs them.

Tolerances, from the roundings (u = 2^-8 to bf16, 2^-24 to fp32; magnitudes as
the references give them):

* prefill output: its own rounding u |o|, S and P rounded to bf16 once each,
  u * magnitudes; everything else is fp32 (32 roundings of partial sums).
* prefill state: a chunk's sum runs over 12 accumulating products of 16 terms and
  a few fp32 factors, 32 roundings; every later chunk adds one.  2 * 2^-24 each,
  as the tensor core may truncate.
* decode: one rounding of the output, 32 fp32 roundings; states 4 roundings
  (exp's two among them).
* tree: states and scores in two bf16 terms, 2^-16 of the magnitudes together,
  and 32 fp32 roundings; the log decays of a path are summed in fp32, up to 64 of
  up to 104: 2^-24 * 64 * 104 / 2 = 2e-4 where decays are that strong, else below
  2^-16 with the decays used here.
"""
import pytest
import torch

from decay_reference import U_BF16, U_F32, close, decays, heads, paths, prefill, step

pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5


@pytest.fixture(autouse=True)
def _status():
    yield
    from rocm_flashinfer_contest_b200._lib import lib
    assert lib().gdn_device_status(0) == 0


def rnd(gen, *shape, s=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=gen, device="cuda") * s).to(dtype)


def gates(gen, lead, HV, kind):
    if kind == "head":
        return torch.log1p(-torch.exp2(-torch.linspace(1, 9, HV, device="cuda")))
    g = -torch.nn.functional.softplus(torch.randn(*lead, HV, generator=gen, device="cuda")) * 0.2
    if kind == "strong":      # from nearly none to hundreds, and some that forget all
        g = g * torch.exp(3 * torch.randn(*lead, HV, generator=gen, device="cuda"))
        g = torch.where(torch.rand(g.shape, generator=gen, device="cuda") < 0.05, float("-inf"), g)
    if kind == "none":
        g = torch.zeros_like(g)
    return g.float()


def prefill_case(lens, H, HV, kind, seed, lead=0, behind=0, state=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T = lead + sum(lens) + behind
    cu = [lead]
    for n in lens:
        cu.append(cu[-1] + n)
    q, k, v = rnd(gen, T, H, 128), rnd(gen, T, H, 128, s=0.2), rnd(gen, T, HV, 128)
    st = rnd(gen, len(lens), HV, 128, 128, s=0.5, dtype=torch.float32) if state else None
    return q, k, v, st, gates(gen, (T,), HV, kind), cu


def check_prefill(o, s, case, scale=SCALE):
    q, k, v, st, g, cu = case
    ro, rm, rs, rsm = prefill(q, k, v, st, g, cu, scale)
    close(o, ro, U_BF16 * ro.abs() + (U_BF16 + 32 * U_F32) * 1.01 * rm + 1e-30, "output")
    chunks = max([0] + [-(-(b - a) // 64) for a, b in zip(cu, cu[1:])])
    close(s, rs, (32 + chunks) * 2 * U_F32 * rsm + 1e-30, "new_state")


@pytest.mark.parametrize("lens,H,HV,kind", [
    ([1], 1, 1, "token"),
    ([2, 1], 2, 4, "head"),
    ([63], 1, 2, "token"),
    ([64], 3, 3, "strong"),
    ([65], 2, 2, "none"),
    ([0, 5, 0], 1, 3, "token"),
    ([128, 0, 1, 130], 4, 8, "token"),
    ([255, 257], 2, 4, "head"),
    ([256, 3], 1, 1, "strong"),
    ([900], 1, 2, "token"),               # several segments, with what lies between them carried
    ([257, 1700, 0, 63], 1, 2, "head"),   # sequences of two and of seven segments, and of one
    ([1290], 2, 2, "strong"),
    ([3] * 40 + [0] * 3 + [70] * 30, 1, 2, "token"),  # more sequences than one look at them takes
    ([150, 149], 15, 150, "token"),       # more v-heads than CTAs: no segments
    ([300, 301, 302], 8, 16, "none"),
])
@pytest.mark.parametrize("state", [True, False])
def test_prefill(lens, H, HV, kind, state):
    from rocm_flashinfer_contest_b200 import decay_prefill
    case = prefill_case(lens, H, HV, kind, seed=sum(lens) + HV, state=state)
    q, k, v, st, g, cu = case
    o, s = decay_prefill.run(q, k, v, st, g, torch.tensor(cu, dtype=torch.int32, device="cuda"), None)
    check_prefill(o, s, case)


@pytest.mark.parametrize("scale", [1.0, -0.25, 3e-5])
def test_prefill_scale(scale):
    from rocm_flashinfer_contest_b200 import decay_prefill
    case = prefill_case([70, 3], 1, 2, "token", seed=3)
    q, k, v, st, g, cu = case
    o, s = decay_prefill.run(q, k, v, st, g, torch.tensor(cu, device="cuda"), scale)
    check_prefill(o, s, case, scale)


def test_prefill_in_place_and_bitwise_repeatable():
    from rocm_flashinfer_contest_b200 import decay_prefill
    case = prefill_case([777, 20, 0, 300], 2, 4, "token", seed=5)
    q, k, v, st, g, cu = case
    cu_t = torch.tensor(cu, device="cuda")
    o, s = decay_prefill.run(q, k, v, st, g, cu_t, SCALE)
    check_prefill(o, s, case)
    for _ in range(3):
        st2, o2 = st.clone(), torch.empty_like(o)
        decay_prefill.run_into(q, k, v, st2, g, cu_t, SCALE, o2, st2)
        assert torch.equal(o2, o) and torch.equal(st2, s)


@pytest.mark.parametrize("lens", [[100, 37], [600, 1], [0]])
def test_prefill_tokens_of_no_sequence(lens):
    """Tokens before the first and behind the last sequence get zeros, whatever they hold, and so does nothing else."""
    from rocm_flashinfer_contest_b200 import decay_prefill
    case = prefill_case(lens, 2, 4, "token", seed=9, lead=70, behind=130)
    q, k, v, st, g, cu = case
    for x in (q, k, v, g):
        x[:70] = float("nan")
        x[cu[-1]:] = float("inf")
    out = torch.full_like(v, 7.0)
    s = torch.empty_like(st)
    decay_prefill.run_into(q, k, v, st, g, torch.tensor(cu, device="cuda"), SCALE, out, s)
    assert (out[:70] == 0).all() and (out[cu[-1]:] == 0).all()
    clean = tuple(x.clone() for x in (q, k, v, g))
    for x in clean:
        x[:70] = 0
        x[cu[-1]:] = 0
    check_prefill(out, s, (*clean[:3], st, clean[3], cu))


def test_prefill_neighbours_do_not_mix():
    """A sequence's NaN stays in that sequence."""
    from rocm_flashinfer_contest_b200 import decay_prefill
    q, k, v, st, g, cu = prefill_case([50, 30, 20], 1, 2, "token", seed=11)
    cu_t = torch.tensor(cu, device="cuda")
    o, s = decay_prefill.run(q, k, v, st, g, cu_t, SCALE)
    for x in (q, k, v):
        x[50:80] = float("nan")
    st2 = st.clone()
    st2[1] = float("nan")
    o2, s2 = decay_prefill.run(q, k, v, st2, g, cu_t, SCALE)
    for part in (slice(0, 50), slice(80, 100)):
        assert torch.equal(o2[part], o[part])
    assert torch.equal(s2[[0, 2]], s[[0, 2]]) and s2[1].isnan().all()


def test_prefill_views_and_int64():
    from rocm_flashinfer_contest_b200 import decay_prefill
    q, k, v, st, g, cu = case = prefill_case([90, 33], 2, 4, "token", seed=13)
    T = q.shape[0]
    fused = torch.zeros(T, 2 + 2 + 4, 128, dtype=torch.bfloat16, device="cuda")
    fused[:, :2], fused[:, 2:4], fused[:, 4:] = q, k, v
    off = torch.zeros(st.numel() + 1, device="cuda")[1:].view(st.shape)   # starts 4 bytes off
    off.copy_(st)
    o, s = decay_prefill.run(fused[:, :2], fused[:, 2:4], fused[:, 4:], off, g.T.contiguous().T,
                             torch.tensor(cu, dtype=torch.int64, device="cuda"), torch.tensor(SCALE))
    check_prefill(o, s, case)


def test_prefill_no_tokens_and_no_sequences():
    from rocm_flashinfer_contest_b200 import decay_prefill
    gen = torch.Generator(device="cuda").manual_seed(1)
    st = rnd(gen, 3, 2, 128, 128, dtype=torch.float32)
    e = torch.zeros(0, 1, 128, dtype=torch.bfloat16, device="cuda")
    ev = torch.zeros(0, 2, 128, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(2, device="cuda")
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    o, s = decay_prefill.run(e, e, ev, st, g, cu, None)
    assert o.shape == (0, 2, 128) and torch.equal(s, st)
    o, s = decay_prefill.run(e, e, ev, None, g, cu, None)
    assert (s == 0).all()
    o, s = decay_prefill.run(e, e, ev, st, g.expand(0, 2), cu, None)   # a decay for each of no tokens
    assert torch.equal(s, st)
    q, v = rnd(gen, 9, 1, 128), rnd(gen, 9, 2, 128)
    o, s = decay_prefill.run(q, q, v, None, g, cu[:1], None)
    assert (o == 0).all() and s.shape[0] == 0


@pytest.mark.parametrize("cu", [[0, 500, 300, 700], [-5, 2000, 700], [700, 0, 10], [3, 3, 10 ** 9]])
def test_prefill_malformed_offsets_stay_in_bounds(cu):
    """Offsets are clamped on the device; a well-formed call beside it is not disturbed."""
    from rocm_flashinfer_contest_b200 import decay_prefill
    T, N = 700, len(cu) - 1
    q, k, v, _, g, good = case = prefill_case([T], 1, 2, "token", seed=2, state=False)
    guard = torch.zeros(T + 128, 2, 128, dtype=torch.bfloat16, device="cuda")
    s = torch.empty(N, 2, 128, 128, device="cuda")
    decay_prefill.run_into(q, k, v, None, g, torch.tensor(cu, device="cuda"), SCALE, guard[64:64 + T], s)
    assert (guard[:64] == 0).all() and (guard[64 + T:] == 0).all()
    o, s = decay_prefill.run(q, k, v, None, g, torch.tensor(good, device="cuda"), SCALE)
    check_prefill(o, s, case)


def test_prefill_graphs_and_streams():
    """Captured calls replay on new inputs; two graphs and another stream keep to their own workspaces."""
    from rocm_flashinfer_contest_b200 import decay_prefill
    a = prefill_case([900], 1, 2, "token", seed=21)
    b = prefill_case([400, 500], 1, 2, "head", seed=22)
    cases, graphs, outs = [a, b], [], []
    for q, k, v, st, g, cu in cases:
        cu_t = torch.tensor(cu, device="cuda")
        decay_prefill.run(q, k, v, st, g, cu_t, SCALE)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(decay_prefill.run(q, k, v, st, g, cu_t, SCALE))
        graphs.append((graph, cu_t))
    for _ in range(2):
        for (graph, _cu), (o, s), case in zip(graphs, outs, cases):
            o.zero_(), s.zero_()
            case[2].copy_(case[2].flip(0))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for (o, s), case in zip(outs, cases):
            check_prefill(o, s, case)


# ---------------------------------------------------------------- decode

def pool_case(B, T, H, HV, kind, seed, bf16, slots):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pool = rnd(gen, slots, HV, 128, 128, s=0.5, dtype=torch.bfloat16 if bf16 else torch.float32)
    idx = torch.randperm(slots, generator=gen, device="cuda")[:B]
    q, k, v = rnd(gen, B, T, H, 128), rnd(gen, B, T, H, 128, s=0.2), rnd(gen, B, T, HV, 128)
    return gen, pool, idx, q, k, v, gates(gen, (B, T), HV, kind)


@pytest.mark.parametrize("B,H,HV,kind", [(1, 1, 1, "token"), (3, 2, 4, "head"), (9, 5, 15, "strong"), (70, 2, 16, "token")])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
def test_decode_pool(B, H, HV, kind, bf16, idt):
    from rocm_flashinfer_contest_b200 import decay_decode
    _, pool, idx, q, k, v, g = pool_case(B, 1, H, HV, kind, B + HV, bf16, B + 3)
    idx = idx.to(idt)
    before = pool.clone()
    pad = [i for i in (1, 4) if i < B]
    for i, x in zip(pad, (-1, B + 3)):
        idx[i] = x
    o, p = decay_decode.run_pool(q, k, v, pool, idx, g, SCALE)
    assert p is pool
    live = [i for i in range(B) if i not in pad]
    at = idx.cpu().long()[live]
    a = decays(g.cpu(), (B, 1), HV).exp()[live, 0]
    S = before.cpu().double()[at]
    ro, om, rs, rm = step(S, heads(q.cpu(), HV)[live, 0], heads(k.cpu(), HV)[live, 0], v.cpu().double()[live, 0], a, SCALE)
    close(o[live, 0], ro, U_BF16 * ro.abs() + 32 * U_F32 * om + 1e-30, "output")
    close(pool[at.cuda()], rs, 4 * U_F32 * rm + (U_BF16 * rs.abs() if bf16 else 0) + 1e-30, "state")
    assert (o[pad] == 0).all()
    rest = [s for s in range(B + 3) if s not in at.tolist()]
    assert torch.equal(pool[rest], before[rest])


def test_decode_run_forms():
    from rocm_flashinfer_contest_b200 import decay_decode
    _, pool, _, q, k, v, g = pool_case(5, 1, 2, 4, "token", 7, False, 5)
    a = decays(g.cpu(), (5, 1), 4).exp()[:, 0]
    args = (heads(q.cpu(), 4)[:, 0], heads(k.cpu(), 4)[:, 0], v.cpu().double()[:, 0], a, SCALE)
    for state in (pool, None):
        S = torch.zeros(5, 4, 128, 128, dtype=torch.float64) if state is None else pool.cpu().double()
        ro, om, rs, rm = step(S, *args)
        o, s = decay_decode.run(q, k, v, state, g, None)
        close(o[:, 0], ro, U_BF16 * ro.abs() + 32 * U_F32 * om + 1e-30, "output")
        close(s, rs, 4 * U_F32 * rm + 1e-30, "state")
    st = pool.clone()
    o2, s2 = decay_decode.run_into(q, k, v, st, g, SCALE, torch.empty_like(v), st)
    o, s = decay_decode.run(q, k, v, pool, g, SCALE)
    assert s2 is st and torch.equal(st, s) and torch.equal(o2, o)


def test_decode_output_slots():
    from rocm_flashinfer_contest_b200 import decay_decode
    _, pool, _, q, k, v, g = pool_case(3, 1, 1, 2, "head", 8, False, 8)
    before = pool.clone()
    idx = torch.tensor([2, 2, 5], device="cuda")          # a slot may be read twice
    dst = torch.tensor([0, 1, -1], device="cuda", dtype=torch.int32)
    decay_decode.run_pool(q, k, v, pool, idx, g, SCALE, output_state_indices=dst)
    a = decays(g.cpu(), (3, 1), 2).exp()[:, 0]
    _, _, rs, rm = step(before.cpu().double()[[2, 2, 5]], heads(q.cpu(), 2)[:, 0], heads(k.cpu(), 2)[:, 0],
                        v.cpu().double()[:, 0], a, SCALE)
    close(pool[:2], rs[:2], 4 * U_F32 * rm[:2] + 1e-30, "state")
    assert torch.equal(pool[2:], before[2:])


def test_decode_slots_past_32_bits():
    """A pool of more than 2^32 bytes and 2^31 elements: the last slot's offset needs 64 bits."""
    from rocm_flashinfer_contest_b200 import decay_decode
    slots, HV = 2 ** 31 // (32 * 128 * 128) + 2, 32
    pool = torch.zeros(slots, HV, 128, 128, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(4)
    last = rnd(gen, HV, 128, 128, s=0.5)
    pool[-1] = last
    q, k, v = rnd(gen, 1, 1, 16, 128), rnd(gen, 1, 1, 16, 128, s=0.2), rnd(gen, 1, 1, HV, 128)
    g = gates(gen, (1, 1), HV, "token")
    o, _ = decay_decode.run_pool(q, k, v, pool, torch.tensor([slots - 1], device="cuda"), g, SCALE)
    ro, om, rs, rm = step(last.cpu().double()[None], heads(q.cpu(), HV)[:, 0], heads(k.cpu(), HV)[:, 0],
                          v.cpu().double()[:, 0], decays(g.cpu(), (1, 1), HV).exp()[:, 0], SCALE)
    close(o[:, 0], ro, U_BF16 * ro.abs() + 32 * U_F32 * om + 1e-30, "output")
    close(pool[-1:], rs, 4 * U_F32 * rm + U_BF16 * rs.abs() + 1e-30, "state")
    assert not pool[:-1].any()


# ---------------------------------------------------------------- trees

def tree_parents(gen, B, T, kind):
    t = torch.arange(T, device="cuda")
    if kind == "chain":
        return (t - 1).expand(B, T).to(torch.int32).contiguous()
    if kind == "star":
        return torch.full((B, T), -1, dtype=torch.int32, device="cuda")
    back = (torch.rand(B, T, generator=gen, device="cuda") * torch.clamp(t + 1, max=4)).long()
    par = (t - 1 - back).to(torch.int32)
    bad = torch.rand(B, T, generator=gen, device="cuda")
    par = torch.where(bad < 0.1, -2, par)
    return torch.where((bad > 0.95), 63, par).to(torch.int32)   # at or behind the node: padding too


def verify_reference(pool, idx, parents, q, k, v, g, scale):
    B, T, HV = v.shape[:3]
    qh, kh, vh, gg = heads(q.cpu(), HV), heads(k.cpu(), HV), v.cpu().double(), decays(g.cpu(), (B, T), HV)
    out = torch.zeros(B, T, HV, 128, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for b in range(B):
        s = int(idx[b])
        if not 0 <= s < pool.shape[0]:
            continue
        S = pool[s].cpu().double()
        for t, path in enumerate(paths(parents[b].tolist())):
            if path is None:
                continue
            c = gg[b, path].cumsum(0)
            w = (c[-1] - c).exp()                                            # [L, HV]
            P = (qh[b, t] * kh[b, path]).sum(-1) * w
            e = c[-1].exp()[:, None]
            inter = (S @ qh[b, t][:, :, None])[..., 0]
            out[b, t] = scale * (e * inter + (P[..., None] * vh[b, path]).sum(0))
            mag[b, t] = abs(scale) * (e * (S.abs() @ qh[b, t].abs()[:, :, None])[..., 0]
                                      + (P.abs()[..., None] * vh[b, path].abs()).sum(0))
    return out, mag


@pytest.mark.parametrize("B,T,H,HV,kind,tree", [
    (1, 1, 1, 1, "token", "chain"), (2, 7, 2, 4, "head", "mixed"), (3, 16, 1, 2, "token", "chain"),
    (2, 17, 5, 5, "token", "mixed"), (1, 33, 1, 3, "head", "star"), (2, 48, 2, 2, "token", "mixed"),
    (2, 64, 1, 2, "token", "chain"), (3, 64, 2, 4, "head", "mixed"), (4, 5, 1, 2, "strong", "mixed"),
])
@pytest.mark.parametrize("bf16", [False, True])
def test_tree_verify_and_commit(B, T, H, HV, kind, tree, bf16):
    from rocm_flashinfer_contest_b200 import decay_tree
    gen, pool, idx, q, k, v, g = pool_case(B, T, H, HV, kind, 31 * T + HV, bf16, B + 2)
    parents = tree_parents(gen, B, T, tree)
    if B > 2:
        idx[1] = -1
    ro, rm = verify_reference(pool, idx, parents, q, k, v, g, SCALE)
    ps = [paths(parents[b].tolist()) for b in range(B)]
    for b in range(B):       # what padding nodes hold is not used
        for t in range(T):
            if ps[b][t] is None:
                q[b, t] = k[b, t] = v[b, t] = float("nan")
    before = pool.clone()
    o = decay_tree.run(q, k, v, pool, idx, parents, g, SCALE)
    assert torch.equal(pool, before)
    # sums of decays up to 104 * T off by a rounding of the sum each, where decays are strong
    slack = 2.0 ** -16 + 32 * U_F32 + (T * 104 * T * U_F32 if kind == "strong" else 0)
    close(o, ro, U_BF16 * ro.abs() + slack * rm + 1e-30, "output")
    dead = torch.tensor([[p is None for p in row] for row in ps])
    dead[idx.cpu() < 0] = True
    assert (o.cpu()[dead] == 0).all()

    accepted = torch.randint(-1, T, (B,), generator=gen, device="cuda").to(torch.int32)
    if B > 2:
        accepted[2] = T + 3                  # no such node
    kept = decay_tree.commit(k, v, pool, idx, parents, accepted, g)
    assert kept is pool
    kh, vh, gg = heads(k.cpu(), HV), v.cpu().double(), decays(g.cpu(), (B, T), HV)
    for b in range(B):
        s, a = int(idx[b]), int(accepted[b])
        path = ps[b][a] if 0 <= a < T else None
        if s < 0:
            continue
        if not path:
            assert torch.equal(pool[s], before[s])
            continue
        S = before[s].cpu().double()
        Sm = S.abs()
        for t in path:
            e = gg[b, t].exp()[:, None, None]
            kv = vh[b, t][:, :, None] * kh[b, t][:, None, :]
            S, Sm = e * S + kv, e * Sm + kv.abs()
        tol = (4 * len(path) + 8) * 2 * U_F32 * Sm + (U_BF16 * S.abs() if bf16 else 0) + 1e-30
        close(pool[s], S, tol, "state")
    rest = [s for s in range(B + 2) if s not in idx.tolist()]
    assert torch.equal(pool[rest], before[rest])


def test_commit_output_slots():
    from rocm_flashinfer_contest_b200 import decay_tree
    _, pool, _, q, k, v, g = pool_case(4, 6, 1, 2, "token", 77, False, 9)
    parents = torch.arange(-1, 5, device="cuda").expand(4, 6).to(torch.int32).contiguous()
    idx = torch.tensor([0, 0, 1, 2], device="cuda", dtype=torch.int32)
    dst = torch.tensor([5, 6, 7, -1], device="cuda", dtype=torch.int32)
    acc = torch.tensor([5, 2, -1, 4], device="cuda", dtype=torch.int32)
    alone = pool.clone()
    decay_tree.commit(k[:1], v[:1], alone, idx[:1], parents[:1], acc[:1], g[:1])
    before = pool.clone()
    decay_tree.commit(k, v, pool, idx, parents, acc, g, output_state_indices=dst)
    assert torch.equal(pool[5], alone[0])
    assert torch.equal(pool[7], before[1])        # nothing accepted: a copy
    assert torch.equal(pool[[0, 1, 2, 3, 4, 8]], before[[0, 1, 2, 3, 4, 8]])
    assert not torch.equal(pool[6], before[6])


def test_tree_shares_slots_and_takes_views():
    from rocm_flashinfer_contest_b200 import decay_tree
    _, pool, _, q, k, v, g = pool_case(3, 9, 2, 4, "token", 5, False, 4)
    parents = torch.arange(-1, 8, device="cuda").expand(3, 9).to(torch.int32)
    idx = torch.tensor([1, 1, 3], device="cuda")
    ro, rm = verify_reference(pool, idx, parents, q, k, v, g, SCALE)
    o = decay_tree.run(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, pool, idx, parents, g, None)
    close(o, ro, U_BF16 * ro.abs() + 2.0 ** -15 * rm + 1e-30, "output")


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("bf16", [False, True])
def test_prompt_tree_decode_together(bf16):
    """A prompt, its state parked and resumed, a drafted tree, the accepted path, a decode step: the tokens' recurrence."""
    from rocm_flashinfer_contest_b200 import decay_decode, decay_prefill, decay_tree
    H, HV, T, N = 2, 4, 8, 2
    gen = torch.Generator(device="cuda").manual_seed(99)
    lens = [300, 41]
    q, k, v, _, g, cu = prefill_case(lens, H, HV, "token", 99, state=False)
    o, s = decay_prefill.run(q, k, v, None, g, torch.tensor(cu, device="cuda"), None)
    pool = torch.zeros(5, HV, 128, 128, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    idx = torch.tensor([3, 1], device="cuda", dtype=torch.int32)
    pool[idx.long()] = s.to(pool.dtype)
    tq, tk, tv = rnd(gen, N, T, H, 128), rnd(gen, N, T, H, 128, s=0.2), rnd(gen, N, T, HV, 128)
    tg = gates(gen, (N, T), HV, "token")
    parents = torch.tensor([[-1, 0, 0, 1, 2, 3, 4, 4]] * N, device="cuda", dtype=torch.int32)
    ov = decay_tree.run(tq, tk, tv, pool, idx, parents, tg)
    decay_tree.commit(tk, tv, pool, idx, parents, torch.tensor([7, 5], device="cuda", dtype=torch.int32), tg)
    dq, dk, dv = rnd(gen, N, 1, H, 128), rnd(gen, N, 1, H, 128, s=0.2), rnd(gen, N, 1, HV, 128)
    dg = gates(gen, (N, 1), HV, "token")
    od, _ = decay_decode.run_pool(dq, dk, dv, pool, idx, dg)
    # the same tokens one after the other through the prefill
    for n, path in enumerate(([0, 2, 4, 7], [0, 1, 3, 5])):
        seq = slice(cu[n], cu[n + 1])
        cat = lambda a, b, c: torch.cat([a[seq], b[n, path], c[n]])  # noqa: E731
        case = (cat(q, tq, dq), cat(k, tk, dk), cat(v, tv, dv), None, cat(g, tg, dg), [0, lens[n] + 5])
        ro, rm, rs, rsm = prefill(*case, SCALE)
        got = torch.cat([o[seq], ov[n, path], od[n]])
        # a pooled state in bf16 is rounded when it is written: twice before the last output, and then once more
        more = U_BF16 if bf16 else 0
        close(got, ro, U_BF16 * ro.abs() + (U_BF16 + 2.0 ** -14 + 2 * more) * rm + 1e-30, "output")
        close(pool[int(idx[n])][None], rs, (2.0 ** -16 + 3 * 1.01 * more) * rsm + 1e-30, "state")


def test_graph_of_a_whole_step():
    """Verify, commit and decode captured together and replayed give what the calls give."""
    from rocm_flashinfer_contest_b200 import decay_decode, decay_tree
    gen, pool, idx, q, k, v, g = pool_case(4, 6, 1, 2, "token", 3, False, 6)
    parents = tree_parents(gen, 4, 6, "mixed")
    acc = torch.tensor([5, 0, -1, 3], device="cuda", dtype=torch.int32)
    start = pool.clone()

    def one():
        o = decay_tree.run(q, k, v, pool, idx, parents, g, SCALE)
        decay_tree.commit(k, v, pool, idx, parents, acc, g)
        d, _ = decay_decode.run_pool(q[:, :1].contiguous(), k[:, :1].contiguous(), v[:, :1].contiguous(), pool, idx,
                                     g[:, :1].contiguous(), SCALE)
        return o, d

    want = one()
    end = pool.clone()
    pool.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = one()
    pool.copy_(start)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(pool, end) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_at_once_on_streams():
    """Prefills (of several launches), trees and the delta rule's prefill on streams of their own give what each gives alone."""
    from rocm_flashinfer_contest_b200 import decay_prefill, decay_tree, gdn_prefill
    jobs = []
    for seed in (1, 2):
        q, k, v, st, g, cu = prefill_case([3000, 65, 0, 700], 2, 8, "token", seed)
        jobs.append((decay_prefill.run, (q, k, v, st, g, torch.tensor(cu, device="cuda"), None)))
    for bf16, T in ((False, 9), (True, 40)):
        gen, pool, idx, q, k, v, g = pool_case(40, T, 2, 8, "token", T, bf16, 44)
        jobs.append((decay_tree.run, (q, k, v, pool, idx, tree_parents(gen, 40, T, "mixed"), g)))
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = rnd(gen, 900, 4, 128), rnd(gen, 900, 4, 128, s=0.1), rnd(gen, 900, 8, 128)
    a, b = rnd(gen, 900, 8), rnd(gen, 900, 8)
    al, dt = rnd(gen, 8, dtype=torch.float32), rnd(gen, 8, dtype=torch.float32)
    jobs.append((gdn_prefill.run, (q, k, v, None, al, a, dt, b, torch.tensor([0, 900], device="cuda"), None)))
    flat = lambda x: x if isinstance(x, tuple) else (x,)  # noqa: E731
    alone = [flat(f(*args)) for f, args in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for (f, args), stream in zip(jobs, streams):
            with torch.cuda.stream(stream):
                got.append(flat(f(*args)))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert all(torch.equal(y, z) for y, z in zip(x, alone[i % len(jobs)])), i


def test_trees_without_nodes():
    from rocm_flashinfer_contest_b200 import decay_tree
    _, pool, idx, q, k, v, g = pool_case(3, 0, 1, 2, "token", 6, False, 6)
    parents = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    assert decay_tree.run(q, k, v, pool, idx, parents, g).shape == (3, 0, 2, 128)
    before = pool.clone()
    dst = torch.tensor([i for i in range(6) if i not in idx.tolist()], device="cuda")
    decay_tree.commit(k, v, pool, idx, parents, torch.tensor([-1, 0, 5], dtype=torch.int32, device="cuda"), g, dst)
    assert torch.equal(pool[dst], before[idx]) and torch.equal(pool[idx], before[idx])


def test_one_entry_of_many_heads_and_padding_around_it():
    """A padded batch: one entry in use, first, in the middle or last; more v-heads than CTAs."""
    from rocm_flashinfer_contest_b200 import decay_decode, decay_tree
    gen, pool, idx, q, k, v, g = pool_case(3, 2, 1, 200, "token", 8, True, 4)
    parents = torch.tensor([[-1, 0]] * 3, dtype=torch.int32, device="cuda")
    full = decay_tree.run(q, k, v, pool, idx, parents, g)
    one = lambda x: x[:, :1].contiguous()  # noqa: E731
    end = pool.clone()
    step_full, _ = decay_decode.run_pool(one(q), one(k), one(v), end, idx, one(g))
    for i in range(3):
        some = torch.full_like(idx, -1)
        some[i] = idx[i]
        q2, k2, v2, g2 = (torch.where((some < 0).view(-1, *[1] * (x.dim() - 1)), float("nan"), x) for x in (q, k, v, g))
        o = decay_tree.run(q2, k2, v2, pool, some, parents, g2)
        mine = pool.clone()
        d, _ = decay_decode.run_pool(one(q2), one(k2), one(v2), mine, some, one(g2))
        rest = [j for j in range(3) if j != i]
        assert torch.equal(o[i], full[i]) and (o[rest] == 0).all()
        assert torch.equal(d[i], step_full[i]) and (d[rest] == 0).all()
        assert torch.equal(mine[idx[i]], end[idx[i]])
        left = [s for s in range(4) if s != int(idx[i])]
        assert torch.equal(mine[left], pool[left])

"""Two index tensors of different types: the narrower one is widened, so an index
outside the pool stays outside it (2^32 as int32 would be slot 0)."""
import pytest
import torch

from rocm_flashinfer_contest_b200 import _common as C

CPU = torch.device("cpu")
FAR = 2 ** 32          # 0 in its low 32 bits


@pytest.mark.parametrize("swap", [False, True])
def test_a_pair_of_two_types_is_widened(swap):
    a = torch.tensor([0, 1], dtype=torch.int32)
    b = torch.tensor([FAR, -1], dtype=torch.int64)
    x, y = C.require_index_pair(*((b, a) if swap else (a, b)), 2, CPU, ("one", "other"))
    if swap:
        x, y = y, x
    assert x.dtype == y.dtype == torch.int64
    assert x.tolist() == [0, 1] and y.tolist() == [FAR, -1]


@pytest.mark.parametrize("dt", [torch.int32, torch.int64])
def test_a_pair_of_one_type_is_taken_as_it_is(dt):
    a, b = torch.tensor([0, 1], dtype=dt), torch.tensor([3, -1], dtype=dt)
    x, y = C.require_index_pair(a, b, 2, CPU, ("one", "other"))
    assert x is a and y is b
    x, y = C.require_index_pair(a, None, 2, CPU, ("one", "other"))
    assert x is a and y is None


def test_a_pair_is_checked():
    a = torch.tensor([0, 1], dtype=torch.int32)
    for bad in (a.float(), a[:1], a[None], "x", a.to(torch.int16)):
        with pytest.raises(ValueError, match="other"):
            C.require_index_pair(a, bad, 2, CPU, ("one", "other"))
        with pytest.raises(ValueError, match="one"):
            C.require_index_pair(bad, a, 2, CPU, ("one", "other"))


@pytest.mark.gpu
@pytest.mark.parametrize("far_first", [False, True])
def test_an_index_past_32_bits_touches_no_slot(far_first):
    from rocm_flashinfer_contest_b200 import decay_decode, decay_tree, state_cache
    gen = torch.Generator(device="cuda").manual_seed(0)
    bf = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(torch.bfloat16)  # noqa: E731
    q, k, v = bf(2, 1, 1, 128), bf(2, 1, 1, 128), bf(2, 1, 2, 128)
    g = torch.full((2,), -0.5, device="cuda")
    pool = torch.randn(4, 2, 128, 128, generator=gen, device="cuda")
    narrow = torch.tensor([2, 3], dtype=torch.int32, device="cuda")
    far = torch.tensor([FAR, FAR + 1], dtype=torch.int64, device="cuda")
    idx, dst = (far, narrow) if far_first else (narrow, far)
    before = pool.clone()
    o, _ = decay_decode.run_pool(q, k, v, pool, idx, g, output_state_indices=dst)
    assert torch.equal(pool, before)
    if far_first:
        assert (o == 0).all()
    parents = torch.full((2, 1), -1, dtype=torch.int32, device="cuda")
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    decay_tree.commit(k, v, pool, idx, parents, zero, g, dst)
    assert torch.equal(pool, before)
    codes, exps = state_cache.empty(4, (2, 128, 128))
    codes.fill_(5), exps.fill_(127)
    state_cache.store(pool, idx, codes, exps, dst)
    assert (codes == 5).all() and (exps == 127).all()
    state_cache.load(codes, exps, idx, pool, dst)
    assert torch.equal(pool, before)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [3, 64])
def test_mtp_output_index_past_32_bits_touches_no_slot(B):
    from rocm_flashinfer_contest_b200 import gdn_mtp, inputs
    args = inputs.to_device(inputs.mtp_inputs(B, 2, B + 2, 2, 4, seed=1), torch.device("cuda"))   # int32 indices
    pool, before = args[3], args[3].clone()
    far = torch.arange(B, device="cuda") + FAR
    out = torch.empty(B, 2, 4, 128, dtype=torch.bfloat16, device="cuda")
    gdn_mtp.run_into(*args[:10], out, pool, output_state_indices=far)
    assert torch.equal(pool, before)
    want, _ = gdn_mtp.run(*args[:10])
    assert torch.equal(out, want)

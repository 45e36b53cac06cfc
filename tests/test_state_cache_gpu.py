"""8-bit state cache on the GPU: codes, exponents and values bit for bit against
the definition in 64 bits (the scales are powers of two, so the codes' own
rounding is the only one)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def reference(x, dtype):
    """(values, exponent bytes) of x [..., n]: e is the smallest integer >= -127 with max|x| <= top * 2^e."""
    x = x.cpu().double()
    x = x.view(*x.shape[:-1], -1, 32)
    top = x.abs().amax(-1)
    e = torch.full_like(top, -127.0)
    fin = torch.isfinite(top)
    while True:
        up = fin & (top > TOP[dtype] * torch.exp2(e))
        if not up.any():
            break
        e[up] += 1
    y = torch.where(fin[..., None], x / torch.exp2(e)[..., None], 0.0)
    if dtype == torch.int8:
        y = torch.round(y)
    else:
        unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        y = torch.round(y / unit) * unit
    val = torch.where(fin[..., None], y * torch.exp2(e)[..., None], float("nan"))
    return val.flatten(-2), torch.where(fin, e + 127, 255.0).to(torch.uint8)


def make(shape, dtype, seed, special=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, generator=gen, device="cuda")
    x = x * torch.exp(4 * torch.randn(*shape[:-1], 1, generator=gen, device="cuda"))
    if special:
        flat = x.view(-1, 32)
        rows = [(0, 0.0), (1, float("inf")), (2, float("nan")), (3, -float("inf"))]
        for r, val in rows:
            if r == 0:
                flat[r] = 0.0
            else:
                flat[r, (7 * r) % 32] = val
        flat[4] = 0.0
        flat[4, 3] = 127.0                   # exactly top * 2^0
        flat[5] = 0.0
        flat[5, 3] = 448.0
        flat[6, :] = 1.5e-45                 # subnormal
        flat[7, 0] = 3.3e38
        flat[8] = torch.arange(32, device="cuda") + 0.5      # ties
        flat[8, 31] = 127.0
        flat[9] = 2.0 ** -130
        flat[10] = torch.linspace(-3, 3, 32, device="cuda") * 2.0 ** -120
        flat[11, 0] = -127.0000076293945
    return x.to(dtype)


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("pdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 128, 128), (1, 3, 32), (5, 7, 96), (1, 128, 128), (33, 32), (1, 32)])
def test_store_and_load(fmt, pdt, shape):
    from rocm_flashinfer_contest_b200 import state_cache
    slots, cslots = 6, 5
    n = 1
    for s in shape:
        n *= s
    pool = make((slots, *shape), pdt, seed=n, special=slots * n >= 32 * 12)
    codes, exps = state_cache.empty(cslots, shape, fmt)
    codes.view(torch.uint8).fill_(3), exps.fill_(9)
    src = torch.tensor([4, -1, 0, 2, 6, 1], device="cuda", dtype=torch.int32)
    dst = torch.tensor([0, 1, 3, 5, 2, 4], device="cuda", dtype=torch.int64)   # another type: converted
    keep = pool.clone()
    assert state_cache.store(pool, src, codes, exps, dst)[0] is codes
    assert torch.equal(pool.view(torch.uint8), keep.view(torch.uint8))
    pairs = [(4, 0), (0, 3), (1, 4)]          # the others: -1, a cache slot past the end, a pool slot past the end
    for a, c in pairs:
        val, eb = reference(pool[a].float(), fmt)
        assert torch.equal(exps[c].cpu(), eb)
        e = eb.double() - 127
        stored = codes[c].float().cpu().double().view(*eb.shape, 32)
        ok = (eb != 255)[..., None].expand_as(stored)
        assert torch.equal((stored * torch.exp2(e)[..., None])[ok], val.view_as(stored)[ok])
        assert (stored[~ok] == 0).all()
    for c in (1, 2):
        assert (codes[c].view(torch.uint8) == 3).all() and (exps[c] == 9).all()

    back = torch.full_like(pool, 5.0)
    assert state_cache.load(codes, exps, torch.tensor([0, 3, 4, -1], device="cuda"), back,
                            torch.tensor([1, 5, 0, 2], device="cuda")) is back
    for (a, c), to in zip(pairs, (1, 5, 0)):
        val, _ = reference(pool[a].float(), fmt)
        want = val.float().to(pdt).cpu()
        got = back[to].cpu()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[~want.isnan()], want[~want.isnan()])
    assert (back[[2, 3, 4]] == 5.0).all()


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn])
def test_every_code_reads_back(fmt):
    from rocm_flashinfer_contest_b200 import state_cache
    raw = torch.arange(256, device="cuda", dtype=torch.int32).to(torch.uint8).view(1, 8, 32)
    codes = raw.view(fmt).clone()
    for byte in (0, 1, 100, 127, 140, 246, 255):
        exps = torch.full((1, 8, 1), byte, dtype=torch.uint8, device="cuda")
        pool = torch.zeros(1, 8, 32, device="cuda")
        z = torch.zeros(1, dtype=torch.int32, device="cuda")
        state_cache.load(codes, exps, z, pool, z)
        want = (codes.float().cpu().double() * 2.0 ** (byte - 127)).float()
        if byte == 255:
            want.fill_(float("nan"))
        got = pool.cpu()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[~want.isnan()], want[~want.isnan()])


def test_store_twice_is_stable():
    """What was read back is stored again without a change: the codes are the values'."""
    from rocm_flashinfer_contest_b200 import state_cache
    for fmt in (torch.int8, torch.float8_e4m3fn):
        pool = make((3, 4, 128, 128), torch.float32, seed=1, special=False)
        codes, exps = state_cache.empty(3, (4, 128, 128), fmt)
        i = torch.arange(3, device="cuda")
        state_cache.store(pool, i, codes, exps, i)
        state_cache.load(codes, exps, i, pool, i)
        first = pool.clone()
        state_cache.store(pool, i, codes, exps, i)
        state_cache.load(codes, exps, i, pool, i)
        assert torch.equal(first, pool)


def test_offsets_past_32_bits():
    from rocm_flashinfer_contest_b200 import state_cache
    shape = (32, 128, 128)
    slots = 2 ** 32 // (32 * 128 * 128) + 2           # codes past 2^32 bytes
    codes, exps = state_cache.empty(slots, shape, torch.int8)
    pool = make((1, *shape), torch.float32, seed=8)
    z, last = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.tensor([slots - 1], device="cuda")
    state_cache.store(pool, z, codes, exps, last)
    back = torch.empty_like(pool)
    state_cache.load(codes, exps, last, back, z)
    want, _ = reference(pool[0], torch.int8)
    ok = ~want.isnan()
    assert torch.equal(back[0].cpu().double()[ok], want[ok]) and back[0].cpu()[~ok].isnan().all()


def test_parks_states_of_both_recurrences():
    """A gated-delta-rule state and a decay state parked in one cache continue from what was read back."""
    from rocm_flashinfer_contest_b200 import decay_decode, gdn_decode, inputs, state_cache
    dev = torch.device("cuda")
    args = inputs.to_device(inputs.decode_inputs(2, 2, 4, seed=0), dev)
    _, s = gdn_decode.run(*args)
    codes, exps = state_cache.empty(4, (4, 128, 128), torch.int8)
    i = torch.arange(2, device=dev)
    state_cache.store(s, i, codes, exps, i + 2)
    resumed = torch.zeros_like(s)
    state_cache.load(codes, exps, i + 2, resumed, i)
    want = torch.stack([reference(x, torch.int8)[0] for x in s]).float()
    assert torch.equal(resumed.cpu(), want)
    q, k, v = args[0], args[1], args[2]
    o, _ = decay_decode.run(q, k, v, resumed, torch.full((4,), -0.1, device=dev), None)
    o2, _ = decay_decode.run(q, k, v, want.to(dev), torch.full((4,), -0.1, device=dev), None)
    assert torch.equal(o, o2)


def test_no_pairs():
    from rocm_flashinfer_contest_b200 import state_cache
    pool = torch.ones(2, 1, 32, device="cuda")
    codes, exps = state_cache.empty(2, (1, 32))
    codes.zero_(), exps.zero_()
    e = torch.zeros(0, dtype=torch.int32, device="cuda")
    state_cache.store(pool, e, codes, exps, e)
    state_cache.load(codes, exps, e, pool, e)
    assert (codes == 0).all() and (pool == 1).all()

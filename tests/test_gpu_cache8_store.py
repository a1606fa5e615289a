"""store_kvcache_q8 against the 64-bit statement: every value and every scale of both caches, bit for bit (quantising is a
rounding of an exact quotient: the scale is a power of two)."""
import numpy as np
import pytest

from cache8_helpers import random_cache, values_of
from oracle import cache8

pytestmark = pytest.mark.gpu


def check(k, v, cache, slots, what=""):
    import torch
    from nanovllm_jax_b200 import ops
    kvh, block = k.shape[1], cache[0].shape[1]
    before = [values_of(c) for c in cache[:2]] + [s.double().cpu().numpy() for s in cache[2:]]
    ops.store_kvcache_q8(k, v, *cache, slots)
    torch.cuda.synchronize()
    for x, rows in enumerate((k, v)):
        flat, grid = before[x].reshape(-1, kvh, 128), before[2 + x].reshape(-1, kvh)
        values, scales = cache8.store(rows.double().cpu().numpy(), flat, grid, slots.cpu().numpy())
        assert np.array_equal(cache[2 + x].double().cpu().numpy().reshape(scales.shape), scales, equal_nan=True), f"{what}: scales {'kv'[x]}"
        got = values_of(cache[x]).reshape(values.shape)
        assert np.array_equal(got, values, equal_nan=True), f"{what}: {'kv'[x]}, slots {np.unique(np.nonzero(~((got == values) | (np.isnan(got) & np.isnan(values))))[0])[:8]}"


def rows(rng, t, kvh, dtype, spread=4):
    import torch
    x = rng.normal(size=(2, t, kvh, 128)) * 2.0 ** rng.integers(-spread, spread + 1, (2, t, kvh, 1))
    return [torch.from_numpy(a.astype(np.float32)).to(dtype).cuda() for a in x]


def prompt_slots(rng, lens, block, nb):
    pages = rng.permutation(nb)
    out, at = [], 0
    for n in lens:
        need = -(-n // block)
        tok = np.arange(n)
        out.append(pages[at:at + need][tok // block] * block + tok % block)
        at += need
    return np.concatenate(out).astype(np.int32)


@pytest.mark.parametrize("f32", (False, True))
@pytest.mark.parametrize("kvh, block, lens", [
    (1, 64, [1]), (8, 256, [1]), (2, 64, [63, 64, 65, 1, 200]), (8, 256, [300, 17]), (3, 192, [100, 400]), (5, 128, [1, 2, 3, 129]),
    (2, 256, [1024]), (2, 256, [1025]), (1, 64, [900, 700, 1]), (4, 512, [3000])])
def test_prompts(kvh, block, lens, f32):
    import torch
    rng = np.random.default_rng(hash((kvh, block, len(lens), f32)) % 1000)
    nb = sum(-(-n // block) for n in lens) + 2
    slots = prompt_slots(rng, lens, block, nb)
    k, v = rows(rng, len(slots), kvh, torch.float32 if f32 else torch.bfloat16)
    check(k, v, random_cache(rng, nb, block, kvh), torch.from_numpy(slots).cuda())


@pytest.mark.parametrize("t, kvh, block", [(1, 1, 64), (5, 8, 256), (64, 2, 128), (256, 1, 256), (1500, 2, 64)])
def test_appended_rows_let_the_scale_grow(t, kvh, block):
    """One row each for blocks that hold others, of magnitudes from far below to far above theirs."""
    import torch
    rng = np.random.default_rng(t)
    nb = -(-t * 64 // block) + 1
    grains = rng.permutation(nb * block // 64)[:t]
    slots = (grains * 64 + rng.integers(0, 64, t)).astype(np.int32)
    k, v = rows(rng, t, kvh, torch.bfloat16, spread=9)
    check(k, v, random_cache(rng, nb, block, kvh), torch.from_numpy(slots).cuda())


@pytest.mark.parametrize("f32", (False, True))
@pytest.mark.parametrize("t, kvh", [(128, 8), (129, 8), (600, 8), (1024, 3), (400, 5)])
def test_rows_alone_in_their_blocks(t, kvh, f32):
    """A decode step's rows, few and many: first slots of blocks and later ones, scales that are none, values that are not finite, and among
    them a few blocks that other rows of the call go to as well."""
    import torch
    rng = np.random.default_rng(t + kvh)
    block, nb = 128, t + 1
    grains = rng.permutation(2 * nb)[:t]
    grains[t // 2], grains[t - 1] = grains[3], grains[3]  # one block three times, far apart
    slots = (grains * 64 + np.where(rng.random(t) < 0.2, 0, rng.integers(0, 64, t))).astype(np.int32)
    slots[5] = -1
    k, v = rows(rng, t, kvh, torch.float32 if f32 else torch.bfloat16, spread=9)
    k[7, 0, 3], k[8, 1], v[9, :, 100], v[10] = float("inf"), float("nan"), -float("inf"), 0
    cache = random_cache(rng, nb, block, kvh)
    cache[2].view(-1)[::7] = 0
    cache[3].view(-1)[::5] = float("nan")
    cache[3].view(-1)[1::5] = -1
    check(k, v, cache, torch.from_numpy(slots).cuda())


@pytest.mark.parametrize("t", (7, 700, 1024, 1030, 4000))
def test_any_slots_in_any_order(t):
    """Slots dealt at random: several of a block far apart in the call, some twice, some of no slot, some beyond the cache."""
    import torch
    rng = np.random.default_rng(t)
    nb, block, kvh = 9, 128, 2
    slots = rng.integers(-40, nb * block + 40, t).astype(np.int32)
    k, v = rows(rng, t, kvh, torch.bfloat16)
    check(k, v, random_cache(rng, nb, block, kvh), torch.from_numpy(slots).cuda())


def test_the_same_slot_many_times():
    import torch
    rng = np.random.default_rng(3)
    for t in (300, 2000):
        slots = np.repeat(np.array([70, 64, 5, 70], np.int32), t // 4)
        k, v = rows(rng, len(slots), 2, torch.bfloat16)
        check(k, v, random_cache(rng, 2, 64, 2), torch.from_numpy(slots).cuda())


@pytest.mark.parametrize("t", (60, 1100))
def test_values_at_the_ends(t):
    """Zeros, subnormals, the largest finite numbers, infinities and NaN, rows of nothing else among them."""
    import torch
    rng = np.random.default_rng(5)
    for f32 in (False, True):
        k, v = rows(rng, t, 2, torch.float32 if f32 else torch.bfloat16, spread=0)
        odd = torch.tensor([0.0, -0.0, 1e-40, -2.0 ** -126, 3.3e38, -3e38, float("inf"), -float("inf"), float("nan"), 448.0, 449.0])
        for x in (k, v):
            pick = torch.from_numpy(rng.integers(0, len(odd), (t, 2, 128)))
            where = torch.from_numpy(rng.random((t, 1, 1)) < 0.5) & torch.from_numpy(rng.random((t, 2, 128)) < 0.3)
            x.copy_(torch.where(where, odd[pick], x.float().cpu()).to(x.dtype))
            x[3] = 0
            x[t // 2] = float("nan")
        nb = -(-t // 64) + 1
        slots = torch.arange(t, dtype=torch.int32).cuda()
        check(k, v, random_cache(rng, nb, 64, 2), slots, f"f32={f32}")
        # a block of nothing finite
        k[:64], v[:64] = float("inf"), float("nan")
        check(k, v, random_cache(rng, nb, 64, 2), slots)


def test_scales_that_are_none_or_no_power_of_two():
    import torch
    rng = np.random.default_rng(6)
    cache = random_cache(rng, 4, 64, 2)
    cache[2].copy_(torch.tensor([[[0.0, -1.0]], [[float("nan"), 0.0]], [[2.0 ** -120, 1.0]], [[0.0, 2.0]]]))
    cache[3].zero_()
    k, v = rows(rng, 4, 2, torch.bfloat16)
    check(k, v, cache, torch.tensor([1, 65, 130, 195], dtype=torch.int32).cuda())


def test_prompt_token_by_token_stays_within_a_rounding():
    """Rows appended one call at a time end within half a step of e4m3 each time their scale grew, and under the same scale."""
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(7)
    k, v = rows(rng, 130, 2, torch.bfloat16)
    cache = random_cache(rng, 3, 64, 2)
    once = [c.clone() for c in cache]
    slots = torch.arange(130, dtype=torch.int32).cuda()
    for t in range(130):
        ops.store_kvcache_q8(k[t:t + 1], v[t:t + 1], *cache, slots[t:t + 1])
    ops.store_kvcache_q8(k, v, *once, slots)
    assert torch.equal(cache[2], once[2]) and torch.equal(cache[3], once[3])
    for x, src in enumerate((k, v)):
        scale = cache[2 + x].repeat_interleave(64, dim=1).reshape(-1, 2, 1)[:130].double()
        got = cache[x].double().reshape(-1, 2, 128)[:130] * scale
        # the first rounding and, where the scale grew, the last one: 2^-4 each, or half a subnormal step 2^-10 of the scale
        bound = 2 * torch.maximum(2.0 ** -4 * src.double().abs() * (1 + 2.0 ** -4), 2.0 ** -10 * scale)
        assert ((got - src.double()).abs() <= bound).all()


def test_captured_and_replayed_on_another_stream():
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(8)
    for t in (40, 1300):
        k, v = rows(rng, t, 2, torch.bfloat16)
        nb = -(-t // 64) + 1
        slots = torch.arange(t, dtype=torch.int32).cuda()
        cache = random_cache(rng, nb, 64, 2)
        start = [c.clone() for c in cache]
        ops.store_kvcache_q8(k, v, *cache, slots)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.store_kvcache_q8(k, v, *cache, slots)
        k2, v2 = rows(rng, t, 2, torch.bfloat16)
        k.copy_(k2), v.copy_(v2)
        slots.copy_(slots.flip(0))
        for c, s in zip(cache, start):
            c.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        for x, src in enumerate((k2, v2)):
            values, scales = cache8.store(src.double().cpu().numpy(), values_of(start[x]).reshape(-1, 2, 128),
                                          start[2 + x].double().cpu().numpy().reshape(-1, 2), slots.cpu().numpy())
            assert np.array_equal(values_of(cache[x]).reshape(values.shape), values)
            assert np.array_equal(cache[2 + x].double().cpu().numpy().reshape(scales.shape), scales)


def test_no_tokens_and_slots_at_an_odd_address():
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(9)
    cache = random_cache(rng, 30, 64, 2)
    k, v = rows(rng, 1200, 2, torch.bfloat16)
    before = [values_of(c) for c in cache[:2]]
    ops.store_kvcache_q8(k[:0], v[:0], *cache, torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert all(np.array_equal(values_of(c), b) for c, b in zip(cache[:2], before))
    slots = torch.arange(-1, 1200, dtype=torch.int32).cuda()[1:]
    check(k, v, cache, slots)

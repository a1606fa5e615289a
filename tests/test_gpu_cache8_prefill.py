"""paged_prefill_q8 against the 64-bit statement."""
import math

import numpy as np
import pytest

from cache8_helpers import attention_bound, random_cache, values_of
from oracle import cache8

pytestmark = pytest.mark.gpu


def make(rng, new, pre, h, kvh, block, mb=None):
    import torch
    lens = [a + b for a, b in zip(new, pre)]
    need = [-(-n // block) for n in lens]
    nb = sum(need) + 2
    pages = rng.permutation(nb).astype(np.int32)
    tables = np.full((len(lens), mb or max(1, max(need))), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = pages[at:at + n]
        at += n
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    cu_k = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    q = torch.from_numpy(rng.normal(size=(int(cu[-1]), h, 128)).astype(np.float32)).to(torch.bfloat16).cuda()
    return q, torch.from_numpy(tables).cuda(), torch.from_numpy(cu).cuda(), torch.from_numpy(cu_k).cuda(), cu, nb, lens


def expect(q, cache, tables, new, lens, scale, block):
    k, v = (cache8.dequantised(values_of(c), s.cpu().numpy()) for c, s in zip(cache[:2], cache[2:]))
    return cache8.attention(q.double().cpu().numpy(), k, v, tables.cpu().numpy(), new, lens, scale, block)


def close(got, want, q, scale, largest_key, what=""):
    """The bound of fp16 probabilities and, on top, a score's error from q, 2^-18 of the row's largest component for each of the 128
    products, which moves a probability, and its normaliser, by as much."""
    out, weight = want[:2]
    top = np.abs(q.double().cpu().numpy()).max(-1, keepdims=True)
    slip = 2.0 ** -18 * top * 128 * largest_key * abs(scale)
    bound = attention_bound(*want) + 2 * slip * weight
    off = np.abs(got.double().cpu().numpy() - out) / bound
    assert off.max(initial=0) <= 1, f"{what}: {off.max():.2f} times the bound at {np.unravel_index(off.argmax(), off.shape)}"
    rms = np.sqrt(np.mean((got.double().cpu().numpy() - out) ** 2) / np.mean(out ** 2))
    # one rounding to bf16, at most 2^-8 and half of that on average over a step of equal width
    assert rms < 2.0 ** -8, f"{what}: {rms:.2e} on average"


def key_size(cache):
    return float((cache[0].float().abs().amax(dim=-1).view(cache[2].shape[0], -1, 64, cache[2].shape[2]).amax(2) * cache[2]).max())


@pytest.mark.parametrize("host", (False, True))
@pytest.mark.parametrize("h, kvh, block, new, pre", [
    (2, 1, 128, [1], [0]), (8, 2, 128, [5, 1, 16], [100, 0, 130]), (32, 8, 256, [17, 70], [300, 4]), (16, 2, 128, [5] * 8, [100 * i for i in range(8)]),
    (10, 2, 256, [33, 129, 1], [0, 127, 128]), (7, 1, 512, [100], [700]), (12, 1, 128, [40, 3], [5, 250]), (9, 3, 384, [200], [500]),
    (64, 8, 128, [20], [1500]), (4, 4, 256, [300, 1, 260], [0, 600, 255]), (8, 1, 128, [3], [6000]), (16, 8, 128, [60], [3000]),
    (3, 1, 128, [129, 400], [1000, 2000])])
def test_against_64_bits(h, kvh, block, new, pre, host):
    import torch
    from nanovllm_jax_b200 import _lib, ops
    rng = np.random.default_rng(h * 1000 + len(new))
    q, tables, cu, cu_k, cu_host, nb, lens = make(rng, new, pre, h, kvh, block)
    cache = random_cache(rng, nb, block, kvh)
    scale = 1 / math.sqrt(128)
    out = torch.full_like(q, float("nan"))
    ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, max(new), scale, block, out=out, cu_seqlens_host=cu_host if host else None)
    assert _lib.device_status() == 0
    close(out, expect(q, cache, tables, new, lens, scale, block), q, scale, key_size(cache))
    again = ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, max(new), scale, block, cu_seqlens_host=cu_host if host else None)
    assert torch.equal(out, again)


def test_many_items_per_cta():
    """More token blocks than SMs, of one tile and of several: the rings run through many items."""
    import torch
    from nanovllm_jax_b200 import _lib, ops
    rng = np.random.default_rng(1)
    new = [int(x) for x in rng.integers(1, 60, 300)]
    pre = [int(x) * int(rng.integers(0, 2)) for x in rng.integers(0, 400, 300)]
    q, tables, cu, cu_k, _, nb, lens = make(rng, new, pre, 4, 2, 128)
    cache = random_cache(rng, nb, 128, 2)
    out = ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, 60, 0.09, 128)
    assert _lib.device_status() == 0
    close(out, expect(q, cache, tables, new, lens, 0.09, 128), q, 0.09, key_size(cache))


def test_against_the_bf16_kernel_over_the_same_values():
    """Long sequences, where the 64-bit statement would take minutes: against attention over the dequantised cache."""
    import torch
    from nanovllm_jax_b200 import _lib, ops
    rng = np.random.default_rng(2)
    for h, kvh, new, pre in ((32, 8, [1000, 300], [9000, 20000]), (8, 1, [2500], [0]), (40, 8, [700, 64], [3000, 100])):
        q, tables, cu, cu_k, _, nb, _ = make(rng, new, pre, h, kvh, 256)
        cache = random_cache(rng, nb, 256, kvh)
        wide = [(c.float() * s.repeat_interleave(64, 1)[..., None]).to(torch.bfloat16) for c, s in zip(cache[:2], cache[2:])]
        out = ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, max(new), 0.0884, 256).float()
        want = ops.paged_prefill(q, *wide, tables, cu, cu_k, max(new), 0.0884, 256).float()
        assert _lib.device_status() == 0
        # results of both are rounded to bf16, there the probabilities, too: 2^-8 at most each time, with weights that sum to 1
        assert ((out - want).norm() / want.norm()) < 2.0 ** -8 * math.sqrt(2)
        assert (out - want).abs().max() < 2.0 ** -6 * wide[1].float().abs().max()


@pytest.mark.parametrize("kv_scale, q_scale", [(2.0 ** -90, 1.0), (2.0 ** 80, 2.0 ** -80), (1.0, 2.0 ** 40), (2.0 ** -40, 2.0 ** -60)])
def test_magnitudes(kv_scale, q_scale):
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(3)
    new, pre = [30, 5], [200, 0]
    q, tables, cu, cu_k, _, nb, lens = make(rng, new, pre, 8, 2, 128)
    cache = random_cache(rng, nb, 128, 2)
    cache[2].mul_(kv_scale)
    cache[3].mul_(2.0 ** -20)
    cache[3][::3] *= 2.0 ** 30
    q.mul_(q_scale)
    q[3] = 0
    scale = 0.1 / (kv_scale * q_scale)
    out = ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, 30, scale, 128)
    close(out, expect(q, cache, tables, new, lens, scale, 128), q, scale, key_size(cache))


def test_rows_behind_the_keys_and_nan():
    """Any bytes and scales behind every sequence's end; a NaN query and a NaN value reach their own rows only; rows of the packed
    output behind the last sequence stay as they are."""
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(4)
    new, pre = [3, 40, 1], [0, 21, 64]
    q, tables, cu, cu_k, cu_host, nb, lens = make(rng, new, pre, 8, 2, 128, mb=5)
    cache = random_cache(rng, nb, 128, 2)
    clean = ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, 40, 0.09, 128)
    trash = random_cache(rng, nb, 128, 2, garbage=True)
    owned = torch.zeros((nb, 128), dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(n):
            owned[tables[b, t // 128], t % 128] = True
    for i in range(2):
        cache[i].view(torch.uint8).copy_(torch.where(owned[:, :, None, None].cuda(), cache[i].view(torch.uint8), trash[i].view(torch.uint8)))
        cache[2 + i].copy_(torch.where(owned.view(nb, 2, 64).any(-1)[:, :, None].cuda(), cache[2 + i], float("nan")))
    longer = torch.cat([q, torch.full((7, 8, 128), float("nan"), dtype=torch.bfloat16, device="cuda")])
    out = torch.full_like(longer, 7.0)
    ops.paged_prefill_q8(longer, *cache, tables, cu, cu_k, 40, 0.09, 128, out=out)
    assert torch.equal(out[:44], clean) and (out[44:] == 7).all()
    ops.paged_prefill_q8(longer, *cache, tables, cu, cu_k, 40, 0.09, 128, out=out, cu_seqlens_host=cu_host)
    assert torch.equal(out[:44], clean) and (out[44:] == 0).all()  # as paged_prefill: where the host knows the lengths
    q[5, 2, 9] = float("nan")
    q[6, 3, 1] = float("inf")
    out = ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, 40, 0.09, 128)
    assert out[5, 2].isnan().all() and out[6, 3].isnan().all()
    rest = torch.ones((44, 8), dtype=torch.bool)
    rest[5, 2] = rest[6, 3] = False
    assert torch.equal(out[rest], clean[rest])


def test_inconsistent_lengths_compute_nothing():
    import torch
    from nanovllm_jax_b200 import _lib, ops
    rng = np.random.default_rng(5)
    q, tables, cu, cu_k, _, nb, _ = make(rng, [5, 6], [10, 0], 4, 2, 128)
    cache = random_cache(rng, nb, 128, 2)
    out = torch.full_like(q, 3.0)
    ops.paged_prefill_q8(q, *cache, tables, cu, torch.tensor([0, 4, 10], dtype=torch.int32).cuda(), 6, 0.09, 128, out=out)
    assert (out == 3).all() and _lib.device_status() == 32
    _lib.device_status_reset()


def test_captured_and_replayed_with_other_lengths():
    import torch
    from nanovllm_jax_b200 import _lib, ops
    rng = np.random.default_rng(6)
    q, tables, cu, cu_k, _, nb, _ = make(rng, [40, 41, 19], [600, 500, 700], 8, 2, 128)
    cache = random_cache(rng, nb, 128, 2)
    out = torch.empty_like(q)
    call = lambda o=None: ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, 100, 0.09, 128, out=o)  # noqa: E731
    call(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for new, total in (([40, 41, 19], [640, 541, 719]), ([1, 98, 1], [1, 98, 700]), ([100, 0, 0], [640, 0, 0]), ([33, 33, 34], [33, 533, 34])):
        cu.copy_(torch.tensor([0, *np.cumsum(new)], dtype=torch.int32))
        cu_k.copy_(torch.tensor([0, *np.cumsum(total)], dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        assert _lib.device_status() == 0
        close(out, expect(q, cache, tables, new, total, 0.09, 128), q, 0.09, key_size(cache), str(new))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = call()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(again, out)


def test_refusals():
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(7)
    q, tables, cu, cu_k, _, nb, _ = make(rng, [5], [10], 4, 2, 128)
    cache = random_cache(rng, nb, 128, 2)
    ok = dict(q=q, k=cache[0], v=cache[1], ks=cache[2], vs=cache[3], t=tables, cu=cu, cu_k=cu_k, m=5, s=0.1, b=128)
    call = lambda **n: ops.paged_prefill_q8(*{**ok, **n}.values())  # noqa: E731
    call()
    for bad, error in ((dict(q=q.float()), TypeError), (dict(k=cache[0].view(torch.uint8)), TypeError), (dict(ks=cache[2][:1]), ValueError),
                       (dict(b=256), ValueError), (dict(cu_k=cu_k[:1]), ValueError), (dict(t=tables[:0]), ValueError), (dict(s=0.0), RuntimeError),
                       (dict(m=0), RuntimeError), (dict(q=q[:, :3].contiguous()), RuntimeError), (dict(cu=cu[:0]), ValueError)):
        with pytest.raises(error):
            call(**bad)
    small = random_cache(rng, 2, 64, 2)
    with pytest.raises(RuntimeError, match="multiple of 128"):
        call(k=small[0], v=small[1], ks=small[2], vs=small[3], b=64)


@pytest.mark.parametrize("exponents", [(-117, 0, 0), (0, -117, 0, -117, -117), (-60, 40, -117, 0, -30), (40, -117, -60)])
@pytest.mark.parametrize("pre", (0, 700, 6000))
def test_value_scales_far_apart(exponents, pre):
    """Blocks of zeros, whose scale is the least there is, between others; and values of any magnitude next to one another."""
    import torch
    from nanovllm_jax_b200 import _lib, ops
    rng = np.random.default_rng(pre + len(exponents))
    q, tables, cu, cu_k, _, nb, lens = make(rng, [200, 9], [pre, 3], 4, 1, 128)
    cache = random_cache(rng, nb, 128, 1)
    of = torch.tensor(exponents)
    for b in range(2):
        for i, page in enumerate(tables[b, :-(-lens[b] // 128)].tolist()):
            for half in range(2):
                e = int(of[(2 * i + half) % len(exponents)])
                cache[3][page, half] = 2.0 ** e
                if e == -117 and exponents[0] <= 0:
                    cache[1].view(torch.uint8)[page, 64 * half:64 * half + 64] = 0
    out = ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, 200, 0.09, 128)
    close(out, expect(q, cache, tables, [200, 9], lens, 0.09, 128), q, 0.09, key_size(cache))
    assert _lib.device_status() == 0


def test_nan_query_of_a_split_sequence():
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(9)
    q, tables, cu, cu_k, _, nb, _ = make(rng, [5], [6000], 8, 1, 128)
    cache = random_cache(rng, nb, 128, 1)
    clean = ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, 5, 0.09, 128)
    q[2, 3] = float("nan")
    out = ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, 5, 0.09, 128)
    assert out[2, 3].isnan().all()
    q[2, 3] = 0
    out[2, 3] = clean[2, 3]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("h, kvh, new, pre", [
    (8, 8, [1] * 10, [8000 - 64 * i for i in range(10)]),                # 80 items: one round, all of them in runs
    (8, 8, [1, 2, 130, 300] * 5, [5000, 4100, 2000, 129] * 5),           # a round and a few items, of unlike length
    (16, 2, [40] * 45, [1500 + 40 * (i % 20) for i in range(45)]),       # both tiles of the same keys; a round and most of another
    (3, 1, [12000], [300])])                                             # a long prompt: three tokens' heads in turn over the tiles
def test_last_round_in_runs(h, kvh, new, pre):
    """More items than half the SMs, in few rounds, with many keys each: against attention over the dequantised cache and, where it is
    quick, the 64-bit statement; the same bits when called again and when captured with other lengths."""
    import torch
    from nanovllm_jax_b200 import _lib, ops
    rng = np.random.default_rng(h + len(new))
    q, tables, cu, cu_k, cu_host, nb, lens = make(rng, new, pre, h, kvh, 256)
    cache = random_cache(rng, nb, 256, kvh)
    out = ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, max(new), 0.0884, 256)
    if sum(new) <= 20:
        close(out, expect(q, cache, tables, new, lens, 0.0884, 256), q, 0.0884, key_size(cache))
    wide = [(c.float() * s.repeat_interleave(64, 1)[..., None]).to(torch.bfloat16) for c, s in zip(cache[:2], cache[2:])]
    want = ops.paged_prefill(q, *wide, tables, cu, cu_k, max(new), 0.0884, 256).float()
    # as in test_against_the_bf16_kernel_over_the_same_values
    assert ((out.float() - want).norm() / want.norm()) < 2.0 ** -8 * math.sqrt(2)
    assert (out.float() - want).abs().max() < 2.0 ** -6 * wide[1].float().abs().max()
    for _ in range(5):
        assert torch.equal(out, ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, max(new), 0.0884, 256))
    # captured where every sequence has one new token, replayed with these: more items than the host could foresee, or fewer
    one = torch.arange(len(new) + 1, dtype=torch.int32).cuda()
    at, at_k, got = one.clone(), torch.cat([one[:1], (one[1:] * 0 + 2100).cumsum(0, dtype=torch.int32)]), torch.zeros_like(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_prefill_q8(q, *cache, tables, at, at_k, max(new), 0.0884, 256, out=got)
    at.copy_(cu), at_k.copy_(cu_k)
    graph.replay()
    assert ((got.float() - want).norm() / want.norm()) < 2.0 ** -8 * math.sqrt(2)
    assert _lib.device_status() == 0

"""paged_decode_q8 and decode_step_q8 against the 64-bit statement, and the attention layer's decode step over an 8-bit cache."""
import math

import numpy as np
import pytest

from cache8_helpers import assert_attention, random_cache, values_of
from oracle import cache8

pytestmark = pytest.mark.gpu


def make(rng, lens, h, kvh, block, mb=None, spare=2):
    """(q, tables, lens) on the device and the pool's size; the tables' unused entries are -1."""
    import torch
    need = [-(-n // block) for n in lens]
    nb = sum(need) + spare
    pages = rng.permutation(nb).astype(np.int32)
    tables = np.full((len(lens), mb or max(1, max(need, default=1))), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = pages[at:at + n]
        at += n
    q = torch.from_numpy(rng.normal(size=(len(lens), h, 128)).astype(np.float32)).to(torch.bfloat16).cuda()
    return q, torch.from_numpy(tables).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), nb


def expect(q, cache, tables, lens, scale, block):
    k, v = (cache8.dequantised(values_of(c), s.cpu().numpy()) for c, s in zip(cache[:2], cache[2:]))
    n = [min(max(int(x), 0), tables.shape[1] * block) for x in lens]
    return cache8.attention(q.double().cpu().numpy(), k, v, tables.cpu().numpy(), [1] * len(n), n, scale, block)


@pytest.mark.parametrize("h, kvh, block, lens", [
    (1, 1, 64, [1]), (16, 8, 256, [300]), (8, 8, 128, [1, 63, 64, 65, 127, 128, 129]), (10, 2, 64, [0, 1, 200, 0, 777]),
    (64, 8, 256, [5, 1030, 256]), (7, 1, 512, [513, 511]), (6, 2, 192, [191, 192, 193, 1000]), (12, 4, 256, [4000, 1]),
    (8, 1, 64, [20000]), (16, 2, 128, list(range(1, 70)))])
def test_decode(h, kvh, block, lens):
    import torch
    from nanovllm_jax_b200 import _lib, ops
    rng = np.random.default_rng(h * 100 + len(lens))
    q, tables, ctx, nb = make(rng, lens, h, kvh, block)
    cache = random_cache(rng, nb, block, kvh)
    out = torch.full_like(q, float("nan"))
    got = ops.paged_decode_q8(q, *cache, tables, ctx, 1 / math.sqrt(128), block, out=out)
    assert got is out
    assert_attention(out, expect(q, cache, tables, lens, 1 / math.sqrt(128), block))
    again = ops.paged_decode_q8(q, *cache, tables, ctx, 1 / math.sqrt(128), block)
    assert torch.equal(out, again) and _lib.device_status() == 0


def test_many_sequences_and_one_long_one():
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(1)
    lens = [int(x) for x in rng.integers(0, 90, 400)] + [9000]
    q, tables, ctx, nb = make(rng, lens, 4, 2, 64)
    cache = random_cache(rng, nb, 64, 2)
    out = ops.paged_decode_q8(q, *cache, tables, ctx, 0.1, 64)
    assert_attention(out, expect(q, cache, tables, lens, 0.1, 64))


@pytest.mark.parametrize("kv_scale, q_scale", [(2.0 ** -100, 1.0), (2.0 ** 90, 2.0 ** -90), (1.0, 2.0 ** 30), (1.0, 2.0 ** -60)])
def test_magnitudes_beyond_fp16(kv_scale, q_scale):
    """Keys, values and queries whose products, not they themselves, are of ordinary size; V scales 2^40 apart within a sequence."""
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(2)
    lens = [700, 64, 3]
    q, tables, ctx, nb = make(rng, lens, 8, 2, 64)
    cache = random_cache(rng, nb, 64, 2)
    cache[2].mul_(kv_scale)
    cache[3].mul_(2.0 ** -20)
    cache[3][::3] *= 2.0 ** 40
    q.mul_(q_scale)
    scale = 0.1 / (kv_scale * q_scale)
    out = ops.paged_decode_q8(q, *cache, tables, ctx, scale, 64)
    assert_attention(out, expect(q, cache, tables, lens, scale, 64))


def test_scores_far_apart():
    """Scores that rise along the sequence (the maximum moves at every tile), and a negative scale."""
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(3)
    lens = [1000, 640]
    q, tables, ctx, nb = make(rng, lens, 4, 1, 64)
    cache = random_cache(rng, nb, 64, 1)
    q.fill_(1.0)
    for b in range(2):
        for i, page in enumerate(tables[b].tolist()):
            if page >= 0:
                cache[0][page] = torch.full((64, 1, 128), 1.0, device="cuda").to(torch.float8_e4m3fn)
                cache[2][page] = float(i + 1)
    for scale in (0.3, -0.3, 3.0, 1e-6):
        out = ops.paged_decode_q8(q, *cache, tables, ctx, scale, 64)
        assert_attention(out, expect(q, cache, tables, lens, scale, 64), str(scale))


def test_rows_behind_the_context_may_hold_anything():
    """Any bytes, NaN among them, behind every sequence's end and in pages of nobody; wide tables; page ids out of the pool."""
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(4)
    lens = [1, 17, 64, 100, 0]
    q, tables, ctx, nb = make(rng, lens, 8, 2, 128, mb=7)
    cache = random_cache(rng, nb, 128, 2)
    clean = [c.clone() for c in cache]
    trash = random_cache(rng, nb, 128, 2, garbage=True)
    owned = torch.zeros((nb, 128), dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(n):
            owned[tables[b, t // 128], t % 128] = True
    grains = owned.view(nb, 2, 64).any(-1)
    for i in range(2):
        rows = owned[:, :, None, None].cuda()
        cache[i].view(torch.uint8).copy_(torch.where(rows, cache[i].view(torch.uint8), trash[i].view(torch.uint8)))
        cache[2 + i].copy_(torch.where(grains[:, :, None].cuda(), cache[2 + i], float("nan")))
    out = ops.paged_decode_q8(q, *cache, tables, ctx, 0.09, 128)
    assert torch.equal(out, ops.paged_decode_q8(q, *clean, tables, ctx, 0.09, 128))
    assert_attention(out, expect(q, clean, tables, lens, 0.09, 128))
    # a context beyond the table's width is cut, a negative one is empty, page ids are clamped
    ctx.copy_(torch.tensor([-5, 17, 64, 100000, 0]))
    tables.copy_(torch.tensor([[0] * 7, [nb + 9] * 7, [-3] * 7, list(range(7)), [1] * 7]))
    out = ops.paged_decode_q8(q, *clean, tables, ctx, 0.09, 128)
    assert_attention(out, expect(q, clean, tables, ctx.tolist(), 0.09, 128))


@pytest.mark.parametrize("f32", (False, True))
@pytest.mark.parametrize("batch, block", [(1, 64), (5, 128), (40, 256), (300, 64), (1100, 64), (4200, 64)])
def test_step_is_store_then_decode(batch, block, f32):
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(batch)
    lens = [int(x) for x in rng.integers(0 if batch > 1 else 1, 400 if batch < 100 else 90, batch)]
    q, tables, ctx, nb = make(rng, lens, 8, 2, block)
    slots = torch.tensor([-1 if n == 0 else int(tables[b, (n - 1) // block]) * block + (n - 1) % block for b, n in enumerate(lens)],
                         dtype=torch.int32).cuda()
    dtype = torch.float32 if f32 else torch.bfloat16
    k, v = (torch.from_numpy((rng.normal(size=(batch, 2, 128)) * 2.0 ** rng.integers(-3, 6, (batch, 1, 1))).astype(np.float32)).to(dtype).cuda() for _ in range(2))
    cache = random_cache(rng, nb, block, 2)
    other = [c.clone() for c in cache]
    ops.store_kvcache_q8(k, v, *other, slots)
    want = ops.paged_decode_q8(q, *other, tables, ctx, 0.09, block)
    got = ops.decode_step_q8(q, k, v, *cache, slots, tables, ctx, 0.09, block)
    assert torch.equal(got, want)
    for a, b in zip(cache, other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    if batch <= 40:
        assert_attention(got, expect(q, cache, tables, lens, 0.09, block))


def test_steps_in_a_row_and_replayed():
    """A conversation of 150 steps through a captured step, against eager calls on another stream."""
    import torch
    from nanovllm_jax_b200 import _lib, ops
    rng = np.random.default_rng(5)
    lens = [1, 60, 130]
    q, tables, ctx, nb = make(rng, [n + 150 for n in lens], 8, 2, 64)
    cache = random_cache(rng, nb, 64, 2)
    other = [c.clone() for c in cache]
    k, v = (torch.zeros((3, 2, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = torch.zeros(3, dtype=torch.int32, device="cuda")
    data = [torch.from_numpy(rng.normal(size=(150, 3, 2, 128)).astype(np.float32)).to(torch.bfloat16).cuda() for _ in range(2)]
    out = torch.empty_like(q)
    ctx.zero_()
    slots.fill_(-1)
    ops.decode_step_q8(q, k, v, *cache, slots, tables, ctx, 0.09, 64, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.decode_step_q8(q, k, v, *cache, slots, tables, ctx, 0.09, 64, out=out)
    side = torch.cuda.Stream()
    for i in range(150):
        n = [x + i for x in lens]
        at = [int(tables[b, (x - 1) // 64]) * 64 + (x - 1) % 64 for b, x in enumerate(n)]
        k.copy_(data[0][i]), v.copy_(data[1][i])
        slots.copy_(torch.tensor(at, dtype=torch.int32))
        ctx.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = ops.decode_step_q8(q, data[0][i], data[1][i], *other, slots.clone(), tables, ctx.clone(), 0.09, 64)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, want), i
    for a, b in zip(cache, other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert _lib.device_status() == 0


def test_nan_stays_in_its_sequence():
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(6)
    q, tables, ctx, nb = make(rng, [200, 200], 4, 1, 64)
    cache = random_cache(rng, nb, 64, 1)
    cache[0].view(torch.uint8)[tables[0, 1], 5, 0, 7] = 0x7F
    out = ops.paged_decode_q8(q, *cache, tables, ctx, 0.09, 64)
    assert out[0].isnan().all() and out[1].isfinite().all()


@pytest.mark.parametrize("n", (40, 9000))
def test_nan_query_and_nan_keys(n):
    """A head whose scores are all NaN gives NaN, in one run of keys or in many; so does a run whose keys all are."""
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(n)
    q, tables, ctx, nb = make(rng, [n, n], 4, 2, 64)
    cache = random_cache(rng, nb, 64, 2)
    clean = ops.paged_decode_q8(q, *cache, tables, ctx, 0.09, 64)
    q[0, 1] = float("nan")
    out = ops.paged_decode_q8(q, *cache, tables, ctx, 0.09, 64)
    assert out[0, 1].isnan().all()
    out[0, 1] = clean[0, 1]
    assert torch.equal(out, clean)
    q[0, 1] = 0
    pages = tables[1, :min(20, -(-n // 64))].long()
    cache[0].view(torch.uint8)[pages, :, 1] = 0x7F
    out = ops.paged_decode_q8(q, *cache, tables, ctx, 0.09, 64)
    assert out[1, 2:].isnan().all() and out[1, :2].isfinite().all() and out[0].isfinite().all()


def test_cache_beyond_4_gb():
    """Offsets of the last pages pass 32 bits: 5 GB of keys, 8 kv heads, a sequence in the first and the last pages."""
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(7)
    nb, block, kvh = 18000, 256, 8
    q, _, _, _ = make(rng, [600], 16, kvh, block)
    small = random_cache(rng, 4, block, kvh)
    cache = [torch.zeros((nb, *c.shape[1:]), dtype=c.dtype, device="cuda") for c in small]
    ids = [nb - 1, 0, nb - 2, 1]
    for c, s in zip(cache, small):
        c.view(torch.uint8)[ids] = s.view(torch.uint8) if c.dtype == torch.float8_e4m3fn else s.view(torch.uint8)
    k, v = (torch.from_numpy(rng.normal(size=(1, kvh, 128)).astype(np.float32)).to(torch.bfloat16).cuda() for _ in range(2))
    ctx = torch.tensor([900], dtype=torch.int32).cuda()
    slot = torch.tensor([899 % 256], dtype=torch.int32).cuda()
    got = ops.decode_step_q8(q, k, v, *cache, slot + 1 * block, torch.tensor([ids], dtype=torch.int32).cuda(), ctx, 0.09, block)
    want = ops.decode_step_q8(q, k, v, *small, slot + 3 * block, torch.arange(4, dtype=torch.int32).cuda()[None], ctx, 0.09, block)
    assert torch.equal(got, want)
    ops.store_kvcache_q8(k, v, *cache, torch.tensor([nb * block - 1], dtype=torch.int32).cuda())
    assert cache[0][nb - 1, block - 1].float().abs().max() > 0

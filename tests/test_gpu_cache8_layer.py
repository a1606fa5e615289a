"""The attention layer over an 8-bit cache, and the operators on it together as a serving loop uses them."""
import math

import numpy as np
import pytest

from cache8_helpers import assert_attention, values_of
from oracle import cache8

pytestmark = pytest.mark.gpu

H, KVH, BLOCK = 8, 2, 128
SCALE = 1 / math.sqrt(128)


def new_layer(nb):
    import torch
    from nanovllm_jax_b200.layers.attention import Attention
    attn = Attention(H, 128, SCALE, KVH, BLOCK)
    attn.set_kv_cache_q8(*(torch.zeros((nb, BLOCK, KVH, 128), device="cuda").to(torch.float8_e4m3fn) for _ in range(2)),
                         *(torch.zeros((nb, BLOCK // 64, KVH), device="cuda") for _ in range(2)))
    return attn


def caches(attn):
    return [attn.k_cache, attn.v_cache, attn.k_scale, attn.v_scale]


def rows(rng, t):
    import torch
    return [torch.from_numpy(rng.normal(size=(t, h, 128)).astype(np.float32)).to(torch.bfloat16).cuda() for h in (H, KVH, KVH)]


def slots_of(pages, lo, hi):
    return [pages[t // BLOCK] * BLOCK + t % BLOCK for t in range(lo, hi)]


def dev(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def expect(attn, q, tables, len_q, len_k):
    k, v = (cache8.dequantised(values_of(c), s.cpu().numpy()) for c, s in zip(caches(attn)[:2], caches(attn)[2:]))
    return cache8.attention(q.double().cpu().numpy(), k, v, tables, len_q, len_k, SCALE, BLOCK)


def decode(attn, rng, tables, lens):
    """A step that makes the sequences `lens` long."""
    from nanovllm_jax_b200.utils.context import create_decode_context
    q, k, v = rows(rng, len(lens))
    slots = [t[(n - 1) // BLOCK] * BLOCK + (n - 1) % BLOCK for t, n in zip(tables, lens)]
    out = attn(q, k, v, create_decode_context(dev(lens), dev(slots), dev(tables)))
    assert_attention(out, expect(attn, q, tables, [1] * len(lens), lens), f"step to {lens}")


def test_prompt_steps_prefix_fork_and_compaction():
    import torch
    from nanovllm_jax_b200 import _lib, ops
    from nanovllm_jax_b200.utils.context import create_prefill_context
    rng = np.random.default_rng(1)
    attn = new_layer(24)
    # two prompts: they attend to the rows that they bring
    pages = [[20, 3, 17, -1], [9, 22, -1, -1]]
    lens = [300, 130]
    q, k, v = rows(rng, 430)
    cu = dev([0, 300, 430])
    slots = slots_of(pages[0], 0, 300) + slots_of(pages[1], 0, 130)
    out = attn(q, k, v, create_prefill_context(cu, cu, 300, 300, dev(slots)))
    plain = ops.varlen_prefill(q, k, v, cu, 300, SCALE)
    assert torch.equal(out, plain)
    values, scales = cache8.store(k.double().cpu().numpy(), np.zeros((24 * BLOCK, KVH, 128)), np.zeros((24 * BLOCK // 64, KVH)), slots)
    assert np.array_equal(values_of(attn.k_cache).reshape(values.shape), values)
    assert np.array_equal(attn.k_scale.double().cpu().numpy().reshape(scales.shape), scales)
    # steps across the end of a page
    for _ in range(3):
        lens = [n + 1 for n in lens]
        decode(attn, rng, pages, lens)
    # a new question behind what is cached, in the last, partly filled page
    q, k, v = rows(rng, 60)
    new = [40, 20]
    slots = slots_of(pages[0], lens[0], lens[0] + 40) + slots_of(pages[1], lens[1], lens[1] + 20)
    total = [a + b for a, b in zip(lens, new)]
    context = create_prefill_context(dev([0, 40, 60]), dev([0, total[0], sum(total)]), 40, max(total), dev(slots), block_tables=dev(pages))
    out = attn(q, k, v, context)
    want = expect(attn, q, pages, new, total)
    off = np.abs(out.double().cpu().numpy() - want[0])
    assert np.sqrt((off ** 2).mean() / (want[0] ** 2).mean()) < 2.0 ** -8 * math.sqrt(2)
    lens = total
    # a fork of the first conversation: whole pages are shared, the last one is copied as far as it is filled
    child = [20, 3, 5, -1]
    ops.copy_pages(caches(attn), dev([17]), dev([5]), BLOCK, tokens=dev([lens[0] - 2 * BLOCK]))
    decode(attn, rng, [pages[0], pages[1], child], [lens[0] + 1, lens[1] + 1, lens[0] + 1])
    for c, s in zip(caches(attn)[:2], caches(attn)[2:]):  # what was copied is what the parent still holds
        n = lens[0] - 2 * BLOCK
        a, b = (cache8.dequantised(values_of(c[p:p + 1]), s[p:p + 1].cpu().numpy())[0, :n] for p in (17, 5))
        assert np.abs(a - b).max() <= 2.0 ** -4 * np.abs(a).max()  # either may have been rounded again by its own step
    lens = [lens[0] + 1, lens[1] + 1, lens[0] + 1]
    # a compaction: the pages in use go to the front, the tables follow
    tables = dev([pages[0], pages[1], child])
    used = sorted({p for t in (pages[0], pages[1], child) for p in t if p >= 0})
    free = [p for p in range(24) if p not in used]
    moves = [(s, d) for s, d in zip(reversed(used), free) if d < s]
    q = rows(rng, 3)[0]
    before = ops.paged_decode_q8(q, *caches(attn), tables, dev(lens), SCALE, BLOCK)
    ops.copy_pages(caches(attn), dev([s for s, _ in moves]), dev([d for _, d in moves]), BLOCK, block_tables=tables)
    for c in caches(attn):
        c[[s for s, _ in moves]] = torch.zeros_like(c[:len(moves)])
    assert torch.equal(before, ops.paged_decode_q8(q, *caches(attn), tables, dev(lens), SCALE, BLOCK))
    assert int(tables.max()) < len(used) + len([p for p in used if p < len(used)])
    # the pages are given to a new sequence: what they held counts no longer
    decode(attn, rng, tables.tolist(), [n + 1 for n in lens])
    fresh = [int(moves[0][0])]
    q, k, v = rows(rng, 1)
    attn.k_scale[fresh[0]] = 2.0 ** 60
    from nanovllm_jax_b200.utils.context import create_decode_context
    out = attn(q, k * 0.01, v, create_decode_context(dev([1]), dev([fresh[0] * BLOCK]), dev([fresh])))
    assert_attention(out, expect(attn, q, [fresh], [1], [1]))
    assert float(attn.k_scale[fresh[0], 0].max()) < 1
    assert _lib.device_status() == 0


def test_layer_takes_any_strides_and_types_and_both_caches():
    import torch
    from nanovllm_jax_b200.utils.context import create_decode_context
    rng = np.random.default_rng(2)
    attn = new_layer(4)
    q, k, v = rows(rng, 3)
    ctx = create_decode_context(dev([1, 1, 1]), dev([0, BLOCK, 2 * BLOCK]), dev([[0], [1], [2]]))
    want = attn(q, k, v, ctx)
    other = [x.float().repeat_interleave(2, -1)[..., ::2] for x in (q, k, v)]
    assert not other[0].is_contiguous()
    assert torch.equal(attn(*other, ctx), want)
    held = caches(attn)
    attn.set_kv_cache(*(torch.zeros((4, BLOCK, KVH, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    wide = attn(q, k, v, ctx)  # one key: the value itself
    assert torch.equal(wide, v.repeat_interleave(H // KVH, 1))
    attn.set_kv_cache_q8(*held)
    assert torch.equal(attn(q, k, v, ctx), want)
    assert (want - wide).abs().max() <= 2.0 ** -4 * wide.abs().max()


def test_prompt_without_a_cache_entry_and_padded_rows():
    """Rows of no slot in a prompt and a padded decode batch leave the cache alone."""
    import torch
    from nanovllm_jax_b200.utils.context import create_decode_context
    rng = np.random.default_rng(3)
    attn = new_layer(3)
    q, k, v = rows(rng, 4)
    ctx = create_decode_context(dev([1, 0, 0, 0]), dev([64, -1, -1, -1]), dev([[0, -1], [-1, -1], [-1, -1], [-1, -1]]))
    before = [c.clone() for c in caches(attn)]
    attn.k_cache.view(torch.uint8)[0, 0] = 8
    attn.k_scale[0, 0] = 1.0
    before[0].view(torch.uint8)[0, 0] = 8
    out = attn(q, k, v, ctx)
    assert (out[1:] == 0).all() and out[0].isfinite().all()
    changed = (attn.k_cache.view(torch.uint8) != before[0].view(torch.uint8)).nonzero()[:, :2].unique(dim=0).tolist()
    assert changed == [[0, 64]]

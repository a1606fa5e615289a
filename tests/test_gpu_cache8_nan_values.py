"""NaN in the 8-bit cache at tokens that count (the store writes one for every NaN or infinity it is given): a row of a prefill gets
NaN exactly where the formula has it, and the tokens in front of it keep their bits."""
import numpy as np
import pytest

from cache8_helpers import random_cache
from test_gpu_cache8_prefill import make

pytestmark = pytest.mark.gpu

# (h, kvh, block, new, pre): every way of packing heads and tokens into tiles, items whole, cut into runs, and a last round in runs
CASES = [
    (8, 2, 128, [3, 40, 1], [0, 21, 64]),
    (4, 4, 256, [300, 1, 260], [0, 600, 255]),
    (3, 1, 128, [129, 400], [1000, 2000]),
    (7, 1, 512, [100, 37], [700, 1]),
    (64, 8, 128, [20, 150], [1500, 90]),
    (16, 2, 128, [5] * 8, [100 * i for i in range(8)]),
    (8, 1, 128, [90], [6000]),
    (8, 8, 256, [1, 2, 130, 300] * 5, [5000, 4100, 2000, 129] * 5),
    (4, 2, 128, [17] * 300, [60] * 300),
]


def poison(rng, cache, tables, new, pre, block, which, how_many):
    """NaN codes at a few live places of `which` (0: K, 1: V); returns [(sequence, position, kv head, dims)]."""
    import torch
    codes = cache[which].view(torch.uint8)
    host = tables.cpu().numpy()
    put = []
    for b in rng.permutation(len(new))[:how_many]:
        for where in ("new", "any"):
            lo, hi = (pre[b], pre[b] + new[b]) if where == "new" else (0, pre[b] + new[b])
            at, head = int(rng.integers(lo, hi)), int(rng.integers(0, codes.shape[2]))
            dims = np.arange(128) if rng.random() < 0.3 else rng.choice(128, 5, replace=False)
            page = int(host[b, at // block])
            for d in dims:
                codes[page, at % block, head, int(d)] = 0x7f if d % 2 else 0xff
            put.append((int(b), at, head, dims))
    return put


@pytest.mark.parametrize("h, kvh, block, new, pre", CASES)
def test_nan_values_reach_the_rows_that_see_them(h, kvh, block, new, pre):
    import torch
    from nanovllm_jax_b200 import _lib, ops
    rng = np.random.default_rng(h * 100 + len(new))
    q, tables, cu, cu_k, cu_host, nb, _ = make(rng, new, pre, h, kvh, block)
    cache = random_cache(rng, nb, block, kvh)
    call = lambda **more: ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, max(new), 0.0884, block, **more)  # noqa: E731
    forms = ({}, {"cu_seqlens_host": cu_host})  # what the host knows may change how items are cut, and with it the bits
    clean = [call(**more) for more in forms]
    put = poison(rng, cache, tables, new, pre, block, 1, 4)
    odd = torch.zeros(q.shape, dtype=torch.bool)
    for b, at, head, dims in put:
        first = int(cu_host[b]) + max(0, at - pre[b])  # the first new token that sees it
        rows = odd[first:int(cu_host[b + 1]), head * (h // kvh):(head + 1) * (h // kvh)]
        rows[..., torch.from_numpy(np.sort(dims))] = True
    odd = odd.cuda()
    for more, without in zip(forms, clean):
        out = call(**more)
        assert torch.equal(out.isnan(), odd), f"{int((out.isnan() ^ odd).sum())} of {odd.numel()} elements"
        assert torch.equal(out[~odd], without[~odd])
    assert _lib.device_status() == 0


@pytest.mark.parametrize("h, kvh, block, new, pre", CASES[:7])
def test_nan_keys_reach_the_rows_that_see_them(h, kvh, block, new, pre):
    import torch
    from nanovllm_jax_b200 import _lib, ops
    rng = np.random.default_rng(h * 100 + len(new) + 1)
    q, tables, cu, cu_k, cu_host, nb, _ = make(rng, new, pre, h, kvh, block)
    cache = random_cache(rng, nb, block, kvh)
    clean = ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, max(new), 0.0884, block)
    put = poison(rng, cache, tables, new, pre, block, 0, 2)
    odd = torch.zeros(clean.shape[:2], dtype=torch.bool)
    for b, at, head, _ in put:
        odd[int(cu_host[b]) + max(0, at - pre[b]):int(cu_host[b + 1]), head * (h // kvh):(head + 1) * (h // kvh)] = True
    out = ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, max(new), 0.0884, block)
    odd = odd.cuda()
    assert torch.equal(out.isnan().all(-1), odd) and torch.equal(out.isnan().any(-1), odd)
    # A key that counts for nothing may change when a neighbouring row's maximum moves, and with it the bits: both results are within
    # 2^-8 |out| + 2^-9 max |v| of the exact one (half a step of bf16 and of the fp16 probabilities, twice).
    most = (cache[1].float().abs().amax(dim=(1, 3)) * cache[3].amax(dim=1)).max()
    off = (out.float() - clean.float())[~odd].abs()
    assert (off <= 2 * (2.0 ** -8 * clean.float()[~odd].abs() + 2.0 ** -9 * most)).all()
    assert _lib.device_status() == 0


def test_stored_infinities_do_not_reach_earlier_tokens():
    """Through the store: a chunk whose last token holds an infinity and a NaN, behind a cached prefix."""
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(5)
    new, pre = [50], [300]
    q, tables, cu, cu_k, _, nb, _ = make(rng, new, pre, 8, 2, 128)
    cache = random_cache(rng, nb, 128, 2)
    k, v = (torch.from_numpy(rng.normal(size=(50, 2, 128)).astype(np.float32)).to(torch.bfloat16).cuda() for _ in range(2))
    at = torch.arange(300, 350)
    slots = (tables[0].cpu()[at // 128] * 128 + at % 128).to(torch.int32).cuda()
    for last in (0.0, float("inf")):
        v[49, 0, 7], v[49, 1, 9] = last, last
        ops.store_kvcache_q8(k, v, *cache, slots)
        out = ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, 50, 0.0884, 128)
        assert out[:49].isfinite().all()
    assert out[49, :4, 7].isnan().all() and out[49, 4:, 9].isnan().all() and int(out.isnan().sum()) == 8


@pytest.mark.parametrize("h, kvh, new, pre", [(32, 8, 2048, 700), (3, 1, 700, 5000), (8, 1, 40, 9000)])
def test_values_of_nothing_but_nan(h, kvh, new, pre):
    """Every row has to look for its own in every tile that it shares: no wait runs out meanwhile."""
    import torch
    from nanovllm_jax_b200 import _lib, ops
    rng = np.random.default_rng(h)
    q, tables, cu, cu_k, _, nb, _ = make(rng, [new], [pre], h, kvh, 128)
    cache = random_cache(rng, nb, 128, kvh)
    cache[1].view(torch.uint8)[:, :, 0] = 0x7f
    out = ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, new, 0.0884, 128)
    assert out[:, :h // kvh].isnan().all() and out[:, h // kvh:].isfinite().all()
    assert _lib.device_status() == 0

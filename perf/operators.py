"""The operators on a cache held in 8 bits and on its pages: what their speed and their results are judged by.

  store   ``store_kvcache_q8``: a step's K/V rows into the 8-bit cache, a scale for every 64 slots and kv head
  decode  ``paged_decode_q8``: one query token per sequence over the pages of the 8-bit cache
  step    ``decode_step_q8``: both in one call, as the attention layer's decode step makes them
  prefix  ``paged_prefill_q8``: the new tokens of a batch over their whole sequences in the 8-bit cache
  copy    ``copy_pages``: pages of many caches copied (a fork) or moved with their block tables (a compaction)

The cache's format: e4m3 values [pages, page size, kv heads, 128] and fp32 scales [pages, page size / 64, kv heads]; an
element stands for value * scale.  The store takes as scale the smallest power of two under which the block's largest
finite magnitude is at most 448; a block whose first slot is written begins anew, another one's scale only grows, and
when it does the rows that the block holds already are rounded again.

Where ``own`` is false ``run`` computes this with elementary torch operations in 32 bits.

Sequence lengths are the evenly spaced quantiles of the stated range, so that a case has the same work whatever the seed;
the seed shuffles them over the batch, deals the pages and draws every tensor.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

D = 128
GRAIN = 64  # slots of a scale
DEVICE = "cuda"
E4M3 = torch.float8_e4m3fn
TOP = 448.0  # largest e4m3 value


def _case(name, kind, **more):
    return {"name": name, "kind": kind, **more}


def listed():
    return [
        # a decode step's new rows, 64 conversations on 8 kv heads: a few microseconds, the call's latency counts
        _case("store-append-b64-kvh8", "store", form="append", batch=64, lo=512, hi=8192, kv_heads=8, block=256, kv="bf16",
              padding=0),
        # the rows of a prefill batch: 16 prompts of 128 to 4096 tokens, 8 kv heads
        _case("store-16-prompts-kvh8", "store", form="prompts", batch=16, lo=128, hi=4096, kv_heads=8, block=256, kv="bf16",
              padding=0),
        # a burst of short prompts in fp32 on a shard, small pages, the batch padded with rows of no slot
        _case("store-48-short-f32-kvh2", "store", form="prompts", batch=48, lo=5, hi=300, kv_heads=2, block=64, kv="f32",
              padding=37),
        # one user's chat on a small model (16 / 8 heads): the shortest attention call there is
        _case("decode-b1-h16", "decode", batch=1, heads=16, kv_heads=8, lo=300, hi=300, log=False, block=256, empty=0),
        # 64 conversations of 512 to 8192 tokens, 32 / 8 heads
        _case("decode-b64-h32", "decode", batch=64, heads=32, kv_heads=8, lo=512, hi=8192, log=False, block=256, empty=0),
        # 256 sequences of very different lengths, 64 / 8 heads
        _case("decode-b256-h64-skewed", "decode", batch=256, heads=64, kv_heads=8, lo=16, hi=16384, log=True, block=256, empty=0),
        # a whole decode step on a shard with an odd number of query heads per kv head, small pages, padded rows
        _case("step-b24-h10", "step", batch=24, heads=10, kv_heads=2, lo=1, hi=2000, log=False, block=64, empty=3, kv="f32"),
        # five drafted tokens of eight conversations to be looked at, 16 / 2 heads
        _case("prefix-8x5-h16", "prefix", batch=8, heads=16, kv_heads=2, lo=5, hi=5, pre_lo=100, pre_hi=3000, block=128,
              host=True),
        # new questions behind cached conversations, 32 / 8 heads
        _case("prefix-12-h32", "prefix", batch=12, heads=32, kv_heads=8, lo=17, hi=700, pre_lo=500, pre_hi=5000, block=256,
              host=True),
        # a chunk of a long document behind what is in the cache already, lengths on the device only
        _case("prefix-1x2048-h32", "prefix", batch=1, heads=32, kv_heads=8, lo=2048, hi=2048, pre_lo=16384, pre_hi=16384,
              block=256, host=False),
        # a conversation forked into four: its last, partly filled page in every layer of an 8-bit cache
        _case("copy-fork-4-36-layers", "copy", form="fork", held="8 bits", layers=36, pairs=4, kv_heads=8, block=256, pool=24,
              batch=8),
        # pages moved to the front of the pool, K and V of four bf16 layers, and every table that names one of them
        _case("copy-compact-96-4-layers", "copy", form="compact", held="bf16", layers=4, pairs=96, kv_heads=8, block=256,
              pool=256, batch=64),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("store", "store", "decode", "decode", "step", "prefix", "prefix", "copy"))
    kv_heads = rng.choice((1, 2, 4, 8, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 4, 5, 7, 8, 8))
    if kind == "store":
        c = {"kind": kind, "form": rng.choice(("append", "prompts")), "kv_heads": kv_heads,
             "block": rng.choice((64, 128, 256, 256, 512)), "kv": rng.choice(("bf16", "bf16", "f32")),
             "padding": rng.choice((0, 0, rng.randint(1, 40)))}
        c["batch"] = _log_int(rng, 1, 256 if c["form"] == "append" else 48)
        c["hi"] = _log_int(rng, 2, 16384 if c["form"] == "append" else min(8192, 32768 // c["batch"]))
        c["lo"] = _log_int(rng, 1, c["hi"])
        return c
    if kind in ("decode", "step"):
        batch = _log_int(rng, 1, 256)
        # the padded keys of the plain form stay below 17 GB, the live rows below those of the largest listed case
        most = min(16384, 4194304 * 8 // (batch * kv_heads))
        c = {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "hi": _log_int(rng, 2, most),
             "log": rng.random() < 0.5, "block": rng.choice((64, 128, 256, 256, 512)), "empty": rng.choice((0, 0, rng.randint(1, 9)))}
        c["lo"] = _log_int(rng, 1, c["hi"])
        if kind == "step":
            c["kv"] = rng.choice(("bf16", "bf16", "f32"))
        while work(c)["bytes"] > 1.1e9:
            c["hi"] = max(2, c["hi"] // 2)
            c["lo"] = min(c["lo"], c["hi"])
        return c
    if kind == "prefix":
        c = {"kind": kind, "batch": _log_int(rng, 1, 32), "heads": heads, "kv_heads": kv_heads,
             "block": rng.choice((128, 256, 256, 512)), "host": rng.random() < 0.7}
        c["hi"] = _log_int(rng, 1, 2048)
        c["lo"] = _log_int(rng, 1, c["hi"])
        c["pre_hi"] = _log_int(rng, 1, 16384)
        c["pre_lo"] = rng.randint(0, c["pre_hi"])
        # operations of the largest listed case, and the plain form's scores below 8 GB
        while work(c)["flops"] > 5.0e11 or c["batch"] * c["heads"] * c["hi"] * (c["hi"] + c["pre_hi"]) > 2.0e9:
            c["batch"], c["pre_hi"] = max(1, c["batch"] // 2), max(1, c["pre_hi"] * 3 // 4)
            c["pre_lo"] = min(c["pre_lo"], c["pre_hi"])
        return c
    c = {"kind": kind, "form": rng.choice(("fork", "compact")), "held": rng.choice(("8 bits", "bf16")),
         "layers": _log_int(rng, 1, 36), "kv_heads": kv_heads, "block": rng.choice((64, 128, 256, 512)), "batch": _log_int(rng, 1, 64)}
    row = 2 * kv_heads * D * (1 if c["held"] == "8 bits" else 2) * c["layers"] * c["block"]  # bytes of a page in all caches
    c["pairs"] = _log_int(rng, 1, max(1, min(96, int(4.0e8 / row))))
    c["pool"] = 2 * c["pairs"] + rng.randint(4, 40)
    return c


# ---- lengths, pages, tensors ---------------------------------------------------------------------------------------


def _lengths(n, lo, hi, log=False):
    at = (np.arange(n) + 0.5) / n
    x = np.exp(math.log(lo) + at * (math.log(hi) - math.log(lo))) if log else lo + at * (hi - lo)
    return np.clip(np.rint(x), lo, hi).astype(np.int64)


def _pages(rng, lens, block):
    """(page ids per sequence, padded block tables, pool): pages dealt at random from a pool with an eighth more."""
    need = -(-lens // block)
    pool = int(need.sum() + need.sum() // 8 + 2)
    perm = rng.permutation(pool).astype(np.int32)
    cut = np.concatenate([[0], np.cumsum(need)])
    lists = [perm[cut[i]:cut[i + 1]] for i in range(len(lens))]
    tables = np.full((len(lens), max(1, int(need.max()))), -1, np.int32)
    for i, ids in enumerate(lists):
        tables[i, :len(ids)] = ids
    return lists, tables, pool


def _slots(lists, first, last, block):
    """Cache slots of tokens first[b] .. last[b] - 1 of every sequence, packed."""
    parts = [np.zeros(0, np.int64)]
    for ids, a, z in zip(lists, first, last):
        tok = np.arange(a, z)
        parts.append(np.asarray(ids, np.int64)[tok // block] * block + tok % block)
    return np.concatenate(parts).astype(np.int32)


def _dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEVICE)


def _normal(gen, shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)


def _kv_dtype(case):
    return torch.float32 if case["kv"] == "f32" else torch.bfloat16


def _held(gen, pool, block, kvh):
    """A cache of rows behind a norm in 8 bits: N(0, 1), every head and block with a magnitude of its own."""
    size = torch.exp2(_normal(gen, (1, 1, kvh), torch.float32) * 0.5 + _normal(gen, (pool, block // GRAIN, kvh), torch.float32) * 0.3)
    x = _normal(gen, (pool, block // GRAIN, GRAIN, kvh, D)) * size[:, :, None, :, None].to(torch.bfloat16)
    scale = _scale_of(x.abs().amax(dim=(2, 4)).float())
    values = (x / scale[:, :, None, :, None].to(torch.bfloat16)).to(E4M3)  # a division by a power of two: the same in bf16
    return values.reshape(pool, block, kvh, D), scale


def prepare(case, seed):
    rng = np.random.Generator(np.random.PCG64(seed))
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    kind, kvh, block = case["kind"], case["kv_heads"], case["block"]
    s = {"kind": kind, "block": block, "scale": 1.0 / math.sqrt(D)}
    if kind == "copy":
        layers, pool, n = case["layers"], case["pool"], case["pairs"]
        s["form"] = case["form"]
        if case["held"] == "8 bits":
            held = [_held(gen, pool * layers, block, kvh) for _ in range(2)]
            s["caches"] = [x.reshape(layers, pool, *x.shape[1:]) for pair in held for x in pair]
        else:
            s["caches"] = [_normal(gen, (layers, pool, block, kvh, D)) for _ in range(2)]
        s["each"] = [x for c in s["caches"] for x in c.unbind(0)]
        pages = rng.permutation(pool).astype(np.int32)
        if case["form"] == "fork":  # few pages, each copied to several
            parents = pages[:max(1, n // 4)]
            s["src"], s["dst"] = _dev(parents[np.arange(n) % len(parents)]), _dev(pages[len(parents):len(parents) + n])
            s["tokens"] = _dev(rng.permutation(_lengths(n, 1, block)).astype(np.int32))
            s["tables"] = None
        else:  # pages at the end of the pool to free ones at its front
            s["src"], s["dst"] = _dev(rng.permutation(np.arange(pool - n, pool)).astype(np.int32)), _dev(rng.permutation(n).astype(np.int32))
            s["tokens"] = None
            tables = rng.integers(n, pool, (case["batch"], 32)).astype(np.int32)
            tables[np.arange(32)[None, :] >= rng.integers(0, 33, (case["batch"], 1))] = -1
            s["tables"] = _dev(tables)
        return s

    if kind == "store":
        lens = rng.permutation(_lengths(case["batch"], case["lo"], case["hi"]))
        if case["form"] == "append":  # a token per sequence, in its newest page (the older ones are elsewhere)
            lens = (lens - 1) % block + 1
        lists, _, pool = _pages(rng, lens, block)
        slots = _slots(lists, lens - 1 if case["form"] == "append" else 0 * lens, lens, block)
        if case["padding"]:
            slots = np.concatenate([slots, np.full(case["padding"], -1, np.int32)])
        s["slots"] = _dev(slots)
        s["k"], s["v"] = (_normal(gen, (len(slots), kvh, D), _kv_dtype(case)) for _ in range(2))
        (s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"]) = (_held(gen, pool, block, kvh) for _ in range(2))
        return s

    batch, h = case["batch"], case["heads"]
    if kind == "prefix":
        new = rng.permutation(_lengths(batch, case["lo"], case["hi"]))
        pre = rng.permutation(_lengths(batch, case["pre_lo"], case["pre_hi"]))
        lens = pre + new
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        s["cu_q"], s["cu_k"] = _dev(cu), _dev(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
        s["cu_host"], s["max_q"] = (cu if case["host"] else None), int(new.max())
        s["q"] = _normal(gen, (int(cu[-1]), h, D))
        # for the plain form: where a packed row belongs
        s["row_seq"], s["row_at"] = _dev(np.repeat(np.arange(batch), new)), _dev(np.concatenate([np.arange(x) for x in new]))
    else:
        lens = rng.permutation(np.concatenate([_lengths(batch, case["lo"], case["hi"], case["log"]), np.zeros(case["empty"], np.int64)]))
        s["q"] = _normal(gen, (len(lens), h, D))
    lists, tables, pool = _pages(rng, lens, block)
    (s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"]) = (_held(gen, pool, block, kvh) for _ in range(2))
    s["tables"], s["lens"] = _dev(tables), _dev(lens.astype(np.int32))
    if kind == "step":
        slots = np.full(len(lens), -1, np.int32)
        live = np.nonzero(lens)[0]
        slots[live] = _slots([lists[i] for i in live], lens[live] - 1, lens[live], block)
        s["slots"] = _dev(slots)
        s["k"], s["v"] = (_normal(gen, (len(lens), kvh, D), _kv_dtype(case)) for _ in range(2))
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _scale_of(amax):
    """The smallest power of two s with amax <= 448 s (448 = 0.875 * 2^9), its exponent within -117 .. 119."""
    part, exponent = torch.frexp(amax)
    e = exponent - 9 + (part > 0.875).to(exponent.dtype)
    e = torch.where(amax > 0, e, e - 1000).clamp(-117, 119)
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _to_e4m3(x):
    return x.clamp(-TOP, TOP).to(E4M3)


def _store(rows, cache, scale, slots):
    """The rows into the cache, in place."""
    kvh = rows.shape[1]
    grains = cache.view(-1, GRAIN, kvh, D)
    flat_scale = scale.view(-1, kvh)
    n = grains.shape[0]
    x = rows.float()
    live = slots >= 0
    at = torch.where(live, slots, n * GRAIN).long()  # rows of no slot go to a place behind the cache
    grain = at // GRAIN
    finite = torch.where(x.isfinite(), x.abs(), torch.zeros((), device=x.device)).amax(dim=-1)
    amax = torch.zeros((n + 1, kvh), device=x.device).scatter_reduce(0, grain[:, None].expand(-1, kvh), finite, "amax")[:n]
    written = torch.zeros((n + 1) * GRAIN, dtype=torch.bool, device=x.device).index_fill(0, at, True)[:n * GRAIN].view(n, GRAIN)
    touched, begins = written.any(dim=1, keepdim=True), written[:, :1]
    old = torch.where(begins, torch.zeros_like(flat_scale), flat_scale)
    new = torch.where(touched, torch.maximum(old, _scale_of(amax)), flat_scale)
    again = (new > old) & (old > 0) & touched  # rows that are in the block already are rounded again
    ratio = torch.where(again, old / new, torch.ones_like(new))
    values = torch.where(again[:, None, :, None] & ~written[:, :, None, None], grains.float() * ratio[:, None, :, None], grains.float())
    values = torch.cat([values.reshape(n * GRAIN, kvh, D), values.new_zeros((1, kvh, D))])
    per_row = torch.cat([new, new.new_ones((1, kvh))])[grain.clamp(max=n)]
    values[at.clamp(max=n * GRAIN)] = x / per_row[:, :, None]
    cache.view(-1, kvh, D).copy_(_to_e4m3(values[:n * GRAIN]))
    flat_scale.copy_(new)


def _gathered(cache, scale, tables):
    """Keys or values of every sequence in 32 bits, [batch, kv heads, tokens of the widest table, 128]."""
    kvh = cache.shape[2]
    page = tables.clamp(min=0).long()
    x = cache.view(torch.uint8)[page].view(E4M3).float()  # [batch, pages, page size, kv heads, 128]
    x = x.view(*x.shape[:2], -1, GRAIN, kvh, D) * scale[page][:, :, :, None, :, None]
    return x.reshape(tables.shape[0], -1, kvh, D).transpose(1, 2)


def _attend(q, k, v, seen, scale):
    """q [batch, kv heads, rows, 128], k and v [batch, kv heads, tokens, 128], seen [batch, 1, rows, tokens]."""
    w = q.float() @ k.transpose(2, 3) * scale
    w = w.masked_fill(~seen, -math.inf)
    top = w.amax(dim=-1, keepdim=True)
    w = torch.exp(w - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = w.sum(dim=-1, keepdim=True)
    return (w @ v) / torch.where(total > 0, total, torch.ones_like(total))


def _decode(s):
    b, h, _ = s["q"].shape
    kvh = s["k_cache"].shape[2]
    k, v = (_gathered(s[x + "_cache"], s[x + "_scale"], s["tables"]) for x in ("k", "v"))
    seen = torch.arange(k.shape[2], device=k.device)[None, None, None, :] < s["lens"][:, None, None, None]
    out = _attend(s["q"].view(b, kvh, h // kvh, D), k, v, seen, s["scale"])
    return out.reshape(b, h, D).to(torch.bfloat16)


def _prefix(s):
    t, h, _ = s["q"].shape
    kvh, g = s["k_cache"].shape[2], h // s["k_cache"].shape[2]
    b, rows = s["tables"].shape[0], s["max_q"]
    k, v = (_gathered(s[x + "_cache"], s[x + "_scale"], s["tables"]) for x in ("k", "v"))
    q = torch.zeros((b, rows, kvh, g, D), device=k.device)
    q[s["row_seq"], s["row_at"]] = s["q"].view(t, kvh, g, D).float()
    new = (s["cu_q"][1:] - s["cu_q"][:-1])[:, None]
    last = s["lens"][:, None] - new + torch.arange(rows, device=k.device)[None, :]  # position of a row's token
    seen = torch.arange(k.shape[2], device=k.device)[None, None, :] <= torch.where(
        torch.arange(rows, device=k.device)[None, :] < new, last, -torch.ones_like(last))[:, :, None]
    seen = seen[:, None].repeat_interleave(g, dim=2)
    out = _attend(q.permute(0, 2, 1, 3, 4).reshape(b, kvh, rows * g, D), k, v, seen, s["scale"])
    out = out.view(b, kvh, rows, g, D).permute(0, 2, 1, 3, 4)
    return out[s["row_seq"], s["row_at"]].reshape(t, h, D).to(torch.bfloat16)


def _copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for cache in s["caches"]:
        c = cache.view(torch.uint8) if cache.dtype == E4M3 else cache
        rows = c[:, src]
        if s["tokens"] is not None:
            per = s["block"] // c.shape[2]  # tokens of a row of this cache
            live = torch.arange(c.shape[2], device=c.device)[None, :] * per < s["tokens"][:, None]
            rows = torch.where(live.view(1, *live.shape, *([1] * (c.dim() - 3))), rows, c[:, dst])
        c[:, dst] = rows
    if s["tables"] is not None:
        to = torch.arange(s["caches"][0].shape[1], device=src.device, dtype=torch.int32)
        to[src] = s["dst"]
        s["tables"].copy_(torch.where(s["tables"] >= 0, to[s["tables"].clamp(min=0).long()], s["tables"]))


# ---- one pass ------------------------------------------------------------------------------------------------------


def run(s):
    kind = s["kind"]
    if own:
        from nanovllm_jax_b200 import ops
        cache = [s.get(x) for x in ("k_cache", "v_cache", "k_scale", "v_scale")]
        if kind == "store":
            ops.store_kvcache_q8(s["k"], s["v"], *cache, s["slots"])
        elif kind == "decode":
            out = ops.paged_decode_q8(s["q"], *cache, s["tables"], s["lens"], s["scale"], s["block"])
        elif kind == "step":
            out = ops.decode_step_q8(s["q"], s["k"], s["v"], *cache, s["slots"], s["tables"], s["lens"], s["scale"], s["block"])
        elif kind == "prefix":
            out = ops.paged_prefill_q8(s["q"], *cache, s["tables"], s["cu_q"], s["cu_k"], s["max_q"], s["scale"], s["block"],
                                       cu_seqlens_host=s["cu_host"])
        else:
            ops.copy_pages(s["each"], s["src"], s["dst"], s["block"], tokens=s["tokens"], block_tables=s["tables"])
    else:
        if kind in ("store", "step"):
            _store(s["k"], s["k_cache"], s["k_scale"], s["slots"])
            _store(s["v"], s["v_cache"], s["v_scale"], s["slots"])
        if kind in ("decode", "step"):
            out = _decode(s)
        elif kind == "prefix":
            out = _prefix(s)
        elif kind == "copy":
            _copy(s)
    if kind == "copy":
        return {"caches": s["caches"], "tables": s["tables"]}
    if kind in ("decode", "prefix"):
        return {"out": out}
    held = {x: s[x] for x in ("k_cache", "v_cache", "k_scale", "v_scale")}
    return held if kind == "store" else {"out": out, **held}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    kind, kvh, block = case["kind"], case["kv_heads"], case["block"]
    if kind == "copy":  # bytes copied, in and out
        tokens = int(_lengths(case["pairs"], 1, block).sum()) if case["form"] == "fork" else case["pairs"] * block
        row = kvh * D * (1 if case["held"] == "8 bits" else 2) + (kvh * 4 / GRAIN if case["held"] == "8 bits" else 0)
        tables = 0 if case["form"] == "fork" else case["batch"] * 32 * 4
        return {"bytes": int(2 * 2 * case["layers"] * tokens * row) + 8 * case["pairs"] + 2 * tables, "flops": 0}
    src = 4 if case.get("kv") == "f32" else 2
    if kind == "store":  # rows in and out, the slots, a scale in and out for every block
        lens = _lengths(case["batch"], case["lo"], case["hi"])
        t = case["batch"] if case["form"] == "append" else int(lens.sum())
        grains = case["batch"] if case["form"] == "append" else int((-(-lens // GRAIN)).sum())
        return {"bytes": t * 2 * kvh * D * (src + 1) + 4 * (t + case["padding"]) + grains * 2 * kvh * 8, "flops": 0}
    h = case["heads"]
    lens = _lengths(case["batch"], case["lo"], case["hi"], case.get("log", False))
    row = 2 * kvh * D + 2 * kvh * 4 / GRAIN  # K and V of a token in the cache, its share of their scales
    if kind in ("decode", "step"):
        b, ctx = case["batch"] + case["empty"], int(lens.sum())
        size = ctx * row + 2 * b * h * D * 2 + 4 * (b + int((-(-lens // block)).sum()))
        if kind == "step":
            size += case["batch"] * 2 * kvh * D * src + 4 * b  # the new rows come from k and v and go to the cache
        return {"bytes": int(size), "flops": 4 * ctx * h * D}
    pre = _lengths(case["batch"], case["pre_lo"], case["pre_hi"])
    # the shuffles pair lengths and prefixes at random: their mean product
    keys = float(lens.sum() * pre.mean() + (lens * (lens + 1) // 2).sum())
    t = int(lens.sum())
    return {"bytes": int((t + int(pre.sum())) * row + 2 * t * h * D * 2), "flops": 4 * D * h * keys}


# ---- the same in 64 bits ---------------------------------------------------------------------------------------------


def _rounded(x):
    """The e4m3 value next to x, ties to even: steps of 2^-9 below 2^-6, else eight to a power of two."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-TOP, TOP)


def _exact_store(rows, cache, scale, slots):
    kvh = rows.shape[1]
    values, grid = cache.double().view(-1, kvh, D).clone(), scale.double().view(-1, kvh).clone()
    x, at = rows.double(), slots.long()
    x, at = x[at >= 0], at[at >= 0]
    order = torch.argsort(at)
    x, at = x[order], at[order]
    blocks, count = torch.unique_consecutive(at // GRAIN, return_counts=True)
    ends = torch.cumsum(count, 0).tolist()
    for blk, z, n in zip(blocks.tolist(), ends, count.tolist()):
        part, place = x[z - n:z], at[z - n:z]
        need = torch.exp2(torch.ceil(torch.log2(part.abs().amax(dim=(0, 2)) / TOP)))
        lo = blk * GRAIN
        if int(place[0]) != lo:
            old = grid[blk].clone()
            need = torch.maximum(need, old)
            values[lo:lo + GRAIN] = _rounded(values[lo:lo + GRAIN] * (old / need)[None, :, None])
        values[place] = _rounded(part / need[None, :, None])
        grid[blk] = need
    return values.view(cache.shape), grid.view(scale.shape)


def _exact_attention(q, cache, scale, tables, first, last, sm):
    """q [rows, heads, 128] at positions first .. last - 1 of one sequence, its pages in `tables`, in 64 bits."""
    block, kvh = cache[0].shape[1], cache[0].shape[2]
    page = tables[:-(-last // block)].long()
    k, v = (c[page].double().view(-1, GRAIN, kvh, D) * s[page].double().view(-1, 1, kvh, 1) for c, s in zip(cache, scale))
    k, v = (x.reshape(-1, kvh, D)[:last] for x in (k, v))
    w = torch.einsum("rkgd,tkd->kgrt", q.double().view(q.shape[0], kvh, -1, D), k) * sm
    late = torch.arange(last, device=q.device)[None, :] > torch.arange(first, last, device=q.device)[:, None]
    w = torch.softmax(w.masked_fill(late, -math.inf), dim=-1)
    return torch.einsum("kgrt,tkd->rkgd", w, v).reshape(q.shape)


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "copy":
        return None
    got = {}
    if kind in ("store", "step"):
        for x in ("k", "v"):
            got[x + "_cache"], got[x + "_scale"] = _exact_store(s[x], s[x + "_cache"], s[x + "_scale"], s["slots"])
    if kind != "store":
        cache = [got.get(x, s[x]) for x in ("k_cache", "v_cache")]
        if cache[0].dtype == E4M3:  # pages are gathered as bytes otherwise
            cache = [c.to(torch.float16) for c in cache]  # e4m3 values are fp16 values
        scale = [got.get(x, s[x]) for x in ("k_scale", "v_scale")]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
        lens = s["lens"].tolist()
        cu = s["cu_q"].tolist() if kind == "prefix" else list(range(len(lens) + 1))
        for b, n in enumerate(lens):
            if n:
                out[cu[b]:cu[b + 1]] = _exact_attention(s["q"][cu[b]:cu[b + 1]], cache, scale, s["tables"][b], n - cu[b + 1] + cu[b], n,
                                                        s["scale"])
        got["out"] = out
    return got

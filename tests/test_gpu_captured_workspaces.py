"""Scratch buffers: two graphs that were captured on one stream are replayed side by side on two others, beside eager calls on the
capture's own stream; two threads call on one stream."""
import gc
import time

import numpy as np
import pytest

from cache8_helpers import random_cache

pytestmark = pytest.mark.gpu


def work(seed):
    """Operators that use scratch (chains of runs, tickets and partial results, a work list) on tensors of their own: what to call,
    and the tensors it writes."""
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(seed)
    nb, block, kvh, h = 40, 256, 2, 8
    cache = random_cache(rng, nb, block, kvh)
    wide = [(c.float() * s.repeat_interleave(64, 1)[..., None]).to(torch.bfloat16) for c, s in zip(cache[:2], cache[2:])]
    q = torch.from_numpy(rng.normal(size=(4, h, 128)).astype(np.float32)).to(torch.bfloat16).cuda()
    rows = torch.from_numpy(rng.normal(size=(3000, kvh, 128)).astype(np.float32)).to(torch.bfloat16).cuda()
    target = [torch.zeros_like(c) for c in cache]
    slots = torch.from_numpy(np.concatenate([rng.permutation(64 * 150)[:2000], np.arange(1000)]).astype(np.int32)).cuda()
    tables = torch.from_numpy(rng.permutation(nb)[:40].reshape(4, 10).astype(np.int32)).cuda()
    lens = torch.from_numpy(rng.integers(1000, 2500, 4).astype(np.int32)).cuda()
    cu = torch.arange(5, dtype=torch.int32).cuda()
    cu_k = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), lens.cumsum(0, dtype=torch.int32)])
    outs = [torch.empty_like(q) for _ in range(4)]

    def call():
        ops.store_kvcache_q8(rows, rows, *target, slots)
        ops.paged_decode_q8(q, *cache, tables, lens, 0.09, block, out=outs[0])
        ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, 1, 0.09, block, out=outs[1])
        ops.paged_decode(q, *wide, tables, lens, 0.09, block, out=outs[2])
        ops.paged_prefill(q, *wide, tables, cu, cu_k, 1, 0.09, block, out=outs[3])

    return call, outs + [target[0].view(torch.uint8), target[1].view(torch.uint8)] + target[2:]


def test_two_graphs_and_an_eager_call_at_once():
    import torch
    from nanovllm_jax_b200 import _lib
    jobs = [work(s) for s in range(3)]
    side = [torch.cuda.Stream() for _ in range(3)]
    want = []
    for call, written in jobs:
        call()
        torch.cuda.synchronize()
        want.append([t.clone() for t in written])
    graphs = []
    for call, _ in jobs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side[2]):
            call()
        graphs.append(graph)
    for _, written in jobs:
        for t in written:
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(30):
        for i in range(3):
            with torch.cuda.stream(side[i]):
                graphs[i].replay() if i < 2 else jobs[2][0]()
    torch.cuda.synchronize()
    for (_, written), expected in zip(jobs, want):
        assert all(torch.equal(a, b) for a, b in zip(written, expected))
    assert _lib.device_status() == 0


def test_buffers_go_with_their_graph():
    import torch
    call, _ = work(5)
    call()
    torch.cuda.synchronize()

    def capture():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graph.replay()
        torch.cuda.synchronize()

    capture()
    gc.collect()
    held = []
    for _ in range(6):
        capture()
        gc.collect()
        until = time.monotonic() + 5
        call()  # gives back what the driver has let go of
        while held and torch.cuda.memory_allocated() > held[0] and time.monotonic() < until:
            time.sleep(0.05)
            call()
        held.append(torch.cuda.memory_allocated())
    assert max(held) <= held[0], held


def test_two_threads_on_one_stream():
    import threading
    import torch
    from nanovllm_jax_b200 import _lib
    jobs = [work(s) for s in (7, 8)]
    want = []
    for call, written in jobs:
        call()
        torch.cuda.synchronize()
        want.append([t.clone() for t in written])
    wrong = []

    def loop(i):
        call, written = jobs[i]
        try:
            for _ in range(60):
                call()
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(written, want[i])):
                wrong.append(i)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and _lib.device_status() == 0

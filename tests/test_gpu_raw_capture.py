"""Calls inside a capture that was begun through the runtime, without torch's private pool."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class RawGraph:
    """A capture of `stream` in the strictest mode, replayed on any stream."""

    def __init__(self, stream):
        self.rt, self.stream = ctypes.CDLL("libcudart.so.12"), ctypes.c_void_p(stream.cuda_stream)
        self.graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()

    def ok(self, rc):
        assert rc == 0, f"CUDA error {rc}"

    def __enter__(self):
        self.ok(self.rt.cudaStreamBeginCapture(self.stream, 0))  # cudaStreamCaptureModeGlobal
        return self

    def __exit__(self, kind, *_):
        rc = self.rt.cudaStreamEndCapture(self.stream, ctypes.byref(self.graph))
        if kind is None:
            self.ok(rc)
            self.ok(self.rt.cudaGraphInstantiate(ctypes.byref(self.exec), self.graph, ctypes.c_ulonglong(0)))
        else:
            self.rt.cudaGetLastError()

    def replay(self, stream):
        self.ok(self.rt.cudaGraphLaunch(self.exec, ctypes.c_void_p(stream.cuda_stream)))

    def close(self):
        self.ok(self.rt.cudaGraphExecDestroy(self.exec))
        self.ok(self.rt.cudaGraphDestroy(self.graph))


def calls():
    """name -> (call into `out`, out) over the operators that need scratch."""
    import torch
    from cache8_helpers import random_cache
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(11)
    cache = random_cache(rng, 64, 128, 2)
    wide = [torch.from_numpy(rng.normal(size=(64, 128, 2, 128)).astype(np.float32)).to(torch.bfloat16).cuda() for _ in range(2)]
    q = torch.from_numpy(rng.normal(size=(4, 8, 128)).astype(np.float32)).to(torch.bfloat16).cuda()
    tables = torch.from_numpy(rng.permutation(64).reshape(4, 16).astype(np.int32)).cuda()
    lens = torch.tensor([2000, 3, 700, 1500], dtype=torch.int32).cuda()
    cu = torch.arange(5, dtype=torch.int32).cuda()
    cu_k = torch.cat([cu[:1], lens.cumsum(0, dtype=torch.int32)])
    outs = {name: torch.zeros_like(q) for name in ("paged_decode", "paged_decode_q8", "paged_prefill", "paged_prefill_q8")}
    return {
        "paged_decode": (lambda: ops.paged_decode(q, *wide, tables, lens, 0.09, 128, out=outs["paged_decode"]), outs["paged_decode"]),
        "paged_decode_q8": (lambda: ops.paged_decode_q8(q, *cache, tables, lens, 0.09, 128, out=outs["paged_decode_q8"]),
                            outs["paged_decode_q8"]),
        "paged_prefill": (lambda: ops.paged_prefill(q, *wide, tables, cu, cu_k, 1, 0.09, 128, out=outs["paged_prefill"]),
                          outs["paged_prefill"]),
        "paged_prefill_q8": (lambda: ops.paged_prefill_q8(q, *cache, tables, cu, cu_k, 1, 0.09, 128, out=outs["paged_prefill_q8"]),
                             outs["paged_prefill_q8"]),
    }


@pytest.mark.parametrize("pending", (False, True))
@pytest.mark.parametrize("name", ("paged_decode", "paged_decode_q8", "paged_prefill", "paged_prefill_q8"))
def test_raw_capture(name, pending):
    """`pending`: torch's allocator waits for another stream's use of memory that was given back, and asks for it when it is called next."""
    import torch
    call, out = calls()[name]
    stream, side = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        call()
        stream.synchronize()
        want = out.clone()
        out.zero_()
        if pending:
            used = torch.zeros(1 << 20, device="cuda")
            with torch.cuda.stream(side):
                torch.cuda._sleep(200_000_000)
            used.record_stream(side)
            del used
        with RawGraph(stream) as graph:
            call()
    torch.cuda.synchronize()
    assert (out == 0).all()
    for s in (stream, side):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay(s)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    graph.close()

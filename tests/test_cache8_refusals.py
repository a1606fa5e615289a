"""What the operators on the 8-bit cache and copy_pages refuse: through the C ABI without a GPU, through the torch operators on one."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from nanovllm_jax_b200 import _lib
    from nanovllm_jax_b200.csrc import build
    build.build()
    return _lib.load()


P = 1 << 20  # an aligned address that nothing reads: every call here is refused before it launches


def store(lib, k=P, cache=P, scale=P, slots=P, ws=None, wsn=0, t=4, kvh=2, d=128, n=128, dtype=0):
    return lib.nvllm_b200_store_kvcache_q8(k, P, cache, P, scale, P, slots, ws, wsn, t, kvh, d, n, dtype, None)


def test_store(lib):
    from nanovllm_jax_b200 import _lib
    assert store(lib, t=-1) == store(lib, kvh=0) == store(lib, n=-64) == _lib.EINVAL
    assert store(lib, d=64) == store(lib, n=100) == store(lib, dtype=7) == store(lib, t=1 << 31) == store(lib, n=1 << 31) == _lib.EUNSUPPORTED
    assert b"multiple of 64" in (store(lib, n=100), lib.nvllm_b200_last_error_string())[1]
    assert store(lib, k=None) == store(lib, cache=None) == store(lib, scale=None) == store(lib, slots=None) == _lib.EINVAL
    assert store(lib, k=P + 8) == store(lib, cache=P + 1) == store(lib, scale=P + 2) == store(lib, slots=P + 1) == _lib.EINVAL
    need = lib.nvllm_b200_store_kvcache_q8_workspace_bytes(1025)
    assert need > 1025 * 16
    assert store(lib, t=1025) == store(lib, t=1025, ws=P, wsn=need - 1) == store(lib, t=1025, ws=P + 8, wsn=need) == _lib.EWORKSPACE
    assert store(lib, t=0, k=None) == store(lib, n=0, k=None) == _lib.OK


def decode(lib, q=P, cache=P, scale=P, ws=P, wsn=1 << 30, b=4, h=8, kvh=2, d=128, nb=4, block=64, mb=2):
    return lib.nvllm_b200_paged_decode_q8(q, cache, P, scale, P, P, P, P, ws, wsn, b, h, kvh, d, nb, block, mb, 0.1, None)


def test_decode(lib):
    from nanovllm_jax_b200 import _lib
    assert decode(lib, d=64) == decode(lib, block=96) == decode(lib, h=7) == decode(lib, h=18) == decode(lib, nb=1 << 30) == _lib.EUNSUPPORTED
    assert decode(lib, b=-1) == decode(lib, mb=0) == decode(lib, q=None) == decode(lib, scale=None) == decode(lib, cache=P + 4) == _lib.EINVAL
    assert decode(lib, scale=P + 1) == _lib.EINVAL
    need = lib.nvllm_b200_paged_decode_q8_workspace_bytes(4, 8, 2)
    assert decode(lib, ws=None) == decode(lib, wsn=need // 2) == decode(lib, ws=P + 16) == _lib.EWORKSPACE
    assert decode(lib, b=0, q=None) == _lib.OK
    assert lib.nvllm_b200_paged_decode_q8_workspace_bytes(5000, 8, 2) > need + lib.nvllm_b200_store_kvcache_q8_workspace_bytes(5000)


def test_decode_step(lib):
    from nanovllm_jax_b200 import _lib

    def step(k=P, slots=P, b=4, d=128, dtype=0, wsn=1 << 30):
        return lib.nvllm_b200_decode_step_q8(P, k, P, P, P, P, P, slots, P, P, P, P, wsn, b, 8, 2, d, 4, 64, 2, 0.1, dtype, None)
    assert step(d=64) == step(dtype=3) == _lib.EUNSUPPORTED
    assert step(k=None) == step(k=P + 4) == step(slots=None) == _lib.EINVAL
    assert step(wsn=100) == _lib.EWORKSPACE
    assert step(b=0) == _lib.OK


def test_copy_pages(lib):
    from nanovllm_jax_b200 import _lib

    def copy(base=P, rows=64, row=256, src=P, dst=P, tokens=None, n=2, nb=8, block=64, tables=None, entries=0, count=1):
        return lib.nvllm_b200_copy_pages((ctypes.c_void_p * 1)(base), (ctypes.c_int32 * 1)(rows), (ctypes.c_int64 * 1)(row), count, src, dst,
                                         tokens, n, nb, block, tables, entries, None)
    assert copy(n=-1) == copy(nb=-1) == copy(block=0) == copy(entries=-1) == copy(count=-1) == _lib.EINVAL
    assert copy(rows=48) == copy(rows=0) == copy(row=6) == copy(row=0) == copy(nb=1 << 31) == _lib.EUNSUPPORTED
    assert copy(base=None) == copy(base=P + 2) == copy(src=None) == copy(dst=None) == copy(src=P + 1) == copy(tokens=P + 2) == _lib.EINVAL
    assert copy(entries=4) == copy(entries=4, tables=P + 2) == _lib.EINVAL
    assert lib.nvllm_b200_copy_pages(None, None, None, 1, P, P, None, 1, 8, 64, None, 0, None) == _lib.EINVAL
    assert copy(n=0, src=None) == copy(nb=0, src=None) == _lib.OK


def test_host_tensors():
    import torch
    from nanovllm_jax_b200 import ops
    x = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.store_kvcache_q8(x, x, x, x, x, x, i), lambda: ops.paged_decode_q8(x, x, x, x, x, i, i, 0.1, 64),
                 lambda: ops.decode_step_q8(x, x, x, x, x, x, x, i, i, i, 0.1, 64), lambda: ops.copy_pages([x], i, i, 64)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.gpu
def test_shapes_types_and_strides():
    import torch
    from nanovllm_jax_b200 import ops
    dev = "cuda"
    k = torch.zeros((3, 2, 128), dtype=torch.bfloat16, device=dev)
    q = torch.zeros((3, 8, 128), dtype=torch.bfloat16, device=dev)
    c = torch.zeros((4, 64, 2, 128), dtype=torch.float8_e4m3fn, device=dev)
    s = torch.zeros((4, 1, 2), device=dev)
    i = torch.zeros(3, dtype=torch.int32, device=dev)
    t = torch.zeros((3, 2), dtype=torch.int32, device=dev)
    store = lambda **n: ops.store_kvcache_q8(*{**dict(k=k, v=k, kc=c, vc=c.clone(), ks=s, vs=s.clone(), i=i - 1), **n}.values())  # noqa: E731
    store()
    for bad, error in ((dict(k=k.half()), TypeError), (dict(v=k.float()), TypeError), (dict(kc=c.float()), TypeError), (dict(kc=c[:, :, :1]), ValueError),
                       (dict(vc=c[:3]), ValueError), (dict(ks=s[:, :, :1].contiguous()), ValueError), (dict(vs=s[0]), ValueError), (dict(ks=s.double()), TypeError),
                       (dict(i=i[:2]), ValueError), (dict(i=i.long()), TypeError), (dict(k=k[:2]), ValueError), (dict(i=i.cpu()), TypeError),
                       (dict(k=k[:, :1].contiguous(), v=k[:, :1].contiguous()), ValueError)):
        with pytest.raises(error):
            store(**bad)
    decode = lambda **n: ops.paged_decode_q8(*{**dict(q=q, kc=c, vc=c, ks=s, vs=s, t=t, i=i, scale=0.1, block=64, out=None), **n}.values())  # noqa: E731
    assert (decode() == 0).all()
    for bad, error in ((dict(q=q.float()), TypeError), (dict(block=128), ValueError), (dict(t=t[:2]), ValueError), (dict(i=i[:2]), ValueError),
                       (dict(q=q.transpose(0, 1)), ValueError), (dict(out=q[:2]), ValueError), (dict(out=q.float()), TypeError), (dict(kc=c.view(torch.uint8)), TypeError)):
        with pytest.raises(error):
            decode(**bad)
    with pytest.raises(RuntimeError, match="H/KVH"):
        decode(q=torch.zeros((3, 7, 128), dtype=torch.bfloat16, device=dev))
    with pytest.raises(ValueError):
        ops.decode_step_q8(q, k[:2], k[:2], c, c, s, s, i, t, i, 0.1, 64)
    copy = lambda caches=(c, s), src=i - 1, dst=i, block=64, **n: ops.copy_pages(caches, src, dst, block, **n)  # noqa: E731
    copy()
    for bad, error in ((dict(caches=[]), ValueError), (dict(caches=[c, s[:3]]), ValueError), (dict(caches=[c.transpose(1, 2)]), ValueError),
                       (dict(caches=[c[0, 0, 0]]), ValueError), (dict(caches=[c.cpu()]), TypeError), (dict(block=96), ValueError), (dict(dst=i[:2]), ValueError),
                       (dict(tokens=i[:2]), ValueError), (dict(block_tables=i), ValueError), (dict(src=i.long()), TypeError), (dict(caches=3), TypeError),
                       (dict(block=0), ValueError)):
        with pytest.raises(error):
            copy(**bad)


def test_prefill(lib):
    from nanovllm_jax_b200 import _lib

    def prefill(q=P, cache=P, scale=P, tables=P, ws=P, wsn=1 << 30, t=5, b=1, m=5, h=8, kvh=2, d=128, nb=4, block=128, mb=2, s=0.1):
        return lib.nvllm_b200_paged_prefill_q8(q, cache, P, scale, P, P, P, tables, None, P, ws, wsn, t, b, m, h, kvh, d, nb, block, mb, s, None)
    assert prefill(d=64) == prefill(block=64) == prefill(block=192) == prefill(h=7) == prefill(b=70000) == _lib.EUNSUPPORTED
    assert prefill(t=-1) == prefill(nb=0) == prefill(mb=0) == prefill(s=0.0) == prefill(m=0) == _lib.EINVAL
    assert prefill(q=None) == prefill(scale=None) == prefill(scale=P + 2) == prefill(tables=None) == prefill(cache=P + 8) == _lib.EINVAL
    assert prefill(ws=None) == prefill(wsn=16) == _lib.EWORKSPACE
    assert prefill(t=0, q=None) == prefill(b=0, q=None) == _lib.OK

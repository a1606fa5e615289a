"""copy_pages against a statement of it on the host, bit for bit."""
import numpy as np
import pytest

from oracle import cache8

pytestmark = pytest.mark.gpu


def caches(rng, nb, block, kvh, held, layers=1):
    import torch
    out = []
    for _ in range(layers):
        for _ in range(2):
            if held == "bf16":
                out.append(torch.from_numpy(rng.integers(0, 1 << 15, (nb, block, kvh, 128)).astype(np.int16)).cuda().view(torch.bfloat16))
            else:
                out.append(torch.from_numpy(rng.integers(0, 256, (nb, block, kvh, 128)).astype(np.uint8)).cuda().view(torch.float8_e4m3fn))
                out.append(torch.from_numpy(rng.random((nb, block // 64, kvh)).astype(np.float32)).cuda())
    return out


def host(t):
    import torch
    return t.view(torch.int16).cpu().numpy() if t.dtype == torch.bfloat16 else t.view(torch.uint8).cpu().numpy().reshape(*t.shape, -1)


def check(c, src, dst, block, tokens=None, tables=None):
    import torch
    from nanovllm_jax_b200 import _lib, ops
    _lib.device_status_reset()
    want, want_tables, bad = cache8.copy_pages([host(x) for x in c], src, dst, block, tokens, tables)
    dev = lambda x: None if x is None else torch.from_numpy(np.asarray(x, np.int32)).cuda()  # noqa: E731
    t = dev(tables)
    ops.copy_pages(c, dev(src), dev(dst), block, tokens=dev(tokens), block_tables=t)
    torch.cuda.synchronize()
    for i, (x, w) in enumerate(zip(c, want)):
        assert np.array_equal(host(x), w), f"cache {i}"
    if tables is not None:
        assert np.array_equal(t.cpu().numpy(), want_tables)
    assert _lib.device_status() == (128 if bad else 0)
    _lib.device_status_reset()
    return bad


@pytest.mark.parametrize("held", ("bf16", "8 bits"))
@pytest.mark.parametrize("kvh, block, nb, n, layers", [(1, 64, 2, 1, 1), (8, 256, 9, 4, 3), (3, 128, 40, 18, 2), (2, 512, 6, 2, 40), (1, 64, 700, 300, 1), (1, 64, 3, 1, 300)])
def test_fork_and_move(held, kvh, block, nb, n, layers):
    rng = np.random.default_rng(n)
    c = caches(rng, nb, block, kvh, held, layers)
    p = rng.permutation(nb)
    assert not check(c, p[:n], p[nb - n:], block)
    tokens = rng.integers(0, block + 1, n)
    tokens[0] = rng.choice([0, 1, block])
    assert not check(c, np.resize(p[:max(1, n // 3)], n), p[nb - n:], block, tokens=tokens)
    tables = rng.integers(-1, nb + 1, (5, 13))
    assert not check(c, p[:n], p[nb - n:], block, tables=tables)


def test_tokens_out_of_range_and_padding_pairs():
    rng = np.random.default_rng(1)
    c = caches(rng, 12, 128, 2, "8 bits", 2)
    assert not check(c, [0, 1, -1, 3, 12, 4, 5], [6, 7, 8, -1, 9, 40, 5], 128, tokens=[-3, 1000, 5, 6, 7, 8, 9],
                     tables=[[0, 1, 2, 3, 4, 5, -1]])
    assert not check(c, [0], [1], 128, tokens=[64], tables=np.zeros((0, 4), np.int32))
    assert not check(c, [], [], 128)


@pytest.mark.parametrize("held", ("bf16", "8 bits"))
def test_pairs_that_contradict_one_another_are_left_out(held):
    rng = np.random.default_rng(2)
    c = caches(rng, 16, 64, 2, held, 1)
    tables = rng.integers(0, 16, (4, 9))
    assert check(c, [0, 1, 2], [1, 2, 3], 64, tables=tables)              # a chain: only its end is carried out
    assert check(c, [4, 5], [5, 4], 64, tables=tables)                    # a swap: neither
    assert check(c, [6, 7, 8], [9, 9, 9], 64, tables=tables)              # the last of three
    assert check(c, [6, 6, 10, 11, -1], [12, 13, 11, 12, 6], 64, tokens=[3, 64, 1, 5, 2], tables=tables)


@pytest.mark.parametrize("n", (3, 700))
def test_many_random_pairs(n):
    rng = np.random.default_rng(n)
    c = caches(rng, 2000, 64, 1, "8 bits", 1)
    for _ in range(3):
        check(c, rng.integers(-20, 2020, n), rng.integers(-20, 2020, n), 64, tokens=rng.integers(0, 65, n), tables=rng.integers(-1, 2000, (3, 50)))


def test_a_tensor_twice_and_views():
    """The same tensor, and another shape of it, in one list: every copy of a page writes what the others write."""
    rng = np.random.default_rng(4)
    c = caches(rng, 9, 64, 2, "bf16", 1)
    assert not check([c[0], c[1], c[0], c[0].view(9, 64, 256)], [0, 1, 7], [2, 3, 8], 64, tokens=[64, 5, 0])
    assert not check([c[0].view(9, 32, 512), c[0]], [0], [5], 64)
    assert np.array_equal(host(c[0][5]), host(c[0][0]))  # bits: there are NaNs among them


def test_captured_and_replayed():
    import torch
    from nanovllm_jax_b200 import ops
    rng = np.random.default_rng(3)
    c = caches(rng, 10, 64, 2, "8 bits", 3)
    src, dst = (torch.full((4,), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    tokens = torch.zeros(4, dtype=torch.int32, device="cuda")
    ops.copy_pages(c, src, dst, 64, tokens=tokens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_pages(c, src, dst, 64, tokens=tokens)
    for s, d, t in (([0, 1], [5, 6], [10, 64]), ([2, 2, 3], [7, 8, 9], [1, 2, 3])):
        want, _, _ = cache8.copy_pages([host(x) for x in c], s, d, 64, t)
        for x, y in ((src, s), (dst, d), (tokens, t)):
            x.copy_(torch.tensor(y + [-1] * (4 - len(y)), dtype=torch.int32))
        graph.replay()
        for x, w in zip(c, want):
            assert np.array_equal(host(x), w)


def test_pool_beyond_4_gb():
    import torch
    from nanovllm_jax_b200 import ops
    nb = 20000
    c = torch.zeros((nb, 256, 8, 128), dtype=torch.float8_e4m3fn, device="cuda")
    c.view(torch.uint8)[nb - 1] = 77
    c.view(torch.uint8)[3] = 5
    ops.copy_pages([c], torch.tensor([nb - 1, 3], dtype=torch.int32).cuda(), torch.tensor([0, nb - 2], dtype=torch.int32).cuda(), 256)
    v = c.view(torch.uint8)
    assert (v[0] == 77).all() and (v[nb - 2] == 5).all() and (v[1] == 0).all() and (v[nb - 3] == 0).all()

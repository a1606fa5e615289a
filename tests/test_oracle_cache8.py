"""The 64-bit statement of the 8-bit cache against torch's own e4m3 and against itself (CPU)."""
import numpy as np
import pytest
import torch

from oracle import cache8


def test_table_is_torchs():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(t, cache8.TABLE, equal_nan=True)


def test_rounding_is_torchs():
    rng = np.random.default_rng(1)
    x = np.concatenate([rng.normal(size=4000) * 2.0 ** rng.integers(-12, 8, 4000), cache8.TABLE[~np.isnan(cache8.TABLE)],
                        (cache8.TABLE[:126] + cache8.TABLE[1:127]) / 2, [0.0, -0.0, 2.0 ** -10, 3 * 2.0 ** -11]])
    x = np.clip(x, -448, 448).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(cache8.to_e4m3(x), want)
    assert np.array_equal(cache8.to_e4m3([1e9, -460.0, np.nan]), [448.0, -448.0, np.nan], equal_nan=True)


@pytest.mark.parametrize("amax, k", [(448.0, 0), (448.0001, 1), (224.0, -1), (1.75, -8), (1.7500001, -7), (1.0, -8), (0.0, -117),
                                     (3.3e38, 119), (2.0 ** -130, -117)])
def test_scale(amax, k):
    assert cache8.scale_for(amax) == 2.0 ** k


def test_store_begins_grows_and_keeps():
    values, scales = np.zeros((128, 1, 128)), np.zeros((2, 1))
    row = np.ones((1, 1, 128))
    values, scales = cache8.store(row * 448, values, scales, [64])
    assert scales[1, 0] == 1.0 and scales[0, 0] == 0.0 and (values[64] == 448).all()
    values, scales = cache8.store(row * 3, values, scales, [65])      # smaller: the scale stays
    assert scales[1, 0] == 1.0 and (values[65] == 3).all()
    values, scales = cache8.store(row * 900, values, scales, [66])    # larger: 4 * 448 >= 900 > 2 * 448
    assert scales[1, 0] == 4.0 and (values[64] == 112).all() and (values[65] == 0.75).all() and (values[66] == 224).all()
    values, scales = cache8.store(row, values, scales, [64])          # the first slot begins the block
    assert scales[1, 0] == 2.0 ** -8


def test_attention_is_softmax():
    rng = np.random.default_rng(2)
    k, v = rng.normal(size=(2, 3, 64, 1, 128))
    q = rng.normal(size=(2, 2, 128))
    out, weight, score, small = cache8.attention(q, k, v, [[2, 0]], [2], [100], 0.1, 64)
    kk, vv = np.concatenate([k[2], k[0]])[:, 0], np.concatenate([v[2], v[0]])[:, 0]
    for i, n in enumerate((99, 100)):
        p = torch.softmax(torch.from_numpy(q[i] @ kk[:n].T * 0.1), -1)
        assert np.allclose(out[i], p.numpy() @ vv[:n], rtol=0, atol=1e-13)
    assert (np.abs(out) <= weight + 1e-15).all() and (score > 0).all() and (small <= weight).all()


def test_copy_pages():
    c = np.arange(24.0).reshape(6, 4)
    out, tables, bad = cache8.copy_pages([c], [0, 1, -1, 3], [2, 4, 5, 9], 4, tables=np.array([[0, 3, -1, 1]], np.int32))
    assert not bad and np.array_equal(out[0][2], c[0]) and np.array_equal(out[0][4], c[1]) and np.array_equal(out[0][5], c[5])
    assert tables.tolist() == [[2, 3, -1, 4]]
    out, _, bad = cache8.copy_pages([c], [0, 2, 1], [2, 3, 3], 4, tokens=[4, 4, 2])  # 0 -> 2 would change a source, 3 has two
    assert bad and np.array_equal(out[0][2], c[2]) and out[0][3].tolist() == [4, 5, 14, 15]

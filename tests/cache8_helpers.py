"""What the tests of the 8-bit cache share."""
import numpy as np

from oracle import cache8


def values_of(t):
    """A float8_e4m3fn tensor's values in 64 bits, on the host."""
    import torch
    return cache8.TABLE[t.contiguous().view(torch.uint8).cpu().numpy()]


def random_cache(rng, nb, block, kvh, device="cuda", garbage=False):
    """(k_cache, v_cache, k_scale, v_scale) on the device: N(0, 1) rows, every 64 slots and head with a magnitude of its own.
    garbage: any byte (NaN too) and scales of any power of two within 2^-20 .. 2^20 instead."""
    import torch
    out, scales = [], []
    for _ in range(2):
        size = 2.0 ** rng.integers(-3, 4, (nb, block // 64, kvh))
        if garbage:
            codes = torch.from_numpy(rng.integers(0, 256, (nb, block, kvh, 128)).astype(np.uint8)).to(device)
            out.append(codes.view(torch.float8_e4m3fn))
            size = 2.0 ** rng.integers(-20, 21, size.shape)
        else:
            x = torch.from_numpy((rng.normal(size=(nb, block, kvh, 128)) * 64).astype(np.float32))
            out.append(x.clamp(-448, 448).to(torch.float8_e4m3fn).to(device))
            size = size / 64
        scales.append(torch.from_numpy(size.astype(np.float32)).to(device))
    return out[0], out[1], scales[0], scales[1]


def attention_bound(out, weight, score, small):
    """How far a bf16 result of fp16 probabilities may be from the 64-bit one.

    Half a step of bf16 of the result, 2^-8 |out|; of every probability half a step of fp16 and as much again for its
    normaliser's share, 2^-10 of sum p |v|; a score error of fp32 sums of 128 products and of the exponential, at most 2^-18 of
    sum |q||k|, which moves a probability (and the normaliser) by as much; and what underflows.  fp16 numbers below 2^-14 are
    multiples of 2^-24, off by 2^-25 at most.  Decode: of a probability relative to its warp's tile of 16 tokens, whose largest
    is 2^-4 or more, 2^-21.  Prefill: of a probability times its V scale, relative to 2^7 times the row's largest
    probability and the largest V scale so far, which is 2^-32 of max p times a value of up to 448 under that scale, 448 /
    (largest value / scale) <= 2 of max |v| where the scale is the least possible.
    """
    return 2.0 ** -8 * np.abs(out) + (2.0 ** -10 + 2.0 ** -17 * score) * weight + 1.01 * small + 1e-30


def assert_attention(got, want, what=""):
    out = want[0]
    got = got.detach().double().cpu().numpy()
    off = np.abs(got - out) / attention_bound(*want)
    assert np.isfinite(got).all(), f"{what}: not finite"
    assert off.max(initial=0) <= 1, f"{what}: {off.max():.2f} times the bound at {np.unravel_index(off.argmax(), off.shape)}"

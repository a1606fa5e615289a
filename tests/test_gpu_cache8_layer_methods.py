"""The attention layer's own decode method over an 8-bit cache, called by itself."""
import numpy as np
import pytest

from cache8_helpers import random_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ("bf16", "fp32", "strided"))
def test_decode_attention_of_the_layer(form):
    import torch
    from nanovllm_jax_b200 import ops
    from nanovllm_jax_b200.layers.attention import Attention
    from nanovllm_jax_b200.utils.context import create_decode_context
    rng = np.random.default_rng(3)
    cache = random_cache(rng, 12, 128, 2)
    q = torch.from_numpy(rng.normal(size=(3, 8, 128)).astype(np.float32)).to(torch.bfloat16).cuda()
    tables = torch.from_numpy(rng.permutation(12).reshape(3, 4).astype(np.int32)).cuda()
    lens = torch.tensor([500, 1, 129], dtype=torch.int32).cuda()
    attn = Attention(8, 128, 0.09, 2, block_size=128)
    attn.set_kv_cache_q8(*cache)
    given = {"bf16": q, "fp32": q.float(), "strided": torch.stack([q, q], -1)[..., 0]}[form]
    context = create_decode_context(lens, torch.full((3,), -1, dtype=torch.int32).cuda(), tables)
    out = attn._decode_attention(given, context)
    assert torch.equal(out, ops.paged_decode_q8(q, *cache, tables, lens, 0.09, 128))

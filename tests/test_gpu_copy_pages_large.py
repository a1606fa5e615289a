"""Pages of more than 2^31 bytes."""
import pytest

pytestmark = pytest.mark.gpu

ROW = (1 << 25) + (1 << 20)  # bytes; 64 of them are 2^31 + 2^26


@pytest.mark.parametrize("tokens", (1, 0, 63, None))
def test_rows_behind_the_tokens_stay(tokens):
    """The piece behind the live rows that is farthest from them begins 2^31 bytes and more behind their end."""
    import torch
    from nanovllm_jax_b200 import _lib, ops
    cache = torch.empty((2, 64, ROW), dtype=torch.uint8, device="cuda")
    cache[0], cache[1] = 3, 5
    cache[0, :, -1] = torch.arange(64, dtype=torch.uint8, device="cuda")
    of = lambda x: torch.tensor([x], dtype=torch.int32, device="cuda")  # noqa: E731
    ops.copy_pages([cache], of(0), of(1), 64, tokens=None if tokens is None else of(tokens))
    n = 64 if tokens is None else tokens
    for i in range(64):
        assert torch.equal(cache[1, i], cache[0, i]) if i < n else bool((cache[1, i] == 5).all()), f"row {i}"
    assert _lib.device_status() == 0

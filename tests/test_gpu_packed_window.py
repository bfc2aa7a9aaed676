"""Windows of packed attention of any size (GPU)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [1 << 29, (1 << 31) + 3, (1 << 32) + 5, (1 << 63) - 1, 1 << 63, 1 << 64, (1 << 64) + 5])
def test_a_window_past_all_keys_is_none(window):
    import ltxk

    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(200, 128, device="cuda", generator=g).to(torch.bfloat16) for _ in range(3))
    offsets = torch.tensor([0, 150, 200], dtype=torch.int32, device="cuda")
    assert torch.equal(ltxk.packed_attention(q, k, v, 2, offsets, window=window), ltxk.packed_attention(q, k, v, 2, offsets))

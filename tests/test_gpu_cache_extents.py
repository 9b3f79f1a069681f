"""Broadcast dimensions of more than 2^32 rows: refused, not taken for their remainder."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_extents_beyond_32_bits():
    import torch_neuronx_b200 as T

    n = (1 << 32) + 8
    x = torch.ones(1, 1, 1, 16, dtype=torch.bfloat16, device="cuda")
    pos, freq = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.ones(8, device="cuda")
    for big in (x.expand(1, 1, n, 16), x.expand(1, n, 1, 16)):
        with pytest.raises(RuntimeError, match="32 bits"):
            T.rotary_embedding(big, None, pos, freq)
    with pytest.raises(RuntimeError, match="32 bits"):
        T.rotary_embedding(x, x.expand(1, n, 1, 16), pos, freq)
    pools = [torch.zeros(4, 2, 1, 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.zeros(4, 2, 1, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
    with pytest.raises(RuntimeError, match="32 bits"):
        T.paged_write(x.expand(1, 1, n, 16), x.expand(1, 1, n, 16), *pools, *scales, torch.zeros(1, 2, dtype=torch.int32, device="cuda"), pos)
    T.check_device_status()
    assert all((s.view(torch.uint8) == 0).all() for s in scales)

"""bf16's largest numbers in an 8-bit cache: from 248 * 2^120 on they round to 2^128."""

import math

import pytest
import torch

from tests import cache_util as U

pytestmark = pytest.mark.gpu

TOP = torch.finfo(torch.bfloat16).max   # 255 * 2^120


def _pools(n, page, H, D):
    k, v = (torch.zeros(n, page, H, D, dtype=torch.uint8, device="cuda").view(U.F8) for _ in range(2))
    ks, vs = (torch.full((n, page, H), 127, dtype=torch.uint8, device="cuda").view(U.E8) for _ in range(2))
    return k, v, ks, vs


def test_read_back():
    import torch_neuronx_b200 as T

    x = torch.ones(1, 1, 4, 64, dtype=torch.bfloat16)
    x[0, 0, 0, 3], x[0, 0, 1, 5], x[0, 0, 2, 7], x[0, 0, 3, 9] = TOP, -TOP, 248 * 2.0**120, -247 * 2.0**120
    pools = _pools(1, 4, 1, 64)
    table, four = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.full((1,), 4, dtype=torch.int32, device="cuda")
    T.paged_write(x.cuda(), x.cuda(), *pools, table, four - 4)
    assert (pools[2].view(torch.uint8) == 247).all()
    for got in T.paged_read(*pools, table, four):
        got = got[0, 0].cpu().float()
        assert got[0, 3] == got[2, 7] == math.inf and got[1, 5] == -math.inf and got[3, 9] == -240 * 2.0**120
        assert (got.isinf().sum(), got.isnan().sum()) == (3, 0)


@pytest.mark.parametrize("D", [64, 128])
def test_under_a_gathered_prefix(D):
    """Keys with such an element where the query has a zero, and values with one: an infinity in their place would make NaN of the
    first and an infinity of every result of the second.  Counting as 255 * 2^120 is 2^-8 less than 2^128."""
    import torch_neuronx_b200 as T

    B, Hq, Hkv, page, P = 128, 4, 2, 16, 4000
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(1, Hkv, P, D, generator=g).bfloat16() for _ in range(2))
    k[:, :, ::7, 3] = -TOP
    v[:, 0, 11, 5], v[:, 1, 3999, 6] = TOP, -TOP
    q = torch.randn(B, Hq, 1, D, generator=g).bfloat16()
    q[..., 3] = 0
    n = P // page + B
    pools = _pools(n, page, Hkv, D)
    order = torch.randperm(n, generator=g).to(torch.int32).cuda()
    prefix, table = order[: P // page].contiguous(), order[P // page:].view(B, 1)
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    T.paged_write(k.cuda(), v.cuda(), *pools, prefix.view(1, -1), lens[:1])
    T.reset_launch_counts()
    out, lse = T.shared_prefix_decode(q.cuda(), pools[0], pools[1], prefix, P, table, lens, need_lse=True, k_scales=pools[2], v_scales=pools[3])
    T.check_device_status()
    assert T.launch_counts()["cache_read"] == 1
    ref, ref_l, _ = U.attend(q, *(t.cpu() for t in pools), table.cpu(), lens.cpu(), "NHD", prefix=prefix.cpu(), P=P)
    out, lse = out.cpu().double(), lse.cpu().double()
    assert ((lse - ref_l).abs() <= 2.0**-16 * (1 + ref_l.abs())).all()
    assert out.isfinite().all()
    top = torch.zeros(B, Hq, 1, D, dtype=torch.bool)
    top[:, :2, 0, 5] = top[:, 2:, 0, 6] = True
    # (at the other columns the rows with the large element are zeros: their scale is 2^120)
    assert ((out - ref).abs()[~top] <= (2.0**-8 * ref.abs() + 2.0**-16 * 8)[~top]).all()
    assert ((out - ref).abs()[top] <= ((2.0**-8 + 2.0**-8 + 2.0**-14) * ref.abs() + 2.0**-16 * 8)[top]).all()

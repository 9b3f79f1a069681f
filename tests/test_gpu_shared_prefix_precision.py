"""Decode under a prefix of an 8-bit cache that is multiplied once for the whole batch: as exact as the decode of that cache alone,
whose probabilities have 22 bits."""

import math

import pytest
import torch

from tests import cache_util as U
from tests.test_gpu_shared_prefix import _cuda, _setup

pytestmark = pytest.mark.gpu

CASES = [
    # dtype, B, Hq, Hkv, D, page, P, own pages, layout
    (torch.bfloat16, 130, 8, 2, 128, 16, 2000, 2, "NHD"),     # pairs of row tiles
    (torch.float16, 130, 8, 2, 128, 32, 1999, 1, "HND"),
    (torch.bfloat16, 200, 4, 2, 64, 16, 4100, 1, "HND"),
    (torch.float16, 200, 4, 2, 64, 4, 4096, 2, "NHD"),
    (torch.bfloat16, 16, 32, 8, 128, 16, 3001, 2, "NHD"),     # one row tile against even and odd key tiles
    (torch.float16, 16, 32, 8, 128, 16, 2900, 2, "HND"),
    (torch.bfloat16, 32, 32, 8, 64, 16, 4500, 1, "NHD"),
    (torch.float16, 32, 32, 8, 64, 16, 4501, 1, "NHD"),
]


@pytest.mark.parametrize("dtype,B,Hq,Hkv,D,page,P,pages,layout", CASES)
def test_probabilities_are_not_rounded_to_16_bits(dtype, B, Hq, Hkv, D, page, P, pages, layout):
    """The tolerance of the 8-bit decode alone.  hi + lo leaves 2^-17 (bf16) of half a step of a probability, 2^-18 of it, and 2^-22
    (fp16), or 2^-25 of the largest one: with all weights together at least a 128th of the number of keys (asserted), 2^-18."""
    import torch_neuronx_b200 as T

    q, k, v, ks, vs, prefix, table, lens = _setup(B + P, dtype, True, B, Hq, Hkv, D, page, P, pages, layout)
    if dtype == torch.float16:
        q = q / 2   # (no few keys have all the weight)
    want = U.attend(q, k, v, ks, vs, table, lens, layout, prefix=prefix, P=P)
    keys = U.rows_of(k, ks, prefix, P, layout).repeat_interleave(Hq // Hkv, 1)
    top = torch.einsum("bhd,shd->bhs", q[:8, :, 0].double(), keys).amax(-1) / math.sqrt(D)
    assert dtype == torch.bfloat16 or ((want[1][:8, :, 0] - top).exp() >= P / 128).all()
    dq, dk, dv, dks, dvs, dp, dt, dl = _cuda(q, k, v, ks, vs, prefix, table, lens)
    T.reset_launch_counts()
    out, lse = T.shared_prefix_decode(dq, dk, dv, dp, P, dt, dl, layout=layout, need_lse=True, k_scales=dks, v_scales=dvs)
    T.check_device_status()
    assert T.launch_counts()["cache_read"] == 1      # (gathered: once for all)
    U.check(out.cpu(), lse.cpu(), want)

"""The 8-bit cache at the ends of its range: scores are ordinary numbers while keys, queries or the scale are not."""

import math

import pytest
import torch

from tests import cache_util as U
from tests.test_gpu_shared_prefix import _cuda, _setup

pytestmark = pytest.mark.gpu


def _decode(q, k, v, ks, vs, table, lens, **kw):
    import torch_neuronx_b200 as T

    dq, dk, dv, dks, dvs, dt, dl = _cuda(q, k, v, ks, vs, table, lens)
    got = T.paged_decode(dq, dk, dv, dt, dl, need_lse=True, k_scales=dks, v_scales=dvs, **kw)
    T.check_device_status()
    return [t.cpu() for t in got]


@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 2, 128, 16), (16, 1, 64, 4), (3, 3, 64, 32)])
@pytest.mark.parametrize("every", [1, 3])
def test_very_large_keys_under_very_small_queries(Hq, Hkv, D, page, every):
    """Keys of about 2^114, all or every third of them, under queries of 2^-114: their products are ordinary numbers (the others'
    are next to zero)."""
    q, k, v, ks, vs, _, table, lens = _setup(9, torch.bfloat16, True, 3, Hq, Hkv, D, page, 0, 300 // page, "NHD")
    lens[0] = table.shape[1] * page
    rows = ks.view(torch.uint8).view(-1, Hkv)[::every]
    rows += 114
    q *= 2.0**-114
    assert ks.view(torch.uint8).max() <= 247 and q.abs().max() > 0
    out, lse = _decode(q, k, v, ks, vs, table, lens)
    U.check(out, lse, U.attend(q, k, v, ks, vs, table, lens, "NHD"))


def test_largest_keys():
    """The largest scale that is written, 2^120, with the largest values that stay finite; scores of up to 240, 350 in
    log2 units, some of them negative.  A score is two rounded products and its maximum another such: 4 x 350 x 2^-24 of an exponent of
    two, so weights are off by at most ln 2 x 1400 x 2^-24 < 2^-14 -- more than the 2^-16 that exponents of up to 2^5 have, and less
    than the half step of 2^-11 that is granted where probabilities were rounded to fp16."""
    q, k, v, ks, vs, _, table, lens = _setup(10, torch.bfloat16, True, 3, 8, 2, 64, 16, 0, 9, "NHD")
    ks.view(torch.uint8).fill_(247)
    k.view(torch.uint8)[..., 1:] = 0
    k.view(torch.uint8)[..., 0] = torch.randint(0x70, 0x78, k.shape[:3], generator=torch.Generator().manual_seed(3)).to(torch.uint8)   # 128 .. 240
    k.view(torch.uint8)[..., 0] += 128 * (torch.arange(k.shape[1]) % 2 == 0).to(torch.uint8)[None, :, None]
    q[..., 0] = 2.0**-120 * torch.linspace(-8, 8, q.shape[0] * q.shape[1]).view(q.shape[:3]).bfloat16()
    out, lse = _decode(q, k, v, ks, vs, table, lens)
    U.check(out, lse, U.attend(q, k, v, ks, vs, table, lens, "NHD"), p_bits=torch.float16)


def test_a_scale_that_makes_all_scores_zero():
    """Scale and queries so small that their product is no number: every key has the same weight."""
    q, k, v, ks, vs, _, table, lens = _setup(11, torch.bfloat16, True, 3, 8, 2, 128, 16, 0, 9, "NHD")
    q *= 2.0**-60
    want = U.attend(q, k, v, ks, vs, table, lens, "NHD", scale=2.0**-100)
    out, lse = _decode(q, k, v, ks, vs, table, lens, scale=2.0**-100)
    U.check(out, lse, want)

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


def _abs_check(out, lse, q, k, v, ks, vs, table, lens):
    """Against the weights times the values' magnitudes, which no large row without weight is part of: one rounding of the result,
    probabilities of 16 bits or more (2^-17 of each) and the fp32 arithmetic of exponents up to 2^5 (see cache_util.check): 2^-16 of
    that sum covers both.  A block without a row 2^-10 of the largest has 2^-25 of the largest probability's 2^9 2^-10 at worst, for
    each key: 300 keys, 2^-16 once more."""
    ref, ref_l, _ = U.attend(q, k, v, ks, vs, table, lens, "NHD")
    size, _, _ = U.attend(q, k, (v.view(torch.uint8) & 127).view(U.F8), ks, vs, table, lens, "NHD")
    got = out.double()
    room = torch.finfo(out.dtype).eps / 2 * ref.abs() + 2.0**-15 * size + (2.0**-25 if out.dtype == torch.float16 else 0.0)
    assert torch.isfinite(got).all() and ((got - ref).abs() <= room).all(), ((got - ref).abs() - room).max()
    dead = ref_l == -math.inf
    assert torch.equal(lse == -math.inf, dead)
    assert ((lse.double() - ref_l).abs() <= 2.0**-16 * (1 + ref_l.abs()))[~dead].all()


@pytest.mark.parametrize("dtype,Hq,Hkv,D,page", [(torch.bfloat16, 8, 2, 128, 16), (torch.float16, 16, 1, 128, 32), (torch.bfloat16, 20, 1, 64, 4), (torch.float16, 3, 3, 64, 32)])
@pytest.mark.parametrize("power", [12, 20, 27, 40, 90])
def test_a_large_value_row_without_weight(dtype, Hq, Hkv, D, page, power):
    """Some keys with value rows 2^power above the others have scores 300 and more below: none of their bits, and all of the others', are seen,
    whether such a row comes before the others, among them, or last."""
    q, k, v, ks, vs, _, table, lens = _setup(12, dtype, True, 3, Hq, Hkv, D, page, 0, 288 // page, "NHD")
    lens[0] = 288 // page * page
    q[..., 0] = 1024
    rows_k, rows_v, codes = k.view(torch.uint8), v.view(torch.uint8), vs.view(torch.uint8)
    rows_k[..., 0] = 0
    ks.view(torch.uint8).fill_(127 - 7)
    for b, where in enumerate(((0, 1, 2), (40, 100, 170), (3, int(lens[2]) - 1))):
        for s in where:
            if 0 <= s < int(lens[b]) - (b == 2 and s == 3):
                at = (int(table[b, s // page]), s % page)
                rows_k[at][:, 0] = 0xFE                      # -448 / 128: scores of -3584 / sqrt(D)
                codes[at] += power
    out, lse = _decode(q, k, v, ks, vs, table, lens)
    _abs_check(out, lse, q, k, v, ks, vs, table, lens)


def test_rows_of_zeros_among_very_small_ones():
    """A row of zeros has the scale 1; the others' are 2^-60."""
    q, k, v, ks, vs, _, table, lens = _setup(13, torch.bfloat16, True, 3, 8, 2, 128, 16, 0, 18, "NHD")
    vs.view(torch.uint8)[:] -= 52
    v.view(torch.uint8)[:, ::5] = 0
    vs.view(torch.uint8)[:, ::5] = 127
    out, lse = _decode(q, k, v, ks, vs, table, lens)
    _abs_check(out, lse, q, k, v, ks, vs, table, lens)


@pytest.mark.parametrize("which", ["key", "value"])
def test_nan_bytes_where_the_product_is_a_bf16_one(which):
    q, k, v, ks, vs, _, table, lens = _setup(14, torch.bfloat16, True, 2, 4, 1, 64, 16, 0, 4, "NHD")
    lens[:] = 64
    if which == "key":
        q[..., 1] = 2.0**-100                                # (fp16 does not hold the row)
        k.view(torch.uint8)[int(table[0, 1]), 3, 0, 7] = 0x7F
    else:
        vs.view(torch.uint8)[int(table[0, 0]), 0] += 30
        v.view(torch.uint8)[int(table[0, 1]), 3, 0, 7] = 0xFF
    out, _ = _decode(q, k, v, ks, vs, table, lens)
    assert out[1].isfinite().all() and out[0, :, 0, 7].isnan().all()
    assert which == "key" or out[0, :, 0, :7].isfinite().all()

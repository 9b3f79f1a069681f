"""A page number outside the pool: which kernel reads the page is a matter of sizes, what is reported and read instead is not."""

import pytest
import torch

from tests import cache_util as U
from tests.test_gpu_shared_prefix import _cuda, _setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quantised,page,B,P", [
    (False, 16, 3, 80), (False, 4, 3, 20), (True, 16, 3, 80), (True, 4, 3, 20), (True, 256, 3, 1280),   # before each sequence's keys
    (False, 16, 500, 80), (False, 256, 300, 1280),                                                     # once for all, in its pages
    (False, 4, 2000, 20), (True, 16, 1500, 80),                                                        # ... and gathered
    (True, 16, 3, 0), (True, 4, 3, 0),                                                                 # no prefix
])
def test_what_is_reported_and_read_instead(quantised, page, B, P):
    import torch_neuronx_b200 as T

    q, k, v, ks, vs, prefix, table, lens = _setup(5, torch.bfloat16, quantised, B, 4, 2, 64, page, P, 3, "NHD")
    lens[0] = 3 * page
    n = k.shape[0]
    dev = _cuda(q, k, v, ks, vs)
    for which, number in (("prefix", n), ("prefix", -1), ("own", n + 7), ("own", -2147483648)):
        if which == "prefix" and P == 0:
            continue
        bad_p, bad_t, got_p, got_t = prefix.clone(), table.clone(), prefix.clone(), table.clone()
        if which == "prefix":
            bad_p[2], got_p[2], said = number, 0, f"role=-1 step={2 * page} extra={n}$"
        else:
            bad_t[0, 1], got_t[0, 1], said = number, 0, f"role=0 step={page} extra={n}$"
        out, lse = T.shared_prefix_decode(*dev[:3], bad_p.cuda(), P, bad_t.cuda(), lens.cuda(), need_lse=True, k_scales=dev[3], v_scales=dev[4])
        with pytest.raises(RuntimeError, match=said):
            T.check_device_status()
        U.check(out.cpu(), lse.cpu(), U.attend(q, k, v, ks, vs, got_t, lens, "NHD", prefix=got_p, P=P), p_bits=torch.bfloat16)


def test_rows_read_back_are_zeros():
    import torch_neuronx_b200 as T

    _, k, v, ks, vs, _, table, _ = _setup(6, torch.bfloat16, True, 2, 4, 2, 64, 8, 0, 3, "NHD")
    bad = table.clone()
    bad[1, 2] = k.shape[0]
    lens = torch.full((2,), 24, dtype=torch.int32)
    got = T.paged_read(*_cuda(k, v, ks, vs), bad.cuda(), lens.cuda())
    with pytest.raises(RuntimeError, match=f"role=1 step=16 extra={k.shape[0]}$"):
        T.check_device_status()
    for x, pool, scale in zip(got, (k, v), (ks, vs)):
        for b in range(2):
            want = U.rows_of(pool, scale, table[b], 24, "NHD").transpose(0, 1)
            if b == 1:
                want[:, 16:] = 0
            assert torch.equal(x[b].cpu().double(), want)

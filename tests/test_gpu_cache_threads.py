"""Decode of a cache from several threads that share a stream: their launches may interleave, their scratch must not be the same."""

import threading

import pytest
import torch

from tests.test_gpu_shared_prefix import _cuda, _setup

pytestmark = pytest.mark.gpu

FORMS = {   # quantised, B, P
    "8-bit": (True, 6, 0), "8-bit, prefix before each": (True, 3, 200), "8-bit, prefix once": (True, 300, 3000), "16-bit, prefix once": (False, 300, 1500),
}


@pytest.mark.parametrize("direct", [False, True])
@pytest.mark.parametrize("form", FORMS)
def test_two_threads_on_one_stream(form, direct):
    """Every call gives the bits that it gives alone.  (An integer as scale is not for the direct route.)"""
    import torch_neuronx_b200 as T

    quantised, B, P = FORMS[form]
    sets = [_cuda(*_setup(s, torch.bfloat16, quantised, B, 8, 2, 128, 16, P, 3 + s, "NHD")) for s in (1, 2)]

    def call(d):
        return T.shared_prefix_decode(d[0], d[1], d[2], d[5], P, d[6], d[7], scale=1.0 if direct else 1, need_lse=True, k_scales=d[3], v_scales=d[4])

    want = [call(d) for d in sets]
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(2)

    def work(i):
        try:
            start.wait(30)
            for n in range(150):
                out, lse = call(sets[i])
                if n % 10 == 0 or n > 140:
                    same = torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])
                    if not same:
                        wrong.append((i, n))
        except Exception as e:   # noqa: BLE001
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    torch.cuda.synchronize()
    T.check_device_status()
    assert not wrong, wrong

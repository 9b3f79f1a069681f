"""A wait that runs out in the decode kernels of an 8-bit cache: the CTA lets its copies land and returns, the merge behind it follows no
slot that was not noted, and the context stays usable.  As in test_gpu_timeout.py nothing is injected: a child process sets a
wait limit of a few dozen cycles, so the first wait for a copy runs out."""

import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r"""
import json, sys, torch
sys.path.insert(0, {root!r})
import torch_neuronx_b200 as T
from oracle import sdpa_oracle as O
from tests import cache_util as U
from tests.test_gpu_shared_prefix import _cuda, _setup

res = []
# keys alone (pages by tensor copies, and rows of small pages), sixteen query heads, and a prefix before each sequence's keys or
# once for all
for dtype, B, Hq, Hkv, D, page, P, pages in ((torch.bfloat16, 5, 8, 2, 128, 16, 0, 40), (torch.float16, 4, 6, 3, 64, 4, 0, 150),
                                             (torch.bfloat16, 2, 16, 1, 128, 32, 0, 30), (torch.bfloat16, 3, 4, 2, 64, 16, 300, 20),
                                             (torch.float16, 130, 4, 2, 64, 16, 2048, 3)):
    q, k, v, ks, vs, prefix, table, lens = _setup(3, dtype, True, B, Hq, Hkv, D, page, P, pages, "NHD")
    dq, dk, dv, dks, dvs, dp, dt, dl = _cuda(q, k, v, ks, vs, prefix, table, lens)
    got = []
    for _ in range(3):   # (the scratch of the second and third holds what the one before left)
        out, lse = T.shared_prefix_decode(dq, dk, dv, dp, P, dt, dl, need_lse=True, k_scales=dks, v_scales=dvs)
        torch.cuda.synchronize()
        try:
            T.check_device_status()
            got.append("ok")
        except RuntimeError as e:
            got.append(str(e))
    right = ""
    if got[-1] == "ok":
        try:
            U.check(out.cpu(), lse.cpu(), U.attend(q, k, v, ks, vs, table, lens, "NHD", prefix=prefix, P=P), p_bits=dtype)
        except AssertionError as e:
            right = str(e)
    x = torch.arange(1000, device="cuda").sum().item()
    f = torch.randn(1, 1, 128, 128, generator=torch.Generator().manual_seed(1))
    o2, _ = T.sdpa_forward(f.cuda(), f.cuda(), f.cuda(), scale=0.1)   # (a kernel without barrier waits)
    torch.cuda.synchronize()
    res.append(dict(status=got, right=right, torch_ok=x == 499500, after=float((o2.cpu() - O.sdpa_forward(f, f, f, scale=0.1)[0]).abs().max())))
print("RESULT " + json.dumps(res))
"""


def _run_child(extra_env):
    env = dict(os.environ)
    env.pop("B200_SDPA_WAIT_LIMIT", None)
    env.update(extra_env)
    proc = subprocess.run([sys.executable, "-c", CHILD.format(root=ROOT)], env=env, capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stdout + proc.stderr
    line = [ln for ln in proc.stdout.splitlines() if ln.startswith("RESULT ")][-1]
    return json.loads(line[len("RESULT "):])


def test_a_wait_that_runs_out_is_reported_and_the_context_survives():
    for res in _run_child({"B200_SDPA_WAIT_LIMIT": "64"}):
        assert all("device status 10" in s and "gave up" in s for s in res["status"]), res
        assert res["torch_ok"] and res["after"] <= 1e-5, res


def test_the_same_calls_with_the_default_limit_are_correct():
    for res in _run_child({}):
        assert res["status"] == ["ok"] * 3 and res["right"] == "", res
        assert res["torch_ok"] and res["after"] <= 1e-5, res

"""Rotary embedding and the cache operators under tracers and transforms, which see nothing of a call by pointers: recorded or
refused, never lost."""

import pytest
import torch

from tests.test_gpu_rotary import _freqs
from tests.test_gpu_shared_prefix import _cuda, _setup

pytestmark = pytest.mark.gpu


def _calls():
    """name -> (function of one tensor, that tensor)"""
    import torch_neuronx_b200 as T

    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 4, 8, 64, generator=g).bfloat16().cuda()
    pos, freq = torch.arange(8, device="cuda"), _freqs(64).cuda()
    q, k, v, ks, vs, prefix, table, lens = _cuda(*_setup(3, torch.bfloat16, True, 3, 4, 2, 64, 16, 40, 3, "NHD"))
    q16, k16, v16, _, _, prefix16, table16, lens16 = _cuda(*_setup(3, torch.bfloat16, False, 3, 4, 2, 64, 16, 40, 3, "NHD"))
    pools16 = (k16, v16)
    rows = torch.randn(3, 2, 5, 64, generator=g).bfloat16().cuda()

    def write(t):
        T.paged_write(t, rows, k, v, ks, vs, table, torch.zeros_like(lens))
        return t * 2

    return {
        "rotary": (lambda t: T.rotary_embedding(t, t, pos, freq)[1], x),
        "write": (write, rows),
        "read": (lambda t: T.paged_read(k, v, ks, t, table, lens)[1], vs.view(torch.uint8)),
        "decode": (lambda t: T.paged_decode(t, k, v, table, lens, k_scales=ks, v_scales=vs)[0], q),
        "shared": (lambda t: T.shared_prefix_decode(t, k, v, prefix, 40, table, lens, k_scales=ks, v_scales=vs)[0], q),
        "shared16": (lambda t: T.shared_prefix_decode(t, *pools16, prefix16, 40, table16, lens16)[0], q16),
    }


NAMES = ["rotary", "write", "read", "decode", "shared", "shared16"]


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("tracer", ["jit", "make_fx", "make_fx_fake"])
def test_a_trace_is_refused(name, tracer):
    """(It used to record the allocation of a result and nothing else.)"""
    f, x = _calls()[name]
    f(x)
    with pytest.raises(Exception if tracer == "make_fx_fake" else RuntimeError, match="" if tracer == "make_fx_fake" else "a trace cannot record"):
        if tracer == "jit":
            torch.jit.trace(f, (x,), check_trace=False)
        else:
            from torch.fx.experimental.proxy_tensor import make_fx

            make_fx(f, tracing_mode="real" if tracer == "make_fx" else "fake")(x)
    f(x)   # nothing of the trace is left
    torch.cuda.synchronize()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("transform", ["grad", "vjp", "vmap", "jvp"])
def test_function_transforms_are_refused(name, transform):
    f, x = _calls()[name]
    if name == "read" and transform in ("vjp", "jvp"):
        return   # (bytes have neither)
    with pytest.raises(RuntimeError, match="transform"):
        if transform == "grad":
            torch.func.grad(lambda t: t * f(x).float().sum())(torch.tensor(3.0, device="cuda"))   # (nor inside one of something else)
        elif transform == "vjp":
            torch.func.vjp(f, x)
        elif transform == "jvp":
            torch.func.jvp(f, (x,), (torch.ones_like(x),))
        else:
            torch.func.vmap(f)(torch.stack((x, x)))

"""Rotary embedding and the cache operators under tracers and transforms, which see nothing of a call by pointers: recorded or
refused, never lost."""

import pytest
import torch

from tests.test_gpu_rotary import _check, _freqs, _want
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


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_tangents(interleaved):
    """A rotation is linear: the tangent is rotated like its tensor, and the gradient flows beside it."""
    import torch.autograd.forward_ad as fw

    import torch_neuronx_b200 as T

    g = torch.Generator().manual_seed(5)
    q, k, tq, tk = (torch.randn(2, h, 7, 32, generator=g) for h in (3, 2, 3, 2))
    pos, freq, sections = torch.randint(0, 900, (2, 2, 7), generator=g), _freqs(24), (5, 7)
    args = (pos.cuda(), freq.cuda())
    kw = dict(sections=sections, interleaved=interleaved)
    with fw.dual_level():
        for which in ("both", "query", "key", "alone"):
            dq = fw.make_dual(q.cuda(), tq.cuda()) if which != "key" else q.cuda()
            dk = fw.make_dual(k.cuda(), tk.cuda()) if which in ("both", "key") else k.cuda()
            y, z = T.rotary_embedding(dq, None if which == "alone" else dk, *args, **kw)
            for got, x, t, has in ((y, q, tq, which != "key"), (z, k, tk, which in ("both", "key"))):
                if got is None:
                    assert which == "alone"
                    continue
                primal, tangent = fw.unpack_dual(got)
                _check(primal.cpu(), _want(x, pos, freq, sections, interleaved))
                assert (tangent is not None) == has
                if has:
                    _check(tangent.cpu(), _want(t, pos, freq, sections, interleaved))
        leaf = q.cuda().requires_grad_()
        y, _ = T.rotary_embedding(fw.make_dual(leaf * 1, tq.cuda()), None, *args, **kw)
        (d,) = torch.autograd.grad(y, leaf, tq.cuda())
        _check(d.cpu(), _want(tq, pos, freq, sections, interleaved, -1.0))
        with pytest.raises(RuntimeError, match="forward-mode"):
            T.rotary_embedding(q.cuda(), None, args[0], fw.make_dual(args[1], args[1]), **kw)


def test_tangents_of_the_cache_operators_are_refused():
    import torch.autograd.forward_ad as fw

    for name, (f, x) in _calls().items():
        if name in ("rotary", "read"):
            continue
        with fw.dual_level(), pytest.raises((NotImplementedError, RuntimeError)):
            f(fw.make_dual(x, torch.ones_like(x)))


def test_a_gradient_of_the_frequencies_is_refused():
    import torch_neuronx_b200 as T

    q, pos = torch.randn(1, 2, 5, 32, device="cuda"), torch.arange(5, device="cuda")
    freq = torch.rand(16, device="cuda", requires_grad=True)
    for x in (q, q.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="inv_freq"):
            T.rotary_embedding(x, None, pos, freq)
        with torch.no_grad():
            T.rotary_embedding(x, None, pos, freq)
        T.rotary_embedding(x, None, pos, freq.detach())

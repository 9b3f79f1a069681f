"""Rotary embedding with several axes: against 64 bits, its gradient against the formula and against differences."""

import contextlib
import gc
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _want(x, positions, inv_freq, sections, interleaved, sign=1.0):
    """The rotation in 64 bits on the CPU; positions (axes, B, L)."""
    R = 2 * inv_freq.shape[0]
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)])
    angle = sign * positions.double()[axis].permute(1, 2, 0) * inv_freq.double()   # (B, L, R/2)
    t = torch.polar(torch.ones_like(angle), angle)[:, None]
    y = x.double().clone()
    i = torch.arange(R // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    z = torch.complex(y[..., a], y[..., b]) * t
    y[..., a], y[..., b] = z.real, z.imag
    pair = torch.zeros_like(y)
    pair[..., a] = pair[..., b] = x.double()[..., a].abs() + x.double()[..., b].abs()
    return y, pair


def _check(got, want):
    """One rounding (eps / 2), and sine, cosine and two products in fp32: 2^-21 of the pair's size."""
    y, pair = want
    room = torch.finfo(got.dtype).eps / 2 * y.abs() + 2.0**-21 * pair
    if got.dtype == torch.float16:
        room = room + 2.0**-25
    over = ((got.double() - y).abs() - room).max().item()
    assert over <= 0, over


def _freqs(R, base=10000.0):
    return torch.tensor([base ** (-2 * i / R) for i in range(R // 2)], dtype=torch.float64)


CASES = [
    # dtype, B, Hq, Hkv, L, D, R, sections, interleaved, far
    (torch.bfloat16, 2, 8, 2, 37, 128, 128, (16, 24, 24), False, 4096),
    (torch.float16, 3, 4, 4, 1, 64, 64, (32,), True, 1000000),
    (torch.float32, 1, 6, 2, 130, 80, 80, (10, 20, 10), False, 500000),
    (torch.bfloat16, 2, 3, 1, 5, 96, 32, (4, 4, 4, 4), True, 100),
    (torch.float32, 2, 5, 5, 3, 18, 6, (0, 3), False, 50),          # nothing is a whole piece, an axis without pairs
    (torch.bfloat16, 1, 1, 1, 700, 256, 256, (128,), False, 10),
    (torch.float16, 65, 12, 12, 41, 64, 48, (24,), False, 9000),    # 2665 tokens: four to a CTA, ragged
    (torch.float32, 2, 3, 2, 9, 7, 4, (2,), False, 70),             # odd head dims: one element to copy, and three
    (torch.bfloat16, 3, 2, 1, 6, 5, 4, (1, 1), True, 70),
    (torch.float16, 1, 30, 7, 11, 33, 2, (1,), False, 700),
]


@pytest.mark.parametrize("dtype,B,Hq,Hkv,L,D,R,sections,interleaved,far", CASES)
def test_rotation_and_its_gradient(dtype, B, Hq, Hkv, L, D, R, sections, interleaved, far):
    import torch_neuronx_b200 as T

    g = torch.Generator().manual_seed(L * D)
    q, k = (torch.randn(B, L, h, D, generator=g).to(dtype).transpose(1, 2) for h in (Hq, Hkv))
    gq, gk = (torch.randn(B, h, L, D, generator=g).to(dtype) for h in (Hq, Hkv))
    pos = torch.randint(-3, far, (len(sections), B, L), generator=g)
    freq = _freqs(R)
    qd, kd = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    yq, yk = T.rotary_embedding(qd, kd, pos.cuda(), freq.cuda(), sections=sections, interleaved=interleaved)
    assert yq.stride() == qd.stride() and yk.stride() == kd.stride()
    dq, dk = torch.autograd.grad((yq, yk), (qd, kd), (gq.cuda(), gk.cuda()))
    T.check_device_status()
    for got, x, sign in ((yq, q, 1), (yk, k, 1), (dq, gq, -1), (dk, gk, -1)):
        _check(got.detach().cpu(), _want(x, pos, freq, sections, interleaved, sign))
    # int32 positions, fp32 frequencies, the keys left out
    y32, none = T.rotary_embedding(q.cuda(), None, pos.int().cuda(), freq.float().cuda(), sections=sections, interleaved=interleaved)
    assert none is None
    _check(y32.cpu(), _want(q, pos, freq.float(), sections, interleaved))


def test_gradient_against_differences():
    """The scalar sum(w * y) changes by its gradient times a step; the function is linear, so only fp32 rounding is left: a
    sum of n terms of about 1 carries some n 2^-24."""
    import torch_neuronx_b200 as T

    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn(1, h, 4, 32, generator=g).cuda().requires_grad_() for h in (2, 1))
    pos = torch.randint(0, 99, (2, 1, 4), generator=g).cuda()
    freq = _freqs(24).cuda()
    wq, wk = torch.randn(q.shape, generator=g).cuda(), torch.randn(k.shape, generator=g).cuda()

    def f(a, b):
        y, z = T.rotary_embedding(a, b, pos, freq, sections=(5, 7))
        return (wq * y).double().sum() + (wk * z).double().sum()

    dq, dk = torch.autograd.grad(f(q, k), (q, k))
    for x, d, n in ((q, dq, 0), (k, dk, 1)):
        step = torch.randn(x.shape, generator=g).cuda()
        at = [q.detach(), k.detach()]
        up, down = list(at), list(at)
        up[n], down[n] = at[n] + step, at[n] - step
        slope = (f(*up) - f(*down)) / 2
        assert abs(slope.item() - (d.double() * step).sum().item()) <= x.numel() * 2.0**-22
    # twice differentiable: the gradient of the gradient is the rotation again
    y, _ = T.rotary_embedding(q, k, pos, freq, sections=(5, 7))
    g1 = torch.randn(y.shape, generator=g).cuda().requires_grad_()
    (d,) = torch.autograd.grad(y, q, g1, create_graph=True)
    (again,) = torch.autograd.grad(d, g1, wq)
    _check(again.cpu(), _want(wq.cpu(), pos.cpu(), freq.cpu(), (5, 7), False))
    # the query alone, and only the keys' gradient
    y, _ = T.rotary_embedding(q, None, pos, freq, sections=(5, 7))
    (d,) = torch.autograd.grad(y, q, wq)
    _check(d.cpu(), _want(wq.cpu(), pos.cpu(), freq.cpu(), (5, 7), False, -1.0))
    _, z = T.rotary_embedding(q.detach(), k, pos, freq, sections=(5, 7))
    (d,) = torch.autograd.grad(z, k, wk)
    _check(d.cpu(), _want(wk.cpu(), pos.cpu(), freq.cpu(), (5, 7), False, -1.0))


def test_strides_broadcasts_and_single_gradients():
    import torch_neuronx_b200 as T

    g = torch.Generator().manual_seed(2)
    B, L, D = 2, 9, 64
    qkv = torch.randn(B, L, 3, 4, D + 1, generator=g)[..., 1:]           # unaligned rows
    q = qkv[:, :, 0].transpose(1, 2)
    k = torch.randn(1, 1, L, D, generator=g).expand(B, 2, L, D)          # stride 0
    pos = torch.arange(L)                                                # (L,)
    freq = _freqs(D)
    full = pos.expand(1, B, L)
    qd, kl = q.cuda(), torch.randn(1, 1, L, D, generator=g).cuda().requires_grad_()
    qd = qkv.cuda()[:, :, 0].transpose(1, 2)
    yq, yk = T.rotary_embedding(qd, k.cuda()[:, :1].expand(B, 2, L, D), pos.cuda(), freq.cuda())
    _check(yq.cpu(), _want(q, full, freq, (D // 2,), False))
    _check(yk.cpu(), _want(k, full, freq, (D // 2,), False))
    # a broadcast leaf, its gradient from an expanded scalar; the query wants none
    _, yk = T.rotary_embedding(qd, kl.expand(B, 3, L, D), pos.cuda(), freq.cuda())
    (dk,) = torch.autograd.grad(yk.sum(), kl)
    one, pair = _want(torch.ones(B, 3, L, D), full, freq, (D // 2,), False, -1.0)
    # six fp32 terms are added: six roundings of the running sum
    assert ((dk.cpu().double() - one.sum((0, 1), keepdim=True)).abs() <= 6 * (2.0**-21 * 2 + 2.0**-24 * 9)).all()
    # (B, L) positions, and the transposed result of the far dimension order
    y, _ = T.rotary_embedding(qd, None, pos.expand(B, L).contiguous().cuda(), freq.cuda())
    assert torch.equal(y, yq)
    # nothing to do
    e, f = T.rotary_embedding(qd[:, :, :0], None, pos[:0].cuda(), freq.cuda())
    assert e.shape == (B, 4, 0, D) and f is None


def test_other_stream_and_captured_graph():
    import torch_neuronx_b200 as T

    g = torch.Generator().manual_seed(3)
    q = torch.randn(4, 8, 1, 128, generator=g).bfloat16()
    pos = torch.randint(0, 5000, (3, 4, 1), generator=g)
    freq = _freqs(128)
    dq, dp, df = q.cuda(), pos.cuda(), freq.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, _ = T.rotary_embedding(dq, None, dp, df, sections=(16, 24, 24))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            z, _ = T.rotary_embedding(dq, None, dp, df, sections=(16, 24, 24))
    side.synchronize()
    _check(y.cpu(), _want(q, pos, freq, (16, 24, 24), False))
    dp.add_(7)
    graph.replay()
    torch.cuda.synchronize()
    _check(z.cpu(), _want(q, pos + 7, freq, (16, 24, 24), False))


def _capture_parts():
    import torch_neuronx_b200 as T

    g = torch.Generator().manual_seed(8)
    q, k = (torch.randn(2, 5, h, 64, generator=g).transpose(1, 2) for h in (4, 2))
    gq, gk = (torch.randn(2, h, 5, 64, generator=g) for h in (4, 2))
    pos = torch.randint(0, 300, (2, 5), generator=g)
    freq = _freqs(64)
    dev = [t.cuda() for t in (q, k, gq, gk, pos, freq)]
    lq, lk = dev[0].requires_grad_(), dev[1].requires_grad_()

    def forward():
        return T.rotary_embedding(lq, lk, dev[4], dev[5])

    def step():
        out = forward()
        return out + torch.autograd.grad(out, (lq, lk), (dev[2], dev[3]))

    def replayed(graph, got):
        with torch.no_grad():
            lq.mul_(-2)
            dev[3].add_(1)
        graph.replay()
        torch.cuda.synchronize()
        full = pos.expand(1, 2, 5)
        for y, x, sign in zip(got, (q * -2, k, gq, gk + 1), (1, 1, -1, -1)):
            _check(y.detach().cpu(), _want(x, full, freq, (32,), False, sign))

    return forward, step, replayed


def test_gradient_captured_while_an_eager_graph_lives():
    """A training step's rotation and its gradient are captured and replayed with new inputs; an eager graph of the same
    leaves, built on the stream that is captured, is alive all the while."""
    forward, step, replayed = _capture_parts()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = forward()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    side.synchronize()
    replayed(graph, got)
    assert alive[0].grad_fn is not None


@pytest.mark.parametrize("direct", [True, False])
def test_gradient_captured_while_a_default_stream_graph_lives_is_refused(direct):
    """The engine would make the default stream wait for the capture.  The call is refused while the capture is whole: it
    ends without an error of its own, and once the eager graph is gone the same leaves are captured and replayed.  Under a
    mode that sees every call the Python layer's function does the same."""
    from torch_neuronx_b200 import _lib

    if _lib.native is None:
        pytest.skip("without the direct entry points the engine's own error ends the capture")
    forward, plain_step, replayed = _capture_parts()

    def step():
        with contextlib.nullcontext() if direct else torch.device("cuda"):
            return plain_step()

    alive = forward()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with pytest.raises(RuntimeError, match="eager graph from the default stream"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                step()
        step()   # eager, the older graph still alive
        side.synchronize()
        del alive
        gc.collect()   # (the refused step's frames, which the exception holds)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    side.synchronize()
    replayed(graph, got)


def test_refusals():
    import torch_neuronx_b200 as T

    q = torch.zeros(2, 4, 8, 64, device="cuda")
    pos = torch.zeros(2, 8, dtype=torch.int64, device="cuda")
    freq = torch.ones(32, device="cuda")
    bad = [
        ((q[0], None, pos, freq), {}, "4-D"),
        ((q.double(), None, pos, freq), {}, "float32, float16"),
        ((q, q[:, :, :7], pos, freq), {}, "share"),
        ((q, None, pos.float(), freq), {}, "int32 or int64"),
        ((q, None, pos[:, :7], freq), {}, "broadcast"),
        ((q, None, pos.expand(3, 2, 8), freq), {}, "sections"),
        ((q, None, pos.expand(3, 2, 8), freq), {"sections": (16, 16)}, "sections"),
        ((q, None, pos.expand(2, 2, 8), freq), {"sections": (16, 17)}, "sections"),
        ((q, None, pos.expand(2, 2, 8), freq), {"sections": (-1, 33)}, "sections"),
        ((q, None, pos.expand(5, 2, 8), freq), {"sections": (8, 8, 8, 8, 0)}, "sections"),
        ((q, None, pos, torch.ones(33, device="cuda")), {}, "room"),
        ((q, None, pos, freq.half()), {}, "float32 or float64"),
        ((q, None, pos, torch.ones(64, device="cuda")[::2]), {}, "contiguous"),
    ]
    for args, kw, text in bad:
        with pytest.raises(RuntimeError, match=text):
            T.rotary_embedding(*args, **kw)
    with pytest.raises(ValueError, match="CUDA"):
        T.rotary_embedding(q.cpu(), None, pos, freq)
    assert math.isfinite(T.rotary_embedding(q, None, pos, freq)[0].sum().item())

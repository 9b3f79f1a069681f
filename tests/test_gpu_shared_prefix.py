"""Decode for a batch that shares a prefix: against 64 bits, and the operators of a serving step run together."""

import math

import pytest
import torch

from tests import cache_util as U

pytestmark = pytest.mark.gpu

CASES = [
    # dtype, quantised, B, Hq, Hkv, D, page, P, own pages, layout
    (torch.bfloat16, False, 5, 8, 2, 128, 16, 300, 3, "NHD"),
    (torch.float16, True, 3, 4, 4, 64, 64, 129, 2, "HND"),
    (torch.bfloat16, True, 40, 32, 8, 128, 32, 1000, 2, "NHD"),     # several row tiles
    (torch.float16, False, 70, 4, 1, 64, 8, 640, 4, "HND"),
    (torch.bfloat16, False, 1, 6, 2, 64, 1, 37, 5, "NHD"),
    (torch.float16, True, 2, 48, 1, 128, 16, 1, 1, "NHD"),          # a prefix of one key, 48 query heads
    (torch.bfloat16, True, 130, 2, 2, 64, 128, 2048, 1, "HND"),
    (torch.bfloat16, False, 7, 5, 1, 128, 16, 0, 3, "NHD"),         # no prefix
    (torch.bfloat16, True, 7, 5, 1, 128, 16, 0, 3, "NHD"),
    (torch.float16, False, 4, 8, 2, 128, 16, 77, 0, "NHD"),         # nothing but the prefix
    (torch.float16, True, 300, 3, 3, 64, 4, 50, 2, "HND"),
    (torch.bfloat16, True, 64, 16, 8, 64, 4, 900, 2, "NHD"),        # small pages, gathered
    (torch.float16, True, 1, 40, 2, 128, 16, 3000, 0, "HND"),       # one sequence with nothing of its own, twenty query heads
    (torch.bfloat16, False, 64, 16, 2, 128, 16, 1000, 3, "NHD"),    # 16-bit, the prefix once for all: in its pages ...
    (torch.float16, False, 70, 8, 4, 64, 8, 643, 4, "HND"),
    (torch.bfloat16, False, 40, 6, 2, 64, 1, 1501, 5, "NHD"),       # ... and gathered
    (torch.float16, False, 3, 40, 2, 64, 2, 333, 40, "HND"),        # 16-bit likewise, twenty query heads
    (torch.bfloat16, False, 1, 8, 1, 128, 16, 5001, 7, "NHD"),      # many ranges, most of the prefix
    (torch.bfloat16, True, 6, 8, 2, 128, 2, 333, 40, "NHD"),        # small pages, the prefix before each sequence's keys
]


def _setup(seed, dtype, quantised, B, Hq, Hkv, D, page, P, pages, layout):
    g = torch.Generator().manual_seed(seed)
    shared = -(-P // page)
    n = B * pages + shared + 2
    order = torch.randperm(n, generator=g).to(torch.int32)
    table, prefix = order[: B * pages].view(B, pages), order[B * pages: B * pages + shared].contiguous()
    k, v, ks, vs = U.make_pools(g, n, page, Hkv, D, dtype, quantised, layout)
    lens = torch.randint(0, pages * page + 1, (B,), generator=g).to(torch.int32)
    lens[-1] = 0
    return torch.randn(B, Hq, 1, D, generator=g).to(dtype), k, v, ks, vs, prefix, table, lens


def _cuda(*ts):
    return tuple(t.cuda() if t is not None else None for t in ts)


@pytest.mark.parametrize("dtype,quantised,B,Hq,Hkv,D,page,P,pages,layout", CASES)
def test_against_64_bits(dtype, quantised, B, Hq, Hkv, D, page, P, pages, layout):
    import torch_neuronx_b200 as T

    q, k, v, ks, vs, prefix, table, lens = _setup(B + P, dtype, quantised, B, Hq, Hkv, D, page, P, pages, layout)
    want = U.attend(q, k, v, ks, vs, table, lens, layout, prefix=prefix, P=P)
    # nothing behind the prefix's end or a sequence's end is looked at
    used = torch.zeros(k.shape[0], page, dtype=torch.bool)
    for s in range(P):
        used[prefix[s // page], s % page] = True
    for b in range(B):
        for s in range(int(lens[b])):
            used[table[b, s // page], s % page] = True
    for pool in (k, v):
        at = pool if layout == "NHD" else pool.transpose(1, 2)
        if quantised:
            at.view(torch.uint8)[~used] = 0x7F
        else:
            at[~used] = math.nan
    dev = _cuda(q, k, v, prefix)
    T.reset_launch_counts()
    out, lse = T.shared_prefix_decode(*dev, P, *_cuda(table, lens), layout=layout, need_lse=True, k_scales=_cuda(ks)[0], v_scales=_cuda(vs)[0])
    T.check_device_status()
    U.check(out.cpu(), lse.cpu(), want, p_bits=dtype)
    assert T.launch_counts()["generic"] == 0
    # without the log-sum-exp, into a given result; the same bits
    mine = torch.full_like(out, math.nan)
    got, none = T.shared_prefix_decode(*dev, P, *_cuda(table, lens), layout=layout, out=mine, k_scales=_cuda(ks)[0], v_scales=_cuda(vs)[0])
    assert none is None and got is mine and torch.equal(mine, out)


def test_largest_fp16_rows_of_an_8_bit_prefix():
    """e4m3 makes 65536 of fp16's largest numbers.  Such keys and values, in a prefix that is gathered as fp16, count as 65504, 2^-11
    less: scores q k / 8 of at most 2^-14 * 65536 / 8 = 1/2 are off by at most 2^-12 each, probabilities by a factor within e^(2^-11), so
    the result by 2^-11 of the largest value, and another 2^-11 for the values' own rounding (on top of the usual)."""
    import torch_neuronx_b200 as T

    B, Hkv, D, page, P = 128, 2, 64, 16, 4000
    q, k, v, ks, vs, prefix, table, lens = _setup(5, torch.float16, True, B, 4, Hkv, D, page, P, 1, "NHD")
    for pool, scales in ((k, ks), (v, vs)):
        pool.zero_()
        scales.view(torch.uint8).fill_(127 + 8)
    g = torch.Generator().manual_seed(6)
    k[..., 0] = torch.randint(-1, 2, k.shape[:3], generator=g).float().mul(256).to(U.F8)      # -65536, 0, 65536
    v[..., ::3] = torch.randint(-1, 2, v[..., ::3].shape, generator=g).float().mul(256).to(U.F8)
    q = torch.zeros_like(q)
    q[..., 0] = 2.0**-14 * torch.randint(-1, 2, q.shape[:3], generator=g)
    ref, ref_l, big = U.attend(q, k, v, ks, vs, table, lens, "NHD", prefix=prefix, P=P)
    assert ref.abs().max() < 60000
    dev = _cuda(q, k, v, prefix)
    T.reset_launch_counts()
    out, lse = T.shared_prefix_decode(*dev, P, *_cuda(table, lens), need_lse=True, k_scales=_cuda(ks)[0], v_scales=_cuda(vs)[0])
    assert T.launch_counts()["cache_read"] == 1
    room = 2.0**-11 * ref.abs() + (2.0**-10 + 2.0**-11 + 2.0**-16) * big   # (probabilities in fp16: 2^-11)
    assert torch.all((out.cpu().double() - ref).abs() <= room)
    assert torch.all((lse.cpu().double() - ref_l).abs() <= 2.0**-12 + 2.0**-16 * (1 + ref_l.abs()))


def test_subnormal_key_scales():
    """Keys at 2^-127 under queries of 2^115: their products are ordinary numbers."""
    import torch_neuronx_b200 as T

    q, k, v, ks, vs, prefix, table, lens = _setup(9, torch.bfloat16, True, 3, 4, 2, 128, 16, 0, 9, "NHD")
    ks.view(torch.uint8)[..., 0] = 0
    q *= 2.0**115
    k.view(torch.uint8)[..., 1, :] = 0   # (the other head's keys are zeros: their scale is not so small)
    want = U.attend(q, k, v, ks, vs, table, lens, "NHD")
    out, lse = T.paged_decode(*_cuda(q, k, v, table, lens), need_lse=True, k_scales=_cuda(ks)[0], v_scales=_cuda(vs)[0])
    U.check(out.cpu(), lse.cpu(), want)


@pytest.mark.parametrize("B", [6, 400])   # the prefix for each sequence, and once for all
def test_other_streams_and_captured_graphs(B):
    """Two graphs that were captured one after the other do not share their scratch; replayed with new inputs."""
    import torch_neuronx_b200 as T

    sets = [_setup(s, torch.bfloat16, s == 2, B, 8, 2, 128, 16, 200 * s, 3, "NHD") for s in (1, 2)]
    graphs, outs, devs = [], [], []
    side = torch.cuda.Stream()
    for i, (q, k, v, ks, vs, prefix, table, lens) in enumerate(sets):
        dev = _cuda(q, k, v, ks, vs, prefix, table, lens)
        P = 200 * (i + 1)

        def call(d=dev, P=P):
            return T.shared_prefix_decode(d[0], d[1], d[2], d[5], P, d[6], d[7], need_lse=True, k_scales=d[3], v_scales=d[4])

        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(call())
        side.synchronize()
        graphs.append(graph)
        devs.append(dev)
    for (q, *_), dev in zip(sets, devs):
        q.neg_()
        dev[0].neg_()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    graphs[0].replay()
    with torch.cuda.stream(other):
        graphs[1].replay()
    torch.cuda.synchronize()
    T.check_device_status()
    for i, (q, k, v, ks, vs, prefix, table, lens) in enumerate(sets):
        want = U.attend(q, k, v, ks, vs, table, lens, "NHD", prefix=prefix, P=200 * (i + 1))
        U.check(outs[i][0].cpu(), outs[i][1].cpu(), want, p_bits=torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_serving_step(dtype):
    """Positions of three axes -> rotated rows -> 8-bit cache -> decode, alone and with a shared prefix, and the rows
    back for a chunk of a prompt.  The cache's rows are compared by what was rounded into them."""
    import torch_neuronx_b200 as T

    g = torch.Generator().manual_seed(21)
    B, Hq, Hkv, D, page, L, P = 4, 8, 2, 64, 16, 45, 70
    freq = torch.tensor([10000.0 ** (-2 * i / D) for i in range(D // 2)], dtype=torch.float64).cuda()
    n = 40
    kp, vp = (torch.zeros(n, page, Hkv, D, dtype=torch.uint8, device="cuda").view(U.F8) for _ in range(2))
    ks, vs = (torch.zeros(n, page, Hkv, dtype=torch.uint8, device="cuda").view(U.E8) for _ in range(2))
    order = torch.randperm(n, generator=g).to(torch.int32)
    prefix, table = order[:5].contiguous(), order[5:25].view(B, 5)

    def rows(batch, length, heads):
        return torch.randn(batch, heads, length, D, generator=g).to(dtype).cuda()

    sections = (8, 12, 12)
    pos = torch.arange(P).expand(3, 1, P)
    _, k = T.rotary_embedding(rows(1, P, Hq), rows(1, P, Hkv), pos.cuda(), freq, sections=sections)
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    T.paged_write(k, rows(1, P, Hkv), kp, vp, ks, vs, prefix.view(1, -1).cuda(), zero[:1])
    lens = torch.tensor([L, 3, 17, 44], dtype=torch.int32, device="cuda")
    pos = P + torch.arange(L).expand(3, B, L)
    _, k = T.rotary_embedding(rows(B, L, Hq), rows(B, L, Hkv), pos.cuda(), freq, sections=sections)
    T.paged_write(k, rows(B, L, Hkv), kp, vp, ks, vs, table.cuda(), zero, lens=lens)
    at = (P + lens.long()).view(1, B, 1).expand(3, B, 1)
    q, k = T.rotary_embedding(rows(B, 1, Hq), rows(B, 1, Hkv), at, freq, sections=sections)
    T.paged_write(k, rows(B, 1, Hkv), kp, vp, ks, vs, table.cuda(), lens)
    lens = lens + 1
    out, lse = T.shared_prefix_decode(q, kp, vp, prefix.cuda(), P, table.cuda(), lens, need_lse=True, k_scales=ks, v_scales=vs)
    alone, alone_lse = T.paged_decode(q, kp, vp, table.cuda(), lens, need_lse=True, k_scales=ks, v_scales=vs)
    T.check_device_status()
    host = [t.cpu() for t in (q, kp, vp, ks, vs)]
    U.check(out.cpu(), lse.cpu(), U.attend(*host, table, lens.cpu(), "NHD", prefix=prefix, P=P), p_bits=dtype)
    U.check(alone.cpu(), alone_lse.cpu(), U.attend(*host, table, lens.cpu(), "NHD"))
    # the next chunk of a prompt behind its cached rows
    K, V = T.paged_read(kp, vp, ks, vs, table.cuda(), lens, max_len=48, dtype=dtype)
    chunk = rows(B, 4, Hq)
    got, _ = T.sdpa_forward(chunk, K, V, kv_lens=lens)
    for i in range(4):
        want = U.attend(chunk[:, :, i:i + 1].cpu(), *host[1:], table, lens.cpu(), "NHD")
        U.check(got[:, :, i:i + 1].cpu(), want[1].float(), want, p_bits=dtype)


@pytest.mark.parametrize("quantised,page,B", [(False, 16, 3), (False, 4, 3), (True, 16, 3), (False, 16, 500), (False, 4, 2000), (True, 16, 1500)])
def test_a_bad_page_is_reported(quantised, page, B):
    """A number outside the pool, in the prefix or a sequence's own table, is looked over before it is used: page 0 stands in."""
    import torch_neuronx_b200 as T

    q, k, v, ks, vs, prefix, table, lens = _setup(5, torch.bfloat16, quantised, B, 4, 2, 64, page, 5 * page, 3, "NHD")
    lens[0] = 3 * page
    want = U.attend(q, k, v, ks, vs, table, lens, "NHD", prefix=prefix, P=5 * page)
    dev = _cuda(q, k, v, ks, vs)
    n = k.shape[0]
    for which, number in (("prefix", n), ("prefix", -1), ("own", n + 7), ("own", -2147483648)):
        p2, t2 = prefix.clone(), table.clone()
        if which == "prefix":
            p2[2] = number
        else:
            t2[0, 1] = number
        out, _ = T.shared_prefix_decode(*dev[:3], p2.cuda(), 5 * page, t2.cuda(), lens.cuda(), k_scales=dev[3], v_scales=dev[4])
        with pytest.raises(RuntimeError, match="page"):
            T.check_device_status()
        assert torch.isfinite(out).all()
    out, lse = T.shared_prefix_decode(*dev[:3], prefix.cuda(), 5 * page, table.cuda(), lens.cuda(), need_lse=True, k_scales=dev[3], v_scales=dev[4])
    T.check_device_status()
    U.check(out.cpu(), lse.cpu(), want, p_bits=torch.bfloat16)


def test_refusals():
    import torch_neuronx_b200 as T

    q, k, v, _, _, prefix, table, lens = _cuda(*_setup(1, torch.bfloat16, False, 3, 4, 2, 64, 16, 40, 2, "NHD"))
    ok = dict(zip("q k v p n t l".split(), (q, k, v, prefix, 40, table, lens)))
    for change, text in (({"n": -1}, "negative"), ({"n": 49}, "room"), ({"p": prefix.long()}, "prefix_table"), ({"p": prefix.view(1, -1)}, "prefix_table"),
                         ({"k": k.half(), "v": v.half()}, "pools"), ({"q": q.float()}, "float16"), ({"t": table[:2]}, "block_table"),
                         ({"l": lens[:2]}, "kv_lens"), ({"q": q[..., :32], "k": k[..., :32], "v": v[..., :32]}, "head dim"),
                         ({"q": q[:, :3]}, "heads"), ({"q": torch.cat([q] * 65, 1)}, "no kernel")):
        a = {**ok, **change}
        with pytest.raises(RuntimeError, match=text):
            T.shared_prefix_decode(*(a[x] for x in "qkvpntl"))
    T.shared_prefix_decode(*(ok[x] for x in "qkvpntl"))
    T.check_device_status()

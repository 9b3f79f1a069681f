"""The 8-bit paged cache: rows written and read back bit for bit, decode against 64 bits."""

import math

import pytest
import torch

from tests import cache_util as U

pytestmark = pytest.mark.gpu


def _table(g, B, per_seq, extra=3):
    n = B * per_seq + extra
    return n, torch.randperm(n, generator=g)[: B * per_seq].view(B, per_seq).to(torch.int32)


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("dtype,B,Hkv,L,D,page", [
    (torch.bfloat16, 3, 8, 33, 128, 16), (torch.float16, 2, 3, 50, 64, 1), (torch.bfloat16, 1, 1, 1, 256, 64),
    (torch.float16, 5, 2, 7, 16, 8), (torch.bfloat16, 2, 5, 300, 80, 32),
])
def test_rows_written_and_read_back(dtype, B, Hkv, L, D, page, layout):
    import torch_neuronx_b200 as T

    g = torch.Generator().manual_seed(B * L)
    start = torch.randint(0, 2 * page + 5, (B,), generator=g).to(torch.int32)
    lens = torch.randint(0, L + 1, (B,), generator=g).to(torch.int32)
    lens[0] = L
    per_seq = -(-(int(start.max()) + L) // page)
    n, table = _table(g, B, per_seq)
    k, v = (U.random_rows((B, L, Hkv, D), dtype, g).transpose(1, 2) for _ in range(2))
    k[0, 0, 0] = 0                                              # a row of zeros
    k[0, -1, 0] = torch.full((D,), 1.75).to(dtype)              # largest value exactly 448 * 2^-8
    v[0, 0, 0] = torch.linspace(-1, 1, D).to(dtype) * 6e-8      # fp16 subnormal numbers
    v[0, -1, -1, 0] = 60000.0
    shape = (n, page, Hkv) if layout == "NHD" else (n, Hkv, page)
    pools = [torch.randint(0, 127, shape + (D,), generator=g).to(torch.uint8) for _ in range(2)]
    scales = [torch.randint(100, 130, shape, generator=g).to(torch.uint8) for _ in range(2)]
    dev = [t.cuda().view(U.F8) for t in pools] + [t.cuda().view(U.E8) for t in scales]
    T.reset_launch_counts()
    T.paged_write(k.cuda(), v.cuda(), *dev, table.cuda(), start.cuda(), lens=lens.cuda(), layout=layout)
    T.check_device_status()
    assert T.launch_counts()["cache_write"] == 1
    want = [t.clone() for t in pools + scales]
    for i, x in enumerate((k, v)):
        values, e = U.quantise(x.transpose(1, 2))
        for b in range(B):
            for j in range(int(lens[b])):
                pos = int(start[b]) + j
                at = (int(table[b, pos // page]), pos % page) if layout == "NHD" else (int(table[b, pos // page]), slice(None), pos % page)
                want[i][at] = values[b, j].float().to(U.F8).view(torch.uint8)
                want[2 + i][at] = (e[b, j] + 127).to(torch.uint8)
    for got, ref in zip(dev, want):   # every byte: rows of padding and all other places are left as they were
        assert torch.equal(got.cpu().view(torch.uint8), ref)
    total = start + lens
    S = per_seq * page - 1 if per_seq * page > 1 else 1
    rk, rv = T.paged_read(*dev, table.cuda(), total.cuda(), max_len=S, dtype=dtype, layout=layout)
    T.check_device_status()
    for got, pool, scale in ((rk, want[0].view(U.F8), want[2].view(U.E8)), (rv, want[1].view(U.F8), want[3].view(U.E8))):
        for b in range(B):
            m = min(int(total[b]), S)
            ref = U.rows_of(pool, scale, table[b], m, layout).transpose(0, 1)
            assert torch.equal(got[b, :, :m].cpu(), ref.to(dtype))
            assert (got[b, :, m:] == 0).all()


def test_rows_that_are_not_numbers():
    import torch_neuronx_b200 as T

    x = torch.ones(1, 4, 1, 64, dtype=torch.bfloat16)
    x[0, 1, 0, 5] = math.inf
    x[0, 2, 0, 63] = math.nan
    x[0, 3] = 3e38
    kp, vp = (torch.zeros(1, 1, 4, 64, dtype=torch.uint8, device="cuda").view(U.F8) for _ in range(2))
    ks, vs = (torch.zeros(1, 1, 4, dtype=torch.uint8, device="cuda").view(U.E8) for _ in range(2))
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    T.paged_write(x.cuda(), x.cuda(), kp, vp, ks, vs, table, one - 1)
    k, v = T.paged_read(kp, vp, ks, vs, table, one)
    assert (k[0, 0] == 1).all() and k[0, 1:3].isnan().all() and torch.equal(k.isnan(), v.isnan())
    assert ((k[0, 3].double() - 3e38).abs() <= 2.0**-4 * 3e38 + 2.0**-8 * 3e38).all()


def test_a_full_table_and_a_bad_page_are_reported():
    """Nothing is written outside: rows behind the table's last page are dropped, a page number outside the pool too."""
    import torch_neuronx_b200 as T

    x = torch.ones(2, 1, 6, 16, dtype=torch.float16, device="cuda")
    kp, vp = (torch.zeros(4, 2, 1, 16, dtype=torch.uint8, device="cuda").view(U.F8) for _ in range(2))
    ks, vs = (torch.full((4, 2, 1), 127, dtype=torch.uint8, device="cuda").view(U.E8) for _ in range(2))
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    start = torch.zeros(2, dtype=torch.int32, device="cuda")
    T.paged_write(x, x, kp, vp, ks, vs, table, start)           # six rows, room for four
    with pytest.raises(RuntimeError, match="full"):
        T.check_device_status()
    assert (kp.float() == 256).all()                            # 1 = 256 * 2^-8: the top binade
    bad = torch.tensor([[0, 7], [-1, 3]], dtype=torch.int32, device="cuda")
    kp.view(torch.uint8).zero_()
    T.paged_write(x[:, :, :4], x[:, :, :4], kp, vp, ks, vs, bad, start)
    with pytest.raises(RuntimeError, match="page"):
        T.check_device_status()
    assert (kp.float() != 0).flatten(1).any(1).tolist() == [True, False, False, True]
    lens = torch.full((2,), 4, dtype=torch.int32, device="cuda")
    k, _ = T.paged_read(kp, vp, ks, vs, bad, lens)
    with pytest.raises(RuntimeError, match="page"):
        T.check_device_status()
    assert (k[0, 0, 2:] == 0).all() and (k[1, 0, :2] == 0).all() and (k[0, 0, :2] == 1).all()
    q = torch.ones(2, 1, 1, 64, dtype=torch.float16, device="cuda")
    kd, vd = (torch.zeros(4, 2, 1, 64, dtype=torch.uint8, device="cuda").view(U.F8) for _ in range(2))
    out, _ = T.paged_decode(q, kd, vd, bad, lens, k_scales=ks, v_scales=vs)
    with pytest.raises(RuntimeError, match="page"):
        T.check_device_status()
    assert torch.isfinite(out).all()


DECODE = [
    # dtype, B, Hq, Hkv, D, page, S pages, layout, chunk
    (torch.bfloat16, 5, 32, 8, 128, 16, 40, "NHD", 0),
    (torch.float16, 3, 12, 12, 64, 128, 3, "HND", 0),
    (torch.bfloat16, 4, 8, 8, 64, 1, 77, "NHD", 64),
    (torch.float16, 2, 16, 1, 128, 8, 60, "HND", 128),      # sixteen query heads
    (torch.bfloat16, 2, 20, 1, 64, 32, 9, "NHD", 0),        # twenty: two blocks
    (torch.float16, 3, 10, 2, 128, 64, 4, "NHD", 96),       # five, ranges that are no whole block
    (torch.bfloat16, 3, 7, 1, 128, 2048, 1, "HND", 0),
]


@pytest.mark.parametrize("dtype,B,Hq,Hkv,D,page,pages,layout,chunk", DECODE)
def test_decode_against_64_bits(dtype, B, Hq, Hkv, D, page, pages, layout, chunk):
    import torch_neuronx_b200 as T

    g = torch.Generator().manual_seed(Hq * D + pages)
    n, table = _table(g, B, pages)
    S = page * pages
    lens = torch.randint(0, S + 1, (B,), generator=g).to(torch.int32)
    lens[0], lens[1] = S + 9, 0                              # longer than the table; empty
    if B > 2:
        lens[2] = 1
    k, v, ks, vs = U.make_pools(g, n, page, Hkv, D, dtype, True, layout)
    q = torch.randn(B, Hq, 1, D, generator=g).to(dtype)
    q[0, 0] = 0
    want = U.attend(q, k, v, ks, vs, table, lens, layout)
    # what lies behind a sequence's end is anything: NaN values, NaN scales
    used = torch.zeros(n, page, dtype=torch.bool)
    for b in range(B):
        for s in range(min(int(lens[b]), S)):
            used[table[b, s // page], s % page] = True
    for pool, scale in ((k, ks), (v, vs)):
        at, codes = (pool, scale) if layout == "NHD" else (pool.transpose(1, 2), scale.transpose(1, 2))
        at.view(torch.uint8)[~used], codes.view(torch.uint8)[~used] = 0x7F, 255
    out, lse = T.paged_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), lens.cuda(), layout=layout, need_lse=True, kv_chunk=chunk,
                              k_scales=ks.cuda(), v_scales=vs.cuda())
    T.check_device_status()
    U.check(out.cpu(), lse.cpu(), want)


def test_decode_with_rows_of_very_different_size():
    """Scales from 2^-100 to 2^60 in one sequence: weights and small values keep their bits where they decide the result.  A
    row's value error is at most 2^-34 of the largest row the warp has met; here the largest rows have no weight left."""
    import torch_neuronx_b200 as T

    g = torch.Generator().manual_seed(11)
    D, page, S = 64, 16, 256
    k, v, ks, vs = U.make_pools(g, S // page, page, 1, D, torch.bfloat16, True, "NHD")
    codes = vs.view(torch.uint8).view(-1)
    codes[:] = torch.randint(115, 139, (S,), generator=g).to(torch.uint8)
    codes[::7] = 27                       # 2^-100
    vz = v.view(torch.uint8).view(S, D)
    vz[5::11] = 0                         # rows of zeros carry weight too
    table = torch.arange(S // page, dtype=torch.int32).view(1, -1)
    lens = torch.tensor([S], dtype=torch.int32)
    q = torch.randn(1, 8, 1, D, generator=g).bfloat16()
    want = U.attend(q, k, v, ks, vs, table, lens, "NHD")
    out, lse = T.paged_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), lens.cuda(), need_lse=True, k_scales=ks.cuda(), v_scales=vs.cuda())
    U.check(out.cpu(), lse.cpu(), want)
    # a NaN scale among the keys or the values makes its head's rows NaN, as a NaN in a 16-bit cache does
    codes[3] = 255
    out, _ = T.paged_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), lens.cuda(), k_scales=ks.cuda(), v_scales=vs.cuda())
    assert out.isnan().all()


def test_strided_pools_query_and_results():
    import torch_neuronx_b200 as T

    g = torch.Generator().manual_seed(12)
    B, Hq, Hkv, D, page = 3, 8, 2, 64, 16
    n, table = _table(g, B, 5)
    lens = torch.tensor([80, 17, 33], dtype=torch.int32)
    k, v, ks, vs = U.make_pools(g, n, page, Hkv, D, torch.bfloat16, True, "NHD")
    q = torch.randn(B, Hq, 1, D, generator=g).bfloat16()
    want = U.attend(q, k, v, ks, vs, table, lens, "NHD")
    # keys and values interleaved in one allocation, scales with gaps, a transposed query, a strided result
    both = torch.stack((k.view(torch.uint8), v.view(torch.uint8)), 2).cuda().view(U.F8)
    kd, vd = both[:, :, 0], both[:, :, 1]
    sd = torch.stack((ks.view(torch.uint8), vs.view(torch.uint8)), -1).cuda().view(U.E8)
    qd = q.cuda().transpose(0, 3).contiguous().transpose(0, 3)
    out = torch.full((B, Hq, 1, 2 * D), math.nan, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((Hq, B, 1), math.nan, device="cuda").transpose(0, 1)
    wide = torch.zeros(B, 9, dtype=torch.int32)
    wide[:, :5] = table
    got, gl = T.paged_decode(qd, kd, vd, wide.cuda()[:, :5], lens.cuda(), out=out[..., :D], lse=lse, k_scales=sd[..., 0], v_scales=sd[..., 1])
    T.check_device_status()
    U.check(got.cpu(), gl.cpu(), want)
    assert out[..., D:].isnan().all()


def test_pools_beyond_4_gib():
    import torch_neuronx_b200 as T

    n, page, D = (1 << 21) + 40, 16, 128     # 2^32 bytes and some pages
    kp = torch.empty(n, page, 1, D, dtype=torch.uint8, device="cuda").view(U.F8)
    ks = torch.full((n, page, 1), 127, dtype=torch.uint8, device="cuda").view(U.E8)
    table = torch.arange(n - 20, n, dtype=torch.int32).view(1, -1)
    g = torch.Generator().manual_seed(1)
    x = U.random_rows((1, 1, 300, D), torch.bfloat16, g)
    start = torch.zeros(1, dtype=torch.int32, device="cuda")
    T.paged_write(x.cuda(), x.cuda(), kp, kp, ks, ks, table.cuda(), start)   # (keys and values alike: the same bytes twice)
    lens = start + 300
    k, _ = T.paged_read(kp, kp, ks, ks, table.cuda(), lens, max_len=300)
    values, e = U.quantise(x)
    ref = values * U.two(e)[..., None]
    assert torch.equal(k.cpu().double(), ref)
    q = torch.randn(1, 4, 1, D, generator=g).bfloat16()
    out, lse = T.paged_decode(q.cuda(), kp, kp, table.cuda(), lens, need_lse=True, k_scales=ks, v_scales=ks)
    s = (q[0, :, 0].double() @ ref[0, 0].T) / math.sqrt(D)
    want = (torch.softmax(s, -1) @ ref[0, 0]).view(1, 4, 1, D), torch.logsumexp(s, -1).view(1, 4, 1), ref.abs().max().expand(1, 4, 1, 1)
    U.check(out.cpu(), lse.cpu(), want)
    T.check_device_status()


def test_refusals():
    import torch_neuronx_b200 as T

    kp, vp = (torch.zeros(4, 16, 2, 64, dtype=torch.uint8, device="cuda").view(U.F8) for _ in range(2))
    ks, vs = (torch.zeros(4, 16, 2, dtype=torch.uint8, device="cuda").view(U.E8) for _ in range(2))
    table = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 4, 1, 64, dtype=torch.float16, device="cuda")
    x = torch.zeros(2, 2, 3, 64, dtype=torch.float16, device="cuda")
    for kw, text in (({"k_scales": ks}, "go together"), ({"k_scales": ks, "v_scales": vs.float()}, "v_scales"),
                     ({"k_scales": ks[:3], "v_scales": vs}, "k_scales"),
                     ({"k_scales": ks, "v_scales": vs, "k_new": x, "v_new": x}, "paged_write"),
                     ({"k_scales": ks, "v_scales": vs, "scale": -1.0}, "plan")):
        with pytest.raises(RuntimeError, match=text):
            T.paged_decode(q, kp, vp, table, lens, **kw)
    for args, text in (((q.float(), kp, vp, table, lens), "float16"), ((q[:, :3], kp, vp, table, lens), "heads"),
                       ((q, kp.view(torch.uint8), vp, table, lens), "float8"), ((q, kp, vp, table.long(), lens), "block_table"),
                       ((q, kp, vp, table, lens.long()), "kv_lens"), ((q[..., :48], kp[..., :48], vp[..., :48], table, lens), "head dim"),
                       ((q, kp[:, :12], vp[:, :12], table, lens), "scales"), ((q, kp[..., :32], vp[..., :32], table, lens), "head dim")):
        with pytest.raises(RuntimeError, match=text):
            T.paged_decode(*args, k_scales=ks, v_scales=vs)
    with pytest.raises(RuntimeError):    # a page size that is no power of two
        T.paged_decode(q, kp[:, :12], vp[:, :12], table, lens, k_scales=ks[:, :12], v_scales=vs[:, :12])
    with pytest.raises(ValueError, match="layout"):
        T.paged_write(x, x, kp, vp, ks, vs, table, lens, layout="DHN")
    for args, text in (((x.float(), x.float()), "float16 or bfloat16"), ((x, x[:, :, :2]), "same shape"), ((x[..., :40], x[..., :40]), "multiple of 16"),
                       ((x[:, :1], x[:, :1]), "heads"), ((x.transpose(2, 3).contiguous().transpose(2, 3),) * 2, "unit inner")):
        with pytest.raises(RuntimeError, match=text):
            T.paged_write(*args, kp, vp, ks, vs, table, lens)
    with pytest.raises(RuntimeError, match="start"):
        T.paged_write(x, x, kp, vp, ks, vs, table, lens[:1])
    with pytest.raises(RuntimeError, match="capacity"):
        T.paged_read(kp, vp, ks, vs, table, lens, max_len=33)
    with pytest.raises(RuntimeError, match="dtype"):
        T.paged_read(kp, vp, ks, vs, table, lens, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="16-byte"):   # rows off their boundary
        wide = torch.zeros(4, 16, 2, 72, dtype=torch.uint8, device="cuda").view(U.F8)
        T.paged_write(x, x, wide[..., :64], wide[..., :64], ks, vs, table, lens)
    T.check_device_status()

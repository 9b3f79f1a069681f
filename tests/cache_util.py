"""A plain 8-bit paged cache and attention over it, in 64 bits on the CPU."""

import math

import torch

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def two(n):
    """2^n exactly."""
    return torch.tensor([math.ldexp(1.0, int(i)) for i in n.reshape(-1)], dtype=torch.float64).reshape(n.shape)


def quantise(x):
    """``(values as doubles, exponents)`` of rows: nearest of the e4m3 values, ties to the even code."""
    x = x.double()
    top = x.abs().amax(-1)
    e = torch.zeros(top.shape, dtype=torch.int64)
    for i, t in enumerate(top.reshape(-1).tolist()):
        if t > 0:
            m, n = math.frexp(t)                     # t = m 2^n, 448 = 0.875 2^9
            e.view(-1)[i] = max(-127, n - 9 if m <= 0.875 else n - 8)
    y = x / two(e)[..., None]
    grid = torch.arange(127, dtype=torch.uint8).view(F8).double()
    low = (torch.searchsorted(grid, y.abs().contiguous(), right=True) - 1).clamp(max=125)
    below, above = y.abs() - grid[low], grid[low + 1] - y.abs()
    up = (above < below) | ((above == below) & (low % 2 == 1))
    return torch.copysign(grid[low + up.long()], y), e


def dequantise(values, scales):
    """Rows of pools (e4m3, e8m0) as doubles."""
    return values.double() * two(scales.view(torch.uint8).long() - 127)[..., None]


def random_rows(shape, dtype, g):
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randn(shape[:-1] + (1,), generator=g))
    return x.to(dtype)


def make_pools(g, n_pages, page, Hkv, D, dtype, quantised, layout):
    """Random pools: ``(k, v, k_scales, v_scales)`` in the layout's order, scales None for a 16-bit cache."""
    shape = (n_pages, page, Hkv) if layout == "NHD" else (n_pages, Hkv, page)
    got = []
    for _ in range(2):
        x = random_rows(shape + (D,), dtype, g)
        if not quantised:
            got.append((x, None))
            continue
        codes, e = (torch.randint(0, 127, shape + (D,), generator=g) + 128 * torch.randint(0, 2, shape + (D,), generator=g)), torch.randint(-9, -5, shape, generator=g)
        got.append((codes.to(torch.uint8).view(F8), (e + 127).to(torch.uint8).view(E8)))
    (k, ks), (v, vs) = got
    return k, v, ks, vs


def rows_of(pool, scales, table, n, layout):
    """The first ``n`` rows of a table's pages, (n, Hkv, D), as doubles."""
    idx = table.long()
    x = pool.view(torch.uint8 if pool.dtype == F8 else torch.int16)[idx].view(pool.dtype)
    x = x.double() if scales is None else dequantise(x, scales.view(torch.uint8)[idx].view(E8))
    if layout == "HND":
        x = x.transpose(1, 2)
    return x.flatten(0, 1)[:n]


def attend(q, k, v, ks, vs, table, lens, layout, scale=None, prefix=None, P=0):
    """``(out, lse, largest |v| seen)`` of one query row per sequence, in 64 bits."""
    B, Hq, _, D = q.shape
    Hkv = k.shape[2] if layout == "NHD" else k.shape[1]
    page = k.shape[1] if layout == "NHD" else k.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros((B, Hq, 1, D), dtype=torch.float64)
    lse = torch.full((B, Hq, 1), -math.inf, dtype=torch.float64)
    big = torch.zeros((B, Hq, 1, 1), dtype=torch.float64)
    pk = pv = torch.zeros((0, Hkv, D), dtype=torch.float64)
    if P:
        pk, pv = rows_of(k, ks, prefix, P, layout), rows_of(v, vs, prefix, P, layout)
    for b in range(B):
        n = max(0, min(int(lens[b]), table.shape[1] * page))
        K = torch.cat((pk, rows_of(k, ks, table[b], n, layout))) if n else pk
        V = torch.cat((pv, rows_of(v, vs, table[b], n, layout))) if n else pv
        if K.shape[0] == 0:
            continue
        g = Hq // Hkv
        s = torch.einsum("hgd,shd->hgs", q[b, :, 0].double().view(Hkv, g, D), K) * scale
        out[b, :, 0] = torch.einsum("hgs,shd->hgd", torch.softmax(s, -1), V).reshape(Hq, D)
        lse[b, :, 0] = torch.logsumexp(s, -1).reshape(Hq)
        big[b] = V.abs().amax((0, 2)).repeat_interleave(g).view(Hq, 1, 1)
    return out, lse, big


def check(out, lse, want, *, p_bits=None, tag=""):
    """One rounding of the result (eps / 2 of it) and the fp32 arithmetic before it: exponents of up to about 2^5 carry
    2^-24 of themselves, sums some steps more -- 2^-16 of the largest value covers both.  ``p_bits``: probabilities were rounded
    to this type first, eps / 2 of at most the largest value."""
    ref, ref_l, big = want
    half = torch.finfo(out.dtype).eps / 2
    got = out.double()
    assert not torch.isnan(got).any(), tag
    room = half * ref.abs() + (2.0**-16 + (torch.finfo(p_bits).eps / 2 if p_bits is not None else 0.0)) * big
    if out.dtype == torch.float16:
        room = room + 2.0**-25   # half a step of fp16's subnormal numbers
    over = ((got - ref).abs() - room).max().item()
    assert over <= 0, f"{tag}: {over:.3e} beyond the tolerance"
    dead = ref_l == -math.inf
    assert torch.equal(lse == -math.inf, dead), tag
    assert torch.all(got[dead] == 0), tag
    if (~dead).any():
        err = (lse.double() - ref_l)[~dead].abs() - 2.0**-16 * (1 + ref_l[~dead].abs())
        assert err.max().item() <= 0, f"{tag}: lse"

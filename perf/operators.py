"""The operators around a serving cache, and rotary positions with several axes, as a program calls them.

* ``rotary``  queries and keys rotated by positions with one to four axes (time, height, width): a training step with its
  gradients, or the new tokens of a serving step
* ``write``   key and value rows quantised to 8 bits as they are written into a paged cache
* ``read``    the cached rows of some sequences back in 16 bits, dense, for the next chunk of a prompt
* ``decode``  one token for each sequence against the 8-bit paged cache
* ``shared``  one token for each sequence of a batch whose sequences all start with the same cached prefix

An 8-bit cache holds e4m3 values and one power of two for each (token, head) row, ``2^e`` with the least ``e`` for which
the row's largest magnitude is at most ``448 * 2^e`` (``e = 0`` for a row of zeros, ``e >= -127``).

``listed()`` fixes a few members of each family, ``draw()`` takes others from the same ranges.  With ``own`` the calls are
the package's; without it the same results are made of elementary torch operations.
"""

import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_F8 = torch.float8_e4m3fn
_E8 = torch.float8_e8m0fnu


def listed():
    return [
        # a training step over text and image patches, three axes on half-split pairs, (B, S, H, D) storage
        {"name": "rotary_train", "kind": "rotary", "grad": True, "dtype": "bf16", "B": 2, "L": 4096, "Hq": 32, "Hkv": 8,
         "D": 128, "rot": 128, "axes": 3, "far": 16384, "interleaved": False},
        # the new tokens of a serving batch far into their contexts, half of the head dimension rotated
        {"name": "rotary_step", "kind": "rotary", "grad": False, "dtype": "fp16", "B": 61, "L": 1, "Hq": 12, "Hkv": 12,
         "D": 64, "rot": 32, "axes": 1, "far": 1000000, "interleaved": True},
        # the prompts of a batch enter the cache, padded to the longest
        {"name": "write_prompts", "kind": "write", "dtype": "bf16", "B": 16, "L": 4096, "lo": 512, "hi": 4096, "Hkv": 8,
         "D": 128, "page": 16, "layout": "NHD"},
        # one new token of each sequence enters the cache
        {"name": "write_step", "kind": "write", "dtype": "bf16", "B": 64, "L": 1, "lo": 1, "hi": 1, "Hkv": 8, "D": 128,
         "page": 16, "layout": "NHD"},
        # long prefixes come back for the next chunk of their prompts
        {"name": "read_long", "kind": "read", "dtype": "bf16", "B": 8, "S": 8192, "lo": 4096, "hi": 8192, "Hkv": 8, "D": 128,
         "page": 64, "layout": "HND"},
        # a short chat of a small model comes back, odd length
        {"name": "read_short", "kind": "read", "dtype": "fp16", "B": 1, "S": 577, "lo": 577, "hi": 577, "Hkv": 12, "D": 64,
         "page": 16, "layout": "NHD"},
        # the next token of one chat: launches and host work
        {"name": "decode_one", "kind": "decode", "dtype": "bf16", "B": 1, "Hq": 32, "Hkv": 8, "D": 128, "S": 2048,
         "lo": 2001, "hi": 2001, "page": 16, "layout": "NHD"},
        # the decode step of a full batch of unequal sequences
        {"name": "decode_ragged", "kind": "decode", "dtype": "bf16", "B": 64, "Hq": 32, "Hkv": 8, "D": 128, "S": 8192,
         "lo": 512, "hi": 8192, "page": 16, "layout": "NHD"},
        # a small multi-head model, head dimension 64, long pages
        {"name": "decode_heads", "kind": "decode", "dtype": "fp16", "B": 16, "Hq": 12, "Hkv": 12, "D": 64, "S": 4096,
         "lo": 128, "hi": 4000, "page": 128, "layout": "HND"},
        # a handful of drafts that continue one short text
        {"name": "shared_few", "kind": "shared", "dtype": "fp16", "quant": False, "B": 5, "Hq": 16, "Hkv": 4, "D": 64,
         "P": 1000, "S": 128, "lo": 0, "hi": 100, "page": 16, "layout": "NHD"},
        # a batch of requests under one long instruction, 16-bit cache
        {"name": "shared_batch", "kind": "shared", "dtype": "bf16", "quant": False, "B": 64, "Hq": 32, "Hkv": 8, "D": 128,
         "P": 16384, "S": 1024, "lo": 16, "hi": 1000, "page": 16, "layout": "NHD"},
        # a larger batch over an 8-bit cache
        {"name": "shared_8bit", "kind": "shared", "dtype": "bf16", "quant": True, "B": 128, "Hq": 32, "Hkv": 8, "D": 128,
         "P": 8192, "S": 512, "lo": 16, "hi": 500, "page": 32, "layout": "HND"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "write", "read", "decode", "shared"])
    dtype = rng.choice(["bf16", "fp16"])
    D = rng.choice([64, 128])
    Hkv = rng.choice([1, 2, 3, 4, 8, 12])
    group = rng.choice([1, 2, 3, 4, 5, 8, 16])
    c = {"kind": kind, "dtype": dtype, "D": D, "Hkv": Hkv}
    if kind == "rotary":
        B = _log(rng, 1, 64)
        c.update(dtype=rng.choice(["bf16", "fp16", "fp32"]), grad=rng.random() < 0.6, B=B, Hq=Hkv * min(group, 4),
                 L=_log(rng, 1, max(1, 8192 // B)), D=rng.choice([64, 80, 96, 128]), axes=rng.choice([1, 2, 3, 4]),
                 far=_log(rng, 1000, 1000000), interleaved=rng.random() < 0.4)
        c["rot"] = c["D"] if rng.random() < 0.7 else rng.choice([16, 32, 64])
        return c
    c.update(page=rng.choice([1, 8, 16, 32, 64, 128]), layout=rng.choice(["NHD", "HND"]))
    if kind == "write":
        B = _log(rng, 1, 64)
        L = 1 if rng.random() < 0.3 else _log(rng, 1, max(1, 65536 // B // max(1, Hkv // 4)))
        c.update(B=B, L=L, lo=max(0, L // rng.choice([1, 2, 8]) - 1), hi=L)
        return c
    B = _log(rng, 1, 96)
    if kind == "shared":
        P = _log(rng, 1, 16384)
        S = _log(rng, 1, max(1, min(1024, 65536 * 8 // Hkv // B)))
        group = min(group, 8)
        c.update(quant=rng.random() < 0.5, B=B, Hq=Hkv * group, P=P, S=S, lo=0, hi=S)
        return c
    S = _log(rng, 1, max(1, min(32768, 524288 * 8 // Hkv // B // (8 if kind == "read" else 1))))
    c.update(B=B, Hq=Hkv * group, S=S, lo=S // rng.choice([1, 2, 16]), hi=S)
    if kind == "read":
        del c["Hq"]
    return c


# ----------------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------------


def _sections(c):
    """Frequency pairs of each axis: about a quarter for the first, the rest in equal parts."""
    pairs, axes = c["rot"] // 2, c["axes"]
    if axes == 1:
        return (pairs,)
    first = max(1, pairs // 4)
    rest = [(pairs - first) // (axes - 1)] * (axes - 1)
    rest[-1] += pairs - first - sum(rest)
    return (first, *rest)


def _lens(c, rng):
    lens = rng.integers(c["lo"], c["hi"] + 1, size=c["B"])
    lens[0] = c["hi"]
    return lens.astype(np.int32)


def _rows(shape, dtype, gen, spread):
    """Key or value rows: normal values whose rows differ in size, a few channels larger than the others."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    x *= torch.exp2(spread * torch.randn(shape[:-1] + (1,), generator=gen, device="cuda"))
    x[..., :2] *= 4
    return x.to(dtype)


def _pow2(n):
    """2^n in 32 bits, exactly, for whole n from -127 on."""
    return torch.where(n > -127, (n + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _quantise(x):
    """(e4m3 values, exponents) of rows, whole tensors at a time."""
    x = x.float()
    mantissa, exponent = torch.frexp(x.abs().amax(-1))
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp(min=-127)
    e = torch.where(mantissa == 0, torch.zeros_like(e), e)
    return (x * _pow2(-e).unsqueeze(-1)).to(_F8), e


def _scales(e):
    return (e + 127).to(torch.uint8).view(_E8)


def _pools(c, pages, quant, gen):
    """Key and value pools with content everywhere (what another sequence left behind included)."""
    shape = (pages, c["page"], c["Hkv"]) if c["layout"] == "NHD" else (pages, c["Hkv"], c["page"])
    got = []
    for spread in (0.3, 0.5):
        rows = _rows(shape + (c["D"],), _DTYPES[c["dtype"]], gen, spread)
        if quant:
            values, e = _quantise(rows)
            got.append((values, _scales(e)))
        else:
            got.append((rows, None))
    return got


def prepare(case, seed):
    c = case
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    dtype = _DTYPES[c["dtype"]]
    if c["kind"] == "rotary":
        B, L, D = c["B"], c["L"], c["D"]
        for name, heads in (("q", c["Hq"]), ("k", c["Hkv"])):
            x = torch.randn((B, L, heads, D), generator=gen, device="cuda").to(dtype).transpose(1, 2)
            s[name] = x.requires_grad_() if c["grad"] else x
            if c["grad"]:
                s["g" + name] = torch.randn((B, L, heads, D), generator=gen, device="cuda").to(dtype).transpose(1, 2)
        start = torch.from_numpy(rng.integers(0, c["far"], size=(c["axes"], B, 1)))
        step = torch.from_numpy(rng.integers(0, 3, size=(c["axes"], B, L))).cumsum(-1)
        s["positions"] = (start + step).to(torch.int32).cuda()
        s["sections"] = _sections(c)
        s["inv_freq"] = torch.from_numpy(10000.0 ** (-np.arange(0, c["rot"], 2) / c["rot"])).cuda()
        return s
    B, page = c["B"], c["page"]
    lens = _lens(c, rng)
    if c["kind"] == "write":
        start = rng.integers(0, 4 * page + 50, size=B).astype(np.int32)
        per_seq = -(-(4 * page + 50 + c["L"]) // page)
        s["start"], s["lens"] = torch.from_numpy(start).cuda(), torch.from_numpy(lens).cuda()
        for name, spread in (("k", 0.3), ("v", 0.5)):
            s[name] = _rows((B, c["L"], c["Hkv"], c["D"]), dtype, gen, spread).transpose(1, 2)
    else:
        per_seq = -(-c["S"] // page)
        s["lens"] = torch.from_numpy(lens).cuda()
        if c["kind"] != "read":
            s["q"] = torch.randn((B, c["Hq"], 1, c["D"]), generator=gen, device="cuda").to(dtype)
    shared = -(-c["P"] // page) if c["kind"] == "shared" else 0
    pages = B * per_seq + shared + 3
    order = torch.from_numpy(rng.permutation(pages).astype(np.int32)).cuda()
    s["table"] = order[: B * per_seq].view(B, per_seq).contiguous()
    s["prefix"] = order[B * per_seq: B * per_seq + shared].contiguous()
    if c["kind"] == "write":
        shape = (pages, page, c["Hkv"]) if c["layout"] == "NHD" else (pages, c["Hkv"], page)
        s["k8"], s["v8"] = (torch.zeros(shape + (c["D"],), dtype=_F8, device="cuda") for _ in range(2))
        s["ks"], s["vs"] = (torch.full(shape, 127, dtype=torch.uint8, device="cuda").view(_E8) for _ in range(2))
    else:
        (s["k8"], s["ks"]), (s["v8"], s["vs"]) = _pools(c, pages, c.get("quant", True), gen)
    return s


# ----------------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------------


def _rotate(x, cos, sin, rot, interleaved):
    """Pairs of the first `rot` elements turned by the angles; 32 bits, rounded once."""
    r = x[..., :rot].float()
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., : rot // 2], r[..., rot // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y.to(x.dtype), x[..., rot:]), -1)


def _plain_rotary(s):
    c = s["case"]
    axis = torch.repeat_interleave(torch.arange(c["axes"], device="cuda"), torch.tensor(s["sections"], device="cuda"))
    angle = s["positions"].double()[axis].permute(1, 2, 0) * s["inv_freq"]   # far positions: 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    got = {}
    with torch.no_grad():
        got["q"], got["k"] = (_rotate(s[n], cos, sin, c["rot"], c["interleaved"]) for n in ("q", "k"))
        if c["grad"]:
            got["gq"], got["gk"] = (_rotate(s[n], cos, -sin, c["rot"], c["interleaved"]) for n in ("gq", "gk"))
    return got


def _plain_write(s):
    c = s["case"]
    L, page = c["L"], c["page"]
    at = s["start"].long()[:, None] + torch.arange(L, device="cuda")
    real = torch.arange(L, device="cuda") < s["lens"][:, None]
    slot = at.clamp(max=s["table"].shape[1] * page - 1)
    pages, rows = torch.gather(s["table"].long(), 1, slot // page)[real], (slot % page)[real]
    for x, pool, scale in (("k", "k8", "ks"), ("v", "v8", "vs")):
        values, e = _quantise(s[x].transpose(1, 2)[real])
        view, exps = s[pool].view(torch.uint8), s[scale].view(torch.uint8)
        if c["layout"] == "HND":
            view, exps = view.transpose(1, 2), exps.transpose(1, 2)
        view[pages, rows] = values.view(torch.uint8)
        exps[pages, rows] = (e + 127).to(torch.uint8)
    return {n: s[n] for n in ("k8", "v8", "ks", "vs")}


def _gather(s, name, scale, table, layout):
    """The rows of the table's pages, (..., rows, Hkv, D), in 32 bits."""
    pool = s[name]
    x = pool.view(torch.uint8 if pool.dtype == _F8 else torch.int16)[table.long()].view(pool.dtype).float()
    if s[scale] is not None:
        x = x * _pow2(s[scale].view(torch.uint8)[table.long()].int() - 127).unsqueeze(-1)
    if layout == "HND":
        x = x.transpose(-3, -2)
    return x.flatten(-4, -3)


def _plain_read(s):
    c = s["case"]
    hidden = torch.arange(c["S"], device="cuda") >= s["lens"][:, None]
    got = {}
    for name, scale in (("k8", "ks"), ("v8", "vs")):
        x = _gather(s, name, scale, s["table"], c["layout"])[:, : c["S"]]
        got[name] = x.masked_fill(hidden[..., None, None], 0).to(_DTYPES[c["dtype"]]).transpose(1, 2)
    return got


def _plain_attend(s):
    """Softmax over the prefix's keys (where there is one) and a sequence's own, in 32 bits."""
    c = s["case"]
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    q = s["q"].float().view(B, Hkv, -1, D) / math.sqrt(D)
    k, v = (_gather(s, n, e, s["table"], c["layout"])[:, : c["S"]] for n, e in (("k8", "ks"), ("v8", "vs")))
    hidden = torch.arange(c["S"], device="cuda") >= s["lens"][:, None]
    score = torch.einsum("bhgd,bshd->bhgs", q, k).masked_fill(hidden[:, None, None], -math.inf)
    if c["kind"] == "shared":
        pk, pv = (_gather(s, n, e, s["prefix"], c["layout"])[: c["P"]] for n, e in (("k8", "ks"), ("v8", "vs")))
        score = torch.cat((torch.einsum("bhgd,shd->bhgs", q, pk), score), -1)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    own_p = p[..., -c["S"]:].masked_fill(hidden[:, None, None], 0)
    out = torch.einsum("bhgs,bshd->bhgd", own_p, v.masked_fill(hidden[..., None, None], 0))
    if c["kind"] == "shared":
        out = out + torch.einsum("bhgs,shd->bhgd", p[..., : c["P"]], pv)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    lse = (top + total.log()).masked_fill(total == 0, -math.inf)
    return {"out": out.view(B, -1, 1, D).to(s["q"].dtype), "lse": lse.view(B, -1, 1)}


def _own(s):
    import torch_neuronx_b200 as T

    c = s["case"]
    if c["kind"] == "rotary":
        q, k = T.rotary_embedding(s["q"], s["k"], s["positions"], s["inv_freq"], sections=s["sections"],
                                  interleaved=c["interleaved"])
        if not c["grad"]:
            return {"q": q, "k": k}
        gq, gk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
        return {"q": q, "k": k, "gq": gq, "gk": gk}
    if c["kind"] == "write":
        T.paged_write(s["k"], s["v"], s["k8"], s["v8"], s["ks"], s["vs"], s["table"], s["start"], lens=s["lens"],
                      layout=c["layout"])
        return {n: s[n] for n in ("k8", "v8", "ks", "vs")}
    if c["kind"] == "read":
        k, v = T.paged_read(s["k8"], s["v8"], s["ks"], s["vs"], s["table"], s["lens"], max_len=c["S"], layout=c["layout"],
                            dtype=_DTYPES[c["dtype"]])
        return {"k8": k, "v8": v}
    if c["kind"] == "decode":
        out, lse = T.paged_decode(s["q"], s["k8"], s["v8"], s["table"], s["lens"], layout=c["layout"], need_lse=True,
                                  k_scales=s["ks"], v_scales=s["vs"])
    else:
        out, lse = T.shared_prefix_decode(s["q"], s["k8"], s["v8"], s["prefix"], c["P"], s["table"], s["lens"],
                                          layout=c["layout"], need_lse=True, k_scales=s["ks"], v_scales=s["vs"])
    return {"out": out, "lse": lse}


def run(state):
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "write": _plain_write, "read": _plain_read}.get(state["case"]["kind"], _plain_attend)(state)


# ----------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------------


def work(case):
    c = case
    D, Hkv = c["D"], c["Hkv"]
    if c["kind"] == "rotary":
        n = c["B"] * c["L"] * (c["Hq"] + Hkv) * D * (2 if c["grad"] else 1)
        return {"bytes": 2 * n * _BYTES[c["dtype"]] + 4 * c["axes"] * c["B"] * c["L"], "flops": 3 * n}
    mean = c["hi"] if c["B"] == 1 else (c["hi"] + (c["B"] - 1) * (c["lo"] + c["hi"]) / 2) / c["B"]
    rows = c["B"] * mean * Hkv
    row8 = 2 * (D + 1)
    if c["kind"] == "write":
        return {"bytes": rows * (4 * D + row8), "flops": rows * 6 * D}
    if c["kind"] == "read":
        return {"bytes": rows * row8 + c["B"] * c["S"] * Hkv * 4 * D, "flops": rows * 2 * D}
    row = row8 if c.get("quant", True) else 4 * D
    shared = c.get("P", 0)
    return {"bytes": (rows + shared * Hkv) * row + 4 * c["B"] * c["Hq"] * (D + 1),
            "flops": 4 * D * c["B"] * c["Hq"] * (mean + shared)}


# ----------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------------------------------


def _two64(n):
    """2^n in 64 bits, exactly."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def _row64(pool, scale, page, row, layout):
    """Rows (tokens, Hkv, D) of a pool by page and row number, as doubles."""
    at = (page, row) if layout == "NHD" else (page, slice(None), row)
    at = tuple(i.long() if isinstance(i, torch.Tensor) else i for i in at)
    x = pool.view(torch.uint8)[at].view(_F8).double() if pool.dtype == _F8 else pool[at].double()
    if scale is not None:
        x = x * _two64(scale.view(torch.uint8)[at].long() - 127)[..., None]
    return x


def _tokens(table, n, page):
    i = torch.arange(n, device="cuda")
    return table[i // page], i % page


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "rotary":
        rot, which, i = c["rot"], [], 0
        for a, n in enumerate(s["sections"]):
            which += [a] * n
        pos = torch.stack([s["positions"][a].double() for a in which], -1)
        turn = torch.polar(torch.ones_like(pos), pos * 10000.0 ** (-torch.arange(0, rot, 2, device="cuda").double() / rot))
        half = rot // 2
        even = torch.arange(0, rot, 2, device="cuda") if c["interleaved"] else torch.arange(half, device="cuda")
        odd = even + 1 if c["interleaved"] else even + half

        def turned(x, t):
            y = x.detach().double().clone()
            z = torch.complex(y[..., even], y[..., odd]) * t[:, None]
            y[..., even], y[..., odd] = z.real, z.imag
            return y

        got = {"q": turned(s["q"], turn), "k": turned(s["k"], turn)}
        if c["grad"]:
            got.update(gq=turned(s["gq"], turn.conj()), gk=turned(s["gk"], turn.conj()))
        return got
    if c["kind"] == "write":
        # rounding is part of the definition: the nearest of the 8-bit values, ties to the even code
        codes = torch.arange(127, dtype=torch.uint8, device="cuda")
        grid = codes.view(_F8).double()
        got = {n: s[n].view(torch.uint8).clone().view(_F8).double() for n in ("k8", "v8")}
        got.update({n: _two64(s[n].view(torch.uint8).long() - 127) for n in ("ks", "vs")})
        for x, pool, scale in (("k", "k8", "ks"), ("v", "v8", "vs")):
            for b in range(c["B"]):
                n, first = int(s["lens"][b]), int(s["start"][b])
                rows = s[x][b, :, :n].double()
                top = rows.abs().amax(-1, keepdim=True)
                e = torch.where(top > 0, torch.ceil(torch.log2(top / 448)), torch.zeros_like(top)).clamp(min=-127)
                e = torch.where(top > 448 * _two64(e), e + 1, e)
                e = torch.where((top > 0) & (top <= 448 * _two64(e - 1)) & (e > -127), e - 1, e)
                y = rows / _two64(e)
                lower = (torch.searchsorted(grid, y.abs(), right=True) - 1).clamp(max=125)
                below, above = y.abs() - grid[lower], grid[lower + 1] - y.abs()
                up = (above < below) | ((above == below) & (lower % 2 == 1))
                y = torch.copysign(grid[lower + up.long()], y)
                page, row = _tokens(s["table"][b], first + n, c["page"])
                page, row = page[first:].long(), row[first:]
                at = (page, row) if c["layout"] == "NHD" else (page, slice(None), row)
                got[pool][at] = y.transpose(0, 1)
                got[scale][at] = _two64(e[..., 0].transpose(0, 1))
        return got
    if c["kind"] == "read":
        got = {}
        for name, scale in (("k8", "ks"), ("v8", "vs")):
            y = torch.zeros((c["B"], c["Hkv"], c["S"], c["D"]), dtype=torch.float64, device="cuda")
            for b in range(c["B"]):
                n = int(s["lens"][b])
                y[b, :, :n] = _row64(s[name], s[scale], *_tokens(s["table"][b], n, c["page"]), c["layout"]).transpose(0, 1)
            got[name] = y
        return got
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    group = c["Hq"] // Hkv
    out = torch.zeros((B, c["Hq"], 1, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, c["Hq"], 1), -math.inf, dtype=torch.float64, device="cuda")
    front = [[], []]
    if c["kind"] == "shared":
        front = [[_row64(s[n], s[e], *_tokens(s["prefix"], c["P"], c["page"]), c["layout"])]
                 for n, e in (("k8", "ks"), ("v8", "vs"))]
    for b in range(B):
        n = int(s["lens"][b])
        at = _tokens(s["table"][b], n, c["page"])
        k, v = (torch.cat(f + [_row64(s[x], s[e], *at, c["layout"])])
                for f, (x, e) in zip(front, (("k8", "ks"), ("v8", "vs"))))
        if k.shape[0] == 0:
            continue
        for h in range(Hkv):
            score = (s["q"][b, h * group:(h + 1) * group, 0].double() @ k[:, h].T) / math.sqrt(D)
            lse[b, h * group:(h + 1) * group, 0] = torch.logsumexp(score, -1)
            out[b, h * group:(h + 1) * group, 0] = torch.softmax(score, -1) @ v[:, h]
    return {"out": out, "lse": lse}

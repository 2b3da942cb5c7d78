"""The operators around a paged latent cache: rotary positions, the cache's
write and read back, and the attention of drafted tokens over it; what is
measured of them, with their plain forms in elementary torch operations.

A case is a dict of plain values with a "kind":

  rope    T tokens of H heads of D values, R of them from `offset` on rotated
  write   T latent rows (512 + 64) normed, rotated, quantised and scattered
          into a paged cache
  read    T rows of a paged cache gathered and widened
  attend  B sequences of up to `n` query tokens each (a tree of drafted tokens,
          or with tree = False the last tokens of the sequence in order) over
          up to L cached positions

Formats of a cache: f16 and bf16 rows, or fp8: the 512 latent values in e4m3
with a power-of-two scale for every 128, the 64 rotary ones in bf16.
"""
import math

import torch

own = False

LAT, ROT, GROUP = 512, 64, 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# the attention's score scale: mscale^2 / sqrt(128 + 64), mscale of a context extended 40 times
SCALE = (0.1 * math.log(40.0) + 1.0) ** 2 / math.sqrt(192.0)
YARN = {"base": 10000.0, "scaling": "yarn", "factor": 40.0, "orig": 4096}


def listed():
    return [
        # a decode step of a few sequences: the rotary part of every head's query, out of the projection's fp32 rows
        {"name": "rope_step_t16", "kind": "rope", "T": 16, "H": 128, "D": 192, "R": 64, "offset": 128, "layout": "interleaved",
         "scaling": "yarn", "factor": 40.0, "x": "f32", "y": "bf16", "part": True, "far": 163840},
        # a prompt of a model with whole heads rotated in the half layout, context extended by interpolation
        {"name": "rope_prompt_t4097", "kind": "rope", "T": 4097, "H": 64, "D": 128, "R": 128, "offset": 0, "layout": "half",
         "scaling": "linear", "factor": 4.0, "x": "bf16", "y": "bf16", "part": False, "far": 16384},
        # a decode step's new rows into a quantised cache: one launch, latency
        {"name": "write_step_fp8_t64", "kind": "write", "T": 64, "x": "f32", "format": "fp8", "page": 64, "norm": True},
        # the rows of a batch of long prompts
        {"name": "write_prompt_bf16_t32768", "kind": "write", "T": 32768, "x": "f32", "format": "bf16", "page": 64, "norm": True},
        # a long prompt's quantised rows read back, as a cached prefix is for a layer that wants bf16
        {"name": "read_fp8_t16384", "kind": "read", "T": 16384, "y": "bf16", "format": "fp8", "page": 64},
        # a short exchange moved out of a half-precision cache of small pages, in fp32
        {"name": "read_f16_t1000", "kind": "read", "T": 1000, "y": "f32", "format": "f16", "page": 16},
        # one sequence, one token: latency
        {"name": "attend_one_l1024", "kind": "attend", "B": 1, "n": 1, "H": 128, "L": 1024, "format": "bf16", "page": 64, "tree": False},
        # a serving step of ragged sequences over quantised pages
        {"name": "attend_b64_fp8_l4095", "kind": "attend", "B": 64, "n": 1, "H": 128, "L": 4095, "format": "fp8", "page": 64, "tree": False},
        # eight drafted tokens each, odd lengths
        {"name": "attend_tree8_b16_l8191", "kind": "attend", "B": 16, "n": 8, "H": 128, "L": 8191, "format": "bf16", "page": 64, "tree": True},
        # the heads that one of eight devices holds, a few drafted tokens each
        {"name": "attend_tree3_h16_l2048", "kind": "attend", "B": 128, "n": 3, "H": 16, "L": 2048, "format": "f16", "page": 16, "tree": True},
        # the largest prompt chunk behind a prefix
        {"name": "attend_chunk512_l4608", "kind": "attend", "B": 1, "n": 512, "H": 128, "L": 4608, "format": "bf16", "page": 128, "tree": False},
        # the largest step: long documents, sixteen drafted tokens each
        {"name": "attend_tree16_b32_fp8_l16384", "kind": "attend", "B": 32, "n": 16, "H": 128, "L": 16384, "format": "fp8", "page": 64, "tree": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "write", "read", "attend", "attend", "attend", "attend"])
    page = 2 ** rng.randint(4, 8)
    fmt = rng.choice(["f16", "bf16", "fp8"])
    if kind == "rope":
        D = rng.choice([64, 128, 192, 256])
        R = 2 * rng.randint(8, min(D, 128) // 2)
        H, x = rng.randint(1, 128), rng.choice(["f32", "f16", "bf16"])
        T = min(_log(rng, 1, 8192), 4097 * 64 * 128 // (H * D))
        scaling = rng.choice(["none", "linear", "yarn"])
        return {"kind": kind, "T": T, "H": H, "D": D, "R": R, "offset": rng.choice([0, D - R]), "layout": rng.choice(["interleaved", "half"]),
                "scaling": scaling, "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 40.0]), "x": x,
                "y": rng.choice([x, "bf16"]), "part": rng.random() < 0.3, "far": _log(rng, 4096, 1 << 20)}
    if kind == "write":
        return {"kind": kind, "T": _log(rng, 1, 32768), "x": rng.choice(["f32", "f16", "bf16"]), "format": fmt, "page": page, "norm": rng.random() < 0.8}
    if kind == "read":
        return {"kind": kind, "T": _log(rng, 1, 32768), "y": rng.choice(["f32", "f16", "bf16"]), "format": fmt, "page": page}
    H = rng.choice([16, 32, 40, 64, 128, 128, 128])
    n = 1 if rng.random() < 0.4 else _log(rng, 2, 64)
    L = _log(rng, 64, 16384)
    B = max(1, min(_log(rng, 1, 128), 32 * 16384 // L, 32 * 16 * 128 * 16384 // (n * H * L)))
    return {"kind": kind, "B": B, "n": n, "H": H, "L": max(L, n), "format": fmt, "page": page, "tree": n > 1 and rng.random() < 0.7}


# ---- inputs --------------------------------------------------------------------------
def _gen(case, seed):
    h = seed & 0x7FFFFFFF
    for c in "|".join("%s=%s" % (k, case[k]) for k in sorted(case) if k != "name"):
        h = (h * 1000003 + ord(c) + 1) & 0x7FFFFFFFFFFFFF
    return torch.Generator(device="cuda").manual_seed(h), torch.Generator().manual_seed(h)


def _normal(g, *shape, std=1.0, mean=0.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).add_(mean)


def _filled(fmt, n_pages, page, g):
    """The planes of a cache that earlier steps have filled: (latent, rope, scale)."""
    lat, rot = _normal(g, n_pages, page, LAT), _normal(g, n_pages, page, ROT)
    if fmt != "fp8":
        return lat.to(TYPES[fmt]), rot.to(TYPES[fmt]), None
    lat, scale = _quantise(lat)
    return lat, rot.bfloat16(), scale


def _frequencies(case):
    """Radians a position, in 64 bits: what both forms are given as base, factor and scaling."""
    R, base = case["R"], YARN["base"]
    i = torch.arange(R // 2, device="cuda", dtype=torch.float64)
    f = base ** (-2.0 * i / R)
    if case["scaling"] == "linear":
        f = f / case["factor"]
    if case["scaling"] == "yarn":
        def at(turns):
            return R * math.log(YARN["orig"] / (2.0 * math.pi * turns)) / (2.0 * math.log(base))
        lo = max(math.floor(at(32.0)), 0)
        hi = max(min(math.ceil(at(1.0)), R // 2 - 1), lo + 1)
        keep = 1.0 - ((i - lo) / (hi - lo)).clamp(0.0, 1.0)
        f = f / case["factor"] * (1.0 - keep) + f * keep
    return f


def _table(case):
    import flash_deepseek_amd as fd
    return fd.rope_table(case["R"], base=YARN["base"], layout=case["layout"], scaling=case["scaling"], factor=case["factor"],
                         orig_ctx=YARN["orig"])


CACHE_ROPE = {"R": ROT, "layout": "interleaved", "scaling": "yarn", "factor": YARN["factor"]}


def _cache(s, planes):
    s["latent"], s["rope"], s["scale"] = planes
    if own:
        import flash_deepseek_amd as fd
        s["cache"] = fd.KvCache(*planes)


def _counts(case):
    """Query tokens of each sequence: between half and all of n, the first all."""
    n, B = case["n"], case["B"]
    return n - torch.arange(B) * 7 % (n // 2 + 1)


def prepare(case, seed):
    g, c = _gen(case, seed)
    s = dict(case)
    if own:
        import flash_deepseek_amd as fd
        if not fd.available():
            fd.init(0)
    if case["kind"] == "rope":
        T, H, D = case["T"], case["H"], case["D"]
        x = _normal(g, T, H, D).to(TYPES[case["x"]])
        s["pos"] = torch.randint(0, case["far"], (T,), generator=g, device="cuda", dtype=torch.int32)
        # part: a caller that wants the rotated values alone, read in place out of the heads
        s["q"] = x
        s["view"] = x[:, :, case["offset"]:case["offset"] + case["R"]] if case["part"] else x
        s["at"] = 0 if case["part"] else case["offset"]
        s["out"] = torch.empty(s["view"].shape, dtype=TYPES[case["y"]], device="cuda")
        s["freq"] = _frequencies(case)
        if own:
            s["table"] = _table(case)
        return s
    if case["kind"] in ("write", "read"):
        T, page = case["T"], case["page"]
        n_pages = -(-T // page) + 3
        _cache(s, _filled(case["format"], n_pages, page, g))
        s["slots"] = torch.randperm(n_pages * page, generator=g, device="cuda")[:T].to(torch.int32)
        if case["kind"] == "read":
            s["out"] = torch.empty(T, LAT + ROT, dtype=TYPES[case["y"]], device="cuda")
            return s
        s["kv"] = _normal(g, T, LAT + ROT, std=1.5).to(TYPES[case["x"]])
        s["pos"] = torch.randint(0, 163840, (T,), generator=g, device="cuda", dtype=torch.int32)
        s["norm_w"] = _normal(g, LAT, std=0.1, mean=1.0) if case["norm"] else None
        s["freq"] = _frequencies(CACHE_ROPE)
        if own:
            s["table"] = _table(CACHE_ROPE)
        return s
    B, n, H, L, page = case["B"], case["n"], case["H"], case["L"], case["page"]
    per = -(-L // page)
    _cache(s, _filled(case["format"], B * per + 1, page, g))
    s["pages"] = torch.randperm(B * per + 1, generator=g, device="cuda")[:B * per].to(torch.int32).view(B, per)
    # ragged: lengths between half and all of L, one sequence of the largest
    count = _counts(case)
    length = torch.maximum(torch.randint((L + 1) // 2, L + 1, (B,), generator=c), count)
    length[0] = L
    start = torch.zeros(B + 1, dtype=torch.int64)
    start[1:] = count.cumsum(0)
    N = int(start[-1])
    s["q_start"], s["kv_len"] = start.to(torch.int32).cuda(), length.to(torch.int32).cuda()
    t = TYPES["f16" if case["format"] == "f16" else "bf16"]
    s["q_lat"], s["q_rope"] = _normal(g, N, H, LAT, std=0.6).to(t), _normal(g, N, H, ROT, std=0.6).to(t)
    s["mask"] = None
    if case["tree"]:
        # each token hangs on one of the four before it, or on the prefix; a row has the bits of its branch
        back = torch.randint(1, 5, (B, n), generator=c)
        rows = torch.zeros(B, n, dtype=torch.int64)
        at = torch.arange(B)
        for i in range(n):
            above = torch.where(back[:, i] <= i, rows[at, (i - back[:, i]).clamp(min=0)], torch.zeros(B, dtype=torch.int64))
            rows[:, i] = above | (1 << i if i < 63 else -(1 << 63))
        s["mask"] = rows[torch.arange(n)[None] < count[:, None]].view(N, 1).cuda()
    s["out"] = torch.empty(N, H, LAT, dtype=t, device="cuda")
    s["lse"] = torch.empty(N, H, dtype=torch.float32, device="cuda")
    if own:
        s["workspace"] = fd.mla_workspace(N, H)
    return s


# ---- the plain forms -----------------------------------------------------------------
def _rotate(x, pos, freq, layout):
    """The last dimension of fp32 [T, H, R], the angles in 64 bits."""
    a = pos.double()[:, None, None] * freq
    c, s = a.cos().float(), a.sin().float()
    if layout == "interleaved":
        u, v = x[..., 0::2], x[..., 1::2]
        return torch.stack((u * c - v * s, u * s + v * c), -1).flatten(-2)
    u, v = x.chunk(2, -1)
    return torch.cat((u * c - v * s, u * s + v * c), -1)


def _quantise(x):
    """fp32 [..., 512] -> e4m3 codes and the e8m0 scales of every 128."""
    g = x.unflatten(-1, (-1, GROUP))
    m, e = torch.frexp(g.abs().amax(-1).double() / 448.0)
    e = torch.where(m > 0.5, e, e - 1).clamp(-100, 119)  # the smallest with max <= 448 2^e
    codes = torch.ldexp(g, -e[..., None].to(torch.int32)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).flatten(-2)
    return codes, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _rows(s, slots):
    """Rows of the cache, widened to fp32 [..., 576]."""
    lat = s["latent"].flatten(0, 1).view(torch.uint8 if s["format"] == "fp8" else s["latent"].dtype)[slots]
    rot = s["rope"].flatten(0, 1)[slots].float()
    if s["format"] == "fp8":
        e = s["scale"].flatten(0, 1).view(torch.uint8)[slots].int() - 127
        lat = torch.ldexp(lat.view(torch.float8_e4m3fn).float().unflatten(-1, (-1, GROUP)), e[..., None]).flatten(-2)
    return torch.cat((lat.float(), rot), -1)


def _plain_write(s):
    x = s["kv"].float()
    lat, rot = x[:, :LAT], x[:, LAT:]
    if s["norm_w"] is not None:
        lat = lat * (1.0 / torch.sqrt(lat.square().mean(-1, keepdim=True) + 1e-6)) * s["norm_w"]
    rot = _rotate(rot[:, None], s["pos"], s["freq"], "interleaved")[:, 0]
    slots = s["slots"].long()
    if s["format"] == "fp8":
        codes, e = _quantise(lat)
        s["latent"].flatten(0, 1).view(torch.uint8)[slots] = codes.view(torch.uint8)
        s["scale"].flatten(0, 1).view(torch.uint8)[slots] = e.view(torch.uint8)
    else:
        s["latent"].flatten(0, 1)[slots] = lat.to(s["latent"].dtype)
    s["rope"].flatten(0, 1)[slots] = rot.to(s["rope"].dtype)


def _places(s):
    """Sequence and place of each query token, and the padded lay-out's sizes."""
    N, B = s["q_lat"].shape[0], s["B"]
    t = torch.arange(N, device="cuda")
    b = torch.searchsorted(s["q_start"][1:].long(), t, right=True)
    return t, b, t - s["q_start"].long()[b], B, s["n"]


def _plain_attend(s):
    t, b, i, B, n = _places(s)
    H, L, page = s["H"], s["L"], s["page"]
    p = torch.arange(L, device="cuda")
    slots = s["pages"].long()[:, p // page] * page + p % page
    k = _rows(s, slots)  # [B, L, 576]
    q = torch.zeros(B, n, H, LAT + ROT, device="cuda")
    q[b, i] = torch.cat((s["q_lat"], s["q_rope"]), -1).float()
    score = torch.bmm(q.view(B, n * H, LAT + ROT), k.transpose(1, 2).contiguous()).mul_(SCALE).view(B, n, H, L)
    count = (s["q_start"][1:] - s["q_start"][:-1]).long()
    length = s["kv_len"].long()
    j = p[None] - (length - count)[:, None]  # place among the sequence's tokens, negative in the prefix
    place = torch.arange(n, device="cuda")
    if s["mask"] is not None:
        bits = torch.zeros(B, n, dtype=torch.int64, device="cuda")
        bits[b, i] = s["mask"][:, 0]
        seen = (bits[:, :, None] >> j.clamp(0, 63)[:, None]) & 1 > 0
    else:
        seen = j[:, None] <= place[None, :, None]
    seen = ((j < 0)[:, None] | seen) & (p[None] < length[:, None])[:, None]
    score.masked_fill_(~seen[:, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = score.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    o = torch.bmm(e.view(B, n * H, L), k[..., :LAT].contiguous()).view(B, n, H, LAT)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + total.log())[..., 0]
    return o[b, i].to(s["out"].dtype), lse[b, i]


def run(s):
    kind = s["kind"]
    if own:
        import flash_deepseek_amd as fd
        if kind == "rope":
            fd.rope(s["table"], s["view"], s["pos"], s["out"], offset=s["at"])
            return s["out"]
        if kind == "write":
            fd.kv_write(s["cache"], s["kv"], s["slots"], norm_w=s["norm_w"], table=s["table"], pos=s["pos"])
            return [s["latent"], s["rope"]] + ([s["scale"]] if s["scale"] is not None else [])
        if kind == "read":
            fd.kv_read(s["cache"], s["slots"], s["out"])
            return s["out"]
        fd.mla_attend(s["cache"], s["q_lat"], s["q_rope"], s["q_start"], s["kv_len"], s["pages"], SCALE, s["out"],
                      mask=s["mask"], lse=s["lse"], workspace=s["workspace"])
        return s["out"], s["lse"]
    if kind == "rope":
        x, at, R = s["view"].float(), s["at"], s["R"]
        y = torch.cat((x[..., :at], _rotate(x[..., at:at + R], s["pos"], s["freq"], s["layout"]), x[..., at + R:]), -1)
        return y.to(TYPES[s["y"]])
    if kind == "write":
        _plain_write(s)
        return [s["latent"], s["rope"]] + ([s["scale"]] if s["scale"] is not None else [])
    if kind == "read":
        return _rows(s, s["slots"].long()).to(TYPES[s["y"]])
    return _plain_attend(s)


# ---- what a pass cannot do without ---------------------------------------------------
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
ROW = {"f16": 2 * (LAT + ROT), "bf16": 2 * (LAT + ROT), "fp8": LAT + LAT // GROUP + 2 * ROT}


def work(case):
    if case["kind"] == "rope":
        D = case["R"] if case["part"] else case["D"]
        values = case["T"] * case["H"] * D
        return {"bytes": values * (SIZE[case["x"]] + SIZE[case["y"]]) + 4 * case["T"], "flops": 3 * case["T"] * case["H"] * case["R"]}
    if case["kind"] == "write":
        return {"bytes": case["T"] * ((LAT + ROT) * SIZE[case["x"]] + ROW[case["format"]] + 8), "flops": case["T"] * 4 * (LAT + ROT)}
    if case["kind"] == "read":
        return {"bytes": case["T"] * ((LAT + ROT) * SIZE[case["y"]] + ROW[case["format"]] + 4), "flops": case["T"] * LAT}
    # the lengths as prepare draws them: three quarters of L on the mean, the first sequence whole
    B, n, H, L = case["B"], case["n"], case["H"], case["L"]
    count = _counts(case).double()
    tokens = float(count.sum())
    positions = L + (B - 1) * 0.75 * L
    pairs = n * L + (tokens - n) * 0.75 * L
    if not case["tree"]:  # in order: a token does not see the ones after it
        pairs -= float((count * (count - 1) / 2).sum())
    return {"bytes": positions * ROW[case["format"]] + tokens * H * 2 * (LAT + ROT + LAT), "flops": pairs * H * 2 * (LAT + ROT + LAT)}


# ---- the definitions in 64 bits --------------------------------------------------------
def _turned(x, pos, scaling, factor, layout):
    """The rotation by its definition: each pair a complex number times e^(i a), [T, H, R]."""
    R = x.shape[-1]
    half = R // 2
    freq = []
    for i in range(half):
        f = math.exp(-2.0 * i / R * math.log(YARN["base"]))
        if scaling == "linear":
            f /= factor
        elif scaling == "yarn":
            # the pair whose wave turns `b` times in the original context, for b = 32 and b = 1
            first, last = (math.log(YARN["orig"] / (b * 2.0 * math.pi)) * R / (2.0 * math.log(YARN["base"])) for b in (32.0, 1.0))
            first, last = max(0, math.floor(first)), min(half - 1, math.ceil(last))
            last = max(last, first + 1)
            w = min(1.0, max(0.0, (i - first) / (last - first)))
            f = f * (1.0 - w) + f * w / factor
        freq.append(f)
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), torch.outer(pos.double(), torch.tensor(freq, dtype=torch.float64, device="cuda")))
    x = x.double()
    z = torch.complex(x[..., 0::2].contiguous(), x[..., 1::2].contiguous()) if layout == "interleaved" else torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous())
    z = z * turn[:, None]
    return torch.stack((z.real, z.imag), -1).flatten(-2) if layout == "interleaved" else torch.cat((z.real, z.imag), -1)


def _wide(s):
    """The whole cache in 64 bits, [rows, 576]."""
    lat = s["latent"].double().reshape(-1, LAT // GROUP, GROUP)
    if s["scale"] is not None:
        lat = lat * torch.exp2(s["scale"].view(torch.uint8).double().reshape(-1, LAT // GROUP, 1) - 127.0)
    return torch.cat((lat.reshape(-1, LAT), s["rope"].double().reshape(-1, ROT)), 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        y, a = s["view"].double().clone(), s["at"]
        y[..., a:a + case["R"]] = _turned(y[..., a:a + case["R"]], s["pos"], case["scaling"], case["factor"], case["layout"])
        return y
    if case["kind"] == "read":
        return _wide(s)[s["slots"].long()]
    if case["kind"] == "write":
        x = s["kv"].double()
        lat = x[:, :LAT]
        if s["norm_w"] is not None:
            lat = lat / ((lat * lat).sum(1, keepdim=True) / LAT + 1e-6).sqrt() * s["norm_w"].double()
        rot = _turned(x[:, None, LAT:], s["pos"], "yarn", YARN["factor"], "interleaved")[:, 0]
        at = s["slots"].long()
        whole = [s["latent"].double().reshape(-1, LAT), s["rope"].double().reshape(-1, ROT)]
        whole[1][at] = rot
        if s["scale"] is None:
            whole[0][at] = lat
        else:
            big = lat.reshape(-1, LAT // GROUP, GROUP).abs().max(2, keepdim=True).values
            e = torch.ceil(torch.log2(big / 448.0)).clamp(-100.0, 119.0)
            v = (lat.reshape(-1, LAT // GROUP, GROUP) / torch.exp2(e)).reshape(-1, LAT)
            # e4m3: steps of 2^-3 of the value's power of two, of 2^-9 below 2^-6, ties to even
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3.0)
            whole[0][at] = (torch.round(v / step) * step).clamp(-448.0, 448.0)
            whole.append(s["scale"].double().reshape(-1, LAT // GROUP))
            whole[2][at] = torch.exp2(e)[:, :, 0]
        return [w.reshape(p.shape) for w, p in zip(whole, (s["latent"], s["rope"], s["scale"]))]
    rows, start, length = _wide(s), s["q_start"].tolist(), s["kv_len"].tolist()
    outs, lses = [], []
    for b in range(case["B"]):
        n, L = start[b + 1] - start[b], length[b]
        k = rows[(s["pages"][b].long()[:, None] * case["page"] + torch.arange(case["page"], device="cuda")).reshape(-1)[:L]]
        q = torch.cat((s["q_lat"], s["q_rope"]), -1)[start[b]:start[b + 1]].double()
        z = (q.reshape(n * case["H"], -1) @ k.T * SCALE).reshape(n, case["H"], L)
        among = torch.arange(n, device="cuda")
        if s["mask"] is None:
            dark = among[None, :] > among[:, None]
        else:
            dark = (s["mask"][start[b]:start[b + 1]] >> among[None, :]) & 1 == 0
        z[:, :, L - n:].masked_fill_(dark[:, None], -math.inf)
        lse = torch.logsumexp(z, -1)
        outs.append(((z - lse[..., None]).exp().reshape(n * case["H"], L) @ k[:, :LAT]).reshape(n, case["H"], LAT))
        lses.append(lse)
    return torch.cat(outs), torch.cat(lses)

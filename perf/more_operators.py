"""The operators of a serving step around the paged latent cache: its page
tables and slots, the residual's addition with the norm, and projections with
the requests' low-rank adapters; what is measured of them, with their plain
forms in elementary torch operations.

A case is a dict of plain values with a "kind":

  pages    B sequences give back the pages behind what they keep of up to L
           positions, then get places for up to n new tokens each
  norm     T rows of d values: residual + update, normed, into a wide type or
           into e4m3 with a power-of-two scale for every 128 values
  project  T rows of B requests through a matrix of out x in, and through the
           rank-r adapter of each request, out of `adapters` of them

Formats of a projection: bf16 and f16 rows and matrix, or fp8: e4m3 rows with a
power-of-two scale for every 128 values, an e4m3 matrix with one for every 128 x 128.
"""
import math

import torch

own = False

GROUP = 128
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a decode step of drafted tokens: the last step's rejected ones go, the next ones get places
        {"name": "pages_step_b64", "kind": "pages", "B": 64, "n": 4, "L": 4096, "page": 64, "ended": 0.0},
        # a batch of prompts in place of requests that ended, small pages
        {"name": "pages_prompts_b512", "kind": "pages", "B": 512, "n": 2048, "L": 6000, "page": 16, "ended": 0.75},
        # a decode step's residual stream in fp32, e4m3 rows for the projection behind it
        {"name": "norm_step_t16", "kind": "norm", "T": 16, "d": 7168, "x": "f32", "add": "f32", "y": "fp8"},
        # a query's latent rows normed alone, a ragged number of them
        {"name": "norm_rows_t1001", "kind": "norm", "T": 1001, "d": 1536, "x": "bf16", "add": None, "y": "bf16"},
        # a long prompt's residual stream
        {"name": "norm_prompt_t16384", "kind": "norm", "T": 16384, "d": 7168, "x": "bf16", "add": "bf16", "y": "fp8"},
        # one request's token through the query's first projection: latency
        {"name": "project_one_bf16", "kind": "project", "B": 1, "n": 1, "in": 7168, "out": 1536, "rank": 16, "adapters": 1, "format": "bf16", "y": "bf16"},
        # a decode step of many requests, query and cache rows in one matrix, several adapters
        {"name": "project_step_fp8_b64", "kind": "project", "B": 64, "n": 1, "in": 7168, "out": 2112, "rank": 16, "adapters": 8, "format": "fp8", "y": "f32"},
        # three drafted tokens of eight requests into every head's query
        {"name": "project_step_f16_b8", "kind": "project", "B": 8, "n": 3, "in": 1536, "out": 24576, "rank": 32, "adapters": 4, "format": "f16", "y": "f16"},
        # a chunk of ragged prompts, odd sizes, the adapters' result in fp32
        {"name": "project_chunk_bf16_t500", "kind": "project", "B": 3, "n": 223, "in": 7168, "out": 2111, "rank": 64, "adapters": 2, "format": "bf16", "y": "f32"},
        # a busy step: a token each of 256 requests, 32 adapters, back into the residual stream
        {"name": "project_step_bf16_b256", "kind": "project", "B": 256, "n": 1, "in": 16384, "out": 7168, "rank": 16, "adapters": 32, "format": "bf16", "y": "bf16"},
        # prompts through the attention's output projection
        {"name": "project_prompt_bf16_t4096", "kind": "project", "B": 5, "n": 1024, "in": 16384, "out": 7168, "rank": 32, "adapters": 4, "format": "bf16", "y": "bf16"},
        # the largest: prompts through a dense layer's gate in 8 bits
        {"name": "project_prompt_fp8_t8191", "kind": "project", "B": 7, "n": 1489, "in": 7168, "out": 18432, "rank": 16, "adapters": 4, "format": "fp8", "y": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["pages", "norm", "norm", "project", "project", "project", "project"])
    if kind == "pages":
        B, n = _log(rng, 1, 512), _log(rng, 1, 2048)
        return {"kind": kind, "B": B, "n": n, "L": _log(rng, 16, 6000), "page": 2 ** rng.randint(4, 8), "ended": rng.choice([0.0, 0.25, 0.75])}
    if kind == "norm":
        x = rng.choice(["f32", "f16", "bf16"])
        d = rng.choice([512, 1536, 7168, 8 * _log(rng, 4, 2048), _log(rng, 30, 16384)])
        add = rng.choice([None, x, x, "bf16"])
        return {"kind": kind, "T": min(_log(rng, 1, 16384), 16384 * 7168 // (2 * d)), "d": d, "x": x, "add": add,
                "y": rng.choice(["fp8", "fp8", "bf16", "f16", "f32"])}
    fmt = rng.choice(["fp8", "bf16", "f16"])
    B, n = _log(rng, 1, 256), 1 if rng.random() < 0.5 else _log(rng, 2, 1500)
    inner = rng.choice([1536, 2048, 7168, 16 * _log(rng, 4, 1024)])
    out = rng.choice([576, 2112, 7168, 18432, _log(rng, 33, 24576)])
    most = 8191 * 7168 * 18432 // (2 * inner * out)
    B = max(1, min(B, 8191 // n, most // n))
    return {"kind": kind, "B": B, "n": max(1, min(n, most)), "in": inner, "out": out, "rank": rng.choice([8, 16, 16, 24, 32, 64, 128]),
            "adapters": min(_log(rng, 1, 32), B), "format": fmt, "y": rng.choice(["f32", "f16" if fmt == "f16" else "bf16"])}


# ---- inputs --------------------------------------------------------------------------
def _gen(case, seed):
    h = seed & 0x7FFFFFFF
    for c in "|".join("%s=%s" % (k, case[k]) for k in sorted(case) if k != "name"):
        h = (h * 1000003 + ord(c) + 1) & 0x7FFFFFFFFFFFFF
    return torch.Generator(device="cuda").manual_seed(h), torch.Generator().manual_seed(h)


def _normal(g, *shape, std=1.0, mean=0.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).add_(mean)


def _counts(case):
    """Tokens of each request: between half and all of n, the first all."""
    n, B = case["n"], case["B"]
    return n - torch.arange(B) * 7 % (n // 2 + 1)


def _codes(g):
    """fp32 [..., values that share a scale] -> e4m3 codes and the exponents of their power-of-two scales."""
    m, e = torch.frexp(g.abs().amax(-1).double() / 448.0)
    e = torch.where(m > 0.5, e, e - 1).clamp(-100, 119)  # the smallest with max <= 448 2^e
    return torch.ldexp(g, -e[..., None].to(torch.int32)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), e


def _bytes(e):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _padded(x, dim):
    """x with zeros behind its last values along `dim`, up to whole groups."""
    more = -x.shape[dim] % GROUP
    return torch.cat((x, x.new_zeros(*[more if k == dim % x.dim() else s for k, s in enumerate(x.shape)])), dim) if more else x


def _quantise_rows(x):
    """fp32 [T, d] -> codes [T, d] and a scale for every 128 values of a row."""
    codes, e = _codes(_padded(x, 1).unflatten(1, (-1, GROUP)))
    return codes.view(torch.uint8).flatten(1)[:, :x.shape[1]].contiguous().view(torch.float8_e4m3fn), _bytes(e)


def _quantise_matrix(w):
    """fp32 [out, in] -> codes [out, in] and a scale for every 128 x 128."""
    out, inner = w.shape
    p = _padded(_padded(w, 0), 1)
    tiles = p.view(p.shape[0] // GROUP, GROUP, p.shape[1] // GROUP, GROUP).transpose(1, 2)
    codes, e = _codes(tiles.flatten(2))
    codes = codes.view(torch.uint8).view(tiles.shape).transpose(1, 2).reshape(p.shape)[:out, :inner]
    return codes.contiguous().view(torch.float8_e4m3fn), _bytes(e)


def _prepare_pages(case, s, g, c):
    B, n, L, page = case["B"], case["n"], case["L"], case["page"]
    new = _counts(case)
    keep = torch.randint((L + 1) // 2, L + 1, (B,), generator=c)
    keep[0] = L
    keep[torch.rand(B, generator=c) < case["ended"]] = 0  # requests that ended: others are in their places
    length = keep + new  # as the last step left it
    P = -(-(L + n) // page)
    used = -(-length // page)
    n_pages = B * P + 3
    order = torch.randperm(n_pages, generator=c)
    table = torch.full((B, P), -1, dtype=torch.int64)
    table[torch.arange(P)[None] < used[:, None]] = order[:int(used.sum())]
    spare = order[int(used.sum()):]
    free = torch.zeros(n_pages, dtype=torch.int64)
    free[:spare.numel()] = spare
    N = int(new.sum()) + 5  # a padded batch
    for name, v in (("new", new), ("keep", keep), ("kv_len", length), ("pages", table), ("free", free), ("n_free", torch.tensor([spare.numel()]))):
        s[name] = v.to(torch.int32).cuda()
    for name, k in (("q_start", B + 1), ("pos", N), ("slots", N), ("refused", 1)):
        s[name] = torch.empty(k, dtype=torch.int32, device="cuda")
    if own:
        import flash_deepseek_amd as fd
        s["table"] = fd.KvPages(s["pages"], s["kv_len"], s["free"], s["n_free"], page)


def _prepare_norm(case, s, g):
    T, d = case["T"], case["d"]
    x = _normal(g, T, d, std=2.0)
    x[:, ::97] *= 20.0  # a few channels of a residual stream are far larger
    s["x"] = x.to(TYPES[case["x"]])
    s["add"] = None if case["add"] is None else _normal(g, T, d).to(TYPES[case["add"]])
    s["norm_w"] = _normal(g, d, std=0.1, mean=1.0)
    s["sum"] = None if case["add"] is None else torch.empty_like(s["x"])
    if case["y"] == "fp8":
        s["out"] = torch.empty(T, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        s["scale"] = torch.empty(T, -(-d // GROUP), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    else:
        s["out"], s["scale"] = torch.empty(T, d, dtype=TYPES[case["y"]], device="cuda"), None


def _prepare_project(case, s, g, c):
    B, inner, out, r, fmt = case["B"], case["in"], case["out"], case["rank"], case["format"]
    t = TYPES["f16" if fmt == "f16" else "bf16"]
    start = torch.zeros(B + 1, dtype=torch.int64)
    start[1:] = _counts(case).cumsum(0)
    T = int(start[-1])
    s["q_start"] = start.to(torch.int32).cuda()
    which = torch.randint(0, case["adapters"], (B,), generator=c)
    which[(torch.rand(B, generator=c) < 0.125) & (torch.arange(B) > 0)] = -1  # requests of the model as it is
    s["adapter"] = which.to(torch.int32).cuda()
    x, w = _normal(g, T, inner), _normal(g, out, inner, std=inner ** -0.5)
    if fmt == "fp8":
        (s["x"], s["x_scale"]), (s["w"], s["w_scale"]) = _quantise_rows(x), _quantise_matrix(w)
    else:
        s["x"], s["w"], s["x_scale"], s["w_scale"] = x.to(t), w.to(t), None, None
    s["a"] = _normal(g, case["adapters"], r, inner, std=inner ** -0.5).to(t)
    s["b"] = _normal(g, case["adapters"], out, r, std=0.5 * r ** -0.5).to(t)
    s["times"] = torch.rand(case["adapters"], generator=g, device="cuda", dtype=torch.float32) + 0.5
    s["out_rows"] = torch.empty(T, out, dtype=TYPES[case["y"]], device="cuda")
    if own:
        import flash_deepseek_amd as fd
        s["adapters_of"] = fd.Adapters(s["a"], s["b"], s["times"])
        s["workspace"] = fd.project_workspace(T, inner, out, r)


def prepare(case, seed):
    g, c = _gen(case, seed)
    s = dict(case)
    if own:
        import flash_deepseek_amd as fd
        if not fd.available():
            fd.init(0)
    if case["kind"] == "pages":
        _prepare_pages(case, s, g, c)
    elif case["kind"] == "norm":
        _prepare_norm(case, s, g)
    else:
        _prepare_project(case, s, g, c)
    return s


# ---- the plain forms -----------------------------------------------------------------
def _plain_trim(s):
    pages, page, P = s["pages"], s["page"], s["pages"].shape[1]
    n_pages = s["free"].numel()
    length = s["kv_len"].long().clamp(0, P * page)
    keep = torch.where(s["keep"] < 0, length, torch.minimum(s["keep"].long(), length))
    have, stay = (length + page - 1) // page, (keep + page - 1) // page
    give = have - stay
    before, total = give.cumsum(0) - give, give.sum()
    p = torch.arange(P, device="cuda")[None]
    goes = (p >= stay[:, None]) & (p < have[:, None])
    at = s["n_free"].long() + total - 1 - (before[:, None] + p - stay[:, None])
    free = torch.cat((s["free"], s["free"].new_zeros(1)))  # the last: of the pages that stay
    free[torch.where(goes, at, n_pages)] = pages
    s["free"].copy_(free[:n_pages])
    s["n_free"].add_(total.int())
    s["kv_len"].copy_(keep)


def _plain_grow(s):
    pages, page, (B, P) = s["pages"], s["page"], s["pages"].shape
    N, n_pages = s["slots"].numel(), s["free"].numel()
    length, new = s["kv_len"].long().clamp(0, P * page), s["new"].long().clamp(min=0)
    room = length + new <= P * page
    have = (length + page - 1) // page
    need = torch.where(room, (length + new + page - 1) // page - have, 0)
    taken, tokens = need.cumsum(0), torch.where(room, new, 0).cumsum(0)
    served = room & ((need == 0) | (taken <= s["n_free"].long())) & (tokens <= N)
    n, need = torch.where(served, new, 0), torch.where(served, need, 0)
    end = n.cumsum(0)
    s["q_start"][:1] = 0
    s["q_start"][1:] = end
    p = torch.arange(P, device="cuda")[None]
    first = need.cumsum(0) - need
    at = s["n_free"].long() - 1 - (first[:, None] + p - have[:, None])
    comes = (p >= have[:, None]) & (p < (have + need)[:, None])
    pages.copy_(torch.where(comes, s["free"][at.clamp(0, n_pages - 1)], pages))
    s["kv_len"].copy_(length + n)
    s["n_free"].sub_(need.sum().int())
    s["refused"].copy_(((new > 0) & ~served).sum()[None])
    t = torch.arange(N, device="cuda")
    b = torch.searchsorted(end, t, right=True).clamp(max=B - 1)
    live = t < end[-1]
    pos = length[b] + t - (end - n)[b]
    of = pages.flatten()[(b * P + pos // page).clamp(0, B * P - 1)].long()
    s["pos"].copy_(torch.where(live, pos, 0))
    s["slots"].copy_(torch.where(live, of * page + pos % page, -1))


def _plain_norm(s):
    h = s["x"].float()
    if s["add"] is not None:
        h = h + s["add"].float()
    if s["sum"] is not None:
        s["sum"].copy_(h)
    y = h * (1.0 / torch.sqrt(h.square().mean(1, keepdim=True) + EPS)) * s["norm_w"]
    if s["scale"] is None:
        return [y.to(s["out"].dtype)] + ([s["sum"]] if s["sum"] is not None else [])
    return list(_quantise_rows(y)) + ([s["sum"]] if s["sum"] is not None else [])


def _wide_rows(codes, scale):
    e = scale.view(torch.uint8).int() - 127
    g = _padded(codes.float(), 1).unflatten(1, (-1, GROUP))
    return torch.ldexp(g, e[..., None]).flatten(1)[:, :codes.shape[1]]


def _wide_matrix(codes, scale):
    e = (scale.view(torch.uint8).int() - 127).repeat_interleave(GROUP, 0)[:codes.shape[0]].repeat_interleave(GROUP, 1)[:, :codes.shape[1]]
    return torch.ldexp(codes.float(), e)


def _plain_project(s):
    fp8 = s["format"] == "fp8"
    x = _wide_rows(s["x"], s["x_scale"]) if fp8 else s["x"].float()
    w = _wide_matrix(s["w"], s["w_scale"]) if fp8 else s["w"].float()
    n, r, inner = s["a"].shape
    y = x @ w.T
    # every adapter's product, of which each row keeps its own
    t = torch.arange(x.shape[0], device="cuda")
    mine = s["adapter"][torch.searchsorted(s["q_start"][1:].long(), t, right=True)]
    u = (x @ s["a"].float().view(n * r, inner).T).view(-1, n, r)
    u = u * torch.where(mine[:, None] == torch.arange(n, device="cuda")[None], s["times"], 0.0)[..., None]
    y += u.flatten(1) @ s["b"].float().transpose(1, 2).reshape(n * r, -1)
    return y.to(s["out_rows"].dtype)


def run(s):
    kind = s["kind"]
    if own:
        import flash_deepseek_amd as fd
        if kind == "pages":
            fd.kv_trim(s["table"], s["keep"])
            fd.kv_grow(s["table"], s["new"], s["q_start"], s["pos"], s["slots"], refused=s["refused"])
            return [s[k] for k in ("q_start", "pos", "slots", "refused", "pages", "kv_len", "free", "n_free")]
        if kind == "norm":
            fd.add_rms_norm(s["x"], s["add"], s["norm_w"], s["out"], scale=s["scale"], sum=s["sum"], eps=EPS)
            return [v for v in (s["out"], s["scale"], s["sum"]) if v is not None]
        fd.project(s["x"], s["w"], s["out_rows"], x_scale=s["x_scale"], w_scale=s["w_scale"], adapters=s["adapters_of"],
                   q_start=s["q_start"], adapter=s["adapter"], workspace=s["workspace"])
        return s["out_rows"]
    if kind == "pages":
        _plain_trim(s)
        _plain_grow(s)
        return [s[k] for k in ("q_start", "pos", "slots", "refused", "pages", "kv_len", "free", "n_free")]
    return _plain_norm(s) if kind == "norm" else _plain_project(s)


# ---- what a pass cannot do without ---------------------------------------------------
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "fp8": 1}


def work(case):
    if case["kind"] == "pages":
        new = float(_counts(case).sum())
        moved = new / case["page"]  # pages given back, and taken again
        return {"bytes": 8 * (new + 5) + 4 * (4 * moved + 6 * case["B"]), "flops": 2 * new}
    if case["kind"] == "norm":
        T, d = case["T"], case["d"]
        add = 0 if case["add"] is None else SIZE[case["add"]] + SIZE[case["x"]]  # the update read, the sum written
        scales = -(-d // GROUP) if case["y"] == "fp8" else 0
        return {"bytes": T * (d * (SIZE[case["x"]] + add + SIZE[case["y"]]) + scales) + 4 * d, "flops": 5 * T * d}
    T, inner, out, r = float(_counts(case).sum()), case["in"], case["out"], case["rank"]
    size, used = SIZE[case["format"]], min(case["adapters"], case["B"])
    scales = T * inner / GROUP + inner * out / GROUP ** 2 if case["format"] == "fp8" else 0
    return {"bytes": size * (T + out) * inner + scales + 2 * used * r * (inner + out) + SIZE[case["y"]] * T * out + 8 * case["B"],
            "flops": 2 * T * (inner * out + r * (inner + out))}


# ---- the definitions in 64 bits --------------------------------------------------------
def _value_of(scale):
    return torch.exp2(scale.view(torch.uint8).double() - 127.0)


def _exact_norm(case, s):
    h = s["x"].double()
    if s["add"] is not None:
        h = h + s["add"].double()
    y = h / ((h * h).sum(1, keepdim=True) / case["d"] + EPS).sqrt() * s["norm_w"].double()
    more = [] if s["sum"] is None else [h]
    if case["y"] != "fp8":
        return [y] + more
    T, d = y.shape
    groups = -(-d // GROUP)
    filled = torch.zeros(T, groups * GROUP, dtype=torch.float64, device="cuda")
    filled[:, :d] = y
    filled = filled.reshape(T, groups, GROUP)
    e = torch.ceil(torch.log2(filled.abs().max(2, keepdim=True).values / 448.0)).clamp(-100.0, 119.0)
    v = filled / torch.exp2(e)
    # e4m3: steps of 2^-3 of the value's power of two, of 2^-9 below 2^-6, ties to even
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3.0)
    v = (torch.round(v / step) * step).clamp(-448.0, 448.0).reshape(T, -1)[:, :d]
    return [v, torch.exp2(e)[..., 0]] + more


def _exact_project(case, s):
    x, w = s["x"].double(), s["w"].double()
    if s["x_scale"] is not None:
        at_x = torch.arange(case["in"], device="cuda") // GROUP
        at_w = torch.arange(case["out"], device="cuda") // GROUP
        x = x * _value_of(s["x_scale"])[:, at_x]
        w = w * _value_of(s["w_scale"])[at_w][:, at_x]
    y = torch.mm(x, w.t())
    start = s["q_start"].tolist()
    for b, k in enumerate(s["adapter"].tolist()):
        if k >= 0:
            rows = slice(start[b], start[b + 1])
            y[rows] += float(s["times"][k]) * ((x[rows] @ s["a"][k].double().t()) @ s["b"][k].double().t())
    return y


def exact(case, seed):
    if case["kind"] == "pages":
        return None  # whole numbers: the plain form's are the definition's
    s = prepare(case, seed)
    return _exact_norm(case, s) if case["kind"] == "norm" else _exact_project(case, s)

"""Float64 forms of the operators around the paged latent cache, for the tests
of rope, kv_write / kv_read and mla_attend.  Everything runs on the CPU."""
import math

import torch

LAT, ROT, GROUP = 512, 64, 128
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # relative, to nearest
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def frequencies(dim, base=10000.0, scaling="none", factor=1.0, orig=4096):
    f = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "yarn":
        def c(turns):
            return dim * math.log(orig / (2.0 * math.pi * turns)) / (2.0 * math.log(base))
        lo = max(math.floor(c(32.0)), 0)
        hi = max(min(math.ceil(c(1.0)), dim // 2 - 1), lo + 1)
        ramp = [min(max((i - lo) / (hi - lo), 0.0), 1.0) for i in range(dim // 2)]
        f = [x / factor * r + x * (1.0 - r) for x, r in zip(f, ramp)]
    return torch.tensor(f, dtype=torch.float64)


def turned(x, pos, freq, layout, mul=1.0):
    """x [T, H, R] in float64, and |u| + |v| of each value's pair."""
    a = pos.double()[:, None, None] * freq
    c, s = a.cos() * mul, a.sin() * mul
    half = freq.numel()
    u, v = (x[..., 0::2], x[..., 1::2]) if layout == "interleaved" else (x[..., :half], x[..., half:])
    p, q, size = u * c - v * s, u * s + v * c, (u.abs() + v.abs()) * abs(mul)
    if layout == "interleaved":
        return torch.stack((p, q), -1).flatten(-2), torch.stack((size, size), -1).flatten(-2)
    return torch.cat((p, q), -1), torch.cat((size, size), -1)


# a turned value: the angle is off by 3 2^-24 (pi / 4) of the turn taken off to an eighth, the sine
# and cosine by 2.5e-8 and two roundings more, mul, two products and their difference round once each
TURN_TOL = 10 * 2.0 ** -24


def quantised(x):
    """The codes of float32 [..., 512] and their exponents, by definition: per 128 values the
    smallest e with max <= 448 2^e in -100 .. 119, codes to nearest even."""
    g = x.unflatten(-1, (-1, GROUP))
    m, e = torch.frexp(g.abs().amax(-1).double() / 448.0)
    e = torch.where(m > 0.5, e, e - 1).clamp(-100, 119)
    e = torch.where(g.abs().amax(-1) == 0, torch.full_like(e, -100), e)
    codes = torch.ldexp(g.double(), -e[..., None]).clamp(-448.0, 448.0).float().to(torch.float8_e4m3fn)
    return codes.flatten(-2), e


def normed(x, w):
    return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w


def widened(latent, rope, scale=None):
    """Cache planes -> float64 [rows, 576]."""
    lat = latent.double().reshape(-1, LAT)
    if scale is not None:
        byte = scale.view(torch.uint8).reshape(-1, LAT // GROUP)
        s = torch.where(byte == 255, torch.full(byte.shape, math.nan, dtype=torch.float64), torch.exp2(byte.double() - 127.0))
        lat = (lat.unflatten(-1, (-1, GROUP)) * s[..., None]).flatten(-2)
    return torch.cat((lat, rope.double().reshape(-1, ROT)), 1)


def attend(rows, page, q_lat, q_rope, q_start, kv_len, pages, scale, mask=None):
    """(out, lse, tolerance of out, tolerance of lse) in float64 for every token
    of a sequence; NaN elsewhere.  The tolerances, for results of 16-bit type t:
      scores: 576 fp32 products and sums of exact 16-bit products, the scale and
        exponent: |ds| <= 2^-24 (600 scale sum |q k| + 4 |s|), and two roundings of the exponential's 2^-22
      weights: each off by ds and, before the second product, half a step of t
      out: sum p |c| (half step + 2 ds + 2^-24 len) and half a step of itself"""
    N, H, _ = q_lat.shape
    step = HALF_STEP[q_lat.dtype]
    out = torch.full((N, H, LAT), math.nan, dtype=torch.float64)
    lse = torch.full((N, H), math.nan, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    n_rows = rows.shape[0]
    for b in range(len(kv_len)):
        t0, t1, L = int(q_start[b]), int(q_start[b + 1]), int(kv_len[b])
        n = t1 - t0
        if n == 0:
            continue
        at = torch.tensor([int(pages[b][j // page]) * page + j % page if 0 <= int(pages[b][j // page]) < n_rows // page
                           else -1 for j in range(L)], dtype=torch.int64)
        k = rows[at.clamp(min=0)]
        seen = torch.zeros(n, L, dtype=torch.bool)
        for i in range(n):
            for j in range(L):
                d = j - (L - n)
                if d < 0:
                    seen[i, j] = True
                elif mask is None:
                    seen[i, j] = d <= i
                else:
                    seen[i, j] = d < 64 * mask.shape[1] and (int(mask[t0 + i, d // 64]) >> (d % 64)) & 1 == 1
        seen &= (at >= 0)[None]
        k = torch.where(seen.any(0)[:, None], k, torch.zeros_like(k)) if L else k
        q = torch.cat((q_lat[t0:t1], q_rope[t0:t1]), -1).double()
        s = torch.einsum("nhd,ld->nhl", q, k) * scale
        size = torch.einsum("nhd,ld->nhl", q.abs(), k.abs()) * abs(scale)
        s = s.masked_fill(~seen[:, None], -math.inf)
        size = size.masked_fill(~seen[:, None], 0.0)
        top = s.amax(-1, keepdim=True) if L else torch.full((n, H, 1), -math.inf, dtype=torch.float64)
        e = (s - top.nan_to_num(neginf=0.0)).exp()
        total = e.sum(-1, keepdim=True)
        p = torch.where(total > 0, e / total, torch.zeros_like(e))
        ds = (2.0 ** -24 * (600 * size + 4 * s.abs().masked_fill(~seen[:, None], 0.0))).amax(-1, keepdim=True) + 2.0 ** -21 if L else torch.zeros(n, H, 1)
        o = torch.einsum("nhl,ld->nhd", p, k[:, :LAT])
        out[t0:t1] = o
        lse[t0:t1] = (top + total.log())[..., 0]
        tol[t0:t1] = torch.einsum("nhl,ld->nhd", p, k[:, :LAT].abs()) * (step + 2 * ds + 2.0 ** -24 * L) + o.abs() * step
        ltol[t0:t1] = (ds + 2.0 ** -24 * L + 2.0 ** -22 * (1 + lse[t0:t1, :, None].abs().nan_to_num(posinf=0.0)))[..., 0]
    return out, lse, tol, ltol


def check(got, want, tol, what):
    got = got.double()
    fine = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()), what
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()]), what
    off = (got - want).abs()[fine] - tol.expand_as(want)[fine]
    assert off.numel() == 0 or off.max() <= 0, (what, float(off.max()), float((got - want).abs()[fine].max()))

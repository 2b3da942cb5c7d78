"""Plain forms of what stands between two attentions (kv_grow / kv_trim,
add_rms_norm, project), for their tests.  Everything runs on the CPU, in whole
numbers or in float64."""
import math

import torch

from tests.latent_case import DTYPES, HALF_STEP, check, quantised  # noqa: F401  (for the tests)

GROUP = 128


# ---- the cache's books, sequence by sequence ---------------------------------------------
class Books:
    def __init__(self, pages, kv_len, free, n_free, page):
        self.pages, self.kv_len, self.free = [list(p) for p in pages], list(kv_len), list(free)
        self.n_free, self.page, self.n_pages = n_free, page, len(free)
        self.room = min(len(self.pages[0]) * page, 2 ** 31 - 4097)

    def _count(self):
        self.kv_len = [min(max(n, 0), self.room) for n in self.kv_len]
        self.n_free = min(max(self.n_free, 0), self.n_pages)

    def _of(self, n):
        return -(-n // self.page)

    def trim(self, keep):
        self._count()
        back = []
        for b, k in enumerate(keep):
            stay = self.kv_len[b] if k < 0 else min(k, self.kv_len[b])
            back += [self.pages[b][p] for p in range(self._of(stay), self._of(self.kv_len[b]))]
            self.kv_len[b] = stay
        for p in reversed(back):
            if self.n_free < self.n_pages:
                self.free[self.n_free] = p
                self.n_free += 1

    def grow(self, new, N):
        """(q_start, pos, slots, refused)"""
        self._count()
        q_start, pos, slots, refused = [0], [], [], 0
        pages = tokens = 0  # asked for so far
        top = self.n_free
        for b, n in enumerate(new):
            n, at = max(n, 0), self.kv_len[b]
            served = at + n <= self.room
            if served:
                need = self._of(at + n) - self._of(at)
                pages, tokens = pages + need, tokens + n
                served = (need == 0 or pages <= top) and tokens <= N
            if served:
                for p in range(self._of(at), self._of(at + n)):
                    self.n_free -= 1
                    self.pages[b][p] = self.free[self.n_free]
                for i in range(at, at + n):
                    page = self.pages[b][i // self.page]
                    pos.append(i)
                    slots.append(page * self.page + i % self.page if 0 <= page < self.n_pages else -1)
                self.kv_len[b] += n
            elif n:
                refused += 1
            q_start.append(len(pos))
        return q_start, pos + [0] * (N - len(pos)), slots + [-1] * (N - len(slots)), refused


# ---- the norm ------------------------------------------------------------------------------
# Of the sum of squares: 32 values a thread, 6 + 16 partial sums (54 roundings, halved by the
# root), the sum s itself twice, the mean, the addition of eps, root, quotient, two products
NORM_TOL = (27 + 2 + 7) * 2.0 ** -24


def normed(x, add, w, eps):
    s = x.double() + (0.0 if add is None else add.double())
    y = s / (s.square().mean(-1, keepdim=True) + eps).sqrt()
    return s, y if w is None else y * w.double()


def check_codes(codes, scale, want, tol):
    """e4m3 codes and their scale bytes against values that the kernel had within tol (relative)."""
    T, d = want.shape
    for g in range(-(-d // GROUP)):
        part, got = want[:, g * GROUP:(g + 1) * GROUP], codes[:, g * GROUP:(g + 1) * GROUP].double()
        byte, top = scale[:, g].int(), part.abs().amax(-1)
        bad = ~part.isfinite().all(-1)
        assert torch.equal(byte == 255, bad)
        assert got[bad].isnan().all()
        e = (byte - 127)[~bad]
        top, part, got = top[~bad], part[~bad], got[~bad]
        one = torch.exp2(e.double())
        assert (e >= -100).all() and (e <= 119).all()
        assert ((top <= 448 * one * (1 + tol)) | (e == 119)).all()
        assert ((top >= 224 * one * (1 - tol)) | (e == -100)).all()
        part = part / one[:, None]
        # half a step of e4m3, of its smallest numbers below 2^-6; those past 448 are cut
        off = (got - part).abs() - part.abs() * tol
        assert (off <= torch.clamp(part.abs() * 2.0 ** -4, min=2.0 ** -10)).all()


# ---- the projection --------------------------------------------------------------------------
def quantised_rows(x):
    """float32 [T, d] -> codes [T, d] and scale bytes [T, ceil(d / 128)]."""
    T, d = x.shape
    p = torch.zeros(T, -(-d // GROUP) * GROUP)
    p[:, :d] = x
    g = p.unflatten(1, (-1, GROUP))
    m, e = torch.frexp(g.abs().amax(-1).double() / 448.0)
    e = torch.where(m > 0.5, e, e - 1).clamp(-100, 119)
    codes = torch.ldexp(g.double(), -e[..., None]).clamp(-448.0, 448.0).float().to(torch.float8_e4m3fn)
    return codes.flatten(1)[:, :d].contiguous(), (e + 127).to(torch.uint8)


def quantised_matrix(w):
    """float32 [out, in] -> codes and scale bytes [ceil(out / 128), ceil(in / 128)]."""
    out, inner = w.shape
    codes = torch.zeros(out, inner, dtype=torch.float8_e4m3fn)
    scale = torch.zeros(-(-out // GROUP), -(-inner // GROUP), dtype=torch.uint8)
    for i in range(scale.shape[0]):
        for j in range(scale.shape[1]):
            t = w[i * GROUP:(i + 1) * GROUP, j * GROUP:(j + 1) * GROUP]
            c, s = t.reshape(1, -1), None
            m, e = math.frexp(float(c.abs().max()) / 448.0)
            s = min(max(e if m > 0.5 else e - 1, -100), 119)
            codes[i * GROUP:(i + 1) * GROUP, j * GROUP:(j + 1) * GROUP] = torch.ldexp(t.double(), torch.tensor(-s)).clamp(-448, 448).float().to(torch.float8_e4m3fn)
            scale[i, j] = s + 127
    return codes, scale


def widened_rows(codes, scale):
    v = torch.where(scale == 255, math.nan, torch.exp2(scale.double() - 127.0))
    return codes.double() * v.repeat_interleave(GROUP, 1)[:, :codes.shape[1]]


def widened_matrix(codes, scale):
    v = torch.where(scale == 255, math.nan, torch.exp2(scale.double() - 127.0))
    return codes.double() * v.repeat_interleave(GROUP, 0)[:codes.shape[0]].repeat_interleave(GROUP, 1)[:, :codes.shape[1]]


def projected(x, w, out_type, a=None, b=None, times=None, q_start=None, adapter=None, half=torch.bfloat16, native=False):
    """(y, tolerance) in float64.  Products of the inputs are exact in fp32; they are added eight
    and more at a time, in any order: (K / 8 + 24) roundings of at most 2^-23 of the sum of their
    sizes (parts and splits among them).  u = A x: the same and one product; where it stands as
    two 16-bit numbers, off by their second's half step (bf16 2^-16 of it; f16 2^-22, and 2^-24 of the
    row's largest); B u: rank products in fp32.  The result: half a step.
    native: the fp8 products of the matrix cores add eight neighbours first, each cut off at
    2^-13 of the largest one's power of two: seven of them lose that at most, and the largest is
    at most the eight's sum of sizes."""
    x, w = x.double(), w.double()
    n = x.shape[1] / 8 + 24
    y, size = x @ w.T, x.abs() @ w.abs().T
    tol = size * (n * 2.0 ** -23 + (7 * 2.0 ** -13 if native else 0.0))
    if a is not None:
        for r in range(len(adapter)):
            k = int(adapter[r])
            if not 0 <= k < a.shape[0]:
                continue
            t = slice(max(int(q_start[r]), 0), min(max(int(q_start[r + 1]), 0), x.shape[0]))
            c, A, B = (1.0 if times is None else float(times[k])), a[k].double(), b[k].double()
            u = x[t] @ A.T * c
            du = (x[t].abs() @ A.abs().T) * abs(c) * (n + 2) * 2.0 ** -23
            du += u.abs() * 2.0 ** -16 if half is torch.bfloat16 else u.abs() * 2.0 ** -22 + u.abs().amax(-1, keepdim=True) * 2.0 ** -24
            y[t] += u @ B.T
            tol[t] += du @ B.abs().T + (u.abs() @ B.abs().T) * (a.shape[1] / 8 + 24) * 2.0 ** -23
    tol += y.abs() * HALF_STEP[out_type] + (2.0 ** -25 if out_type is torch.float16 else 0.0)
    return y, tol

"""64-bit statements of counter-based dropout and of the residual seam, with bounds on what a correct 32-bit
evaluation may be off, for the tests."""

import numpy as np
import torch

from ffn_reference import HALF_STEP, U32

TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}   # half of the smallest step


# ------------------------------------------------------------------ the generator
def philox(key, ctr, rounds=7):
    """Philox4x32 on arrays of four counter words and two key words (unsigned 32-bit numbers in uint64)."""
    m, h = np.uint64(0xFFFFFFFF), np.uint64(32)
    ctr, key = [np.asarray(c, np.uint64) for c in ctr], [np.uint64(k) for k in key]
    for _ in range(rounds):
        a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(b >> h) ^ ctr[1] ^ key[0], b & m, (a >> h) ^ ctr[3] ^ key[1], a & m]
        key = [(key[0] + np.uint64(0x9E3779B9)) & m, (key[1] + np.uint64(0xBB67AE85)) & m]
    return ctr


def bits(seed, N, F, stream, row0=0):
    """The 16 bits of every element [N, F], from row `row0` on."""
    s = int(seed) % 2 ** 64
    g = np.arange(-(-F // 8), dtype=np.uint64)[None, :]
    n = (np.arange(N, dtype=np.uint64) + np.uint64(row0))[:, None]
    w = philox((s % 2 ** 32, s >> 32), (g + 0 * n, (n & np.uint64(0xFFFFFFFF)) + 0 * g, (n >> np.uint64(32)) + 0 * g,
                                        np.full((N, g.size), stream, np.uint64)))
    u = np.stack([x for v in w for x in (v & np.uint64(0xFFFF), v >> np.uint64(16))], -1)
    return u.reshape(N, -1)[:, :F].astype(np.int64)


def cut(p):
    return int(np.floor(p * 65536 + 0.5))


def keep(seed, N, F, p, stream=0, row0=0):
    """(kept, factor of the kept ones) in float64."""
    c = cut(p)
    kept = torch.from_numpy(bits(seed, N, F, stream, row0) >= c)
    return kept, (65536 / (65536 - c) if c < 65536 else 0.0)


# ------------------------------------------------------------------ values with what they may be off
class V:
    """A 64-bit value `v` whose 32-bit evaluation is off by at most `e`; every operation adds a half step of fp32."""

    def __init__(self, v, e=None):
        self.v, self.e = v, torch.zeros_like(v) if e is None else e

    def __mul__(self, o):
        o = o if isinstance(o, V) else V(torch.as_tensor(o, dtype=torch.float64, device=self.v.device).expand_as(self.v))
        v = self.v * o.v
        return V(v, self.v.abs() * o.e + o.v.abs() * self.e + self.e * o.e + U32 * v.abs())

    def __add__(self, o):
        v = self.v + o.v
        return V(v, (self.e + o.e) * (1 + U32) + U32 * v.abs())

    def __neg__(self):
        return V(-self.v, self.e)

    def sum(self, dim, depth, keepdim=False):
        """A sum in which no term passes more than `depth` additions."""
        mag = (self.v.abs() + self.e).sum(dim, keepdim=keepdim)
        return V(self.v.sum(dim, keepdim=keepdim), self.e.sum(dim, keepdim=keepdim) + depth * U32 * mag)

    def where(self, mask):
        return V(torch.where(mask, self.v, torch.zeros_like(self.v)), torch.where(mask, self.e, torch.zeros_like(self.e)))

    def rounded(self, dtype):
        return V(self.v, self.e + HALF_STEP[dtype] * (self.v.abs() + self.e) + TINY[dtype])

    def rows(self, like):
        return V(self.v.expand_as(like.v), self.e.expand_as(like.v))


def rs(x, eps, depth):
    """1 / sqrt(mean(x^2) + eps) of rows: half the relative error of what is under the root, a root and a quotient."""
    d = x.v.shape[-1]
    ss = (x * x).sum(-1, depth, keepdim=True)
    under = V(ss.v / d + eps, ss.e / d + 2 * U32 * (ss.v / d + eps))
    rel = under.e / under.v
    v = under.v ** -0.5
    return V(v, v * (0.5 * rel / (1 - rel) + 3 * U32))


DEPTH = 64      # of a row's sums: at most 32 terms in a lane, 64 lanes, 8 waves


def seam(h, y, post=None, gate=None, pre=None, scale=1.0, eps=1e-5, mask=None, keep=1.0, dh=None, dn=None):
    """The forward {'h', 'n'}, and with a gradient the backward {'dh', 'dy', 'dpost', 'dgate', 'dpre'}: V's.  The results
    h and n are before their rounding."""
    H, Y, N, d = V(h.double()), V(y.double()), *h.shape
    scale = float(np.float32(scale))
    x1 = Y
    if post is not None:
        r1 = rs(Y, eps, DEPTH)
        x1 = Y * r1.rows(Y)
        P = V(post.double().expand(N, d))
    z = x1 * P if post is not None else Y
    keep = V(torch.full((N, d), keep, dtype=torch.float64, device=h.device), torch.full((N, d), keep * U32, dtype=torch.float64, device=h.device))
    zd = z if mask is None else (z * keep).where(mask)
    per = 1 if gate is None else N // (1 if gate.dim() == 1 else gate.shape[0])
    G = None if gate is None else V(gate.double().reshape(-1, d).repeat_interleave(per, 0))
    hn = H + (zd if G is None else zd * G) * scale
    out = {"h": hn}
    if pre is not None:
        r2 = rs(hn, eps, DEPTH)
        W = V(pre.double().expand(N, d))
        out["n"] = hn * r2.rows(hn) * W
    if dh is None and dn is None:
        return out
    t = V(torch.zeros_like(H.v)) if dh is None else V(dh.double())
    if dn is not None:
        x2 = hn * r2.rows(hn)
        dN = V(dn.double())
        out["dpre"] = (dN * x2).sum(0, N + 8)
        q = dN * W
        m = (q * x2).sum(-1, DEPTH, keepdim=True)
        m = V(m.v / d, m.e / d + U32 * m.v.abs() / d)
        t = t + (q + -(x2 * m.rows(x2))) * r2.rows(x2)
    out["dh"] = t
    t = t * scale
    if G is not None:
        g = (t * zd)
        rows = 1 if gate.dim() == 1 else gate.shape[0]
        out["dgate"] = V(g.v.reshape(rows, per, d), g.e.reshape(rows, per, d)).sum(1, per + 8)
        t = t * G
    if mask is not None:
        t = (t * keep).where(mask)
    if post is not None:
        out["dpost"] = (t * x1).sum(0, N + 8)
        v = t * P
        m = (v * x1).sum(-1, DEPTH, keepdim=True)
        m = V(m.v / d, m.e / d + U32 * m.v.abs() / d)
        t = (v + -(x1 * m.rows(x1))) * r1.rows(x1)
    out["dy"] = t
    return out


def close(got, want):
    """Every value of `got` is a number within the bound of `want` and the rounding to its type."""
    assert torch.isfinite(want.v).all() and torch.isfinite(want.e).all(), "the reference and its bounds are numbers"
    assert torch.isfinite(got).all(), f"{int((~torch.isfinite(got)).sum())} of {got.numel()} values are no numbers"
    v, bound = want.v.reshape(got.shape), want.rounded(got.dtype).e.reshape(got.shape)
    off = (got.double() - v).abs()
    bad = off > bound
    assert not bool(bad.any()), (int(bad.sum()), got.numel(), float((off / bound)[bad].max()), float(off[bad].max()))

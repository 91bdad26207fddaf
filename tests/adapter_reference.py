"""64-bit statements of the low-rank adapters, with bounds on what a correct 32-bit evaluation may be off, for the
tests."""

import torch

from ffn_reference import U32
from seam_reference import V, close  # noqa: F401

# t' and dt' enter their products as a truncation to 8 bits, exact, and a rest below 2^-7 of them rounded to bf16
SPLIT = 2.0 ** -7 * 2.0 ** -8


def split(t):
    return V(t.v, t.e + SPLIT * (t.v.abs() + t.e))


def mm(a, b, terms):
    """a (V) times the exact b; sums of `terms` products in any order, each product rounded."""
    mag = (a.v.abs() + a.e) @ b.abs()
    return V(a.v @ b, a.e @ b.abs() + (terms + 2) * U32 * mag)


def adapter(y, x, a, b, ids, scales=None, dout=None):
    """{'out'} and with a gradient {'dx', 'dy', 'da', 'db'}: V's before their rounding."""
    y, x, a, b = (t.double() for t in (y, x, a, b))
    n, r, fin = a.shape
    fout = b.shape[1]
    z = torch.zeros_like
    out, eo = y.clone(), z(y)
    g = {"dx": V(z(x), z(x)), "dy": None, "da": V(z(a), z(a)), "db": V(z(b), z(b))} if dout is not None else {}
    for k in range(n):
        rows = torch.nonzero(ids.flatten() == k).flatten()
        if not len(rows):
            continue
        s = 1.0 if scales is None else float(scales[k])
        t = split(mm(V(x[rows]), a[k].T, fin) * s)
        d = mm(t, b[k].T, 2 * r)
        out[rows] = y[rows] + d.v
        eo[rows] = d.e + U32 * (y[rows] + d.v).abs()
        if dout is None:
            continue
        dy = dout[rows].double()
        u = split(mm(V(dy), b[k], fout) * s)
        dx = mm(u, a[k], 2 * r)
        g["dx"].v[rows], g["dx"].e[rows] = dx.v, dx.e
        for name, p, q in (("da", u, x[rows]), ("db", t, dy)):
            d = mm(V(p.v.T, p.e.T), q, 2 * len(rows))
            g[name].v[k], g[name].e[k] = (d.v, d.e) if name == "da" else (d.v.T, d.e.T)
    g["out"] = V(out, eo)
    if dout is not None:
        g["dy"] = V(dout.double())
    return g

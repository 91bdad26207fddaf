"""64-bit statements of the 4-bit and of the dense gated FFN operators, with bounds on what a correct
32-bit evaluation may be off, for the tests."""

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
U32 = 2.0 ** -24


# ------------------------------------------------------------------ quantisation
def scale_exponent(top):
    """floor(log2 top) - 2 in [-127, 127]; top = 0 gives -127."""
    _, e = torch.frexp(top)
    return torch.where(top > 0, (e - 3).clamp(-127, 127), torch.full_like(e, -127))


def round_e2m1(a):
    """Magnitudes -> code 0 .. 7: the nearest value, ties to the even code, beyond 6 to 6."""
    table = E2M1.to(a.device)
    code = torch.zeros_like(a, dtype=torch.int64)
    for k in range(1, 8):
        mid = (table[k - 1] + table[k]) / 2
        code = torch.where((a > mid) | ((a == mid) & (k % 2 == 0)), torch.full_like(code, k), code)
    return code


def mx_quantize(x):
    """x [..., F] -> (codes uint8 [..., F/2], scales uint8 [..., F/32], values float64)."""
    v = x.double().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    bad = ~torch.isfinite(v).all(-1, keepdim=True)
    e = scale_exponent(torch.where(torch.isfinite(v), v, torch.zeros_like(v)).abs().amax(-1, keepdim=True))
    s = torch.ldexp(torch.ones_like(v[..., :1]), e)
    code = round_e2m1(v.abs() / s)
    val = torch.copysign(E2M1.to(v.device)[code], v) * s
    val = torch.where(bad, torch.full_like(val, float("nan")), val)
    code = code + 8 * torch.signbit(v)
    code = code.reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
    scales = torch.where(bad, torch.full_like(e, 255), e + 127).squeeze(-1)
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), scales.to(torch.uint8), val.reshape(x.shape)


def tile_values(codes, scales):
    """codes [R, K, B_out, B_in/2], scales [R, K, B_out, B_in/32] -> float64 [R, K, B_out, B_in]."""
    R, K, B, _ = codes.shape
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(R, K, B, B).long()
    v = E2M1.to(c.device)[c & 7] * (1 - 2 * (c >> 3))
    s = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 127)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return (v.reshape(R, K, B, B // 32, 32) * s[..., None]).reshape(R, K, B, B)


def dense(codes, scales, cols, C):
    """The dense [R * B, C * B] weight; dead and out-of-range slots contribute nothing, repeated columns add."""
    v = tile_values(codes, scales)
    R, K, B, _ = v.shape
    w = torch.zeros(R, C + 1, B, B, dtype=torch.float64, device=v.device)
    at = torch.where((cols < 0) | (cols >= C), torch.full_like(cols, C), cols).long()
    w.scatter_add_(1, at[:, :, None, None].expand_as(v), v)
    return w[:, :C].transpose(1, 2).reshape(R * B, C * B)


def product(x, weight, bias=None, e_x=None):
    """(y, bound on a 32-bit sum's error) of x [N, F] (float64 values) through a 4-bit weight.  A sum of n
    terms in any order is off by at most n 2^-24 times the sum of their magnitudes (n counts the bias
    and the roundings of the scales' products, which are exact)."""
    B = weight[0].shape[2]
    w = dense(*weight, x.shape[1] // B)
    y = x @ w.T
    n = weight[0].shape[1] * B + 2
    mag = x.abs() @ w.abs().T
    if bias is not None:
        y = y + bias.double()
        mag = mag + bias.double().abs()
    err = n * U32 * mag
    if e_x is not None:
        err = err + e_x @ w.abs().T
    return y, err


def silu(z):
    return z * torch.sigmoid(z)


def silu_bound(z, e):
    """|silu| off by: a slope of at most 1.1, and the evaluation: exp of a product rounded at |z| 2^-24
    and good to 2 units, a reciprocal good to 1, two more roundings."""
    return 1.1 * e + silu(z).abs() * (z.abs() + 8) * 2.0 ** -23


def swiglu(x, gate, up, down, residual, bg, bu, bd):
    """(out, bound) of the 4-bit FFN for bf16 x [N, d].  Where the 32-bit hidden state may lie on either
    side of a border between two codes, or of a power of two in its group's maximum, the bound covers
    both choices."""
    xq = mx_quantize(x)[2]
    g, eg = product(xq, gate, bg)
    u, eu = product(xq, up, bu)
    h = silu(g) * u
    eh = u.abs() * silu_bound(g, eg) + silu(g).abs() * eu + eg * eu + h.abs() * 2.0 ** -22
    hg, ehg = (t.reshape(h.shape[0], h.shape[1] // 32, 32) for t in (h, eh))
    lo = ((hg.abs() - ehg).clamp(min=0)).amax(-1, keepdim=True)
    hi = (hg.abs() + ehg).amax(-1, keepdim=True)
    table = E2M1.to(h.device)

    def q(v, top):
        s = torch.ldexp(torch.ones_like(v[..., :1]), scale_exponent(top))
        return torch.copysign(table[round_e2m1(v.abs() / s)], v) * s

    qh = q(hg, hg.abs().amax(-1, keepdim=True))
    cand = torch.stack([q(v, t) for t in (lo, hi) for v in (hg - ehg, hg + ehg)])
    off = (cand - qh).abs().amax(0).reshape(h.shape)
    out, err = product(qh.reshape(h.shape), down, bd, off)
    if residual:
        out = out + x.double()
        err = err + U32 * out.abs()
    return out, err


def close(got, want, err):
    """Every value within its half step of rounding (of a value that may be `err` off), and `err`."""
    hs = HALF_STEP[got.dtype]
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps      # half the smallest subnormal, and more
    bound = err * (1 + hs) + hs * want.abs() + tiny
    far = (got.double() - want).abs() - bound
    assert not (far > 0).any(), (f"{int((far > 0).sum())} of {far.numel()} values off; the worst by "
                                 f"{float(((got.double() - want).abs() / bound).max()):.3g} of its bound")


# ------------------------------------------------------------------ dense gated FFN
def act(z, kind):
    """act, act' and a bound of |act''|."""
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s)), 0.5
    k = (2 / torch.pi) ** 0.5
    t = torch.tanh(k * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z), 1.2


def act_eval(z, a):
    """Evaluation error of act or act' in 32 bits: as silu's; GELU's exponent is up to 1.6 (|z| + 0.05 |z|^3)."""
    return (a.abs() + 1) * (2 * z.abs() + 0.1 * z.abs() ** 3 + 12).clamp(max=400) * 2.0 ** -23


def gated(x, wg, wu, wd, dy, kind, residual):
    """{name: (value, bound)} of the forward, and with dy of the four gradients, from float64 copies of the
    inputs.  The bounds count 32-bit sums and one rounding to the inputs' type of each of h, dg and du,
    and to 24 bits (a half step of 2^-16) of the factors u act'(g) and act(g) that the forward keeps; the last rounding of a result is `close`'s."""
    hs = HALF_STEP[x.dtype]
    dt = x.dtype
    # a rounding near or below the subnormals is off by at most half their step instead
    sub = torch.finfo(dt).tiny * torch.finfo(dt).eps / 2
    X, G, U, D = (t.detach().double() for t in (x, wg, wu, wd))

    def mm(a, b, ea=None, n=None):
        """a @ b with a's error."""
        n = n or a.shape[1] + 2
        e = n * U32 * (a.abs() @ b.abs())
        if ea is not None:
            e = e + (1 + n * U32) * (ea @ b.abs())
        return a @ b, e

    g, eg = mm(X, G.T)
    u, eu = mm(X, U.T)
    a, da, dd = act(g, kind)
    h = a * u
    ea = 1.2 * eg + act_eval(g, a)
    eh = ea * u.abs() + a.abs() * eu + ea * eu + 2 * U32 * h.abs()
    eh = eh * (1 + hs) + hs * h.abs() + sub
    out, eo = mm(h, D.T, eh)
    if residual:
        out = out + X
        eo = eo + U32 * out.abs()
    res = {"out": (out, eo)}
    if dy is None:
        return res
    Y = dy.double()
    dh, edh = mm(Y, D)
    dg, du = dh * u * da, dh * a

    def times(p, ep, q, eq):
        full = (p.abs() + ep) * (q.abs() + eq)
        return full - (p * q).abs() + 2 * U32 * full

    ecg = times(u, eu, da, dd * eg + act_eval(g, da))
    hf = 2.0 ** -16
    ecg = ecg * (1 + hf) + hf * (u * da).abs()
    ecu = ea * (1 + hf) + hf * a.abs()
    edg, edu = times(dh, edh, u * da, ecg), times(dh, edh, a, ecu)
    edg = edg * (1 + hs) + hs * dg.abs() + sub
    edu = edu * (1 + hs) + hs * du.abs() + sub
    F = dg.shape[1]
    x1, e1 = mm(dg, G, edg, 2 * F + 2)
    x2, e2 = mm(du, U, edu, 2 * F + 2)
    dx, ex = x1 + x2, e1 + e2
    if residual:
        dx = dx + Y
        ex = ex + U32 * dx.abs()
    N = X.shape[0] + 2
    res["dx"] = (dx, ex)
    for name, p, ep, q in (("dw_gate", dg, edg, X), ("dw_up", du, edu, X)):
        v, e = mm(q.T, p, None, N)
        e = e + (1 + N * U32) * (q.abs().T @ ep)
        res[name] = (v.T, e.T)
    v, e = mm(Y.T, h, None, N)
    res["dw_down"] = (v, e + (1 + N * U32) * (Y.abs().T @ eh))
    return res

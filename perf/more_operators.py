"""The measured cases of the operators around a block's FFN, with their plain forms.

Three operators: what a looped block is fine-tuned and served with beside its projections.

  dropout  ``dropout``: from a counter-based generator, its mask never stored, forward and backward
  seam     ``residual_norm``: the branch's norm, dropout, gate and scale, the residual sum and the norm ahead of
           the next application in one pass, inference or a training step
  adapter  ``adapter_plan`` and ``adapter_add``: low-rank adapters of many requests beside one shared projection,
           inference or a training step

Sizes come from the repository's benchmark, tests and layer cases.  ``listed()`` holds the fixed cases,
``draw(rng)`` gives more of the same ranges:

  features  500 .. 4096 (dropout and seam: odd ones too), outputs of a projection up to 14336
  tokens    1 .. 16384, odd counts included
  adapters  1 .. 256 of rank 4 .. 64; one per token, per prompt or per sequence, some tokens with none

The generator (see ``_uniform16``) is Philox4x32 with 7 rounds (Salmon, Moraes, Dror and Shaw, "Parallel random
numbers: as easy as 1, 2, 3", 2011); its seed is an input.
"""

from __future__ import annotations

import os
import sys

import numpy as np
import torch

own = False

_DEV = "cuda"
_EPS = 1e-5
_STREAM = 5
# most bytes of a drawn case (the largest listed one takes 4.7e8)
_MAX_DRAW_BYTES = 3e8


def _kernels():
    pkg = os.path.join(os.getcwd(), "looped-blockell-tpu_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from looped_blockell import kernels

    return kernels


# ------------------------------------------------------------------ cases
def _dropout(name, tokens, features, p, dtype="bfloat16"):
    return dict(name=name, kind="dropout", tokens=tokens, features=features, p=p, dtype=dtype)


def _seam(name, tokens, features, *, state="float32", dtype="bfloat16", seqs=1, p=0.0, post=True, gate=True, pre=True,
          train=False):
    """state: type of the residual stream.  seqs: gates, one for each run of tokens / seqs rows."""
    return dict(name=name, kind="seam", tokens=tokens, features=features, state=state, dtype=dtype, seqs=seqs, p=p, post=post,
                gate=gate, pre=pre, train=train)


def _adapter(name, tokens, fin, fout, rank, adapters, *, per="prompt", none=0.0, dtype="bfloat16", train=False, plan=False):
    """per: what an adapter belongs to, 'token' (one step of generation), 'prompt' (runs of ragged length) or
    'sequence' (runs of 512).  none: share of them without.  plan: made in the call, as ahead of a step's
    first layer, instead of kept for the step's other layers."""
    return dict(name=name, kind="adapter", tokens=tokens, fin=fin, fout=fout, rank=rank, adapters=adapters, per=per, none=none,
                dtype=dtype, train=train, plan=plan)


def listed():
    return [
        # a ragged micro-batch of a small odd-sized model in fp16
        _dropout("dropout_1999_fp16", 1999, 1001, 0.25, dtype="float16"),
        # the branch of the headline layer, 32 sequences of 512
        _dropout("dropout_16k", 16384, 1024, 0.1),
        # one token of the wide model between two applications: launch and host work
        _seam("seam_1", 1, 4096),
        # scoring a large batch with the looped headline layer
        _seam("seam_16k", 16384, 1024),
        # training with gates from each sequence's conditioning: 17 sequences of 241 tokens, odd features, fp16
        _seam("seam_train_4097_fp16", 4097, 1001, state="float16", dtype="float16", seqs=17, p=0.1, train=True),
        # one training step through the looped headline layer's seam, fp32 state, dropout
        _seam("seam_train_16k", 16384, 1024, p=0.1, train=True),
        # one request generating with the wide model's up projection
        _adapter("adapter_1", 1, 4096, 14336, 16, 64, per="token"),
        # 64 requests generating, an adapter each; the step's plan made in the call
        _adapter("adapter_64", 64, 4096, 14336, 16, 128, per="token", none=0.1, plan=True),
        # prompts of odd lengths, some without an adapter
        _adapter("adapter_4099_r64", 4099, 2048, 8192, 64, 12, none=0.1),
        # scoring a large batch with few adapters of the headline layer
        _adapter("adapter_16k", 16384, 1024, 4096, 16, 4, per="sequence"),
        # fine-tuning a small model's adapters on a ragged micro-batch in fp16, odd rank
        _adapter("adapter_train_1999_fp16", 1999, 512, 1792, 12, 3, dtype="float16", train=True),
        # fine-tuning four adapters of the headline layer at once, 32 sequences of 512
        _adapter("adapter_train_16k", 16384, 1024, 4096, 16, 4, per="sequence", train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    while True:
        kind = rng.choice(["dropout", "seam", "seam", "adapter", "adapter"])
        tokens = _log_int(rng, 1, 16384)
        if rng.random() < 0.5:
            tokens |= 1
        dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
        if kind == "adapter":
            fin = rng.choice([512, 640, 1024, 1280, 2048, 4096])
            per = "token" if tokens <= 256 else rng.choice(["prompt", "sequence"])
            train = tokens > 256 and rng.random() < 0.5
            c = _adapter(None, tokens, fin, int(fin * rng.choice([1, 2, 3.5])), rng.choice([4, 8, 12, 16, 32, 64]),
                         _log_int(rng, 1, 256), per=per, none=rng.choice([0.0, 0.1]), dtype=dtype, train=train,
                         plan=per == "token")
        else:
            features = _log_int(rng, 500, 4096)
            if rng.random() < 0.6:
                features = features // 64 * 64
            if kind == "dropout":
                c = _dropout(None, tokens, features, rng.choice([0.05, 0.1, 0.3, 0.5]), rng.choice([dtype, "float32"]))
            else:
                state = rng.choice(["float32", dtype])
                dtype = rng.choice([dtype, dtype, state])
                seqs = rng.choice([s for s in range(1, 65) if tokens % s == 0])
                train = rng.random() < 0.5
                c = _seam(None, tokens, features, state=state, dtype=dtype, seqs=seqs, p=rng.choice([0.0, 0.1]) if train else 0.0,
                          post=rng.random() < 0.7, gate=rng.random() < 0.7, pre=rng.random() < 0.8, train=train)
        del c["name"]
        if work(c)["bytes"] <= _MAX_DRAW_BYTES:
            return c


_SIZE = {"bfloat16": 2, "float16": 2, "float32": 4}


def work(c):
    N = c["tokens"]
    if c["kind"] == "dropout":
        # x and the result's gradient in, result and x's gradient out
        return {"bytes": 4.0 * N * c["features"] * _SIZE[c["dtype"]], "flops": 4.0 * N * c["features"]}
    if c["kind"] == "seam":
        e, s, b = N * c["features"], _SIZE[c["state"]], _SIZE[c["dtype"]]
        vectors = c["features"] * (4.0 * c["post"] + 4.0 * c["pre"] + c["gate"] * c["seqs"] * 4.0)
        fwd = e * (2.0 * s + b + b * c["pre"]) + vectors
        if not c["train"]:
            return {"bytes": fwd, "flops": 10.0 * e}
        # and both gradients in and out
        return {"bytes": fwd + e * (2.0 * s + b + b * c["pre"]) + vectors, "flops": 40.0 * e}
    fin, fout, r, n = c["fin"], c["fout"], c["rank"], min(c["adapters"], N)
    weights, flops = 2.0 * n * r * (fin + fout), 2.0 * N * r * (fin + fout)
    if not c["train"]:
        return {"bytes": 2.0 * N * (fin + 2 * fout) + weights + 4.0 * N, "flops": flops}
    # the result's gradient in, x's and the adapters' out
    return {"bytes": 2.0 * N * (2 * fin + 3 * fout) + 2 * weights + 4.0 * N, "flops": 3 * flops}


# ------------------------------------------------------------------ inputs
def _ids(c, gc):
    """The adapter of every token."""
    N, n = c["tokens"], c["adapters"]
    if c["per"] == "token":
        runs = [1] * N
    elif c["per"] == "sequence":
        runs = [512] * (N // 512) + [N % 512]
    else:
        cuts = torch.randint(0, N + 1, (max(1, N // 450),), generator=gc).sort().values.tolist()
        runs = [b - a for a, b in zip([0] + cuts, cuts + [N])]
    ids = torch.randint(0, n, (len(runs),), generator=gc)
    ids[torch.rand(len(runs), generator=gc) < c["none"]] = -1
    return torch.repeat_interleave(ids, torch.tensor(runs)).to(torch.int32)


def prepare(c, seed):
    g = torch.Generator(device=_DEV).manual_seed(int(seed) & 0x7FFFFFFF)
    gc = torch.Generator().manual_seed((int(seed) + 1) & 0x7FFFFFFF)
    N, dt = c["tokens"], getattr(torch, c["dtype"])

    def randn(*shape, scale=1.0, dtype=dt):
        return torch.randn(shape, device=_DEV, generator=g).mul_(scale).to(dtype)

    st = {"case": c}
    if c["kind"] != "adapter":
        d = c["features"]
        st["seed"] = torch.randint(-2 ** 62, 2 ** 62, (1,), generator=gc).to(_DEV)
    if c["kind"] == "dropout":
        st["x"], st["dy"] = randn(N, d).requires_grad_(True), randn(N, d)
        return st
    if c["kind"] == "seam":
        sdt = getattr(torch, c["state"])
        st["h"], st["y"] = randn(N, d, scale=3.0, dtype=sdt), randn(N, d)
        for name in ("post", "pre"):
            st[name] = 1 + 0.1 * randn(d, dtype=torch.float32) if c[name] else None
        st["gate"] = 0.5 + 0.2 * randn(c["seqs"], d, dtype=torch.float32) if c["gate"] else None
        if c["train"]:
            st["dh"], st["dn"] = randn(N, d, dtype=sdt), randn(N, d) if c["pre"] else None
            for name in ("h", "y", "post", "gate", "pre"):
                if st[name] is not None:
                    st[name].requires_grad_(True)
        return st
    fin, fout, r, n = c["fin"], c["fout"], c["rank"], c["adapters"]
    st["ids"] = _ids(c, gc).to(_DEV)
    st["x"], st["y"] = randn(N, fin), randn(N, fout)
    st["a"], st["b"] = randn(n, r, fin, scale=fin ** -0.5), randn(n, fout, r, scale=r ** -0.5)
    st["scales"] = 0.5 + torch.rand(n, device=_DEV, generator=g)
    if c["train"]:
        st["dout"] = randn(N, fout)
        for name in ("x", "y", "a", "b"):
            st[name].requires_grad_(True)
    if own and not c["plan"]:
        st["plan"] = _kernels().adapter_plan(st["ids"], n)
    return st


# ------------------------------------------------------------------ plain forms
def _uniform16(seed, rows, cols, stream):
    """The generator: 16 bits for each element [rows, cols], from 7 rounds of Philox4x32 under the key (seed low,
    seed high) on the counters (column / 8, row low, row high, stream); a block of 128 bits serves 8 columns."""
    m32 = 0xFFFFFFFF
    dev = seed.device
    k0, k1 = seed & m32, (seed >> 32) & m32
    c0 = torch.arange((cols + 7) // 8, device=dev)[None, :].expand(rows, -1)
    row = torch.arange(rows, device=dev)[:, None].expand_as(c0)
    c1, c2, c3 = row & m32, row >> 32, torch.full_like(c0, stream)
    for _ in range(7):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57          # modulo 2^64, whose upper half is masked out below
        c0, c1, c2, c3 = ((p1 >> 32) & m32) ^ c1 ^ k0, p1 & m32, ((p0 >> 32) & m32) ^ c3 ^ k1, p0 & m32
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    words = torch.stack([c0, c1, c2, c3], -1)
    return torch.stack([words & 0xFFFF, words >> 16], -1).reshape(rows, -1)[:, :cols]


def _keep(seed, rows, cols, p):
    """0 where an element is dropped, else the factor that keeps the expectation."""
    t = int(p * 65536 + 0.5)
    return (_uniform16(seed, rows, cols, _STREAM) >= t).float() * (65536 / (65536 - t))


def _plain_dropout(st, c):
    x, dy = st["x"], st["dy"]
    k = _keep(st["seed"], *x.shape, c["p"])
    return {"y": (x.float() * k).to(x.dtype), "dx": (dy.float() * k).to(x.dtype)}


def _plain_seam(st, c):
    h, y = st["h"].float(), st["y"].float()
    N, d = h.shape
    r1 = torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS)
    xh1 = y * r1 if c["post"] else y
    z = xh1 * st["post"] if c["post"] else y
    k = _keep(st["seed"], N, d, c["p"]) if c["p"] > 0 else None
    zd = z if k is None else z * k
    seqs = c["seqs"]
    gate = st["gate"][:, None, :] if c["gate"] else torch.ones(1, 1, 1, device=h.device)
    hn = h + 0.5 * (zd.reshape(seqs, -1, d) * gate).reshape(N, d)
    res = {"h": hn.to(st["h"].dtype)}
    r2 = torch.rsqrt((hn * hn).mean(-1, keepdim=True) + _EPS)
    xh2 = hn * r2
    if c["pre"]:
        res["n"] = (xh2 * st["pre"]).to(st["y"].dtype)
    if not c["train"]:
        return res
    total = st["dh"].float()
    if c["pre"]:
        dn = st["dn"].float()
        q = dn * st["pre"]
        total = total + r2 * (q - xh2 * (q * xh2).mean(-1, keepdim=True))
        res["dpre"] = (dn * xh2).sum(0)
    res["dh"] = total.to(st["h"].dtype)
    scaled = 0.5 * total.reshape(seqs, -1, d)
    if c["gate"]:
        res["dgate"] = (scaled * zd.reshape(seqs, -1, d)).sum(1)
    s = (scaled * gate).reshape(N, d)
    if k is not None:
        s = s * k
    if c["post"]:
        res["dpost"] = (s * xh1).sum(0)
        v = s * st["post"]
        s = r1 * (v - xh1 * (v * xh1).mean(-1, keepdim=True))
    res["dy"] = s.to(st["y"].dtype)
    return res


def _plain_adapter(st, c):
    x, y, a, b = (st[n].float() for n in ("x", "y", "a", "b"))
    ids, dt = st["ids"].long(), st["x"].dtype
    out = y.clone()
    dout = st["dout"].float() if c["train"] else None
    dx, da, db = (torch.zeros_like(t) if c["train"] else None for t in (x, a, b))
    present = torch.unique(ids).tolist()
    for k in present:
        if k < 0:
            continue
        rows = torch.nonzero(ids == k).flatten()
        t = x[rows] @ a[k].T
        s = st["scales"][k]
        out[rows] = y[rows] + s * (t @ b[k].T)
        if c["train"]:
            do = s * dout[rows]
            u = do @ b[k]
            dx[rows], da[k], db[k] = u @ a[k], u.T @ x[rows], do.T @ t
    res = {"out": out.to(dt)}
    if c["train"]:
        res.update(dx=dx.to(dt), dy=dout.to(dt), da=da.to(dt), db=db.to(dt))
    return res


def _own(st):
    K, c = _kernels(), st["case"]
    if c["kind"] == "dropout":
        y = K.dropout(st["x"], c["p"], st["seed"], stream=_STREAM)
        return {"y": y.detach(), "dx": torch.autograd.grad(y, st["x"], st["dy"])[0]}
    if c["kind"] == "seam":
        h, n = K.residual_norm(st["h"], st["y"], post_scale=st["post"], gate=st["gate"], pre_scale=st["pre"],
                               residual_scale=0.5, eps=_EPS, p=c["p"], seed=st["seed"], stream=_STREAM)
        res = {"h": h.detach()}
        if n is not None:
            res["n"] = n.detach()
        if c["train"]:
            names = [k for k in ("h", "y", "post", "gate", "pre") if st[k] is not None]
            outs, grads = ([h], [st["dh"]]) if n is None else ([h, n], [st["dh"], st["dn"]])
            res.update(zip(("d" + k for k in names), torch.autograd.grad(outs, [st[k] for k in names], grads)))
        return res
    plan = K.adapter_plan(st["ids"], c["adapters"]) if c["plan"] else st["plan"]
    out = K.adapter_add(st["y"], st["x"], st["a"], st["b"], plan, scales=st["scales"])
    res = {"out": out.detach()}
    if c["train"]:
        res.update(zip(("dx", "dy", "da", "db"), torch.autograd.grad(out, [st[k] for k in "x y a b".split()], st["dout"])))
    return res


def run(st):
    if own:
        return _own(st)
    with torch.no_grad():
        c = st["case"]
        return {"dropout": _plain_dropout, "seam": _plain_seam, "adapter": _plain_adapter}[c["kind"]](st, c)


# ------------------------------------------------------------------ in 64 bits
def _exact_keep(seed, rows, cols, p):
    """The generator's factors, from its definition in unsigned integers on the host."""
    key = int(seed.item()) % 2 ** 64
    key = [np.uint64(key % 2 ** 32), np.uint64(key >> 32)]
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    groups = -(-cols // 8)
    ctr = [np.zeros((rows, groups), np.uint64) for _ in range(4)]
    ctr[0] += np.arange(groups, dtype=np.uint64)
    ctr[1] += np.arange(rows, dtype=np.uint64)[:, None]
    ctr[3] += np.uint64(_STREAM)
    for _ in range(7):
        even, odd = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(odd >> half) ^ ctr[1] ^ key[0], odd & low, (even >> half) ^ ctr[3] ^ key[1], even & low]
        key = [(key[0] + np.uint64(0x9E3779B9)) & low, (key[1] + np.uint64(0xBB67AE85)) & low]
    u = np.empty((rows, groups, 8), np.int32)
    for k in range(4):
        u[..., 2 * k], u[..., 2 * k + 1] = ctr[k] & np.uint64(0xFFFF), ctr[k] >> np.uint64(16)
    cut = int(np.floor(p * 65536 + 0.5))
    kept = torch.from_numpy(u.reshape(rows, -1)[:, :cols] >= cut).to(_DEV)
    return kept.double() * (65536 / (65536 - cut))


def _exact_seam(st, c):
    leaf = {k: st[k].detach().double().requires_grad_(c["train"]) for k in ("h", "y", "post", "gate", "pre") if st[k] is not None}
    N, d = st["h"].shape

    def norm(v, w):
        return v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + _EPS) * w

    with torch.set_grad_enabled(c["train"]):
        z = norm(leaf["y"], leaf["post"]) if c["post"] else leaf["y"]
        if c["p"] > 0:
            z = z * _exact_keep(st["seed"], N, d, c["p"])
        if c["gate"]:
            z = z * leaf["gate"].repeat_interleave(N // c["seqs"], 0)
        outs = {"h": leaf["h"] + z / 2}
        if c["pre"]:
            outs["n"] = norm(outs["h"], leaf["pre"])
    res = {k: v.detach() for k, v in outs.items()}
    if c["train"]:
        grads = [st["d" + k].double() for k in outs]
        res.update(zip(("d" + k for k in leaf), torch.autograd.grad(list(outs.values()), list(leaf.values()), grads)))
    return res


def _exact_adapter(st, c):
    x, y, a, b = (st[k].detach().double() for k in ("x", "y", "a", "b"))
    ids, s = st["ids"].cpu(), st["scales"].double()
    delta = torch.zeros_like(y)
    grads = [torch.zeros_like(t) for t in (x, a, b)] if c["train"] else None
    for k in range(c["adapters"]):
        sel = (ids == k).to(x.device)
        if not bool(sel.any()):
            continue
        w = s[k] * (b[k] @ a[k])                      # the update of the dense weight that the adapter stands for
        delta[sel] = x[sel] @ w.T
        if c["train"]:
            g = st["dout"][sel].double()
            grads[0][sel] = g @ w
            dw = s[k] * (g.T @ x[sel])
            grads[1][k], grads[2][k] = b[k].T @ dw, dw @ a[k].T
    res = {"out": y + delta}
    if c["train"]:
        res.update(dx=grads[0], dy=st["dout"].double(), da=grads[1], db=grads[2])
    return res


def exact(c, seed):
    st = prepare(c, seed)
    if c["kind"] == "seam":
        return _exact_seam(st, c)
    with torch.no_grad():
        if c["kind"] == "adapter":
            return _exact_adapter(st, c)
        k = _exact_keep(st["seed"], *st["x"].shape, c["p"])
        return {"y": st["x"].double() * k, "dx": st["dy"].double() * k}

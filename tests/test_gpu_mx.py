"""GPU tests of the microscaled 4-bit operators against their 64-bit statements (tests/ffn_reference.py)."""

import pytest
import torch

import ffn_reference as ref
from looped_blockell import kernels

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _acts(N, F, seed, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(N, F, device="cuda", generator=g) * torch.exp(0.7 * torch.randn(F, device="cuda", generator=g))
    return x.to(dtype)


def _weight(R, C, K, B, seed, dead=0.0, lo=118, hi=121):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (R, K, B, B // 2), dtype=torch.uint8, generator=g)
    scales = torch.randint(lo, hi, (R, K, B, B // 32), dtype=torch.uint8, generator=g)
    cols = torch.stack([torch.randperm(max(C, K), generator=g)[:K] % C for _ in range(R)]).int().reshape(R, K)
    if dead:
        cols[torch.rand(R, K, generator=g) < dead] = -1
    return codes.cuda(), scales.cuda(), cols.cuda()


# ------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,F", [(1, 32), (3, 96), (17, 1024), (130, 2048 + 64), (1000, 64)])
def test_quantize_rows(gpu, N, F, dtype):
    x = _acts(N, F, N + F, dtype)
    x[N // 2] = 0
    codes, scales = kernels.mx_quantize(x)
    c, s, v = ref.mx_quantize(x.cpu())
    assert torch.equal(codes.cpu(), c) and torch.equal(scales.cpu(), s)
    for out in DTYPES:
        assert torch.equal(kernels.mx_dequantize(codes, scales, out).cpu(), v.to(out))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_borders_and_extremes(gpu, dtype):
    """Every border between two codes, exactly on it and one step to each side, at several scales; the
    largest and the smallest values of the type; signed zeros."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.0, -0.0, 6.0, 7.0], dtype=dtype)
    near = torch.cat([mids, torch.nextafter(mids, torch.full_like(mids, 9.0)), torch.nextafter(mids, torch.full_like(mids, -9.0))])
    rows = []
    for p in (-12, -3, 0, 5):
        for top in (4.0, 6.0, 7.75):
            r = torch.zeros(64, dtype=dtype)
            r[:33] = near.to(dtype)
            r[33:63] = -r[:30]
            r[31] = r[63] = top
            rows.append((r.float() * 2.0 ** p).to(dtype))
    fi = torch.finfo(dtype)
    for v in (fi.max, fi.tiny, fi.tiny * fi.eps, fi.tiny * 3):
        rows.append(torch.linspace(-1, 1, 64, dtype=torch.float64).mul(v).to(dtype))
    x = torch.stack(rows).cuda()
    codes, scales = kernels.mx_quantize(x)
    c, s, v = ref.mx_quantize(x.cpu())
    assert torch.equal(scales.cpu(), s) and torch.equal(codes.cpu(), c)
    assert torch.equal(kernels.mx_dequantize(codes, scales, torch.float32).cpu(), v.float())


def test_quantize_not_finite(gpu):
    x = _acts(6, 128, 0)
    x[1, 5], x[2, 40], x[3, 127] = float("nan"), float("inf"), -float("inf")
    codes, scales = kernels.mx_quantize(x)
    _, s, v = ref.mx_quantize(x.cpu())
    assert torch.equal(scales.cpu(), s) and int((scales == 255).sum()) == 3
    got = kernels.mx_dequantize(codes, scales, torch.float32).cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(v)) and torch.equal(got.nan_to_num(0), v.float().nan_to_num(0))


def test_quantize_strides_and_leading_dimensions(gpu):
    big = _acts(10, 256, 1)
    for x in (big[:, :96], big[::2, 32:96], big.t()[:64, :].contiguous().t()[:, :64], big.flatten()[4:4 + 9 * 96].view(9, 96),
              big.t()[:96].contiguous().t()[:, :32]):
        a, b = kernels.mx_quantize(x), kernels.mx_quantize(x.clone(memory_format=torch.contiguous_format))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x = _acts(24, 64, 2).reshape(2, 3, 4, 64)
    c, s = kernels.mx_quantize(x)
    assert c.shape == (2, 3, 4, 32) and s.shape == (2, 3, 4, 2)
    assert kernels.mx_dequantize(c, s).shape == x.shape
    c, s = kernels.mx_quantize(x.reshape(24, 64)[:0])
    assert c.shape == (0, 32) and kernels.mx_dequantize(c, s).shape == (0, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,K,B", [(1, 1, 32), (3, 2, 64), (5, 7, 32), (2, 0, 64)])
def test_quantize_tiles(gpu, R, K, B, dtype):
    v = _acts(R * K * B, B, 7, dtype).reshape(R, K, B, B) * 0.02
    if K > 1:
        v[0, 1] = 0
    codes, scales = kernels.mx_quantize_tiles(v)
    c, s, val = ref.mx_quantize(v.cpu().transpose(-1, -2))
    assert torch.equal(codes.cpu(), c) and torch.equal(scales.cpu(), s)
    back = kernels.mx_dequantize_tiles(codes, scales, torch.float32)
    assert torch.equal(back.cpu(), val.transpose(-1, -2).float())
    assert torch.equal(ref.tile_values(c, s), val)


# ------------------------------------------------------------------ product
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("N,R,C,K,B,dead", [
    (1, 2, 2, 1, 32, 0.0), (1, 9, 16, 5, 64, 0.0), (5, 4, 8, 3, 32, 0.4), (16, 8, 64, 6, 64, 0.0), (17, 3, 5, 5, 64, 0.2),
    (33, 7, 33, 8, 32, 0.0), (64, 5, 64, 64, 32, 0.1), (65, 2, 4, 4, 64, 0.0), (130, 16, 32, 8, 32, 0.1),
    (257, 3, 20, 19, 32, 0.0), (300, 33, 16, 4, 64, 0.0), (700, 12, 128, 33, 64, 0.05), (129, 6, 260, 70, 32, 0.3),
    (1025, 10, 16, 4, 32, 0.0), (40, 3, 256, 200, 64, 0.0), (2049, 5, 40, 10, 64, 0.1),
    (150, 5, 320, 7, 32, 0.1), (200, 4, 256, 9, 64, 0.2), (131, 3, 300, 2, 32, 0.0), (260, 3, 150, 3, 64, 0.0)])
def test_matmul(gpu, N, R, C, K, B, dead, bias):
    x, w = _acts(N, C * B, N), _weight(R, C, K, B, R + K, dead)
    x[N // 3] = 0
    b = torch.randn(R * B, device="cuda") * 0.1 if bias else None
    y = kernels.mx_matmul(x, *w, bias=b)
    ref.close(y, *ref.product(ref.mx_quantize(x)[2], w, b))


@pytest.mark.parametrize("N", [3, 100, 200])
@pytest.mark.parametrize("B", [32, 64])
def test_matmul_topology(gpu, N, B):
    """A row of dead slots, columns out of range and repeated columns."""
    R, C, K = 6, 5, 4
    x, (codes, scales, cols) = _acts(N, C * B, 3), _weight(R, C, K, B, 4)
    cols[1] = -1
    cols[2] = torch.tensor([C, C + 7, -5, 2 ** 30], dtype=torch.int32)
    cols[3] = 2
    cols[4] = torch.tensor([-1, 3, 3, -1], dtype=torch.int32)
    y = kernels.mx_matmul(x, codes, scales, cols)
    assert not y[:, B:3 * B].any()
    ref.close(y, *ref.product(ref.mx_quantize(x)[2], (codes, scales, cols)))
    none = kernels.mx_matmul(x, codes[:, :0], scales[:, :0], cols[:, :0], bias=torch.ones(R * B, device="cuda"))
    assert (none == 1).all()


@pytest.mark.parametrize("N", [4, 150])
@pytest.mark.parametrize("B", [32, 64])
def test_matmul_not_finite(gpu, N, B):
    """A NaN or Inf activation reaches the outputs that read its group, those of its token only; dead
    slots and other tokens do not see it."""
    R, C, K = 5, 6, 3
    x, (codes, scales, cols) = _acts(N, C * B, 3), _weight(R, C, K, B, 4)
    cols[0] = torch.tensor([0, 1, 5], dtype=torch.int32)
    cols[1] = torch.tensor([3, -1, 5], dtype=torch.int32)
    cols[2] = torch.tensor([4, 3, 5], dtype=torch.int32)
    clean = kernels.mx_matmul(x, codes, scales, cols)
    y_in = x.clone()
    y_in[2, 3 * B + 1] = float("inf")
    y_in[N - 1, 5 * B] = float("nan")
    y = kernels.mx_matmul(y_in, codes, scales, cols)
    reads = torch.zeros(N, R, dtype=torch.bool)
    reads[2] = (cols == 3).any(1).cpu()
    reads[N - 1] = (cols == 5).any(1).cpu()
    nan = torch.isnan(y).reshape(N, R, B).cpu()
    assert torch.equal(nan.all(2), reads) and torch.equal(nan.any(2), reads)
    assert torch.equal(y[~torch.isnan(y)], clean[~torch.isnan(y)])


def test_matmul_extreme_scales(gpu):
    """Weight and activation scales at the ends of their range whose products are ordinary numbers."""
    x = _acts(20, 128, 0).float()
    big, small = (x * 2.0 ** 100).to(torch.bfloat16), (x * 2.0 ** -100).to(torch.bfloat16)
    for v, lo in ((big, 20), (small, 222)):
        w = _weight(3, 4, 2, 32, 1, lo=lo, hi=lo + 3)
        ref.close(kernels.mx_matmul(v, *w), *ref.product(ref.mx_quantize(v)[2], w))


# ------------------------------------------------------------------ FFN
def _ffn(d, ff, B, kg, ku, kd, seed, dead=0.0):
    return (_weight(ff // B, d // B, kg, B, seed, dead), _weight(ff // B, d // B, ku, B, seed + 1, dead),
            _weight(d // B, ff // B, kd, B, seed + 2, dead))


@pytest.mark.parametrize("N,d,ff,B,kg,ku,kd,dead,extra", [
    (1, 64, 128, 32, 2, 2, 4, 0.0, False), (1, 512, 2048, 64, 2, 2, 8, 0.0, True), (16, 256, 896, 64, 3, 2, 5, 0.0, False),
    (7, 128, 320, 32, 1, 3, 9, 0.3, True), (33, 256, 512, 32, 8, 8, 16, 0.0, True), (64, 512, 1792, 64, 4, 4, 14, 0.1, False),
    (65, 192, 448, 64, 3, 3, 7, 0.0, True), (129, 1024, 4096, 32, 8, 8, 32, 0.0, False),
    (300, 640, 2240, 32, 5, 5, 17, 0.1, True), (515, 256, 1024, 64, 4, 4, 16, 0.0, True),
    (200, 2048, 8192, 64, 4, 4, 16, 0.1, True), (70, 1280, 4480, 64, 20, 20, 70, 0.0, False),
    (140, 256, 9728, 64, 2, 3, 15, 0.1, True), (333, 128, 10240, 32, 2, 2, 9, 0.0, False), (170, 64, 128, 32, 0, 2, 3, 0.0, True),
    (140, 64, 128, 64, 1, 1, 0, 0.0, True)])
def test_swiglu(gpu, N, d, ff, B, kg, ku, kd, dead, extra):
    x, (g, u, dn) = _acts(N, d, N), _ffn(d, ff, B, kg, ku, kd, d + ff, dead)
    b = [torch.randn(n, device="cuda") * 0.1 if extra else None for n in (ff, ff, d)]
    y = kernels.mx_swiglu(x, g, u, dn, add_residual=extra, b_gate=b[0], b_up=b[1], b_down=b[2])
    ref.close(y, *ref.swiglu(x, g, u, dn, extra, *b))


@pytest.mark.parametrize("N", [1, 20, 100, 200])
def test_swiglu_zero_rows_and_repeats(gpu, N):
    """Zero rows give the biases' answer, equal rows equal answers, whatever stands beside them; two calls agree."""
    x, (g, u, dn) = _acts(N, 256, N), _ffn(256, 512, 32, 4, 4, 6, 1)
    x[0] = 0
    y = kernels.mx_swiglu(x, g, u, dn)
    assert not y[0].any()
    again = kernels.mx_swiglu(torch.cat([x, x.flip(0)]), g, u, dn)
    assert N < 200 or torch.equal(again[:N], y)      # few tokens' products sum in another order
    assert torch.equal(kernels.mx_swiglu(x, g, u, dn), y)
    assert kernels.mx_swiglu(x[:0], g, u, dn).shape == (0, 256)
    assert kernels.mx_swiglu(x.reshape(1, N, 256), g, u, dn).shape == (1, N, 256)


@pytest.mark.parametrize("N", [16, 160])
def test_swiglu_captured(gpu, N):
    """Replays of a captured call follow the inputs and the weights, with eager calls of other sizes between."""
    x, w = _acts(N, 256, 5), _ffn(256, 512, 64, 2, 2, 4, 6)
    y = kernels.mx_swiglu(x, *w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = kernels.mx_swiglu(x, *w)
    for k in range(4):
        x.copy_(_acts(N, 256, 10 + k))
        w[2][0].copy_(_ffn(256, 512, 64, 2, 2, 4, 20 + k)[2][0])
        kernels.mx_swiglu(_acts(70, 256, k), *w)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, kernels.mx_swiglu(x, *w))


def test_on_another_stream(gpu):
    x, w = _acts(100, 256, 5), _ffn(256, 512, 32, 2, 2, 4, 6)
    want = kernels.mx_swiglu(x, *w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for t in (x, *w[0], *w[1], *w[2]):
            t.record_stream(s)
        outs = [kernels.mx_swiglu(x, *w) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(o, want) for o in outs)


def test_refusals(gpu):
    x, (c, s, i) = _acts(4, 128, 0), _weight(2, 4, 2, 32, 0)
    for bad in (lambda: kernels.mx_quantize(x[:, :48]), lambda: kernels.mx_quantize(x.double()),
                lambda: kernels.mx_quantize(x.cpu()), lambda: kernels.mx_dequantize(c[0, 0], s[0, 0, :, :0]),
                lambda: kernels.mx_dequantize(*kernels.mx_quantize(x), torch.int8),
                lambda: kernels.mx_quantize_tiles(torch.zeros(2, 2, 16, 16, device="cuda")),
                lambda: kernels.mx_quantize_tiles(torch.zeros(2, 2, 32, 64, device="cuda")),
                lambda: kernels.mx_matmul(x[:, :96 + 16], c, s, i), lambda: kernels.mx_matmul(x, c, s[:1], i),
                lambda: kernels.mx_matmul(x, c, s, i.long()), lambda: kernels.mx_matmul(x, c.char(), s, i),
                lambda: kernels.mx_matmul(x, c, s, i, bias=torch.zeros(3, device="cuda")),
                lambda: kernels.mx_matmul(x, c, s, i.cpu()),
                lambda: kernels.mx_swiglu(x, (c, s, i), (c[:1], s[:1], i[:1]), (c, s, i)),
                lambda: kernels.mx_swiglu(x, (c, s, i), (c, s, i), (c, s, i))):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(RuntimeError):
        kernels.mx_matmul(x.float().requires_grad_(), c, s, i).sum().backward()

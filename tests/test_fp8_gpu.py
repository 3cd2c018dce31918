"""Products in 8-bit floating point (csrc/fp8_*.cu) against float64.

Quantisation: the formula in fp32 (reciprocal, product, rounding) evaluated by torch on the CPU must
give the same bytes and scales.
Products: the operands' e4m3 values are exact, their products are exact in fp32, so an fp32 output is off
by the roundings of the sums and scales: below 2^-20 of sum |a b| (K / 128 additions of at most
2^-24 each, plus those of a block's 128 terms and of the scale product).  16-bit outputs add half an ulp.
"""

import math

import pytest
import torch

from tests.inputs import rel_rms

pytestmark = pytest.mark.gpu

ULP = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E4M3 = torch.float8_e4m3fn


def blocks(n):
    return -(-n // 128)


def plain_rows(x):
    """The row quantisation in fp32 on the CPU."""
    x = x.float().cpu()
    M, K = x.shape
    xp = torch.nn.functional.pad(x, (0, blocks(K) * 128 - K)).view(M, blocks(K), 128)
    a = xp.abs().amax(-1).clamp(min=1e-30)
    q = (xp * (torch.reciprocal(a) * 448.0)[..., None]).view(M, -1)[:, :K].to(E4M3)
    return q, a * torch.tensor(1.0 / 448.0, dtype=torch.float32)


def rows64(q, s):
    return q.cpu().double() * s.cpu().double().repeat_interleave(128, -1)[..., : q.shape[-1]]


def weight64(q, s):
    w = s.cpu().double().repeat_interleave(128, -2)[..., : q.shape[-2], :].repeat_interleave(128, -1)
    return q.cpu().double() * w[..., : q.shape[-1]]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def data(M, K, seed, dtype=torch.float32):
    g = gen(seed)
    x = torch.randn(M, K, device="cuda", generator=g) * torch.exp(torch.randn(M, 1, device="cuda", generator=g) * 3)
    return x.to(dtype)


@pytest.fixture
def impl():
    """Select the product kernel for one test: 1 streaming, 2 one CTA a tile, 3 CTA pairs."""
    from rwkv_mlx_b200 import _native as nat

    def choose(i):
        nat.check(nat.lib().rwkv_fp8_set_gemm_impl(i), "rwkv_fp8_set_gemm_impl")

    yield choose
    choose(0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 127), (7, 129), (130, 776), (33, 1024), (1000, 515), (5, 2056)])
def test_quantize_rows_bytes(dtype, M, K):
    from rwkv_mlx_b200.fp8 import quantize_fp8_rows

    x = data(M, K, M * K, dtype)
    q, s = quantize_fp8_rows(x)
    qr, sr = plain_rows(x)
    assert q.dtype == E4M3 and q.shape == (M, K) and s.shape == (M, blocks(K))
    assert torch.equal(q.cpu().view(torch.uint8), qr.view(torch.uint8))
    assert torch.equal(s.cpu(), sr)


def test_quantize_rows_strides_and_values():
    from rwkv_mlx_b200.fp8 import quantize_fp8_rows

    base = data(40, 300, 5)
    for x in (base[3:37, 1:258], base.t()[:77], base[::2, ::2], base[:, 8:264].half(), base[:1, :200]):
        q, s = quantize_fp8_rows(x)
        qr, sr = plain_rows(x)
        assert torch.equal(q.cpu().view(torch.uint8), qr.view(torch.uint8)) and torch.equal(s.cpu(), sr)
    x = torch.zeros(6, 256, device="cuda")
    x[1, 3], x[1, 130] = 1e-38, -1e-44       # below the smallest block maximum
    x[2] = 3e38                              # a large block: 448 / a is tiny, nothing overflows
    x[3, 7], x[4, 9], x[5] = math.nan, math.inf, -0.0
    x[3, 8] = 2.0
    q, s = quantize_fp8_rows(x)
    v = rows64(q, s)
    assert (v[0] == 0).all() and (s[0] > 0).all() and torch.isfinite(v[1]).all() and v[1].abs().max() <= 1e-38
    assert (s[2] < 1e37).all() and torch.allclose(v[2], torch.tensor(3e38, dtype=torch.float64), rtol=1e-6)
    # a NaN stays in its place: the block's other value, 2, is its maximum and stands as 448 of the scale 2 / 448
    one = torch.tensor(2.0) * torch.tensor(1.0 / 448.0)
    assert torch.isnan(v[3, 7]) and s[3, 0] == one and v[3, 8] == 448 * one.double() and torch.isfinite(v[3, 8:]).all()
    assert torch.isnan(v[4, 9]) and (v[4, 128:] == 0).all()                              # an infinity spoils its block
    assert (v[5] == 0).all()
    assert quantize_fp8_rows(x[:0])[0].shape == (0, 256)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(128, 128), (200, 300), (3, 130, 257), (2, 1, 1), (1, 129, 16)])
def test_quantize_weight_and_transpose(dtype, shape):
    from rwkv_mlx_b200.fp8 import quantize_fp8_weight, transpose_fp8_weight

    w = (torch.randn(*shape, device="cuda", generator=gen(1)) * 0.05).to(dtype)
    q, s = quantize_fp8_weight(w)
    N, K = shape[-2:]
    w3 = w.float().cpu().reshape(-1, N, K)
    p = torch.nn.functional.pad(w3, (0, blocks(K) * 128 - K, 0, blocks(N) * 128 - N))
    a = p.view(-1, blocks(N), 128, blocks(K), 128).abs().amax((2, 4)).clamp(min=1e-30)
    mul = (torch.reciprocal(a) * 448.0).repeat_interleave(128, 1).repeat_interleave(128, 2)[:, :N, :K]
    assert q.shape == shape and s.shape == (*shape[:-2], blocks(N), blocks(K))
    assert torch.equal(q.cpu().contiguous().view(torch.uint8).view(-1, N, K), (w3 * mul).to(E4M3).view(torch.uint8))
    assert torch.equal(s.cpu().view(a.shape), a * torch.tensor(1.0 / 448.0))
    qt, st = transpose_fp8_weight(q, s)
    assert torch.equal(weight64(qt, st), weight64(q, s).transpose(-1, -2))


SHAPES = [(1, 8, 16), (5, 40, 130), (128, 128, 128), (129, 257, 1096), (300, 1000, 640), (31, 1024, 1), (513, 300, 2000),
          (1100, 520, 384)]


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("which", [1, 2, 3, 0])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_matmul_matches_float64(impl, which, M, N, K, out_dtype):
    from rwkv_mlx_b200 import check_device_error
    from rwkv_mlx_b200.fp8 import fp8_matmul, quantize_fp8_rows, quantize_fp8_weight

    impl(which)
    q, s = quantize_fp8_rows(torch.randn(M, K, device="cuda", generator=gen(M)))
    wq, ws = quantize_fp8_weight(torch.randn(N, K, device="cuda", generator=gen(N)))
    a, w = rows64(q, s), weight64(wq, ws)
    ref, mag = a @ w.T, a.abs() @ w.abs().T
    y = fp8_matmul(q, s, wq, ws, out_dtype=out_dtype)
    tiny = 2.0 ** -24 if out_dtype == torch.float16 else 0.0
    assert ((y.cpu().double() - ref).abs() <= 2.0 ** -20 * mag + ULP[out_dtype] * ref.abs() * 1.001 + tiny).all()
    r = fp8_matmul(q, s, wq, ws, relu_sq=True, out_dtype=torch.float32)
    sq = ref.clamp(min=0) ** 2
    assert ((r.cpu().double() - sq).abs() <= 2.0 ** -20 * mag * (2 * ref.abs() + mag * 2.0 ** -20) + 2.0 ** -23 * sq).all()
    check_device_error()


@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_quantised_hidden_rows(impl, which, M, N, K):
    """relu^2 quantised in the epilogue: the scale is that of the float64 rows to 1e-5 (twice the relative error
    of the largest product, which is no small sum), each value within half an e4m3 step of its own."""
    from rwkv_mlx_b200.fp8 import fp8_matmul_relu_sq_quantized, quantize_fp8_rows, quantize_fp8_weight

    impl(which)
    q, s = quantize_fp8_rows(torch.randn(M, K, device="cuda", generator=gen(M + 1)))
    wq, ws = quantize_fp8_weight(torch.randn(N, K, device="cuda", generator=gen(N + 1)))
    a, w = rows64(q, s), weight64(wq, ws)
    h = (a @ w.T).clamp(min=0) ** 2
    mag = (a.abs() @ w.abs().T) ** 2
    hq, hs = fp8_matmul_relu_sq_quantized(q, s, wq, ws)
    assert hq.shape == (M, N) and hs.shape == (M, blocks(N))
    hp = torch.nn.functional.pad(h, (0, blocks(N) * 128 - N)).view(M, blocks(N), 128)
    top = hp.amax(-1).clamp(min=1e-30)
    mp = torch.nn.functional.pad(mag, (0, blocks(N) * 128 - N)).view(M, blocks(N), 128).amax(-1)
    assert ((hs.cpu().double() - top / 448).abs() <= 1e-6 * top / 448 + 2.0 ** -18 * mp / 448).all()
    step = torch.maximum(h * 2.0 ** -4, hs.cpu().double().repeat_interleave(128, 1)[:, :N] * 2.0 ** -10)
    assert ((rows64(hq, hs) - h).abs() <= 1.001 * step + 2.0 ** -17 * mag).all()


GROUPS = [([300, 0, 128, 1, 517], 384, 200, 0), ([0, 0, 5], 264, 128, 0), ([1, 1, 1, 0, 2, 1, 1], 160, 144, 3),
          ([1000, 24, 256, 255, 257, 3], 512, 392, 0), ([700, 900], 300, 256, 11), ([0, 0], 128, 128, 0)]


@pytest.mark.parametrize("which", [1, 2, 3, 0])
@pytest.mark.parametrize("sizes,N,K,first", GROUPS)
def test_grouped_matmul(impl, which, sizes, N, K, first):
    """Empty groups, tiles that end inside another group's rows, rows outside every group left alone."""
    from rwkv_mlx_b200.fp8 import fp8_matmul, fp8_matmul_relu_sq_quantized, quantize_fp8_rows, quantize_fp8_weight

    impl(which)
    G, M = len(sizes), first + sum(sizes) + 9
    offs = torch.tensor([first + sum(sizes[:i]) for i in range(G + 1)], dtype=torch.int32, device="cuda")
    q, s = quantize_fp8_rows(torch.randn(M, K, device="cuda", generator=gen(7)))
    wq, ws = quantize_fp8_weight(torch.randn(G, N, K, device="cuda", generator=gen(8)))
    a, w = rows64(q, s), weight64(wq, ws)
    for dt in (torch.float32, torch.bfloat16):
        out = torch.full((M, N + 24), 7.0, device="cuda", dtype=dt)
        fp8_matmul(q, s, wq, ws, offs, out=out[:, :N])
        o = out.cpu().double()
        assert (o[:, N:] == 7).all() and (o[:first] == 7).all() and (o[first + sum(sizes):] == 7).all()
        for g in range(G):
            lo, hi = int(offs[g]), int(offs[g + 1])
            ref, mag = a[lo:hi] @ w[g].T, a[lo:hi].abs() @ w[g].abs().T
            assert ((o[lo:hi, :N] - ref).abs() <= 2.0 ** -20 * mag + ULP[dt] * 1.001 * ref.abs()).all()
    if which in (0, 2, 3):
        hq, hs = fp8_matmul_relu_sq_quantized(q, s, wq, ws, offs)
        v = rows64(hq, hs)
        for g in range(G):
            lo, hi = int(offs[g]), int(offs[g + 1])
            h = (a[lo:hi] @ w[g].T).clamp(min=0) ** 2
            mag = (a[lo:hi].abs() @ w[g].abs().T) ** 2
            step = torch.maximum(h * 2.0 ** -4, hs.cpu().double().repeat_interleave(128, 1)[lo:hi, :N] * 2.0 ** -10)
            assert ((v[lo:hi] - h).abs() <= 1.001 * step + 2.0 ** -17 * mag).all()


@pytest.mark.parametrize("which", [2, 3])
def test_unaligned_output_rows(impl, which):
    """An output whose rows TMA and 16-byte stores cannot take is written value by value."""
    from rwkv_mlx_b200.fp8 import fp8_matmul, quantize_fp8_rows, quantize_fp8_weight

    impl(which)
    q, s = quantize_fp8_rows(torch.randn(200, 256, device="cuda", generator=gen(1)))
    wq, ws = quantize_fp8_weight(torch.randn(301, 256, device="cuda", generator=gen(2)))
    out = torch.zeros(200, 305, device="cuda", dtype=torch.bfloat16)
    fp8_matmul(q, s, wq, ws, out=out[:, 1:302])
    ref = fp8_matmul(q, s, wq, ws)
    assert torch.equal(out[:, 1:302], ref) and (out[:, 0] == 0).all() and (out[:, 302:] == 0).all()


def test_infinite_and_nan_operands_stay_in_their_rows():
    from rwkv_mlx_b200.fp8 import fp8_matmul, quantize_fp8_rows, quantize_fp8_weight

    x = torch.randn(300, 256, device="cuda", generator=gen(4))
    x[17, 3], x[250, 200] = math.nan, math.inf
    q, s = quantize_fp8_rows(x)
    wq, ws = quantize_fp8_weight(torch.randn(264, 256, device="cuda", generator=gen(5)))
    for rs in (False, True):
        y = fp8_matmul(q, s, wq, ws, relu_sq=rs, out_dtype=torch.float32)
        bad = ~torch.isfinite(y).all(1)
        assert bad.nonzero().flatten().tolist() == [17, 250] and torch.isnan(y[[17, 250]]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 4, 33, 400])
def test_linear_and_its_gradient(dtype, M):
    from rwkv_mlx_b200.fp8 import fp8_linear, quantize_fp8_weight, transpose_fp8_weight

    N, K = 200, 328
    wq, ws = quantize_fp8_weight(torch.randn(N, K, device="cuda", generator=gen(1)) / 18)
    wt, wst = transpose_fp8_weight(wq, ws)
    x = torch.randn(M, 2, K, device="cuda", generator=gen(2)).to(dtype).requires_grad_(True)
    y = fp8_linear(x, wq, ws, wt, wst)
    dy = torch.randn(M, 2, N, device="cuda", generator=gen(3)).to(dtype)
    (dx,) = torch.autograd.grad(y, x, dy)
    w = weight64(wq, ws)
    for got, inp, mat, n in ((y, x, w.T, N), (dx, dy, w, K)):
        v = rows64(*plain_rows(inp.detach().reshape(2 * M, -1)))
        ref, mag = v @ mat, v.abs() @ mat.abs()
        g = got.detach().cpu().double().reshape(2 * M, n)
        tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
        assert got.dtype == dtype and ((g - ref).abs() <= 2.0 ** -20 * mag + ULP[dtype] * 1.001 * ref.abs() + tiny).all()
    with torch.no_grad():
        assert torch.equal(fp8_linear(x, wq, ws), y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("K", [16, 144, 1040, 4096, 8192, 8208])
@pytest.mark.parametrize("M", [1, 3, 8, 9])
def test_linear_of_few_rows(dtype, K, M):
    """Rows that the product's own kernel quantises (up to 8, K a multiple of 16 up to 8192) against the two calls in a row:
    the same bytes and the same sums, so the same result; odd pitches and bases included."""
    from rwkv_mlx_b200.fp8 import fp8_linear, fp8_matmul, quantize_fp8_rows, quantize_fp8_weight

    for N in (40, 300):
        wq, ws = quantize_fp8_weight(torch.randn(N, K, device="cuda", generator=gen(N)))
        wide = data(M, K + 7, M, dtype)
        for x in (wide[:, :K].contiguous(), wide[:, 3:3 + K], wide[:, 1:1 + K]):
            y = fp8_linear(x, wq, ws)
            assert torch.equal(y, fp8_matmul(*quantize_fp8_rows(x), wq, ws, out_dtype=dtype))
    x = torch.randn(M, K, device="cuda", generator=gen(1)).to(dtype)
    x[0] = 0
    x[-1, K // 2] = math.nan
    y = fp8_linear(x, wq, ws)
    assert torch.isnan(y[-1]).all() and (M == 1 or (y[0] == 0).all()) and torch.isfinite(y[:-1]).all()


def test_linear_gradient_against_differences():
    """dy and the steps lie on values that e4m3 holds exactly in every block, so quantisation is the identity and the
    product is linear: differences of float64-exact values."""
    from rwkv_mlx_b200.fp8 import fp8_linear, quantize_fp8_weight, transpose_fp8_weight

    N, K = 128, 128
    grid = torch.tensor([-448.0, -224, -112, 0, 112, 224, 448], device="cuda")
    pick = lambda r, c, s: grid[torch.randint(0, 7, (r, c), device="cuda", generator=gen(s))]  # noqa: E731
    w = pick(N, K, 1)
    w[:, 0] = 448
    wq, ws = quantize_fp8_weight(w)
    wt, wst = transpose_fp8_weight(wq, ws)
    x, dy = pick(4, K, 2), pick(4, N, 3)
    x[:, 0], dy[:, 0] = 448, 448             # every block's maximum, so its scale is 1
    x.requires_grad_(True)
    y = fp8_linear(x, wq, ws, wt, wst)
    (dx,) = torch.autograd.grad(y, x, dy)
    for k in (1, 2, 64, 127):
        up, dn = x.detach().clone(), x.detach().clone()
        up[:, k], dn[:, k] = 448, -448
        d = ((fp8_linear(up, wq, ws) - fp8_linear(dn, wq, ws)).double() * dy.double()).sum(1) / 896
        assert torch.allclose(d, dx[:, k].double(), rtol=1e-5, atol=1e-2 * 448)


@pytest.mark.parametrize("M,E", [(5, 8), (40, 8), (900, 4), (3000, 3)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_experts_match_their_parts(M, E, dtype):
    """The chained call gives what its products give one by one on each expert's rows (the hidden rows'
    quantisation can fall on the other side of a step where fp32 sums differ: 1e-3 relative)."""
    from rwkv_mlx_b200.fp8 import fp8_experts, fp8_matmul, quantize_fp8_rows, quantize_fp8_weight

    C, D = 256, 392
    g = gen(M)
    key, ks = quantize_fp8_weight(torch.randn(E, D, C, device="cuda", generator=g) / 16)
    val, vs = quantize_fp8_weight(torch.randn(E, C, D, device="cuda", generator=g) / 20)
    who = torch.randint(0, max(1, E - 1), (M,), device="cuda", generator=g)     # the last expert gets no row
    sizes = torch.bincount(who, minlength=E)
    offs = torch.cat([sizes.new_zeros(1), sizes.cumsum(0)]).int()
    x = torch.randn(M, C, device="cuda", generator=g).to(dtype)
    y = fp8_experts(x, key, ks, val, vs, offs)
    parts = []
    for e in range(E):
        xe = x[int(offs[e]):int(offs[e + 1])]
        if xe.shape[0]:
            h = fp8_matmul(*quantize_fp8_rows(xe), key[e], ks[e], relu_sq=True, out_dtype=torch.float32)
            parts.append(fp8_matmul(*quantize_fp8_rows(h), val[e], vs[e], out_dtype=dtype))
    ref = torch.cat(parts)
    assert rel_rms(y.double().cpu().numpy(), ref.double().cpu().numpy()) < 1e-3 + 2 * ULP[dtype]


@pytest.mark.parametrize("M,E", [(7, 4), (700, 3)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_experts_gradient(M, E, dtype):
    """dx against the formula in float64 with the quantisations where the operator has them (q(dy), q(du); u and dh are
    rounded to the rows' type on the way: an ulp each, and a few of q(du)'s values on the other side of a
    step of 2^-4: 2^-4 * sqrt(2 ulp)), and against the float64 layer's own gradient, from which the
    quantised dy, du and hidden rows differ by 2^-5 or so each."""
    from rwkv_mlx_b200.fp8 import fp8_experts, quantize_fp8_weight, transpose_fp8_weight

    C, D = 136, 264
    g = gen(M)
    key, ks = quantize_fp8_weight(torch.randn(E, D, C, device="cuda", generator=g) / 12)
    val, vs = quantize_fp8_weight(torch.randn(E, C, D, device="cuda", generator=g) / 16)
    tr = (*transpose_fp8_weight(key, ks), *transpose_fp8_weight(val, vs))
    sizes = torch.bincount(torch.randint(1, E, (M,), device="cuda", generator=g), minlength=E)
    offs = torch.cat([sizes.new_zeros(1), sizes.cumsum(0)]).int()
    x = torch.randn(M, C, device="cuda", generator=g).to(dtype).requires_grad_(True)
    y = fp8_experts(x, key, ks, val, vs, offs, tr)
    with torch.no_grad():
        assert torch.equal(y, fp8_experts(x, key, ks, val, vs, offs))
    dy = torch.randn(M, C, device="cuda", generator=g).to(dtype)
    (dx,) = torch.autograd.grad(y, x, dy)
    K, V = weight64(key, ks), weight64(val, vs)
    xq, dyq = rows64(*plain_rows(x.detach())), rows64(*plain_rows(dy))
    ref, free = torch.zeros(M, C, dtype=torch.float64), torch.zeros(M, C, dtype=torch.float64)
    for e in range(E):
        lo, hi = int(offs[e]), int(offs[e + 1])
        u = (xq[lo:hi] @ K[e].T).to(dtype).double()
        dh = (dyq[lo:hi] @ V[e]).to(dtype).double()
        du = dh * 2 * u.clamp(min=0)
        if hi > lo:
            ref[lo:hi] = rows64(*plain_rows(du)) @ K[e]
        xe = x[lo:hi].detach().cpu().double().requires_grad_(True)
        ((xe @ K[e].T).clamp(min=0) ** 2 @ V[e].T).backward(dy[lo:hi].cpu().double())
        free[lo:hi] = xe.grad
    ulp = max(ULP[dtype], 2.0 ** -20)
    assert dx.dtype == dtype
    assert rel_rms(dx.cpu().double().numpy(), ref.numpy()) < 4 * ulp + 2.0 ** -4 * math.sqrt(2 * ulp)
    assert rel_rms(dx.cpu().double().numpy(), free.numpy()) < 0.08


@pytest.mark.parametrize("M,K", [(3, 127), (130, 776), (33, 1024)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_relu_sq_grad_bytes(dtype, M, K):
    from rwkv_mlx_b200 import _native as nat

    dh, u = data(M, K, 1, dtype), data(M, K, 2, dtype)
    q = torch.zeros(M, -(-K // 16) * 16, device="cuda", dtype=torch.uint8)
    s = torch.zeros(blocks(K), M, device="cuda")
    nat.check(nat.lib().rwkv_quantize_fp8_relu_sq_grad(dh.data_ptr(), u.data_ptr(), K, q.data_ptr(), q.stride(0),
                                                       s.data_ptr(), M, K, nat.dtype_code(dh), nat.stream_ptr(dh.device)),
              "rwkv_quantize_fp8_relu_sq_grad")
    qr, sr = plain_rows(dh.float().cpu() * (2 * u.float().cpu().clamp(min=0)))
    assert torch.equal(q[:, :K].cpu(), qr.view(torch.uint8)) and torch.equal(s.t().cpu(), sr)


def test_second_derivatives_are_refused():
    """The backward passes are not differentiable themselves: asking for that raises instead of leaving terms out."""
    from rwkv_mlx_b200.fp8 import fp8_linear, quantize_fp8_weight, transpose_fp8_weight
    from rwkv_mlx_b200.route import route_experts

    w = quantize_fp8_weight(torch.randn(64, 32, device="cuda"))
    x = torch.randn(3, 32, device="cuda", requires_grad=True)
    c = torch.randn(3, 64, device="cuda", requires_grad=True)
    (d,) = torch.autograd.grad((fp8_linear(x, *w, *transpose_fp8_weight(*w)) * c).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
    (d,) = torch.autograd.grad(route_experts(x, 4)[1].square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


def test_offsets_past_32_bits():
    """Rows whose byte offset exceeds 2^32 in the activations, the e4m3 rows and the outputs."""
    from rwkv_mlx_b200.fp8 import fp8_linear, quantize_fp8_weight

    M, K, N = 140001, 32768, 128
    wq, ws = quantize_fp8_weight(torch.randn(N, K, device="cuda", generator=gen(1)) / 181)
    x = torch.zeros(M, K, device="cuda", dtype=torch.bfloat16)
    rows = [0, 65536, 131073, M - 1]
    x[rows] = torch.randn(4, K, device="cuda", generator=gen(2)).bfloat16()
    y = fp8_linear(x, wq, ws)
    part = fp8_linear(x[rows].contiguous(), wq, ws)
    # another kernel (few rows), so fp32 sums in another order and one bf16 rounding
    assert rel_rms(y[rows].double().cpu().numpy(), part.double().cpu().numpy()) < 2.0 ** -8
    rest = torch.ones(M, dtype=torch.bool, device="cuda")
    rest[rows] = False
    assert (y[rest] == 0).all()


def test_repeatable_and_on_another_stream():
    from rwkv_mlx_b200.fp8 import fp8_experts, fp8_linear, quantize_fp8_weight

    wq, ws = quantize_fp8_weight(torch.randn(512, 384, device="cuda", generator=gen(1)))
    key, ks = quantize_fp8_weight(torch.randn(4, 256, 384, device="cuda", generator=gen(2)))
    val, vs = quantize_fp8_weight(torch.randn(4, 384, 256, device="cuda", generator=gen(3)))
    offs = torch.tensor([0, 100, 100, 350, 500], device="cuda", dtype=torch.int32)
    x = torch.randn(500, 384, device="cuda", generator=gen(4)).half()
    a = [fp8_linear(x, wq, ws), fp8_linear(x[:3], wq, ws), fp8_experts(x, key, ks, val, vs, offs)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = [fp8_linear(x, wq, ws), fp8_linear(x[:3], wq, ws), fp8_experts(x, key, ks, val, vs, offs)]
    s.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_captures_in_a_cuda_graph():
    """Group sizes are read on the device: a captured graph replays correctly after they change."""
    from rwkv_mlx_b200.fp8 import fp8_experts, quantize_fp8_weight

    key, ks = quantize_fp8_weight(torch.randn(4, 256, 128, device="cuda", generator=gen(2)))
    val, vs = quantize_fp8_weight(torch.randn(4, 128, 256, device="cuda", generator=gen(3)))
    for M in (6, 640):
        offs = torch.tensor([0, 1, 2, 3, M], device="cuda", dtype=torch.int32)
        x = torch.randn(M, 128, device="cuda", generator=gen(4)).bfloat16()
        fp8_experts(x, key, ks, val, vs, offs)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fp8_experts(x, key, ks, val, vs, offs)
        for new in ([0, 0, M // 2, M // 2, M], [0, M, M, M, M]):
            offs.copy_(torch.tensor(new, dtype=torch.int32))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, fp8_experts(x, key, ks, val, vs, offs))


@pytest.mark.parametrize("which", [2, 3])
def test_forced_wait_timeout_fills_outputs_with_nan(impl, which):
    """Every bounded wait gives up at once (a flag set from the host): NaN outputs, the error word set, and the next
    call is right again."""
    import rwkv_mlx_b200 as rb
    from rwkv_mlx_b200 import _native
    from rwkv_mlx_b200.fp8 import fp8_matmul, quantize_fp8_rows, quantize_fp8_weight

    impl(which)
    q, s = quantize_fp8_rows(torch.randn(400, 256, device="cuda", generator=gen(1)))
    wq, ws = quantize_fp8_weight(torch.randn(300, 256, device="cuda", generator=gen(2)))
    good = fp8_matmul(q, s, wq, ws)
    rb.check_device_error()
    L = _native.lib()
    _native.check(L.rwkv_debug_force_wait_timeout(1), "rwkv_debug_force_wait_timeout")
    try:
        out = fp8_matmul(q, s, wq, ws)
        torch.cuda.synchronize()
    finally:
        _native.check(L.rwkv_debug_force_wait_timeout(0), "rwkv_debug_force_wait_timeout")
    assert torch.isnan(out).all()
    with pytest.raises(rb.RwkvDeviceError):
        rb.check_device_error()
    assert torch.equal(fp8_matmul(q, s, wq, ws), good)
    rb.check_device_error()


def test_refusals():
    from rwkv_mlx_b200 import RwkvNativeError
    from rwkv_mlx_b200.fp8 import fp8_experts, fp8_linear, fp8_matmul, quantize_fp8_rows, quantize_fp8_weight

    q, s = quantize_fp8_rows(torch.randn(8, 256, device="cuda"))
    wq, ws = quantize_fp8_weight(torch.randn(2, 128, 256, device="cuda"))
    offs = torch.tensor([0, 4, 8], device="cuda", dtype=torch.int32)
    x = torch.randn(8, 256, device="cuda").half()
    for bad in (lambda: fp8_matmul(q, s, wq, ws),                                    # groups without offsets
                lambda: fp8_matmul(q, s, wq, ws, offs.long()), lambda: fp8_matmul(q, s, wq, ws, offs[:2]),
                lambda: fp8_matmul(q, s, wq, ws, offs.cpu()), lambda: fp8_matmul(q, s[:, :1], wq, ws, offs),
                lambda: fp8_matmul(q, s.half(), wq, ws, offs), lambda: fp8_matmul(q.float(), s, wq, ws, offs),
                lambda: fp8_matmul(q[:, :128], s[:, :1], wq, ws, offs), lambda: fp8_matmul(q, s, wq, ws[:1], offs),
                lambda: fp8_matmul(q.view(torch.uint8)[:, 1:].view(E4M3)[:, :128], s[:, :1], wq[..., :128], ws[..., :1], offs),
                lambda: fp8_matmul(q, s, wq, ws, offs, out=torch.empty(8, 127, device="cuda")),
                lambda: fp8_linear(x, wq, ws), lambda: fp8_linear(x[:, :255], wq[0], ws[0]),
                lambda: fp8_linear(x, wq[0], ws[0].double()), lambda: fp8_linear(x.cpu(), wq[0], ws[0]),
                lambda: fp8_experts(x, wq, ws, wq, ws, offs), lambda: quantize_fp8_rows(x[0]),
                lambda: quantize_fp8_weight(x[0]), lambda: quantize_fp8_rows(x[:, :0])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RwkvNativeError):
        quantize_fp8_rows(x.double())
    with pytest.raises(RwkvNativeError):
        fp8_matmul(q, s, wq[0], ws[0], out_dtype=torch.int32)
    with pytest.raises(RuntimeError):
        fp8_linear(x.float().requires_grad_(True), wq[0], ws[0])                     # no transposed weight
    vq, vs = quantize_fp8_weight(torch.randn(2, 256, 128, device="cuda"))
    with pytest.raises(RuntimeError):
        fp8_experts(x.float().requires_grad_(True), wq, ws, vq, vs, offs)
    with pytest.raises(ValueError):
        fp8_experts(x.float().requires_grad_(True), wq, ws, vq, vs, offs, (wq, ws, vq, vs))


@pytest.mark.parametrize("own_router", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_moe_layer_in_8_bits(own_router, dtype):
    """Fp8MoE_CMix against MoE_CMix with the weights that the e4m3 experts stand for: what is left is the
    activations' quantisation (each value off by at most 2^-4, 2^-5 on average at random, on both
    products' inputs; a sum of independent errors: 5 % of the output)."""
    from rwkv_mlx_b200.model import RWKVConfig
    from rwkv_mlx_b200.moe import Fp8MoE_CMix, GroupRouter, MoE_CMix

    torch.manual_seed(1)
    cfg = RWKVConfig(n_layer=1, n_embd=256, vocab_size=64)
    moe = MoE_CMix(cfg, 0, 8, 2).cuda()
    with torch.no_grad():
        moe.expert_val.copy_(torch.randn_like(moe.expert_val) / 30)
        moe.x_k.copy_(torch.rand_like(moe.x_k))
    moe = moe.to(dtype)
    moe.requires_grad_(False)
    router = None if own_router else GroupRouter(256, 8, 2, n_groups=4, topk_groups=2).cuda().requires_grad_(False)
    f8 = Fp8MoE_CMix(moe, router)
    x = torch.randn(3, 50, 256, device="cuda").to(dtype)
    y, aux, z = f8(x)
    assert y.shape == x.shape and y.dtype == dtype
    kq, ks, vq, vs = f8.expert_weights()
    moe.expert_key.data, moe.expert_val.data = weight64(kq, ks).to(dtype).cuda(), weight64(vq, vs).to(dtype).cuda()
    if own_router:
        ref, raux, rz = moe(x)
        assert torch.equal(aux, raux) and torch.equal(z, rz)
        assert rel_rms(y.double().cpu().numpy(), ref.double().cpu().numpy()) < 0.05
        rnn = f8.forward_rnn(x[:, 1].contiguous(), x[:, 0].contiguous())
        # token 1's predecessor is token 0 in both modes: other kernels, one more rounding of the output type
        assert rel_rms(rnn.double().cpu().numpy(), y[:, 1].double().cpu().numpy()) < 4 * ULP[dtype] + 1e-3
    else:
        assert float(aux) == 0 and float(z) == 0
        inds, w, _ = router(x.reshape(150, 256))
        prev = torch.cat([torch.zeros_like(x[:, :1]), x[:, :-1]], 1).reshape(150, 256).double().cpu()
        xd, ref = x.reshape(150, 256).double().cpu(), torch.zeros(150, 256, dtype=torch.float64)
        K, V, xk = weight64(kq, ks), weight64(vq, vs), moe.x_k.double().cpu().reshape(8, 256)
        for t in range(150):
            for j in range(2):
                e = int(inds[t, j])
                h = (K[e] @ (xd[t] + (prev[t] - xd[t]) * xk[e])).clamp(min=0) ** 2
                ref[t] += float(w[t, j]) * (V[e] @ h)
        assert rel_rms(y.double().cpu().numpy().reshape(150, 256), ref.numpy()) < 0.05
    half = f8.half()                          # a module cast leaves the experts' bytes alone
    assert torch.equal(half.expert_weights()[0].view(torch.uint8), kq.view(torch.uint8))


def test_model_with_experts_in_8_bits():
    """quantize_experts swaps a model's full experts: prefill and decode agree with each other and, up to the
    activations' quantisation (as in test_moe_layer_in_8_bits; it reaches the logits through the residual
    stream, which it does not enlarge), with the 16-bit model on the same expert values; a captured decode step equals
    the eager one."""
    from rwkv_mlx_b200.model import RWKV, DecodeGraph, RWKVConfig, cast_for_inference, init_weights
    from rwkv_mlx_b200.moe import Fp8MoE_CMix, MoE_CMix, quantize_experts

    torch.manual_seed(0)
    cfg = RWKVConfig(n_layer=2, n_embd=128, vocab_size=512, dim_ffn=256, moe_num_experts=4, moe_top_k=2, moe_mode="full")
    m = init_weights(RWKV(cfg).cuda(), seed=1)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(torch.randn(p.shape, generator=gen(2), device="cuda") * (0.05 if p.dim() > 1 else 0.02))
        m.emb.weight.mul_(1000.0)
    m = cast_for_inference(m)
    idx = torch.randint(0, cfg.vocab_size, (3, 20), device="cuda", generator=gen(3))
    with torch.no_grad():
        for blk in m.blocks:  # values that e4m3 holds, so both models have the same experts
            f8 = Fp8MoE_CMix(blk.ffn)
            kq, ks, vq, vs = f8.expert_weights()
            blk.ffn.expert_key.data = weight64(kq, ks).half().cuda()
            blk.ffn.expert_val.data = weight64(vq, vs).half().cuda()
        ref, aux = m(idx)
        assert quantize_experts(m) is m and not any(isinstance(x, MoE_CMix) for x in m.modules())
        y, aux8 = m(idx)
        assert rel_rms(y.double().cpu().numpy(), ref.double().cpu().numpy()) < 0.05
        assert abs(float(aux8) - float(aux)) < 0.05 * abs(float(aux)) + 1e-4
        _, _, states = m.forward_with_state(idx[:, :16])
        dec = torch.stack([m.forward_rnn_batch(idx[:, t], states) for t in range(16, 20)], 1)
        assert rel_rms(dec.double().cpu().numpy(), y[:, 16:].double().cpu().numpy()) < 0.02
        _, _, states = m.forward_with_state(idx[:, :16])
        graph = DecodeGraph(m, [{k: v.clone() for k, v in st.items()} for st in states], idx[:, 16])
        graph.step()
        eager = m.forward_rnn_batch(idx[:, 16], states)
        assert rel_rms(graph.logits.double().cpu().numpy(), eager.double().cpu().numpy()) < 1e-3

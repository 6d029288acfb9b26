"""MXFP4 quantisation and linear layers against their definitions in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=F64)


@pytest.fixture(scope="module")
def X():
    import omnivideo.modules.mxfp4 as X
    return X


def randn(shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g) * scale


def ref_quant(x):
    """(codes [M, K], scale bytes [M, K/32], values [M, K] in 64 bits) of the definition, on the CPU: the nearest of the
    eight magnitudes, a tie to the even code"""
    b = x.double().reshape(x.shape[0], -1, 32)
    amax = b.abs().amax(2)
    e = torch.frexp(amax)[1].double() - 1 - 2
    s = torch.where(amax > 0, e + 127, torch.zeros_like(e)).clamp(0, 254)
    scale = torch.exp2(s - 127)[..., None]
    u = (b / scale).abs()
    dist = (u[..., None] - E2M1).abs()
    odd = torch.arange(8) % 2
    code = (dist + odd * 1e-13 * E2M1.clamp(min=1)).argmin(-1)          # codes' distances differ by 0 or by >= 2^-24
    val = torch.where(b < 0, -E2M1[code], E2M1[code]) * scale
    code = code + 8 * torch.signbit(b)
    return code.reshape(x.shape).to(torch.uint8), s.to(torch.uint8), val.reshape(x.shape)


def codes_of(m):
    c, s = m.to_ocp()
    c, s = c.cpu(), s.cpu()
    return torch.stack((c & 15, c >> 4), -1).reshape(m.rows, m.cols), s


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,K", [(1, 32), (1, 1536), (5, 96), (31, 288), (33, 256), (64, 4096), (257, 13824)])
def test_quantize_equals_definition(X, M, K, dtype):
    x = (randn((M, K), M + K) * torch.exp2(torch.randint(-40, 40, (M, K // 32), generator=torch.Generator().manual_seed(3)).float())
         .repeat_interleave(32, 1)).to(dtype)
    x[0, :32] = 0
    m = X.mxfp4_quantize(x.cuda())
    code, s, val = ref_quant(x)
    got_c, got_s = codes_of(m)
    assert torch.equal(got_s, s)
    assert torch.equal(got_c, code)
    for dt in (BF16, F32):
        assert torch.equal(m.dequantize(dt).cpu().double(), val)


def test_quantize_ties_saturation_and_extreme_exponents(X):
    """every midpoint of the grid on both sides of zero, values between 6 and 8 times the scale, the smallest and
    largest exponents of the type, both zeros"""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0, 6.0, 6.5, 7.0, 7.9375, 0.0, 0.5, 1.0, 1.5])
    base = torch.cat((mids, -mids))
    rows = [base * 2.0 ** p for p in (0, 1, -1, 30, -30, 100, -100, 124, -120)]
    rows.append(torch.full((32,), 3.3895e38))                       # the largest bf16: scale 2^125
    rows.append(torch.tensor([2.0 ** -126, -2.0 ** -126] * 16))      # scale byte clamped at 0
    rows.append(torch.tensor([2.0 ** -133, 2.0 ** -127, 0.0, -2.0 ** -130] * 8))
    x = torch.stack(rows).to(BF16)
    for dt in (BF16, F32):
        m = X.mxfp4_quantize(x.to(dt).cuda())
        code, s, val = ref_quant(x)
        got_c, got_s = codes_of(m)
        assert torch.equal(got_s, s)
        assert torch.equal(got_c, code)
        assert torch.equal(m.dequantize(F32).cpu().double(), val)


def test_quantize_infinities_and_nan_stay_in_their_block(X):
    x = randn((4, 96), 5).to(BF16)
    x[1, 33] = math.inf
    x[2, 70] = math.nan
    x[3, 0] = -math.inf
    m = X.mxfp4_quantize(x.cuda())
    v = m.dequantize(F32).cpu()
    bad = torch.zeros(4, 96, dtype=torch.bool)
    bad[1, 32:64] = bad[2, 64:] = bad[3, :32] = True
    assert torch.equal(torch.isnan(v), bad)
    clean = torch.where(bad, torch.zeros_like(x), x)
    assert torch.equal(v[~bad].double(), ref_quant(clean)[2][~bad])
    w = X.mxfp4_quantize(randn((8, 96), 6).cuda())
    y = X.mxfp4_linear(m, w, out_dtype=F32)
    assert torch.isnan(y[1:]).all() and torch.isfinite(y[0]).all()


def test_quantize_strided_and_offset_rows(X):
    big = randn((70, 3 * 160 + 1), 7).to(BF16).cuda()
    for view in (big[:, 160:320], big[::2, 8:136], big[:, 1:97], big[:, :64].t().reshape(64, 70)[:, :64]):
        got, want = X.mxfp4_quantize(view), X.mxfp4_quantize(view.contiguous().clone())
        assert torch.equal(got.dequantize(), want.dequantize())
    x3 = randn((3, 5, 64), 8).to(BF16).cuda()
    assert X.mxfp4_quantize(x3).shape == (15, 64)
    assert X.mxfp4_quantize(x3[:0]).dequantize().shape == (0, 64)
    wide = torch.full((15, 96), 7.0, device="cuda", dtype=BF16)
    X.mxfp4_quantize(x3).dequantize(out=wide[:, 16:80])
    assert (wide[:, :16] == 7).all() and (wide[:, 80:] == 7).all()


def test_ocp_round_trip(X):
    g = torch.Generator().manual_seed(1)
    for rows, cols in ((1, 32), (33, 288), (100, 1536)):
        c = torch.randint(0, 256, (rows, cols // 2), generator=g).to(torch.uint8).cuda()
        s = torch.randint(100, 140, (rows, cols // 32), generator=g).to(torch.uint8).cuda()
        m = X.MXFP4Matrix.from_ocp(c, s)
        c2, s2 = m.to_ocp()
        assert torch.equal(c, c2) and torch.equal(s, s2)
        lut = torch.cat((E2M1, -E2M1))
        nib = torch.stack((c & 15, c >> 4), -1).reshape(rows, cols).cpu().long()
        val = lut[nib] * torch.exp2(s.cpu().double() - 127).repeat_interleave(32, 1)
        assert torch.equal(m.dequantize(F32).cpu().double(), val)


SHAPES = [(1, 4, 32), (1, 5120, 5120), (2, 36, 288), (17, 260, 96), (31, 128, 1024), (32, 1536, 256), (33, 64, 2336),
          (64, 512, 320), (130, 100, 512), (550, 1536, 8960), (700, 772, 4096), (2049, 512, 1536), (1300, 1280, 96),
          (8000, 1100, 512), (3333, 2564, 1056), (4127, 2052, 288), (700, 1252, 544), (20001, 2308, 288)]


def close(got, want, bound, dtype):
    """bound: of the fp32 sum; the stored value is rounded once more by half a step"""
    half = torch.finfo(dtype).eps / 2
    err = (got.double() - want).abs()
    tol = bound + half * (want.abs() + bound) + 1e-37
    assert (err <= tol).all(), f"worst {float((err / tol).max())} of the tolerance"


def operands(X, M, N, K, seed):
    a = X.mxfp4_quantize(randn((M, K), seed).cuda())
    w = X.mxfp4_quantize(randn((N, K), seed + 1, 1 / math.sqrt(K)).cuda())
    A, W = a.dequantize(F32).double(), w.dequantize(F32).double()
    # fp32 sums of K exact products: each of at most K additions is off by at most 2^-23 of the running magnitude
    # (2^-24 rounded to nearest, twice that truncated)
    return a, w, A @ W.t(), K * 2.0 ** -23 * (A.abs() @ W.abs().t())


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_epilogues(X, M, N, K):
    a, w, want, bound = operands(X, M, N, K, M + N)
    bias = randn((N,), 3, 0.1).to(BF16).cuda()
    close(X.mxfp4_linear(a, w), want, bound, BF16)
    close(X.mxfp4_linear(a, w, out_dtype=F32), want, bound, F32)
    wb = want + bias.double()
    bound_b = bound + 2.0 ** -24 * (wb.abs() + bound)
    close(X.mxfp4_linear(a, w, bias), wb, bound_b, BF16)
    u = math.sqrt(2 / math.pi) * (wb + 0.044715 * wb ** 3)
    # |gelu'| <= 1.13; the kernel's form of it is off by the fp32 roundings of exp2's argument: 2^-21 |x|
    close(X.mxfp4_linear(a, w, bias, gelu=True), 0.5 * wb * (1 + torch.tanh(u)), 1.13 * bound_b + 2.0 ** -21 * wb.abs(), BF16)
    x0, gate = randn((M, N), 4).cuda(), randn((N,), 5).cuda()
    for g in (gate, None):
        x = x0.clone()
        r = X.mxfp4_linear(a, w, bias, residual=x, gate=g)
        gd = torch.ones(N, device="cuda", dtype=F64) if g is None else g.double()
        assert r.data_ptr() == x.data_ptr()
        close(x, x0.double() + wb * gd, bound_b * gd.abs(), F32)


@pytest.mark.parametrize("M,N,K", [(1, 32, 64), (5, 96, 512), (33, 544, 288), (550, 1536, 1536), (300, 8960, 512),
                                   (4127, 2080, 288), (8000, 1280, 512), (700, 1248, 544), (20001, 2336, 288)])
def test_linear_with_quantised_output(X, M, N, K):
    """the output operand = the quantisation of the fp32 result: equal where the fp32 value is not within its own error
    of a border of the rounding or of a power of two of the block's largest magnitude"""
    a, w, prod, bound = operands(X, M, N, K, M + 7)
    bias = randn((N,), 3, 0.1).to(BF16).cuda()
    m = X.mxfp4_linear(a, w, bias, gelu=True, quantize_output=True)
    assert isinstance(m, X.MXFP4Matrix) and m.shape == (M, N)
    wb = prod + bias.double()
    want = 0.5 * wb * (1 + torch.tanh(math.sqrt(2 / math.pi) * (wb + 0.044715 * wb ** 3)))
    err = 1.13 * (bound + 2.0 ** -24 * (wb.abs() + bound)) + 2.0 ** -21 * wb.abs() + 1e-37
    code, s, _ = ref_quant(want.cpu())
    got_c, got_s = codes_of(m)
    e = err.cpu().reshape(M, -1, 32)
    top = want.cpu().abs().reshape(M, -1, 32)
    lo, hi = (top - e).amax(2), (top + e).amax(2)
    sure = torch.floor(torch.log2(lo.clamp(min=1e-300))) == torch.floor(torch.log2(hi))      # the block's scale
    assert torch.equal(got_s[sure], s[sure])
    assert float(sure.double().mean()) > 0.9 or N * M < 2000
    assert ((got_s.int() - s.int()).abs() <= 1).all()
    u = (want.cpu().abs().reshape(M, -1, 32) / torch.exp2(s.double() - 127)[..., None])
    du = e / torch.exp2(s.double() - 127)[..., None]
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=F64)
    clear = ((u[..., None] - borders).abs() > du[..., None]).all(-1) & sure[..., None]
    mag = lambda c: (c & 7).reshape(M, -1, 32)
    assert torch.equal(mag(got_c)[clear], mag(code)[clear])
    sign_clear = clear & (mag(code) > 0)
    assert torch.equal((got_c >> 3).reshape(M, -1, 32)[sign_clear], (code >> 3).reshape(M, -1, 32)[sign_clear])
    # it is an operand of the next product, padding included
    w2 = X.mxfp4_quantize(randn((64, N), 9, 1 / math.sqrt(N)).cuda())
    A, W2 = m.dequantize(F32).double(), w2.dequantize(F32).double()
    close(X.mxfp4_linear(m, w2, out_dtype=F32), A @ W2.t(), N * 2.0 ** -23 * (A.abs() @ W2.abs().t()), F32)
    again = X.MXFP4Matrix.empty(M, N, "cuda")
    again.buf.fill_(255)
    assert X.mxfp4_linear(a, w, bias, gelu=True, quantize_output=True, out=again) is again
    assert torch.equal(again.dequantize(F32), m.dequantize(F32))
    close(X.mxfp4_linear(again, w2, out_dtype=F32), A @ W2.t(), N * 2.0 ** -23 * (A.abs() @ W2.abs().t()), F32)


def test_linear_exact_on_small_integers(X):
    """whole numbers with scale 1 have exact sums: a wrong lane, block order, nibble order or scale byte shows as a
    wrong whole number.  Blocks get different scales, so each scale has to meet its own block."""
    for M, N, K in ((40, 68, 608), (1, 132, 1056), (300, 512, 256), (1030, 1536, 768), (5000, 1668, 1312),
                    (16000, 516, 512), (20001, 2308, 288)):
        g = torch.Generator().manual_seed(M)
        lut = torch.tensor([0.0, 1.0, 2.0, 3.0, 4.0, 6.0])
        a = lut[torch.randint(0, 6, (M, K), generator=g)] * (torch.randint(0, 2, (M, K), generator=g) * 2 - 1)
        w = lut[torch.randint(0, 6, (N, K), generator=g)] * (torch.randint(0, 2, (N, K), generator=g) * 2 - 1)
        a[:, ::32], w[:, ::32] = 4, -4                          # the block's largest magnitude is 4 or 6: scale 1
        sa = torch.exp2(torch.randint(-2, 3, (M, K // 32), generator=g).float()).repeat_interleave(32, 1)
        sw = torch.exp2(torch.randint(-2, 3, (N, K // 32), generator=g).float()).repeat_interleave(32, 1)
        a, w = a * sa, w * sw
        y = X.mxfp4_linear(a.cuda(), X.mxfp4_quantize(w.cuda()), out_dtype=F32)
        assert torch.equal(y.cpu().double(), a.double() @ w.double().t())


def test_linear_quantises_its_input(X):
    w = X.mxfp4_quantize(randn((256, 512), 1).cuda())
    x = randn((3, 50, 512), 2).to(BF16).cuda()
    y = X.mxfp4_linear(x, w)
    assert y.shape == (3, 50, 256)
    assert torch.equal(y.view(150, 256), X.mxfp4_linear(X.mxfp4_quantize(x), w))
    assert torch.equal(X.mxfp4_linear(x.float(), w), y)
    assert X.mxfp4_linear(x[:0], w).shape == (0, 50, 256)


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 33])
@pytest.mark.parametrize("K,N", [(32, 4), (512, 256), (1120, 100), (13824, 64), (17408, 36), (30752, 32)])
def test_linear_of_few_rows_equals_quantise_then_product(X, M, K, N):
    """one launch or several: the same codes, and the same order of sums up to 32 rows"""
    w = X.mxfp4_quantize(randn((N, K), 1, 1 / math.sqrt(K)).cuda())
    bias, gate = randn((N,), 4).to(BF16).cuda(), randn((N,), 5).cuda()
    for dt in (BF16, F32):
        x = randn((M, K + 32), K, 3.0).to(dt).cuda()[:, 32:]
        x[0, :40] = 0
        a = X.mxfp4_quantize(x)
        for kw in (dict(), dict(out_dtype=F32), dict(gelu=True)):
            assert torch.equal(X.mxfp4_linear(x, w, bias, **kw), X.mxfp4_linear(a, w, bias, **kw))
        r0 = randn((M, N), 6).cuda()
        assert torch.equal(X.mxfp4_linear(x, w, residual=r0.clone(), gate=gate), X.mxfp4_linear(a, w, residual=r0.clone(), gate=gate))
        A, W = a.dequantize(F32).double(), w.dequantize(F32).double()
        close(X.mxfp4_linear(x, w, out_dtype=F32), A @ W.t(), K * 2.0 ** -23 * (A.abs() @ W.abs().t()), F32)
    x[0, 5] = math.inf
    y = X.mxfp4_linear(x, w)
    assert torch.isnan(y[0]).all() and torch.isfinite(y[1:]).all()


@pytest.mark.parametrize("M", [1, 8, 40, 700])
def test_linear_into_its_own_input(X, M):
    """x = f(x) and x += f(x): what is read is x as it was"""
    C = 1536
    w = X.mxfp4_quantize(randn((C, C), 1, 1 / math.sqrt(C)).cuda())
    for dt in (BF16, F32):
        x = randn((M, C), 2).to(dt).cuda()
        want = X.mxfp4_linear(x, w, out_dtype=dt)
        for _ in range(3):
            y = x.clone()
            assert X.mxfp4_linear(y, w, out=y) is y
            assert torch.equal(y, want)
    x = randn((M, C), 3).cuda()
    want = X.mxfp4_linear(x, w, residual=x.clone())
    buf = torch.zeros(M + 1, C, device="cuda")
    for rows in (buf[:M], buf[1:]):
        rows.copy_(x)
        X.mxfp4_linear(rows, w, residual=rows)
        assert torch.equal(rows, want)


def test_quantised_output_refuses_an_operand(X):
    a, w = X.mxfp4_quantize(randn((40, 64), 1).cuda()), X.mxfp4_quantize(randn((64, 64), 2).cuda())
    with pytest.raises(ValueError, match="operands"):
        X.mxfp4_linear(a, w, gelu=True, quantize_output=True, out=a)


@pytest.mark.parametrize("M,N,K", [(5, 64, 512), (300, 1536, 256), (700, 1252, 512), (1500, 1280, 512), (4100, 2052, 512)])
def test_linear_writes_only_its_rows(X, M, N, K):
    a, w, _, _ = operands(X, M, N, K, 9)
    for dt in (BF16, F32):
        buf = torch.full((M + 3, N + 16), 5.0, device="cuda", dtype=dt)
        X.mxfp4_linear(a, w, out=buf[1:M + 1, 8:N + 8])
        assert torch.equal(buf[1:M + 1, 8:N + 8], X.mxfp4_linear(a, w, out_dtype=dt))
        buf[1:M + 1, 8:N + 8] = 5
        assert (buf == 5).all()


@pytest.mark.parametrize("M,N,K", [(1, 1536, 5120), (550, 1536, 1536), (4096, 2048, 1536)])
def test_linear_is_repeatable_on_streams_and_in_graphs(X, M, N, K):
    w = X.mxfp4_quantize(randn((N, K), 2).cuda())
    x = randn((M, K), 1).to(BF16).cuda()
    x2 = randn((M, K), 3).to(BF16).cuda()
    first, second = X.mxfp4_linear(x, w), X.mxfp4_linear(x2, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(X.mxfp4_linear(x, w), first)
    torch.cuda.current_stream().wait_stream(side)
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = X.mxfp4_linear(static, w)
    for src, want in ((x2, second), (x, first), (x2, second)):
        static.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        assert torch.equal(X.mxfp4_linear(src, w), want)

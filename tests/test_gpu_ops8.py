"""The 8-bit operators against their formulas in 64 bits (needs a B200: -m gpu).

Tolerances count roundings: bf16 u = 2^-8, fp32 2^-24; a tensor-core sum of n products a b is within
(n + 2) 2^-23 sum |a b| of the real one (each addition may truncate).  The GELU itself errs by at most
2^-20 (1 + |gelu|): exp2 and reciprocal are good to a few 2^-23, and |x| p (1 - p) |2 u| < 1 bounds what an error
of the exponent does.
"""
import pytest

torch = pytest.importorskip("torch")

import ptxforge_b200 as pf  # noqa: E402

pytestmark = pytest.mark.gpu

BF, F32, TINY = 2.0 ** -8, 2.0 ** -24, 2.0 ** -126
K0, K1 = 0.7978845608028654, 0.044715
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, device=DEV, generator=gen(seed)).to(dtype)


def gelu64(x):
    return x * torch.sigmoid(2 * K0 * x * (1 + K1 * x * x))


def grad64(x):
    p = torch.sigmoid(2 * K0 * x * (1 + K1 * x * x))
    return p + 2 * K0 * x * p * (1 - p) * (1 + 3 * K1 * x * x)


def codes64(x, axis):
    """Codes and scales from the definition: the real quotient rounded once."""
    scale = (x.double().abs().amax(axis) / 127).float().clamp(min=TINY)
    return torch.round(x.double() / scale.double().unsqueeze(axis)).to(torch.int8), scale


def within(got, want, tol):
    off = (got.double() - want).abs() - tol
    assert got.shape == want.shape and not torch.isnan(got).any()
    assert off.max() <= 0, f"off by {(got.double() - want).abs().max():.3e}, {off.max():.3e} over the tolerance"


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    assert pf.ops8_status() == 0


# ---------------------------------------------------------------------------------------------
# store and restore
# ---------------------------------------------------------------------------------------------
SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 1001), (257, 264), (2, 16390), (70001, 8), (130, 14336), (33, 512), (4097, 96)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("axis", [1, 0])
def test_store(rows, cols, dtype, axis):
    x = randn(rows, cols, seed=rows + cols, dtype=dtype) * torch.exp(randn(cols, seed=3)).to(dtype)
    codes, scale = pf.quantize_s8(x, axis)
    want, want_scale = codes64(x, axis)
    assert torch.equal(scale, want_scale) and torch.equal(codes, want)
    for out in (torch.bfloat16, torch.float32):
        back = pf.dequantize_s8(codes, scale, axis, dtype=out)
        assert torch.equal(back, (codes.float() * scale.unsqueeze(axis)).to(out))


@pytest.mark.parametrize("rows", [5000, 4096])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_store_with_unaligned_scales(rows, dtype):
    """Scales that start anywhere: no wide load of them fits."""
    x = randn(rows, 136, seed=rows, dtype=dtype)
    for axis in (1, 0):
        want, want_scale = codes64(x, axis)
        for first in (1, 2, 3):
            room = torch.zeros(rows + 8, device=DEV)
            s = room[first:first + want_scale.numel()]
            codes, scale = pf.quantize_s8(x, axis, scale=s)
            assert scale.data_ptr() == s.data_ptr() and torch.equal(codes, want) and torch.equal(s, want_scale)
            assert torch.equal(pf.dequantize_s8(codes, s, axis, dtype=dtype), (want.float() * s.unsqueeze(axis)).to(dtype))
            s.zero_()
            assert not room.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("axis", [1, 0])
@pytest.mark.parametrize("first,cols", [(3, 40), (8, 64), (1, 33), (0, 96)])
def test_store_of_a_view_leaves_its_surroundings(dtype, axis, first, cols):
    big = randn(37, 104, seed=5, dtype=dtype)
    x = big[2:35, first:first + cols]
    room = torch.full((37, 104), 77, dtype=torch.int8, device=DEV)
    codes, scale = pf.quantize_s8(x, axis, codes=room[2:35, first:first + cols])
    want, want_scale = codes64(x, axis)
    assert torch.equal(codes, want) and torch.equal(scale, want_scale)
    values = torch.full((37, 104), 55.0, dtype=dtype, device=DEV)
    pf.dequantize_s8(codes, scale, axis, out=values[2:35, first:first + cols])
    assert torch.equal(values[2:35, first:first + cols], (want.float() * want_scale.unsqueeze(axis)).to(dtype))
    for t, v in ((room, 77), (values, 55.0)):
        t[2:35, first:first + cols] = v
        assert (t == v).all()


@pytest.mark.parametrize("axis", [1, 0])
@pytest.mark.parametrize("cols", [64, 65])
def test_store_of_extreme_values(axis, cols):
    x = randn(16, cols, seed=9)
    x[1] = 0
    x[2] *= 1e-42               # below the least scale
    x[3] = 3e38
    x[4, 5] = float("inf")
    x[5, 6] = -float("inf")
    x[6, 7] = float("nan")
    x[7] = torch.arange(cols, device=DEV) - 0.5  # half steps
    x[7, 0] = 127.0
    x[8] *= 1e-38
    y = x if axis else x.t().contiguous()
    codes, scale = pf.quantize_s8(y, axis)
    codes, fine = (codes if axis else codes.t()), [0, 1, 2, 3, 7, 8, 9, 10, 11, 12, 13, 14, 15]
    assert torch.isnan(scale[4:7]).all() and (codes[4:7] == 0).all()
    want, want_scale = codes64(x[fine], 1)
    assert torch.equal(scale[fine], want_scale) and torch.equal(codes[fine], want)
    assert scale[1] == TINY and (codes[7, 1:4] == torch.tensor([0, 2, 2], device=DEV)).all()  # 0.5, 1.5, 2.5


@pytest.mark.parametrize("cols", [8, 1001])
def test_codes_next_to_half_steps(cols):
    """Quotients a step of fp32 to each side of k + 1/2, where a division rounded to fp32 would land on it."""
    s = torch.rand(64, 1, device=DEV, generator=gen(4)) + 0.5
    k = torch.randint(-126, 126, (64, cols), device=DEV, generator=gen(5)) + 0.5
    x = (k * s.double()).float()
    x = torch.nextafter(x, torch.where(torch.rand(64, cols, device=DEV, generator=gen(6)) < 0.5, 1e9, -1e9).float())
    x[:, 0] = 127 * s[:, 0]
    codes, scale = pf.quantize_s8(x)
    want, want_scale = codes64(x, 1)
    assert torch.equal(scale, want_scale) and torch.equal(codes, want)


# ---------------------------------------------------------------------------------------------
# the int8 product
# ---------------------------------------------------------------------------------------------
def s8_operands(M, N, K, seed=0, low=-127):
    g = gen(seed)
    a = torch.randint(low, 128, (M, K), device=DEV, generator=g, dtype=torch.int8)
    b = torch.randint(low, 128, (K, N), device=DEV, generator=g, dtype=torch.int8)
    sa = torch.rand(M, device=DEV, generator=g) * 0.02 / K ** 0.5 + 1e-6
    sb = torch.rand(N, device=DEV, generator=g) * 0.02 + 1e-6
    return a, b, sa, sb, torch.randn(N, device=DEV, generator=g)


def check_s8(c, a, b, sa, sb, bias, gelu):
    x = a.double() @ b.double() * sa.double()[:, None] * sb.double()
    tol = 4 * F32 * x.abs()  # the sum to fp32, the two scales, their product with the sum, the bias
    if bias is not None:
        x = x + bias.double()
        tol = tol + F32 * x.abs()
    if gelu:
        x = gelu64(x)
        tol = 1.13 * tol + 2.0 ** -20 * (1 + x.abs())
    within(c, x, tol + (BF if c.dtype == torch.bfloat16 else F32) * (x.abs() + tol))


PRODUCTS = [(1, 16, 16), (1, 1, 1), (1, 512, 4096), (3, 5, 7), (8, 256, 512), (17, 272, 528), (37, 512, 1040), (64, 64, 2048),
            (127, 129, 131), (128, 128, 128), (129, 256, 144), (200, 136, 80), (256, 256, 256), (300, 1008, 96),
            (333, 1001, 2050), (1000, 1040, 528), (2050, 2064, 272), (5, 4100, 33),
            (24, 64, 4096), (40, 128, 8192), (100, 384, 8192), (256, 2048, 4096),  # split sums, of few and many tokens
            (2500, 2048, 1040), (2500, 2049, 1030)]                                # pairs, and a last wave of single CTAs


@pytest.mark.parametrize("M,N,K", PRODUCTS)
@pytest.mark.parametrize("gelu,with_bias,dtype", [(False, False, torch.bfloat16), (True, True, torch.bfloat16),
                                                  (False, True, torch.float32), (True, False, torch.float32)])
def test_product(M, N, K, gelu, with_bias, dtype):
    a, b, sa, sb, bias = s8_operands(M, N, K, seed=M + N + K)
    bias = bias if with_bias else None
    c = torch.full((M, N), float("nan"), dtype=dtype, device=DEV)
    assert pf.gemm_s8(a, b, sa, sb, bias, c, gelu=gelu) is c
    check_s8(c, a, b, sa, sb, bias, gelu)


@pytest.mark.parametrize("M", [2, 300])
def test_product_sums_are_exact_to_the_largest_k(M):
    a = torch.full((M, 131071), -128, dtype=torch.int8, device=DEV)
    b = torch.full((131071, 32), -128, dtype=torch.int8, device=DEV)
    a[:, ::3] = 127
    one = torch.ones(M, device=DEV), torch.ones(32, device=DEV)
    c = pf.gemm_s8(a, b, *one, dtype=torch.float32)
    assert torch.equal(c.double(), (a.double() @ b.double()).float().double())


@pytest.mark.parametrize("first,n,k", [(0, 64, 64), (16, 48, 80), (3, 41, 65), (1, 64, 64)])
@pytest.mark.parametrize("M", [4, 290])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_product_of_views_leaves_their_surroundings(first, n, k, M, dtype):
    a, b, sa, sb, bias = s8_operands(M + 4, 160, 160, seed=11)
    a, b, sa, sb, bias = a[2:M + 2, first:first + k], b[3:3 + k, first:first + n], sa[2:M + 2], sb[1:n + 1], bias[1:n + 1]
    room = torch.full((M + 4, 160), 9.0, dtype=dtype, device=DEV)
    c = pf.gemm_s8(a, b, sa, sb, bias, room[1:M + 1, first:first + n])
    check_s8(c, a, b, sa, sb, bias, False)
    room[1:M + 1, first:first + n] = 9.0
    assert (room == 9.0).all()


def test_product_of_a_token_with_a_nan_scale_is_nan_there_alone():
    a, b, sa, sb, bias = s8_operands(70, 64, 64)
    sa[3] = float("nan")
    sb[7] = float("nan")
    c = pf.gemm_s8(a, b, sa, sb, bias, gelu=True)
    bad = torch.isnan(c)
    assert bad[3].all() and bad[:, 7].all() and int(bad.sum()) == 64 + 70 - 1


# ---------------------------------------------------------------------------------------------
# the product with an 8-bit checkpoint, and its gradients
# ---------------------------------------------------------------------------------------------
LAYERS = [(1, 8, 8), (1, 136, 72), (7, 64, 256), (77, 512, 512), (128, 128, 64), (129, 264, 136), (200, 136, 72),
          (256, 256, 256), (300, 1024, 520), (515, 776, 1032), (1000, 72, 2048), (2100, 2056, 264), (1601, 1544, 1288),
          (2500, 2304, 2048), (20, 4096, 1024), (60, 256, 4096)]


def layer(M, N, K, seed=0):
    a = randn(M, K, seed=seed, dtype=torch.bfloat16)
    b = (randn(K, N, seed=seed + 1) * 1.5 / K ** 0.5).bfloat16()
    return a, b, randn(N, seed=seed + 2) * 0.5


@pytest.mark.parametrize("M,N,K", LAYERS)
def test_forward(M, N, K):
    a, b, bias = layer(M, N, K, seed=M + N + K)
    c, saved = pf.gemm_bias_gelu_checkpoint(a, b, bias)
    z = a.double() @ b.double() + bias.double()
    dz = (K + 3) * 2.0 ** -23 * (a.double().abs() @ b.double().abs() + bias.double().abs())
    y = gelu64(z)
    within(c, y, 1.13 * dz + 2.0 ** -20 * (1 + y.abs()) + BF * (y.abs() + 1.13 * dz))
    # a half step of 1 / 200, and the second derivative (at most 1.13) times what z is off
    within(saved.gelu_grad(torch.float32), grad64(z), 0.0025 + 1.13 * dz + 2.0 ** -18)
    want, want_scale = codes64(a, 1)
    assert torch.equal(saved.a_codes, want) and torch.equal(saved.a_scale, want_scale)
    assert torch.equal(saved.input(torch.float32), want.float() * want_scale[:, None])
    c2, bare = pf.gemm_bias_gelu_checkpoint(a, b, bias, torch.empty_like(c), keep_input=False)
    assert torch.equal(c, c2) and torch.equal(bare.grad_codes, saved.grad_codes) and bare.a_codes is None


def test_forward_of_extreme_values():
    a, b, bias = layer(40, 64, 64)
    bias[0], bias[1], bias[2], bias[3] = float("inf"), -1e30, 1e30, float("nan")
    bias[4] = -60.0
    a[9, 3] = float("nan")
    c, saved = pf.gemm_bias_gelu_checkpoint(a, b, bias)
    d = saved.gelu_grad(torch.float32)
    rows = [i for i in range(40) if i != 9]
    assert (saved.grad_codes[9] == 255).all() and torch.isnan(c[9]).all() and torch.isnan(saved.a_scale[9])
    assert (d[rows, 0] == 1).all() and (d[rows, 1] == 0).all() and (d[rows, 2] == 1).all() and torch.isnan(d[rows, 3]).all()
    assert (d[rows, 4] == 0).all() and (c[rows, 4] == 0).all() and (c[rows, 1] == 0).all() and (c[rows, 2] == c[0, 2]).all()
    # the backward pass: NaN where a derivative or an input is, and nowhere else
    dA, dB, dbias = pf.gemm_bias_gelu_backward(torch.ones_like(c), b, saved)
    assert torch.isnan(dbias).all()  # token 9 is in every column's sum
    keep = torch.tensor([i for i in range(64) if i != 3], device=DEV)
    rows = torch.tensor(rows, device=DEV)
    part = pf.Checkpoint(saved.a_codes[rows].contiguous(), saved.a_scale[rows].contiguous(),
                         saved.grad_codes[rows][:, keep[:56]].contiguous())
    got = pf.gemm_bias_gelu_backward(torch.ones(39, 56, dtype=torch.bfloat16, device=DEV), b[:, keep[:56]].contiguous(), part)
    assert not any(torch.isnan(t).any() for t in got)


def test_every_grad_code_stands_for_its_step():
    codes = torch.arange(256, dtype=torch.uint8, device=DEV)
    d = pf.dequantize_gelu_grad(codes, dtype=torch.float32)
    want = ((codes.double() - 26) / 200).float()
    assert torch.equal(d[:255], want[:255]) and torch.isnan(d[255])
    assert torch.equal(pf.dequantize_gelu_grad(codes[:255].clone()), want[:255].bfloat16())
    big = torch.randint(0, 253, (1003, 77), dtype=torch.uint8, device=DEV, generator=gen(1))
    assert torch.equal(pf.dequantize_gelu_grad(big, dtype=torch.float32), want[big.long()])
    big = torch.randint(0, 253, (8192 * 1024 + 4333,), dtype=torch.uint8, device=DEV, generator=gen(2))
    for part in (big, big[1:], big[:8192 * 1024 - 8]):  # four vectors a thread; codes that start anywhere; a whole last block less
        for dtype in (torch.bfloat16, torch.float32):
            assert torch.equal(pf.dequantize_gelu_grad(part, dtype=dtype), want[part.long()].to(dtype))


def grads64(dc, b, saved):
    d = (saved.grad_codes.double() - 26) / 200
    dz = dc.double() * d
    a = saved.a_codes.double() * saved.a_scale.double()[:, None]
    return dz, a, dz @ b.double().t(), a.t() @ dz, dz.sum(0)


def saved_of(M, N, K, seed=0):
    q, s = codes64(randn(M, K, seed=seed, dtype=torch.bfloat16), 1)
    d = torch.randint(0, 253, (M, N), dtype=torch.uint8, device=DEV, generator=gen(seed + 1))
    return pf.Checkpoint(q, s, d)


@pytest.mark.parametrize("M,N,K", LAYERS + [(3000, 8, 8), (128, 8, 1024), (2, 2048, 16)])
def test_backward(M, N, K):
    saved = saved_of(M, N, K, seed=M + N + K)
    dc = randn(M, N, seed=5, dtype=torch.bfloat16)
    b = randn(K, N, seed=6, dtype=torch.bfloat16)
    dA, dB, dbias = pf.gemm_bias_gelu_backward(dc, b, saved)
    dz, a, want_a, want_b, want_bias = grads64(dc, b, saved)
    sum_a = dz.abs() @ b.double().abs().t()
    tol = (BF + (N + 2) * 2.0 ** -23) * sum_a  # dz to bf16, the sum
    within(dA, want_a, tol + BF * (want_a.abs() + tol))
    sum_b = a.abs().t() @ dz.abs()
    tol = (BF + (M + 3) * 2.0 ** -23) * sum_b  # dz to bf16, the sum
    within(dB, want_b, tol + BF * (want_b.abs() + tol))
    within(dbias, want_bias, (M + 2) * F32 * dz.abs().sum(0))
    # by the norm: two independent roundings, of rms 2^-8 / sqrt 3 each at most
    for got, want in ((dA, want_a), (dB, want_b)):
        if want.numel() > 1000:
            assert (got.double() - want).norm() <= (2 / 3) ** 0.5 * BF * want.norm()
    again = pf.gemm_bias_gelu_backward(dc, b, saved)
    assert all(torch.equal(x, y) for x, y in zip((dA, dB, dbias), again))


def test_backward_of_what_is_wanted():
    saved, dc, b = saved_of(70, 136, 72), randn(70, 136, seed=1, dtype=torch.bfloat16), randn(72, 136, seed=2, dtype=torch.bfloat16)
    every = dict(zip(("dA", "dB", "dbias"), pf.gemm_bias_gelu_backward(dc, b, saved)))
    for need in (("dA",), ("dB",), ("dbias",), ("dA", "dbias"), ()):
        got = dict(zip(("dA", "dB", "dbias"), pf.gemm_bias_gelu_backward(dc, b, saved, need=need)))
        for k, v in got.items():
            assert (v is None) == (k not in need)
            assert v is None or torch.equal(v, every[k]) or k == "dA"
            if k == "dA" and v is not None:  # without dB, dz is rounded without the input's scale
                assert (v.double() - every[k].double()).norm() <= 2 * BF * every[k].double().norm()
    bare = pf.Checkpoint(None, None, saved.grad_codes)
    assert torch.equal(pf.gemm_bias_gelu_backward(dc, b, bare, need=("dA",))[0],
                       pf.gemm_bias_gelu_backward(dc, b, saved, need=("dA", "dbias"))[0])
    with pytest.raises(ValueError, match="keep_input"):
        pf.gemm_bias_gelu_backward(dc, b, bare)


def test_backward_of_tokens_of_tiny_huge_and_bad_inputs():
    """A token's dA does not depend on its input: a scale of 2^-126, 2.6e36 or NaN leaves it as it is."""
    M, N, K = 20, 64, 40
    saved, dc, b = saved_of(M, N, K), randn(M, N, seed=1, dtype=torch.bfloat16), randn(K, N, seed=2, dtype=torch.bfloat16)
    s = saved.a_scale.clone()
    s[3], s[4], s[5] = TINY, 2.6e36, 0.0
    saved = saved._replace(a_scale=s)
    dz, a, want_a, want_b, _ = grads64(dc, b, saved)
    dA, dB, _ = pf.gemm_bias_gelu_backward(dc, b, saved)
    tol = (BF + (N + 2) * 2.0 ** -23) * (dz.abs() @ b.double().abs().t())
    within(dA, want_a, tol + BF * (want_a.abs() + tol))
    tol = (BF + (M + 3) * 2.0 ** -23) * (a.abs().t() @ dz.abs())
    # token 4 alone adds up to 127 * 2.6e36 |dz| = 3.3e38 |dz|, past bf16's largest 3.39e38 where |dz| > 1.03: inf there
    fits = want_b.abs() + tol < 3.38e38
    assert fits.any() and not fits.all() and (dB[~fits].abs().double() > 3.3e38).all()
    within(dB[fits], want_b[fits], (tol + BF * (want_b.abs() + tol))[fits])
    s[6] = float("nan")
    dA2, dB2, dbias = pf.gemm_bias_gelu_backward(dc, b, saved._replace(a_scale=s))
    tol = (BF + (N + 2) * 2.0 ** -23) * (dz.abs() @ b.double().abs().t())
    within(dA2, want_a, tol + BF * (want_a.abs() + tol))
    assert torch.isnan(dB2).all() and not torch.isnan(dbias).any()


def test_gradients_against_differences():
    """L = sum g gelu(A B + bias): the slope of L along each computed gradient's own direction, by central differences
    in 64 bits.  Tolerances add up what each term may be off: the derivative's half step of 1 / 200 and dz's rounding,
    for dB the input's half step (scale / 2), and the result's rounding."""
    M, N, K, h = 96, 128, 64, 1e-4
    a, b, bias = layer(M, N, K, seed=40)
    g = randn(M, N, seed=44, dtype=torch.bfloat16)
    _, saved = pf.gemm_bias_gelu_checkpoint(a, b, bias)
    grads = [t.double() for t in pf.gemm_bias_gelu_backward(g, b, saved)]
    at = [a.double(), b.double(), bias.double()]
    g = g.double()
    L = lambda a, b, bias: (g * gelu64(a @ b + bias)).sum()  # noqa: E731
    d = grad64(at[0] @ at[1] + at[2])
    step = saved.a_scale.double()[:, None] / 2
    for which, got in enumerate(grads):
        v = got / got.norm()
        up, down = list(at), list(at)
        up[which], down[which] = at[which] + h * v, at[which] - h * v
        slope = (L(*up) - L(*down)) / (2 * h)
        reach = v @ at[1] if which == 0 else at[0] @ v if which == 1 else v.expand(M, N)
        tol = (g.abs() * (0.0025 + BF * d.abs() + 1e-5) * reach.abs()).sum() + BF * (got * v).abs().sum()
        if which == 1:
            tol = tol + (step * ((g * d) @ v.t()).abs()).sum()
        assert tol < 0.2 * slope  # the bound says something
        assert ((got * v).sum() - slope).abs() <= tol


def test_no_tokens():
    b, bias = randn(16, 24, dtype=torch.bfloat16), randn(24)
    a = torch.empty(0, 16, dtype=torch.bfloat16, device=DEV)
    c, saved = pf.gemm_bias_gelu_checkpoint(a, b, bias)
    assert c.shape == (0, 24)
    dA, dB, dbias = pf.gemm_bias_gelu_backward(c, b, saved)
    assert dA.shape == (0, 16) and not dB.any() and not dbias.any()
    q, s = pf.quantize_s8(a)
    assert q.shape == (0, 16) and s.shape == (0,) and pf.dequantize_s8(q, s).shape == (0, 16)
    b8, sb = pf.quantize_s8(b, axis=0)
    assert pf.gemm_s8(q, b8, s, sb, bias).shape == (0, 24)
    # scales over nothing are the least one
    assert (pf.quantize_s8(a, axis=0)[1] == TINY).all()
    assert (pf.quantize_s8(b[:, :0], axis=1)[1] == TINY).all() and pf.quantize_s8(b[:, :0], axis=0)[1].shape == (0,)


# ---------------------------------------------------------------------------------------------
# together, as they are used
# ---------------------------------------------------------------------------------------------
def test_a_served_mlp_block():
    """quantize -> product, GELU -> quantize -> product, against the same steps in 64 bits on the same codes."""
    M, D, H = 45, 192, 656
    x, w1, w2 = randn(M, D, seed=1, dtype=torch.bfloat16), randn(D, H, seed=2) / D ** 0.5, randn(H, D, seed=3) / H ** 0.5
    bias = randn(H, seed=4) * 0.1
    (q1, s1), (q2, s2) = pf.quantize_s8(w1, axis=0), pf.quantize_s8(w2, axis=0)
    xq, xs = pf.quantize_s8(x)
    h = pf.gemm_s8(xq, q1, xs, s1, bias, gelu=True)
    check_s8(h, xq, q1, xs, s1, bias, True)
    hq, hs = pf.quantize_s8(h)
    want, want_scale = codes64(h, 1)
    assert torch.equal(hq, want) and torch.equal(hs, want_scale)
    y = pf.gemm_s8(hq, q2, hs, s2, dtype=torch.float32)
    check_s8(y, hq, q2, hs, s2, None, False)
    full = gelu64(x.double() @ w1.double() + bias.double()) @ w2.double()
    assert (y.double() - full).norm() < 0.05 * full.norm()  # four operands off by at most half a step of amax / 127


def test_a_trained_layer_captured_and_replayed():
    """Forward and backward as one CUDA graph, replayed on new inputs, equal the eager calls' bits; a second graph of
    other sizes, captured meanwhile and replayed beside it, does not disturb it."""
    def step(a, b, bias, g):
        c, saved = pf.gemm_bias_gelu_checkpoint(a, b, bias)
        return (c, *pf.gemm_bias_gelu_backward(g, b, saved))

    sizes = [(300, 520, 264), (64, 1032, 136)]
    held, graphs, outs = [], [], []
    side = torch.cuda.Stream()
    for M, N, K in sizes:
        held.append([*layer(M, N, K), randn(M, N, seed=9, dtype=torch.bfloat16)])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*held[-1])  # first calls come before a capture
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*held[-1]))
        graphs.append(graph)
    for seed in (100, 200):
        for (M, N, K), ops in zip(sizes, held):
            for t, v in zip(ops, [*layer(M, N, K, seed), randn(M, N, seed=seed + 9, dtype=torch.bfloat16)]):
                t.copy_(v)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for ops, got in zip(held, outs):
            assert all(torch.equal(x, y) for x, y in zip(got, step(*ops)))


def test_a_kernel_captured_at_its_first_use():
    """A capture may be the first call of a size, and so of a kernel, once the device was set up by any other call."""
    import subprocess
    import sys
    code = """
import torch, ptxforge_b200 as pf
x = torch.ones(2, 8, device="cuda")
pf.quantize_s8(x)
torch.cuda.synchronize()
a = torch.randint(-127, 128, (700, 1040), dtype=torch.int8, device="cuda")
b = torch.randint(-127, 128, (1040, 2064), dtype=torch.int8, device="cuda")
s, t = torch.ones(700, device="cuda"), torch.ones(2064, device="cuda")
h, w, bias = torch.randn(333, 264, device="cuda").bfloat16(), torch.randn(264, 520, device="cuda").bfloat16(), torch.randn(520, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    c = pf.gemm_s8(a, b, s, t, dtype=torch.float32)
    d = pf.gemm_s8(a[:3], b, s[:3], t, dtype=torch.float32)
    y, saved = pf.gemm_bias_gelu_checkpoint(h, w, bias)
    grads = pf.gemm_bias_gelu_backward(y, w, saved)
    q = pf.quantize_s8(w, axis=0)
    r = pf.quantize_s8(h[:, 1:], axis=0)   # unaligned: a memset and three kernels
    none = pf.gemm_bias_gelu_backward(y[:0], w, pf.Checkpoint(saved.a_codes[:0], saved.a_scale[:0], saved.grad_codes[:0]))
g.replay()
torch.cuda.synchronize()
assert torch.equal(c, (a.double() @ b.double()).float()) and torch.equal(d, c[:3])
y2, saved2 = pf.gemm_bias_gelu_checkpoint(h, w, bias)
assert torch.equal(y, y2) and all(torch.equal(p, r) for p, r in zip(grads, pf.gemm_bias_gelu_backward(y2, w, saved2)))
assert all(torch.equal(p, t) for p, t in zip((*q, *r), (*pf.quantize_s8(w, axis=0), *pf.quantize_s8(h[:, 1:], axis=0))))
assert not none[1].any() and not none[2].any() and pf.ops8_status() == 0
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_calls_of_two_threads():
    """Two host threads, a stream each, products of the same weights: the library keeps nothing that they could share."""
    import threading
    a, b, bias = layer(300, 1032, 520)
    g = randn(300, 1032, seed=3, dtype=torch.bfloat16)
    c0, saved0 = pf.gemm_bias_gelu_checkpoint(a, b, bias)
    want = (c0, *pf.gemm_bias_gelu_backward(g, b, saved0))
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(30):
                c, saved = pf.gemm_bias_gelu_checkpoint(a, b, bias)
                got = (c, *pf.gemm_bias_gelu_backward(g, b, saved))
                s.synchronize()
                if not all(torch.equal(x, y) for x, y in zip(want, got)):
                    bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_a_stream_of_its_own():
    """Calls on a named stream order their work there, with outputs and workspaces of that stream."""
    s = torch.cuda.Stream()
    a, b, bias = layer(700, 1032, 520)
    g = randn(700, 1032, seed=3, dtype=torch.bfloat16)
    c0, saved0 = pf.gemm_bias_gelu_checkpoint(a, b, bias)
    want = (c0, *pf.gemm_bias_gelu_backward(g, b, saved0))
    s.wait_stream(torch.cuda.current_stream())
    for stream in (s, s.cuda_stream):
        for _ in range(5):
            c, saved = pf.gemm_bias_gelu_checkpoint(a, b, bias, stream=stream)
            got = (c, *pf.gemm_bias_gelu_backward(g, b, saved, stream=stream))
            torch.zeros(1 << 22, device=DEV)  # the current stream takes memory meanwhile
        s.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, got))
    q, sc = pf.quantize_s8(a, stream=s)
    v = pf.dequantize_s8(q, sc, stream=s)
    s.synchronize()
    assert torch.equal(v, saved0.input())


def test_operands_that_do_not_fit_are_refused():
    a, b, bias = layer(16, 24, 32)
    with pytest.raises(pf.PFError) as e:
        pf.gemm_bias_gelu_checkpoint(a[:, :20].contiguous(), b[:20], bias)
    assert e.value.code == pf.PF_ESHAPE
    for bad in (lambda: pf.gemm_bias_gelu_checkpoint(a.t().contiguous().t(), b, bias),
                lambda: pf.gemm_bias_gelu_checkpoint(a[:, :16], b[:16], bias),
                lambda: pf.gemm_bias_gelu_checkpoint(a, b, bias.bfloat16()),
                lambda: pf.gemm_bias_gelu_checkpoint(a, b[:16], bias),
                lambda: pf.quantize_s8(a.t()),
                lambda: pf.quantize_s8(a[:1].expand(4, 32)),
                lambda: pf.quantize_s8(a, scale=torch.zeros(16)),
                lambda: pf.quantize_s8(a, codes=torch.zeros(16, 31, dtype=torch.int8, device=DEV))):
        with pytest.raises(ValueError):
            bad()
    q, s = pf.quantize_s8(a)
    w, t = pf.quantize_s8(b, axis=0)
    for bad in (lambda: pf.gemm_s8(q, w, t, s), lambda: pf.gemm_s8(q, w[:8], s, t), lambda: pf.gemm_s8(q, w.t(), s, t),
                lambda: pf.gemm_s8(q, w, s, t, bias.bfloat16()),
                lambda: pf.gemm_s8(q, w, s, t, C=torch.zeros(16, 24, device=DEV), dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            bad()
    saved = pf.gemm_bias_gelu_checkpoint(a, b, bias)[1]
    g = torch.zeros(16, 24, dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: pf.gemm_bias_gelu_backward(g[:8], b, saved), lambda: pf.gemm_bias_gelu_backward(g, b[:16], saved),
                lambda: pf.gemm_bias_gelu_backward(g, b.t(), saved)):
        with pytest.raises(ValueError):
            bad()

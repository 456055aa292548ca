"""The 8-bit operators at the edges of their ranges and of their kernels' tiles, against their formulas in 64 bits (needs
a B200: -m gpu).  Tolerances count roundings as test_gpu_ops8.py does."""
import ctypes
import threading
import time

import pytest

torch = pytest.importorskip("torch")

import ptxforge_b200 as pf  # noqa: E402
from test_gpu_ops8 import (BF, DEV, F32, check_s8, codes64, gelu64, grad64, grads64, layer, no_wait_ran_out,  # noqa: E402,F401
                           randn, s8_operands, saved_of, within)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------
# sums split over a cluster, whose CTAs read one another's shared memory
# ---------------------------------------------------------------------------------------------
# Counts of tokens that end anywhere in a tile of 16 to 128 and in a warp's look-ahead of up to 16; last channel tiles of 1, 8,
# 40 and 104 channels.  Clusters of 2 (8200 channels), 4 (4104 and 4097) and 8 (1000 and 1001).
TOKENS = (1, 2, 3, 5, 6, 7, 9, 13, 15, 17, 18, 21, 25, 29, 31, 33, 37, 38, 41, 45, 49, 50, 53, 57, 61, 63, 65, 66, 69, 77, 97, 101,
          113, 125, 127, 129, 145, 177, 201, 257, 261, 293)


@pytest.mark.parametrize("N,K", [(1001, 2048), (1000, 4096), (4097, 2048), (4104, 4096), (8200, 4096)])
def test_split_int8_sums_of_any_number_of_tokens(N, K):
    a, b, sa, sb, bias = s8_operands(TOKENS[-1], N, K, seed=N)
    for M in TOKENS:
        c = torch.full((M + 1, N), 7.0, device=DEV)
        pf.gemm_s8(a[:M], b, sa[:M], sb, bias, c[:M])
        check_s8(c[:M], a[:M], b, sa[:M], sb, bias, False)
        assert (c[M] == 7.0).all()
        again = pf.gemm_s8(a[:M], b, sa[:M], sb, bias, dtype=torch.float32)
        assert torch.equal(c[:M], again)


@pytest.mark.parametrize("N,K", [(1000, 2048), (4104, 2048), (8200, 2048)])
def test_split_bf16_sums_of_any_number_of_tokens(N, K):
    a, b, bias = layer(TOKENS[-1], N, K, seed=N)
    z = a.double() @ b.double() + bias.double()
    dz = (K + 3) * 2.0 ** -23 * (a.double().abs() @ b.double().abs() + bias.double().abs())
    y, d = gelu64(z), grad64(z)
    tol = 1.13 * dz + 2.0 ** -20 * (1 + y.abs())
    for M in TOKENS:
        c, saved = pf.gemm_bias_gelu_checkpoint(a[:M], b, bias, keep_input=False)
        within(c, y[:M], tol[:M] + BF * (y[:M].abs() + 1.13 * dz[:M]))
        within(saved.gelu_grad(torch.float32), d[:M], 0.0025 + 1.13 * dz[:M] + 2.0 ** -18)


@pytest.mark.parametrize("N,K", [(2048, 1000), (2048, 4104)])
def test_split_sums_of_gradients_of_any_number_of_tokens(N, K):
    saved = saved_of(TOKENS[-1], N, K, seed=K)
    dc, b = randn(TOKENS[-1], N, seed=5, dtype=torch.bfloat16), randn(K, N, seed=6, dtype=torch.bfloat16)
    dz, _, want, _, _ = grads64(dc, b, saved)
    tol = (BF + (N + 2) * 2.0 ** -23) * (dz.abs() @ b.double().abs().t())
    for M in TOKENS:
        part = pf.Checkpoint(*(t[:M].contiguous() for t in saved))
        for need in (("dA",), ("dA", "dB")):
            got = pf.gemm_bias_gelu_backward(dc[:M], b, part, need=need)[0]
            within(got, want[:M], tol[:M] + BF * (want[:M].abs() + tol[:M]))


# ---------------------------------------------------------------------------------------------
# kernels that start before the one that writes their operands has ended
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,D,H", [(3, 264, 520), (300, 1024, 2056), (2500, 264, 2056), (90, 1001, 777)])
def test_a_chain_through_the_same_buffers_reads_what_the_last_launch_wrote(M, D, H):
    """Codes, scales, bias and results of 40 steps go through one set of buffers with no wait between them; every step gives
    the bits of the same calls made one at a time, with the GPU waited for after each."""
    xs = [randn(M, D, seed=i, dtype=torch.bfloat16) * (1 + i) for i in range(40)]
    w8, sw = pf.quantize_s8(randn(D, H, seed=99), axis=0)
    bias8 = torch.randint(-127, 128, (1, H), dtype=torch.int8, device=DEV)
    q, s = torch.empty(M, D, dtype=torch.int8, device=DEV), torch.empty(M, device=DEV)
    bias, one = torch.empty(1, H, device=DEV), torch.empty(1, device=DEV)
    h = torch.empty(M, H, dtype=torch.bfloat16, device=DEV)
    hq, hs = torch.empty(M, H, dtype=torch.int8, device=DEV), torch.empty(H, device=DEV)
    steps = [torch.full((1,), 0.01 * (1 + i), device=DEV) for i in range(40)]

    def step(i, wait):
        out = torch.empty(M, H, device=DEV)
        for call in (lambda: pf.quantize_s8(xs[i], codes=q, scale=s),
                     lambda: pf.dequantize_s8(bias8, steps[i], out=bias),
                     lambda: pf.gemm_s8(q, w8, s, sw, bias[0], h, gelu=True),
                     lambda: pf.quantize_s8(h, 0, codes=hq, scale=hs),
                     lambda: pf.dequantize_s8(hq, hs, 0, out=out)):
            call()
            if wait:
                torch.cuda.synchronize()
        return out

    want = [step(i, True) for i in range(40)]
    got = [step(i, False) for i in range(40)]
    assert all(torch.equal(x, y) for x, y in zip(want, got))


def test_a_backward_pass_reads_the_checkpoint_that_was_just_written():
    M, N, K = 300, 1032, 520
    a, b, bias = layer(M, N, K)
    xs = [randn(M, K, seed=i, dtype=torch.bfloat16) * (1 + i) for i in range(30)]

    def step(x, wait):
        c, saved = pf.gemm_bias_gelu_checkpoint(x, b, bias)
        if wait:
            torch.cuda.synchronize()
        return (c, *pf.gemm_bias_gelu_backward(c, b, saved))

    want = [step(x, True) for x in xs]
    got = [step(x, False) for x in xs]
    assert all(torch.equal(p, r) for x, y in zip(want, got) for p, r in zip(x, y))


# ---------------------------------------------------------------------------------------------
# values near the ends of their types' ranges
# ---------------------------------------------------------------------------------------------
def check_backward(dc, b, saved):
    """All three gradients within the tolerances of test_gpu_ops8.test_backward."""
    (M, N), K = dc.shape, b.shape[0]
    dz, a, want_a, want_b, want_bias = grads64(dc, b, saved)
    dA, dB, dbias = pf.gemm_bias_gelu_backward(dc, b, saved)
    tol = (BF + (N + 2) * 2.0 ** -23) * (dz.abs() @ b.double().abs().t())
    within(dA, want_a, tol + BF * (want_a.abs() + tol))
    tol = (BF + (M + 3) * 2.0 ** -23) * (a.abs().t() @ dz.abs())
    within(dB, want_b, tol + BF * (want_b.abs() + tol))
    within(dbias, want_bias, (M + 2) * F32 * dz.abs().sum(0))
    plain_a, _, plain_bias = pf.gemm_bias_gelu_backward(dc, b, pf.Checkpoint(None, None, saved.grad_codes), need=("dA", "dbias"))
    tol = (BF + (N + 2) * 2.0 ** -23) * (dz.abs() @ b.double().abs().t())
    within(plain_a, want_a, tol + BF * (want_a.abs() + tol))
    assert torch.equal(plain_bias, dbias)


@pytest.mark.parametrize("M,N,K", [(8, 64, 40), (9, 520, 264)])
def test_backward_of_gradients_near_the_largest(M, N, K):
    """dz = dC d is finite up to bf16's 3.39e38, whatever dC times a code on the way to it would be."""
    saved = saved_of(M, N, K)
    codes = torch.randint(0, 227, (M, N), dtype=torch.uint8, device=DEV, generator=torch.Generator(device=DEV).manual_seed(8))
    codes[:, 1], codes[:, 2], codes[1:, 3] = 226, 0, 252  # d = 1, -0.13 and 1.13
    saved = saved._replace(a_scale=torch.full((M,), 2.0 ** -30, device=DEV), grad_codes=codes)
    dc = randn(M, N, seed=1).clamp(-3, 3) * 3e35
    dc[0] = 3.3e38  # with the others' 8 * 1.02e36 below fp32's 3.40e38: dbias is finite
    dc[0, ::2] *= -1
    b = (randn(K, N, seed=2) * 2.0 ** -30).bfloat16()
    check_backward(dc.bfloat16(), b, saved)


@pytest.mark.parametrize("M,N,K", [(8, 64, 40), (9, 520, 264), (300, 2056, 264)])
@pytest.mark.parametrize("scale", [1.99 * 2.0 ** -30, 1.0, 1.5, 1.99 * 2.0 ** -126, 2.0 ** -126])
def test_backward_of_gradients_near_the_largest_with_any_scale(M, N, K, scale):
    """The input's scale takes no part in dA, and dz near bf16's largest is finite with any of its mantissas."""
    saved = saved_of(M, N, K)
    saved = saved._replace(a_scale=torch.full((M,), scale, device=DEV), grad_codes=torch.full((M, N), 226, dtype=torch.uint8, device=DEV))
    if scale >= 1:  # dB = q s dz stays finite
        saved = saved._replace(a_codes=(saved.a_codes == 127).to(torch.int8))
        saved.a_codes[1:] = 0
    dc = torch.zeros(M, N, device=DEV)
    dc[0] = 3.3e38 / max(scale, 1.0)
    dc[0, ::3] = 1.8e38 / max(scale, 1.0)
    dc[M // 2, 1::4] = -3e38 / max(scale, 1.0)
    b = (randn(K, N, seed=2) * 2.0 ** -30).bfloat16()
    check_backward(dc.bfloat16(), b, saved)


@pytest.mark.parametrize("scale", [1.01 * 2.0 ** -7, 1.0, 1.99])
def test_backward_of_gradients_near_the_smallest(scale):
    """dz and dz times a scale's mantissa keep an absolute half step of bf16's smallest, 2^-134, below its normal range."""
    M, N, K = 40, 136, 72
    saved = saved_of(M, N, K)
    saved = saved._replace(a_scale=torch.full((M,), scale, device=DEV))
    dc = (randn(M, N, seed=1) * 2.0 ** -125).bfloat16()
    b = (randn(K, N, seed=2) * 2.0 ** 30).bfloat16()
    dz, a, want_a, want_b, want_bias = grads64(dc, b, saved)
    dA, dB, dbias = pf.gemm_bias_gelu_backward(dc, b, saved)
    off = BF * dz.abs() + 2.0 ** -133  # a step of 2^-134 of m dz is up to two of dz
    tol = off @ b.double().abs().t() + (N + 2) * 2.0 ** -23 * (dz.abs() @ b.double().abs().t())
    within(dA, want_a, tol + BF * (want_a.abs() + tol))
    tol = a.abs().t() @ off + (M + 3) * 2.0 ** -23 * (a.abs().t() @ dz.abs())
    within(dB, want_b, tol + BF * (want_b.abs() + tol) + 2.0 ** -134)
    within(dbias, want_bias, (M + 2) * F32 * dz.abs().sum(0) + M * 2.0 ** -149)


@pytest.mark.parametrize("M,N,K", [(25, 25, 64), (25, 1025, 2048), (2500, 2050, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_products_of_far_scales(M, N, K, dtype):
    """Scales whose product alone is past fp32's range, times a sum that brings the value back into it (or is 0)."""
    a, b, _, _, _ = s8_operands(M, N, K, seed=N)
    a[:M // 2] = a[:M // 2].clamp(-1, 1)
    a[3] = 0
    each = torch.tensor([2.0 ** -126, 1e-30, 3e-20, 1e-9, 0.7, 1.0, 3e7, 1e18, 1e31, 2.6e36], device=DEV)
    sa, sb = each[torch.arange(M, device=DEV) % 10], each[torch.arange(N, device=DEV) // 10 % 10]
    want = a.double() @ b.double() * sa.double()[:, None] * sb.double()
    c = pf.gemm_s8(a, b, sa, sb, dtype=dtype)
    u = BF if dtype == torch.bfloat16 else 2.0 ** -24
    fits = (want.abs() >= 2.0 ** -126) & (want.abs() < 3.3e38) | (want == 0)
    assert fits.float().mean() > 0.4
    tol = 4 * 2.0 ** -24 * want.abs()
    within(c[fits], want[fits], (tol + u * (want.abs() + tol))[fits])
    # below the smallest normal number an absolute half step and a rounding before it; above the largest, infinity
    small, large = want.abs() < 2.0 ** -126, want.abs() > 3.45e38
    assert ((c.double() - want).abs()[small] <= 2.0 ** -133).all() and torch.isinf(c[large]).all()


@pytest.mark.parametrize("N,K", [(1001, 2048), (2056, 512), (4104, 4096)])
def test_a_token_gets_the_same_bits_in_every_batch(N, K):
    """The integer sums are exact and the rest goes by value: neither the number of tokens, and so the kernel, nor a token's
    place among them moves a bit."""
    a, b, sa, sb, bias = s8_operands(2500, N, K, seed=N)
    sa[::7] *= 1e30
    for gelu in (False, True):
        c = pf.gemm_s8(a, b, sa, sb, bias, gelu=gelu, dtype=torch.float32)
        for first, last in ((0, 1), (3, 4), (1, 18), (5, 45), (2, 131), (700, 1003), (11, 1211), (1, 2500)):
            part = pf.gemm_s8(a[first:last], b, sa[first:last], sb, bias, gelu=gelu, dtype=torch.float32)
            assert torch.equal(part, c[first:last])


# ---------------------------------------------------------------------------------------------
# waits that ran out
# ---------------------------------------------------------------------------------------------
def run_out(stream, ns=1000):
    """One bounded wait on `stream` that nothing ends."""
    text = ctypes.create_string_buffer(256)
    rc = pf.load_library().pf_ops8_selftest_wait_timeout(0, ns, stream.cuda_stream, text, 256)
    assert rc == pf.PF_OK, text.value


def test_a_wait_that_ran_out_is_reported_once():
    run_out(torch.cuda.current_stream())
    assert pf.ops8_status() != 0 and pf.ops8_status() == 0
    q, s = pf.quantize_s8(randn(4, 64))  # the context stays usable
    assert s.numel() == 4 and pf.ops8_status() == 0


def test_no_report_is_lost_beside_a_thread_that_reads_them():
    """A bit set while another thread reads and clears the word is seen by this read or by the next one."""
    seen, stop, s = [], threading.Event(), torch.cuda.Stream()

    def read():
        while not stop.is_set():
            if pf.ops8_status():
                seen.append(1)

    reader = threading.Thread(target=read)
    reader.start()
    try:
        for i in range(500):
            before = len(seen)
            run_out(s)
            s.synchronize()
            limit = time.monotonic() + 1
            while len(seen) == before and time.monotonic() < limit:
                time.sleep(1e-5)
            assert len(seen) > before, f"report {i} was lost"
    finally:
        stop.set()
        reader.join()


# ---------------------------------------------------------------------------------------------
# matrices of more than 2^31 values, and more tokens than a grid's second dimension has tiles
# ---------------------------------------------------------------------------------------------
@pytest.fixture
def large():
    """Memory of large tensors goes back to the device afterwards."""
    yield
    torch.cuda.empty_cache()


def some_rows(rows, cols):
    """The first rows, those around value 2^31, and the last ones."""
    at = 2 ** 31 // cols
    return sorted({0, 1, rows - 2, rows - 1} | {r for r in (at - 1, at, at + 1) if 0 <= r < rows})


@pytest.mark.parametrize("rows,cols", [(65537, 32776), (1048577, 2049)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("axis", [1, 0])
def test_store_past_2_to_the_31_values(rows, cols, dtype, axis, large):
    assert rows * cols > 2 ** 31
    x = torch.empty(rows, cols, dtype=dtype, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    x[rows - 1] *= 2  # the last row has most columns' largest values
    codes, scale = pf.quantize_s8(x, axis)
    back = pf.dequantize_s8(codes, scale, axis, dtype=dtype)
    if axis == 0:
        want_scale = torch.zeros(cols, device=DEV)
        for first in range(0, rows, 16384):
            want_scale = torch.maximum(want_scale, x[first:first + 16384].float().abs().amax(0))
        want_scale = (want_scale.double() / 127).float()
        assert torch.equal(scale, want_scale)
    for r in some_rows(rows, cols):
        if axis == 1:
            want, s = codes64(x[r:r + 1], 1)
            assert torch.equal(scale[r:r + 1], s)
        else:
            s = scale
            want = torch.round(x[r:r + 1].double() / s.double()).to(torch.int8)
        assert torch.equal(codes[r:r + 1], want)
        assert torch.equal(back[r], (want[0].float() * s).to(dtype))


def test_derivatives_past_2_to_the_31(large):
    n = 2 ** 31 + 4333
    codes = torch.zeros(n, dtype=torch.uint8, device=DEV)
    ends = torch.tensor([0, 1, 2 ** 31 - 1, 2 ** 31, 2 ** 31 + 1, n - 4097, n - 2, n - 1], device=DEV)
    codes[ends] = torch.arange(100, 108, dtype=torch.uint8, device=DEV)
    d = pf.dequantize_gelu_grad(codes)
    want = ((torch.arange(100, 108, device=DEV).double() - 26) / 200).float().bfloat16()
    assert torch.equal(d[ends], want)
    assert int((d == torch.tensor(-0.13, device=DEV).bfloat16()).sum()) == n - 8


@pytest.mark.parametrize("M,N,K", [(2 ** 21 + 77, 1032, 16), (2 ** 21 + 77, 1033, 17),  # C past 2^31 values
                                   (65537, 16, 32784),                                  # A past it
                                   (40, 65537 * 16, 2064),                              # B past it
                                   (8388481, 16, 16)])                                  # 65,536 tiles of 128 tokens
def test_product_past_2_to_the_31_values(M, N, K, large):
    a, b, sa, sb, bias = s8_operands(M, N, K, seed=3)
    c = pf.gemm_s8(a, b, sa, sb, bias)
    rows = some_rows(M, min(N, 2 ** 30)) if M > 40 else [0, 17, 39]
    rows = sorted(set(rows) | {M // 2, max(0, M - 300)})
    check_s8(c[rows], a[rows], b, sa[rows], sb, bias, False)


@pytest.mark.parametrize("M,N,K", [(2 ** 21 + 77, 1032, 16), (2 ** 21 + 77, 16, 1032), (8388481, 8, 8)])
def test_a_layer_past_2_to_the_31_values(M, N, K, large):
    a, b, bias = layer(M, N, K, seed=4)
    c, saved = pf.gemm_bias_gelu_checkpoint(a, b, bias)
    rows = sorted(set(some_rows(M, max(N, K))) | {M // 2, M - 300})
    z = a[rows].double() @ b.double() + bias.double()
    dz = (K + 3) * 2.0 ** -23 * (a[rows].double().abs() @ b.double().abs() + bias.double().abs())
    y = gelu64(z)
    within(c[rows], y, 1.13 * dz + 2.0 ** -20 * (1 + y.abs()) + BF * (y.abs() + 1.13 * dz))
    part = pf.Checkpoint(*(t[rows] for t in saved))
    within(part.gelu_grad(torch.float32), grad64(z), 0.0025 + 1.13 * dz + 2.0 ** -18)
    want, want_scale = codes64(a[rows], 1)
    assert torch.equal(part.a_codes, want) and torch.equal(part.a_scale, want_scale)
    # a gradient in these rows alone, so that they are all there is to sum
    dc = torch.zeros_like(c)
    dc[rows] = randn(len(rows), N, seed=5, dtype=torch.bfloat16)
    dA, dB, dbias = pf.gemm_bias_gelu_backward(dc, b, saved)
    dz, x, want_a, want_b, want_bias = grads64(dc[rows], b, part)
    tol = (BF + (N + 2) * 2.0 ** -23) * (dz.abs() @ b.double().abs().t())
    within(dA[rows], want_a, tol + BF * (want_a.abs() + tol))
    tol = (BF + (len(rows) + 3) * 2.0 ** -23) * (x.abs().t() @ dz.abs())  # adding zeros rounds nothing
    within(dB, want_b, tol + BF * (want_b.abs() + tol))
    within(dbias, want_bias, (len(rows) + 2) * F32 * dz.abs().sum(0))
    dA[rows] = 0
    assert not dA.any()


# ---------------------------------------------------------------------------------------------
# results over operands
# ---------------------------------------------------------------------------------------------
def carve(raw, first, dtype, rows, cols, ld=None):
    """A matrix (rows None: a vector) of `dtype` whose memory starts at byte `first` of `raw`, rows `ld` bytes apart."""
    flat = raw[first:first + (raw.numel() - first) // 4 * 4].view(dtype)
    if rows is None:
        return flat[:cols]
    return flat.as_strided((rows, cols), ((ld or cols * flat.element_size()) // flat.element_size(), 1))


I8, U8, BF16, FP32 = torch.int8, torch.uint8, torch.bfloat16, torch.float32


def product_into(v, C, scale_a=8192, scale_b=9216, bias=None):
    """gemm_s8 of A at byte 0 and B at byte 4096 into C."""
    return pf.gemm_s8(v(0, I8, 48, 64), v(4096, I8, 64, 64), v(scale_a, FP32, None, 48), v(scale_b, FP32, None, 64),
                      bias and v(bias, FP32, None, 64), C)


def layer_into(v, C, bias=16384):
    return pf.gemm_bias_gelu_checkpoint(v(0, BF16, 48, 64), v(8192, BF16, 64, 64), v(bias, FP32, None, 64), v(C, BF16, 48, 64))


@pytest.mark.parametrize("call", [
    lambda v: pf.quantize_s8(v(0, BF16, 48, 64), codes=v(0, I8, 48, 64, 128), scale=v(8192, FP32, None, 48)),  # in place
    lambda v: pf.quantize_s8(v(0, BF16, 48, 64), codes=v(64, I8, 48, 64, 128), scale=v(8192, FP32, None, 48)),
    lambda v: pf.quantize_s8(v(0, BF16, 48, 64), codes=v(6080, I8, 48, 64), scale=v(16384, FP32, None, 48)),   # the last row
    lambda v: pf.quantize_s8(v(0, FP32, 48, 64), codes=v(16384, I8, 48, 64), scale=v(12284, FP32, None, 48)),  # the last value
    lambda v: pf.quantize_s8(v(0, FP32, 48, 64, 512), 0, codes=v(252, I8, 48, 64, 512), scale=v(32768, FP32, None, 64)),
    lambda v: pf.quantize_s8(v(0, FP32, 48, 64), codes=v(16384, I8, 48, 64), scale=v(16384 + 3068, FP32, None, 48)),
    lambda v: pf.dequantize_s8(v(0, I8, 48, 64, 128), v(8192, FP32, None, 48), out=v(0, BF16, 48, 64)),        # in place
    lambda v: pf.dequantize_s8(v(0, I8, 48, 64), v(16384, FP32, None, 48), out=v(16384, BF16, 48, 64)),
    lambda v: pf.dequantize_s8(v(0, I8, 1, 64), v(80, FP32, None, 1), out=v(64, BF16, 1, 64)),
    lambda v: product_into(v, v(0, BF16, 48, 64)),
    lambda v: product_into(v, v(4096, BF16, 48, 64, 256)),
    lambda v: product_into(v, v(8380, FP32, 48, 64)),
    lambda v: product_into(v, v(12288, BF16, 48, 64), scale_b=12288),
    lambda v: product_into(v, v(16384, BF16, 48, 64), bias=16384 + 4096),
    lambda v: layer_into(v, 0),
    lambda v: layer_into(v, 8208),
    lambda v: layer_into(v, 16384, bias=16640),
    lambda v: pf.dequantize_gelu_grad(v(0, U8, None, 64), out=v(60, BF16, None, 64)),
])
def test_results_over_operands_are_refused(call):
    raw = torch.zeros(1 << 16, dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        call(lambda *a: carve(raw, *a))


def test_results_beside_operands_are_not():
    """One buffer for all: columns beside one another, a single row between rows, the next byte."""
    raw = torch.zeros(1 << 16, dtype=torch.uint8, device=DEV)
    x = carve(raw, 0, BF16, 48, 64, 256)  # a row: 128 bytes of values, 64 of codes, 64 for others
    x.copy_(randn(48, 64, dtype=BF16))
    x0, (want, want_scale) = x.clone(), codes64(x, 1)
    codes, scale = pf.quantize_s8(x, codes=carve(raw, 128, I8, 48, 64, 256), scale=carve(raw, 47 * 256 + 192, FP32, None, 48))
    assert torch.equal(codes, want) and torch.equal(scale, want_scale) and torch.equal(x, x0)
    one = pf.dequantize_s8(codes[:1, :32], scale[:1], out=carve(raw, 192, BF16, 1, 32))
    assert torch.equal(one, (want[:1, :32].float() * want_scale[0]).to(BF16)) and torch.equal(x, x0) and torch.equal(codes, want)
    a, b, bias = layer(48, 64, 64)
    flat = torch.zeros(4 * 4096, dtype=BF16, device=DEV)
    flat[:112 * 64] = torch.cat([a.flatten(), b.flatten()])
    A, B, C = flat[:48 * 64].view(48, 64), flat[48 * 64:112 * 64].view(64, 64), flat[112 * 64:160 * 64].view(48, 64)
    assert torch.equal(pf.gemm_bias_gelu_checkpoint(A, B, bias, C)[0], pf.gemm_bias_gelu_checkpoint(a, b, bias)[0])

"""Refusals of the 8-bit operators, on the CPU: the C ABI's checks that come before any device is touched, and the Python
view's operand checks, which come before the C ABI."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import ptxforge_b200 as pf  # noqa: E402

LL = ctypes.c_longlong
P = 4096  # stands for a device pointer: never read, the call is refused first


def call(name, *args):
    err = ctypes.create_string_buffer(256)
    rc = getattr(pf.load_library(), name)(*args, err, 256)
    return rc, err.value.decode()


def quantize(src=2, rows=4, cols=8, x=P, ldx=8, axis=1, q=P, ldq=8, s=P):
    return call("pf_quantize_s8", 0, src, rows, cols, x, LL(ldx), axis, q, LL(ldq), s, None)


def dequantize(rows=4, cols=8, q=P, ldq=8, s=P, axis=1, dst=2, x=P, ldx=8):
    return call("pf_dequantize_s8", 0, rows, cols, q, LL(ldq), s, axis, dst, x, LL(ldx), None)


def gemm(M=4, N=8, K=16, a=P, lda=16, b=P, ldb=8, sa=P, sb=P, bias=None, out=2, c=P, ldc=8):
    return call("pf_gemm_s8", 0, M, N, K, a, LL(lda), b, LL(ldb), sa, sb, bias, 0, out, c, LL(ldc), None, 0, None)


def unaligned():
    return call("pf_gemm_s8", 0, 4, 8, 16, P, LL(17), P, LL(16), P, P, None, 0, 2, P, LL(8), P, 100, None)


def forward(M=4, N=8, K=16, a=P, b=P, bias=P, c=P, q=P, s=P, d=P):
    return call("pf_gemm_bias_gelu_checkpoint", 0, M, N, K, a, b, bias, c, q, s, d, None)


@pytest.mark.parametrize("got,code,needle", [
    (lambda: quantize(src=3), pf.PF_EINVAL, "f32 or bf16"),
    (lambda: quantize(rows=-1), pf.PF_EINVAL, "0 to 2^30"),
    (lambda: quantize(rows=(1 << 30) + 1), pf.PF_EINVAL, "0 to 2^30"),
    (lambda: quantize(axis=2), pf.PF_EINVAL, "axis"),
    (lambda: quantize(x=None), pf.PF_EINVAL, "null"),
    (lambda: quantize(s=None), pf.PF_EINVAL, "null"),
    (lambda: quantize(ldx=7), pf.PF_EINVAL, "stride"),
    (lambda: quantize(ldq=7), pf.PF_EINVAL, "stride"),
    (lambda: dequantize(dst=1), pf.PF_EINVAL, "f32 or bf16"),
    (lambda: dequantize(cols=-2), pf.PF_EINVAL, "0 to 2^30"),
    (lambda: dequantize(axis=-1), pf.PF_EINVAL, "axis"),
    (lambda: dequantize(q=None), pf.PF_EINVAL, "null"),
    (lambda: dequantize(ldx=3), pf.PF_EINVAL, "stride"),
    (lambda: gemm(M=-1), pf.PF_EINVAL, "0 to 2^30"),
    (lambda: gemm(K=0), pf.PF_EINVAL, "K must be"),
    (lambda: gemm(K=131072, lda=131072), pf.PF_EINVAL, "131071"),
    (lambda: gemm(out=0 + 1), pf.PF_EINVAL, "f32 or bf16"),
    (lambda: gemm(lda=15), pf.PF_EINVAL, "stride"),
    (lambda: gemm(ldb=7), pf.PF_EINVAL, "stride"),
    (lambda: gemm(ldc=7), pf.PF_EINVAL, "stride"),
    (lambda: gemm(sb=None), pf.PF_EINVAL, "null"),
    (lambda: gemm(), pf.PF_EINVAL, "workspace"),         # rows of B are 8 bytes
    (lambda: unaligned(), pf.PF_EINVAL, "workspace holds 100 bytes"),
    (lambda: forward(N=0), pf.PF_EINVAL, "1 to 2^30"),
    (lambda: forward(M=2 ** 31 - 1), pf.PF_EINVAL, "0 to 2^30"),
    (lambda: forward(N=12), pf.PF_ESHAPE, "16 bytes"),
    (lambda: forward(K=20), pf.PF_ESHAPE, "16 bytes"),
    (lambda: forward(d=None), pf.PF_EINVAL, "null"),
    (lambda: forward(s=None), pf.PF_EINVAL, "together"),
    (lambda: forward(c=P + 8), pf.PF_EINVAL, "aligned"),
    (lambda: call("pf_dequantize_gelu_grad", 0, LL(-1), P, 2, P, None), pf.PF_EINVAL, "negative"),
    (lambda: call("pf_dequantize_gelu_grad", 0, LL(1), None, 2, P, None), pf.PF_EINVAL, "null"),
    (lambda: call("pf_ops8_status", 0, None), pf.PF_EINVAL, "null"),
])
def test_c_abi_refusals(got, code, needle):
    rc, text = got()
    assert rc == code and needle in text, (rc, text)


def test_no_rows_is_no_work():
    assert quantize(rows=0)[0] == dequantize(rows=0)[0] == gemm(M=0)[0] == gemm(N=0)[0] == forward(M=0)[0] == pf.PF_OK
    assert call("pf_dequantize_gelu_grad", 0, LL(0), None, 2, None, None)[0] == pf.PF_OK


def test_without_a_gpu_every_call_reports_it():
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    word = ctypes.c_uint()
    for rc, _ in (quantize(), dequantize(), gemm(ldb=16), forward(), call("pf_ops8_status", 0, ctypes.byref(word)),
                  call("pf_dequantize_gelu_grad", 0, LL(1), P, 2, P, None),
                  call("pf_gemm_bias_gelu_backward", 0, 4, 8, 16, P, P, P, P, P, P, P, P, P, 1 << 20, None)):
        assert rc == pf.PF_ENODEV


def test_product_workspace():
    size = pf.load_library().pf_gemm_s8_workspace
    args = lambda M, N, K, a, lda, b, ldb: (M, N, K, a, LL(lda), b, LL(ldb))  # noqa: E731
    assert size(*args(4, 32, 16, P, 16, P, 32)) == 0
    assert size(*args(1, 32, 17, P, 17, P, 32)) == 0                 # one row has no stride
    assert size(*args(4, 32, 17, P, 17, P, 32)) == 256               # A: 4 rows of 32 bytes
    assert size(*args(4, 33, 16, P, 16, P, 33)) == 768               # B: 16 rows of 48 bytes
    assert size(*args(4, 33, 17, P + 1, 32, P, 33)) == 256 + 1024    # both; B: 17 rows of 48 bytes
    assert size(*args(1 << 20, 32, 100001, P, 100001, P, 32)) >= (1 << 20) * 100001  # past 32 bits


def test_backward_workspace():
    size = pf.load_library().pf_gemm_bias_gelu_backward_workspace
    assert size(0, 8, 8) == size(8, 0, 8) == size(-1, 8, 8) == 0
    # at least dz and the input in bf16
    assert size(100, 64, 32) >= 100 * 64 * 2 + 100 * 32 * 2
    assert size(2 ** 20, 2 ** 14, 2 ** 13) >= 2 ** 20 * (2 ** 14 + 2 ** 13) * 2  # past 32 bits


@pytest.mark.parametrize("call,needle", [
    (lambda: pf.quantize_s8(torch.zeros(2, 4)), "CUDA tensor"),
    (lambda: pf.quantize_s8(torch.zeros(2, 4, dtype=torch.float16)), "bfloat16 or torch.float32"),
    (lambda: pf.quantize_s8(torch.zeros(8)), "matrix"),
    (lambda: pf.dequantize_s8(torch.zeros(2, 4), torch.zeros(2)), "int8"),
    (lambda: pf.gemm_s8(torch.zeros(2, 4), torch.zeros(4, 2), torch.zeros(2), torch.zeros(2)), "int8"),
    (lambda: pf.gemm_s8(torch.zeros(2, 4, dtype=torch.int8), torch.zeros(4, 2), torch.zeros(2), torch.zeros(2)), "CUDA tensor"),
    (lambda: pf.gemm_bias_gelu_checkpoint(torch.zeros(8, 8), torch.zeros(8, 8), torch.zeros(8)), "bfloat16"),
    (lambda: pf.gemm_bias_gelu_backward(torch.zeros(8, 8), torch.zeros(8, 8), pf.Checkpoint(None, None, torch.zeros(8, 8))), "bfloat16"),
    (lambda: pf.gemm_bias_gelu_backward(torch.zeros(8, 8), None, None, need=("dA", "dW")), "dW"),
    (lambda: pf.dequantize_gelu_grad(torch.zeros(8)), "uint8"),
    (lambda: pf.dequantize_gelu_grad(torch.zeros(8, dtype=torch.uint8)), "CUDA tensor"),
])
def test_operands_that_do_not_fit_are_refused_before_any_launch(call, needle):
    with pytest.raises(ValueError, match=needle):
        call()

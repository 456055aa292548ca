"""The 8-bit operators of include/pf_b200.h on CUDA torch tensors.

Serving: weights and activations as int8 codes, a scale for each channel and each token.

    B8, sb = pf.quantize_s8(B, axis=0)                       # once, when the weights are loaded
    A8, sa = pf.quantize_s8(A)                               # a scale for each token
    C = pf.gemm_s8(A8, B8, sa, sb, bias, gelu=True)

Training: the bf16 fused product with its activations kept in 8 bits for the backward pass.

    C, saved = pf.gemm_bias_gelu_checkpoint(A, B, bias)
    dA, dB, dbias = pf.gemm_bias_gelu_backward(dC, B, saved)

Matrices have contiguous rows; a row stride above the row's length is fine where a function says so.  Operands that
do not fit raise ValueError before anything is launched, what the library refuses raises PFError.  Work goes on
`stream`, by default torch's current stream of the operands' device; outputs and workspaces that a call makes are
allocated on that stream.  Calls do not wait for the GPU: ops8_status() says whether a bounded device wait ran out.
"""
from __future__ import annotations

import ctypes
import threading
from typing import NamedTuple

import ptxforge_b200 as _pf

_F32, _BF16 = 0, 2  # pf_dtype
_ERR_BYTES = 256
_local = threading.local()  # each thread's error text
_functions = {}  # the library's entry points by name
torch = None  # imported by the first call: the package loads without it
_raw_stream = None  # torch's current stream of a device index, as a handle


def _need_torch():
    global torch, _raw_stream
    if torch is None:
        import torch as t
        # the handle without a Stream object around it, where torch has that: 2 us less a call
        _raw_stream = getattr(t._C, "_cuda_getCurrentRawStream", None) or (lambda i: t.cuda.current_stream(i).cuda_stream)
        torch = t


def _type_code(dtype, what: str) -> int:
    if dtype is torch.bfloat16:
        return _BF16
    if dtype is torch.float32:
        return _F32
    raise ValueError(f"{what} must be torch.bfloat16 or torch.float32, got {dtype}")


def _matrix(x, name: str, dtype=None, shape=None, device=None, contiguous: bool = False):
    """(rows, cols, row stride) of a CUDA matrix with contiguous rows, or ValueError."""
    size = x.shape
    if len(size) != 2:
        raise ValueError(f"{name} must be a matrix, got {tuple(size)}")
    _check(x, name, dtype, shape, device)
    rows, cols = size
    if x.is_contiguous():
        return rows, cols, cols
    ld, step = x.stride()
    if contiguous or (step != 1 and cols > 1) or ld < cols:
        raise ValueError(f"{name} must be contiguous" + ("" if contiguous else " along its rows, which must not overlap")
                         + f", got strides {x.stride()}")
    return rows, cols, ld


def _vector(x, name: str, n: int, device):
    _check(x, name, torch.float32, (n,), device)
    if not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _check(x, name, dtype, shape, device):
    """`device`: the index of the other operands' device, None for the first."""
    if dtype is not None and x.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {x.dtype}")
    if shape is not None and x.shape != shape:
        raise ValueError(f"{name} must be {' x '.join(map(str, shape))}, got {tuple(x.shape)}")
    at = x.get_device()
    if at < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    if device is not None and at != device:
        raise ValueError(f"{name} is on cuda:{at}, other operands on cuda:{device}")


def _on(stream, device):
    """(the stream's handle, the stream on which torch is to allocate, None for the current one)."""
    if stream is None:
        return _raw_stream(device), None
    handle = _pf._stream(stream)
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)
    return handle, stream


def _empty(on, dtype, device, *size):
    if on is None:
        return torch.empty(*size, dtype=dtype, device=device)
    with torch.cuda.stream(on):
        return torch.empty(*size, dtype=dtype, device=device)


def _call(name: str, *args):
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(_pf.load_library(), name)
    err = getattr(_local, "err", None)
    if err is None:
        err = _local.err = ctypes.create_string_buffer(_ERR_BYTES)
    rc = fn(*args, err, _ERR_BYTES)
    if rc:
        raise _pf.PFError(rc, f"{name}: {err.value.decode()}")


def _axis(axis: int, rows: int, cols: int) -> int:
    if axis not in (0, 1):
        raise ValueError(f"axis must be 1 (a scale for each row) or 0 (for each column), got {axis!r}")
    return rows if axis else cols


def quantize_s8(X, axis: int = 1, codes=None, scale=None, *, stream=None):
    """(codes, scale) of a bfloat16 or float32 matrix: int8 codes rint(x / scale) in [-127, 127] and float32 scales
    max(max |x| / 127, 2**-126), one for each row (axis 1, a token) or column (axis 0, a channel).

    A row (column) with an infinity or NaN gets the scale NaN and codes 0.  Row strides are free."""
    _need_torch()
    src = _type_code(X.dtype, "X")
    rows, cols, ldx = _matrix(X, "X")
    n = _axis(axis, rows, cols)
    dev = X.get_device()
    handle, on = _on(stream, dev)
    if codes is None:
        codes = _empty(on, torch.int8, X.device, rows, cols)
    if scale is None:
        scale = _empty(on, torch.float32, X.device, n)
    ldq = _matrix(codes, "codes", torch.int8, (rows, cols), dev)[2]
    _vector(scale, "scale", n, dev)
    _call("pf_quantize_s8", dev, src, rows, cols, X.data_ptr(), ldx, axis, codes.data_ptr(), ldq,
          scale.data_ptr(), handle)
    return codes, scale


def dequantize_s8(codes, scale, axis: int = 1, out=None, *, dtype=None, stream=None):
    """The values codes * scale stand for, in `dtype` (that of `out`, else bfloat16).  Row strides are free."""
    _need_torch()
    rows, cols, ldq = _matrix(codes, "codes", torch.int8)
    dev = codes.get_device()
    _vector(scale, "scale", _axis(axis, rows, cols), dev)
    dtype = dtype or (out.dtype if out is not None else torch.bfloat16)
    dst = _type_code(dtype, "dtype")
    handle, on = _on(stream, dev)
    if out is None:
        out = _empty(on, dtype, codes.device, rows, cols)
    ldx = _matrix(out, "out", dtype, (rows, cols), dev)[2]
    _call("pf_dequantize_s8", dev, rows, cols, codes.data_ptr(), ldq, scale.data_ptr(), axis, dst,
          out.data_ptr(), ldx, handle)
    return out


def gemm_s8(A, B, scale_a, scale_b, bias=None, C=None, *, gelu: bool = False, dtype=None, stream=None):
    """C = f(scale_a[:, None] * scale_b * (A @ B) + bias), A [M, K] and B [K, N] int8 codes, scale_a float32 [M] (a
    scale for each token), scale_b float32 [N] (for each channel), bias float32 [N] or None; f is GELU's tanh form with
    gelu=True, else the identity.  `dtype` of C: bfloat16 (default) or float32.  The integer sums are exact; K is at
    most 131071.  Any M, N, K; row strides are free."""
    _need_torch()
    M, K, lda = _matrix(A, "A", torch.int8)
    dev = A.get_device()
    K2, N, ldb = _matrix(B, "B", torch.int8, None, dev)
    if K2 != K:
        raise ValueError(f"shape mismatch: A {tuple(A.shape)}, B {tuple(B.shape)}")
    _vector(scale_a, "scale_a", M, dev)
    _vector(scale_b, "scale_b", N, dev)
    if bias is not None:
        _vector(bias, "bias", N, dev)
    dtype = dtype or (C.dtype if C is not None else torch.bfloat16)
    out = _type_code(dtype, "dtype")
    handle, on = _on(stream, dev)
    if C is None:
        C = _empty(on, dtype, A.device, M, N)
    ldc = _matrix(C, "C", dtype, (M, N), dev)[2]
    a, b, space = A.data_ptr(), B.data_ptr(), None
    size = _pf.load_library().pf_gemm_s8_workspace(M, N, K, a, lda, b, ldb)  # 0 where rows start on 16-byte boundaries
    if size:
        space = _empty(on, torch.uint8, A.device, size)  # back to the stream's pool on return
    _call("pf_gemm_s8", dev, M, N, K, a, lda, b, ldb, scale_a.data_ptr(), scale_b.data_ptr(),
          None if bias is None else bias.data_ptr(), int(gelu), out, C.data_ptr(), ldc,
          None if space is None else space.data_ptr(), size, handle)
    return C


class Checkpoint(NamedTuple):
    """What gemm_bias_gelu_backward needs of a forward pass, M K + M N bytes and a float for each token: the input's
    codes and scales (None where dB is not wanted), and the GELU derivative's codes rint(200 d) + 26 (255: NaN)."""
    a_codes: object     # int8 [M, K]
    a_scale: object     # float32 [M]
    grad_codes: object  # uint8 [M, N]

    def input(self, dtype=None):
        """The input as the backward pass sees it, in `dtype` (default bfloat16)."""
        return dequantize_s8(self.a_codes, self.a_scale, dtype=dtype)

    def gelu_grad(self, dtype=None):
        """The GELU's derivative as the backward pass sees it, in `dtype` (default bfloat16)."""
        return dequantize_gelu_grad(self.grad_codes, dtype=dtype)


def gemm_bias_gelu_checkpoint(A, B, bias, C=None, *, keep_input: bool = True, stream=None):
    """(C, checkpoint): C = gelu_tanh(A @ B + bias) in bfloat16, for bfloat16 A [M, K] and B [K, N] and float32 bias [N],
    and in 8 bits what gemm_bias_gelu_backward needs.  keep_input=False leaves the input out (no dB then).  Operands
    contiguous, N and K multiples of 8."""
    _need_torch()
    M, K, _ = _matrix(A, "A", torch.bfloat16, contiguous=True)
    dev = A.get_device()
    K2, N, _ = _matrix(B, "B", torch.bfloat16, None, dev, contiguous=True)
    if K2 != K:
        raise ValueError(f"shape mismatch: A {tuple(A.shape)}, B {tuple(B.shape)}")
    _vector(bias, "bias", N, dev)
    handle, on = _on(stream, dev)
    if C is None:
        C = _empty(on, torch.bfloat16, A.device, M, N)
    grad_codes = _empty(on, torch.uint8, A.device, M, N)
    a_codes = _empty(on, torch.int8, A.device, M, K) if keep_input else None
    a_scale = _empty(on, torch.float32, A.device, M) if keep_input else None
    _matrix(C, "C", torch.bfloat16, (M, N), dev, contiguous=True)
    _call("pf_gemm_bias_gelu_checkpoint", dev, M, N, K, A.data_ptr(), B.data_ptr(), bias.data_ptr(), C.data_ptr(),
          a_codes.data_ptr() if keep_input else None, a_scale.data_ptr() if keep_input else None, grad_codes.data_ptr(),
          handle)
    return C, Checkpoint(a_codes, a_scale, grad_codes)


def gemm_bias_gelu_backward(dC, B, checkpoint: Checkpoint, *, need=("dA", "dB", "dbias"), stream=None):
    """(dA, dB, dbias) of C = gelu_tanh(A @ B + bias) from dC [M, N] (bfloat16), B and the forward pass's checkpoint:
    bfloat16 [M, K] and [K, N], float32 [N]; None for those that `need` leaves out.  Sums are in float32, in an order
    that depends on the sizes alone."""
    _need_torch()
    unknown = set(need) - {"dA", "dB", "dbias"}
    if unknown:
        raise ValueError(f"need names dA, dB and dbias, got {sorted(unknown)}")
    M, N, _ = _matrix(dC, "dC", torch.bfloat16, contiguous=True)
    dev = dC.get_device()
    K, _, _ = _matrix(B, "B", torch.bfloat16, (B.shape[0], N), dev, contiguous=True)
    _matrix(checkpoint.grad_codes, "checkpoint.grad_codes", torch.uint8, (M, N), dev, contiguous=True)
    a, s = None, None
    if "dB" in need:
        if checkpoint.a_codes is None:
            raise ValueError("dB needs the input: the checkpoint was made with keep_input=False")
        _matrix(checkpoint.a_codes, "checkpoint.a_codes", torch.int8, (M, K), dev, contiguous=True)
        _vector(checkpoint.a_scale, "checkpoint.a_scale", M, dev)
        a, s = checkpoint.a_codes.data_ptr(), checkpoint.a_scale.data_ptr()
    handle, on = _on(stream, dev)
    size = _pf.load_library().pf_gemm_bias_gelu_backward_workspace(M, N, K)
    dA = _empty(on, torch.bfloat16, dC.device, M, K) if "dA" in need else None
    dB = _empty(on, torch.bfloat16, dC.device, K, N) if "dB" in need else None
    dbias = _empty(on, torch.float32, dC.device, N) if "dbias" in need else None
    space = _empty(on, torch.uint8, dC.device, size)  # back to the stream's pool on return
    _call("pf_gemm_bias_gelu_backward", dev, M, N, K, dC.data_ptr(), B.data_ptr(), a, s,
          checkpoint.grad_codes.data_ptr(), None if dA is None else dA.data_ptr(), None if dB is None else dB.data_ptr(),
          None if dbias is None else dbias.data_ptr(), space.data_ptr(), size, handle)
    return dA, dB, dbias


def dequantize_gelu_grad(codes, out=None, *, dtype=None, stream=None):
    """The GELU derivatives (code - 26) / 200 that uint8 codes stand for (NaN for 255), in `dtype` (default bfloat16)."""
    _need_torch()
    _check(codes, "codes", torch.uint8, None, None)
    if not codes.is_contiguous():
        raise ValueError("codes must be contiguous")
    dev = codes.get_device()
    dtype = dtype or (out.dtype if out is not None else torch.bfloat16)
    dst = _type_code(dtype, "dtype")
    handle, on = _on(stream, dev)
    if out is None:
        out = _empty(on, dtype, codes.device, *codes.shape)
    _check(out, "out", dtype, codes.shape, dev)
    if not out.is_contiguous():
        raise ValueError("out must be contiguous")
    _call("pf_dequantize_gelu_grad", dev, codes.numel(), codes.data_ptr(), dst, out.data_ptr(), handle)
    return out


def ops8_status(device: int = 0) -> int:
    """Waits for the device, then reads and clears the bits of bounded waits that ran out in these operators (0: none)."""
    word = ctypes.c_uint()
    _call("pf_ops8_status", device, ctypes.byref(word))
    return word.value

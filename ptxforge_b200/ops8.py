"""The 8-bit operators of include/pf_b200.h on CUDA torch tensors.

Serving: weights and activations as int8 codes, a scale for each channel and each token.

    B8, sb = pf.quantize_s8(B, axis=0)                       # once, when the weights are loaded
    A8, sa = pf.quantize_s8(A)                               # a scale for each token
    C = pf.gemm_s8(A8, B8, sa, sb, bias, gelu=True)

Training: the bf16 fused product with its activations kept in 8 bits for the backward pass.

    C, saved = pf.gemm_bias_gelu_checkpoint(A, B, bias)
    dA, dB, dbias = pf.gemm_bias_gelu_backward(dC, B, saved)

Matrices have contiguous rows; a row stride above the row's length is fine where a function says so.  Results that a
caller passes must not overlap an operand.  Operands that do not fit raise ValueError before anything is launched, what the
library refuses raises PFError.  Work goes on `stream` (a torch stream or a handle), by default torch's current stream of
the operands' device; outputs and workspaces that a call makes are allocated on that stream, and operands of another
stream have to live until it has used them (Tensor.record_stream), as with torch's own functions.  Calls do not wait for
the GPU: ops8_status() says whether a bounded device wait ran out.  The checks and calls themselves are compiled
(csrc/torch_ops8.cpp).
"""
from __future__ import annotations

import re
from typing import NamedTuple

import ptxforge_b200 as _pf

_module = None


def _ops():
    """The compiled side, loaded by the first call (the package itself loads without torch)."""
    global _module
    if _module is None:
        import torch  # its libraries come first
        try:
            from . import _ops8
        except ImportError as e:
            raise RuntimeError(f"ptxforge_b200/_ops8.so cannot be loaded ({e}): build it with `python -m ptxforge_b200.build`") from e
        if re.match(r"\d+\.\d+\.\d+", torch.__version__)[0] != _ops8.torch_version:
            raise RuntimeError(f"ptxforge_b200/_ops8.so was built for torch {_ops8.torch_version}, this is {torch.__version__}: "
                               "build it again with `python -m ptxforge_b200.build`")
        _module = _ops8
    return _module


def _handle(stream):
    return None if stream is None else _pf._stream(stream)


def quantize_s8(X, axis: int = 1, codes=None, scale=None, *, stream=None):
    """(codes, scale) of a bfloat16 or float32 matrix: int8 codes rint(x / scale) in [-127, 127] and float32 scales
    max(max |x| / 127, 2**-126), one for each row (axis 1, a token) or column (axis 0, a channel).

    A row (column) with an infinity or NaN gets the scale NaN and codes 0.  Row strides are free."""
    return _ops().quantize_s8(X, axis, codes, scale, _handle(stream))


def dequantize_s8(codes, scale, axis: int = 1, out=None, *, dtype=None, stream=None):
    """The values codes * scale stand for, in `dtype` (that of `out`, else bfloat16).  Row strides are free."""
    return _ops().dequantize_s8(codes, scale, axis, out, dtype, _handle(stream))


def gemm_s8(A, B, scale_a, scale_b, bias=None, C=None, *, gelu: bool = False, dtype=None, stream=None):
    """C = f(scale_a[:, None] * scale_b * (A @ B) + bias), A [M, K] and B [K, N] int8 codes, scale_a float32 [M] (a
    scale for each token), scale_b float32 [N] (for each channel), bias float32 [N] or None; f is GELU's tanh form with
    gelu=True, else the identity.  `dtype` of C: bfloat16 (default) or float32.  The integer sums are exact, for
    which K is 1 to 131071.  M and N are free, and so are row strides."""
    return _ops().gemm_s8(A, B, scale_a, scale_b, bias, C, gelu, dtype, _handle(stream))


class Checkpoint(NamedTuple):
    """What gemm_bias_gelu_backward needs of a forward pass, M K + M N bytes and a float for each token: the input's
    codes and scales (None where dB is not wanted), and the GELU derivative's codes rint(200 d) + 26 (255: NaN)."""
    a_codes: object     # int8 [M, K]
    a_scale: object     # float32 [M]
    grad_codes: object  # uint8 [M, N]

    def input(self, dtype=None):
        """The input as the backward pass sees it, in `dtype` (default bfloat16), on torch's current stream."""
        if self.a_codes is None:
            raise ValueError("the checkpoint was made with keep_input=False: it has no input")
        return dequantize_s8(self.a_codes, self.a_scale, dtype=dtype)

    def gelu_grad(self, dtype=None):
        """The GELU's derivative as the backward pass sees it, in `dtype` (default bfloat16), on torch's current stream."""
        return dequantize_gelu_grad(self.grad_codes, dtype=dtype)


def gemm_bias_gelu_checkpoint(A, B, bias, C=None, *, keep_input: bool = True, stream=None):
    """(C, checkpoint): C = gelu_tanh(A @ B + bias) in bfloat16, for bfloat16 A [M, K] and B [K, N] and float32 bias [N],
    and in 8 bits what gemm_bias_gelu_backward needs.  keep_input=False leaves the input out (no dB then).  Operands
    contiguous and 16-byte aligned, N and K multiples of 8."""
    C, a_codes, a_scale, grad_codes = _ops().gemm_bias_gelu_checkpoint(A, B, bias, C, keep_input, _handle(stream))
    return C, Checkpoint(a_codes, a_scale, grad_codes)


def gemm_bias_gelu_backward(dC, B, checkpoint: Checkpoint, *, need=("dA", "dB", "dbias"), stream=None):
    """(dA, dB, dbias) of C = gelu_tanh(A @ B + bias) from dC [M, N] (bfloat16), B and the forward pass's checkpoint:
    bfloat16 [M, K] and [K, N], float32 [N]; None for those that `need` leaves out.  Sums are in float32, in an order
    that depends on the sizes and on `need` alone.  Operands contiguous."""
    unknown = set(need) - {"dA", "dB", "dbias"}
    if unknown:
        raise ValueError(f"need names dA, dB and dbias, got {sorted(unknown)}")
    return _ops().gemm_bias_gelu_backward(dC, B, *checkpoint, "dA" in need, "dB" in need, "dbias" in need, _handle(stream))


def dequantize_gelu_grad(codes, out=None, *, dtype=None, stream=None):
    """The GELU derivatives (code - 26) / 200 that uint8 codes stand for (NaN for 255), in `dtype` (default bfloat16)."""
    return _ops().dequantize_gelu_grad(codes, out, dtype, _handle(stream))


def ops8_status(device: int = 0) -> int:
    """Waits for the device, then reads and clears the bits of bounded waits that ran out in these operators (0: none)."""
    return _ops().ops8_status(device)

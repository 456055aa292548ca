"""The 8-bit operators at the edges of their ranges and of their kernels' tiles, against their formulas in 64 bits (needs
a B200: -m gpu).  Tolerances count roundings as test_gpu_ops8.py does."""
import pytest

torch = pytest.importorskip("torch")

import ptxforge_b200 as pf  # noqa: E402
from test_gpu_ops8 import (BF, DEV, F32, check_s8, gelu64, grad64, grads64, layer, no_wait_ran_out,  # noqa: E402,F401
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

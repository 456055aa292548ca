"""The 8-bit operators, what the CPU can show of them beyond test_ops8.py's refusals: rules that their sources keep, the
build of their torch side, and the checkpoint's own checks."""
import ctypes
import os
import re

import pytest

torch = pytest.importorskip("torch")

from ptxforge_b200 import build as pbuild  # noqa: E402


def code_of(name):
    """A CUDA source without its comments."""
    text = open(os.path.join(pbuild.CSRC, name)).read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


@pytest.mark.parametrize("name", ["ops8.cu", "ops8_epilogue.cuh", "quant_s8.cuh", "gemm8_tc.cuh"])
def test_kernels_that_start_early_read_by_coherent_loads(name):
    """A kernel that may start before its producer has ended must not read what that wrote through the read-only path,
    which asks for data that nobody writes while the kernel lives."""
    assert not re.findall(r"__ldg\w*\s*\(|ld\.global\.(?:\w+\.)*nc\b|__restrict__", code_of(name))


def test_selftest_of_the_waits_refuses_what_is_not_bounded():
    import ptxforge_b200 as pf
    for ns in (0, 10 ** 10 + 1):
        text = ctypes.create_string_buffer(256)
        assert pf.load_library().pf_ops8_selftest_wait_timeout(0, ns, None, text, 256) == pf.PF_EINVAL and b"timeout_ns" in text.value

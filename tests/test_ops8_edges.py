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


# ---------------------------------------------------------------------------------------------
# the build of the torch side
# ---------------------------------------------------------------------------------------------
@pytest.fixture
def torch_build(monkeypatch, tmp_path):
    """build_torch with its outputs in a folder of their own; the commands that it would run, which do nothing."""
    commands = []

    def run(cmd):
        commands.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return ""

    monkeypatch.setattr(pbuild, "_run", run)
    monkeypatch.setattr(pbuild, "TORCH_LIB", str(tmp_path / "_ops8.so"))
    monkeypatch.setattr(pbuild, "OBJ_DIR", str(tmp_path))
    return commands


def test_the_library_builds_beside_a_torch_without_cuda(torch_build, monkeypatch, capsys):
    monkeypatch.setattr(torch.version, "cuda", None)
    assert pbuild.build_torch() is None and not torch_build
    assert "CUDA" in capsys.readouterr().err


def test_the_library_builds_without_a_host_compiler_for_torch(torch_build, monkeypatch, capsys):
    which = pbuild.shutil.which
    monkeypatch.setattr(pbuild.shutil, "which", lambda name, *a, **k: None if name == "g++" else which(name, *a, **k))
    assert pbuild.build_torch() is None and not torch_build
    assert "g++" in capsys.readouterr().err


def test_the_torch_side_is_built_again_for_another_torch_or_python(torch_build, monkeypatch):
    assert pbuild.build_torch() and len(torch_build) == 1
    assert pbuild.build_torch() and len(torch_build) == 1  # nothing changed
    monkeypatch.setattr(torch, "__version__", "9.8.7+cu999")
    assert pbuild.build_torch() and len(torch_build) == 2
    assert pbuild.build_torch() and len(torch_build) == 2
    var = pbuild.sysconfig.get_config_var
    monkeypatch.setattr(pbuild.sysconfig, "get_config_var", lambda name: "cpython-399" if name == "SOABI" else var(name))
    assert pbuild.build_torch() and len(torch_build) == 3


def test_a_torch_side_of_another_torch_is_refused(monkeypatch):
    from ptxforge_b200 import ops8
    monkeypatch.setattr(ops8, "_module", None)
    monkeypatch.setattr(torch, "__version__", "9.8.7+cu999")
    with pytest.raises(RuntimeError, match="9.8.7.*ptxforge_b200.build"):
        ops8.quantize_s8(torch.zeros(2, 4))
    monkeypatch.undo()
    monkeypatch.setattr(ops8, "_module", None)
    monkeypatch.setattr(torch, "__version__", re.match(r"[\d.]+", torch.__version__)[0] + "a0+git123")
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops8.quantize_s8(torch.zeros(2, 4))


def test_a_checkpoint_without_its_input_says_so():
    import ptxforge_b200 as pf
    with pytest.raises(ValueError, match="keep_input=False"):
        pf.Checkpoint(None, None, torch.zeros(4, 8, dtype=torch.uint8)).input()


# ---------------------------------------------------------------------------------------------
# registers of the CTA-pair kernels, as ptxas reports them
# ---------------------------------------------------------------------------------------------
def test_pair_kernels_fit_one_cta_per_sm():
    pbuild.build()
    log = os.path.join(os.path.dirname(pbuild.LIB), "libpf_b200.ptxas.txt")
    if not os.path.exists(log):
        pytest.skip("no ptxas report beside the library")
    seen = []
    for name, regs in re.findall(r"Function properties for (\S*gemm8_pair\S*)\n.*?Used (\d+) registers", open(log).read(), re.S):
        warps = 2 + int(re.search(r"gemm8_pairILi\d+ELi(\d+)E", name)[1])  # producer, MMA and the epilogue warps
        seen.append(warps)
        assert -(-int(regs) * 32 // 512) * 512 * warps <= 65536, (name, regs, warps)  # registers come in blocks of 512 a warp
    assert set(seen) == {10, 18} and len(seen) >= 10

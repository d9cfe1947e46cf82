"""Which build of the layer's torch side a process takes: the present one, or none."""
import pytest

from nsa_from_scratch_b200 import _lib as L, build


@pytest.fixture
def fresh(monkeypatch):
    L.torch_ops()
    monkeypatch.setattr(L, "_torch_ops", None)
    return monkeypatch


def test_source_that_does_not_compile_is_an_error(fresh):
    """A module from before the change lies there; it is not what the sources say."""
    def broken():
        raise RuntimeError("nvcc failed on torch_ops.cpp")
    fresh.setattr(build, "build_torch", broken)
    with pytest.raises(RuntimeError, match="torch_ops.cpp"):
        L.torch_ops()
    assert L._torch_ops is None


def test_machine_without_a_compiler_takes_what_was_built(fresh):
    def none():
        raise build.NoCompiler("nvcc not found; set NVCC")
    fresh.setattr(build, "build_torch", none)
    assert L.torch_ops().abi_version == L.ABI_VERSION
    fresh.setattr(L, "_torch_ops", None)
    fresh.setattr(build, "TORCH_LIB", build.TORCH_LIB + ".missing")
    with pytest.raises(build.NoCompiler):
        L.torch_ops()


def test_no_compiler_is_what_is_raised_without_one(monkeypatch):
    monkeypatch.delenv("NVCC", raising=False)
    monkeypatch.setattr(build.shutil, "which", lambda _: None)
    monkeypatch.setattr(build.os.path, "exists", lambda _: False)
    with pytest.raises(build.NoCompiler):
        build._nvcc()


def test_module_of_another_abi_is_refused(fresh):
    fresh.setattr(L, "ABI_VERSION", L.ABI_VERSION + 1)
    with pytest.raises(RuntimeError, match="ABI version"):
        L.torch_ops()
    assert L._torch_ops is None


def test_versions_agree():
    assert L.load().nsa_abi_version() == L.ABI_VERSION == L.torch_ops().abi_version

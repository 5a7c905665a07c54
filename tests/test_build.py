"""What the library's build needs: the C entry points neither torch nor a host compiler, the torch binding both. The
compilers are scripts that write their output file."""
import sys

import pytest

from interior_amd import build as b

WRITES = "#!/bin/sh\nwhile [ $# -gt 0 ]; do [ \"$1\" = -o ] && echo built > \"$2\"; shift; done\n"


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A source tree of one kernel unit and the binding, with a compiler for each."""
    def script(name, text):
        (tmp_path / name).write_text(text)
        (tmp_path / name).chmod(0o755)
        return str(tmp_path / name)

    (tmp_path / "csrc").mkdir()
    for name in ("unit.hip", "ops_torch.cpp"):
        (tmp_path / "csrc" / name).write_text("")
    for name, value in (("CSRC", tmp_path / "csrc"), ("BUILD", tmp_path / "build"), ("LIB", tmp_path / "lib.so"),
                        ("TORCH_LIB", tmp_path / "_ops_torch.so"), ("HIPCC", script("hipcc", WRITES))):
        monkeypatch.setattr(b, name, value)
    monkeypatch.setenv("CXX", script("cxx", WRITES))
    return script


def test_both_are_built(tree, recwarn):
    assert b.build() == b.LIB and b.LIB.exists() and b.TORCH_LIB.exists() and not recwarn.list


@pytest.mark.parametrize("missing", ["compiler", "torch"])
def test_library_needs_no_torch_and_no_host_compiler(tree, monkeypatch, missing):
    """It is linked with a warning, and a binding of another build does not stay beside it."""
    b.build()
    for out in (b.LIB, b.TORCH_LIB):
        out.write_text("old")
    if missing == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)
    else:
        monkeypatch.setenv("CXX", "/nonexistent/g++")
    with pytest.warns(UserWarning, match="interior_amd.ops cannot be used: .*" + missing):
        assert b.build(force=True) == b.LIB
    assert b.LIB.read_text() == "built\n" and not b.TORCH_LIB.exists()


def test_a_binding_that_does_not_compile_is_an_error(tree, monkeypatch):
    monkeypatch.setenv("CXX", tree("bad", "#!/bin/sh\necho wrong type >&2\nexit 1\n"))
    with pytest.raises(RuntimeError, match="wrong type"):
        b.build()
    assert b.LIB.exists() and not b.TORCH_LIB.exists()


def test_every_unit_is_built_without_packed_fp32(tree, monkeypatch):
    """Some forms of v_pk_{add,mul,fma}_f32 have given wrong results: no unit is excepted."""
    for name in ("norm.hip", "gemm.hip"):
        (b.CSRC / name).write_text("")
    log = b.CSRC / "calls"
    monkeypatch.setattr(b, "HIPCC", tree("logging", f"#!/bin/sh\necho \"$@\" >> {log}\n" + WRITES.split("\n", 1)[1]))
    b.build()
    calls = [c for c in log.read_text().splitlines() if " -c " in c]
    assert len(calls) == 3 and all("-Xclang -target-feature -Xclang -packed-fp32-ops" in c for c in calls)

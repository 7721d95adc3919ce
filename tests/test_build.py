"""vector-rs_b200/build.py: which steps it takes, with the compilers replaced."""
import importlib.util
import os
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def made(tmp_path, monkeypatch):
    """build.py on folders of its own, beside a torch that is a few empty files.
    Commands are written down, succeed (but for g++ where `made.fails`) and leave
    their output behind."""
    spec = importlib.util.spec_from_file_location("vrs_build_test", os.path.join(ROOT, "vector-rs_b200", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    torch = tmp_path / "torch"
    (torch / "lib").mkdir(parents=True)
    (torch / "version.py").write_text("__version__ = '1.0'\n")
    (torch / "lib" / "libc10_cuda.so").write_text("")
    headers = tmp_path / "headers"
    headers.mkdir()
    (headers / "Python.h").write_text("")
    for name in ("BUILD", "LIBDIR"):
        monkeypatch.setattr(b, name, str(tmp_path / name))
    monkeypatch.setattr(b, "LIB", str(tmp_path / "LIBDIR" / "libvrs.so"))
    monkeypatch.setattr(b, "OPS", str(tmp_path / "_ops.so"))
    monkeypatch.setattr(b, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setattr(b.importlib.util, "find_spec",
                        lambda name: types.SimpleNamespace(submodule_search_locations=[str(torch)]))
    monkeypatch.setattr(b.sysconfig, "get_paths", lambda: {"include": str(headers)})
    ran = []

    def run(cmd, **_):
        out = cmd[cmd.index("-o") + 1]
        kind = "ops" if cmd[0] == "g++" else "link" if "-shared" in cmd else "compile"
        ran.append(kind)
        if kind == "ops" and made.fails:
            return types.SimpleNamespace(returncode=1, stdout="", stderr="no")
        with open(out, "w") as f:
            f.write("x")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(b.subprocess, "run", run)
    made = types.SimpleNamespace(b=b, ran=ran, torch=torch, headers=headers, fails=False)
    return made


def test_library_is_linked_whatever_the_extension_does(made):
    made.fails = True
    with pytest.raises(RuntimeError, match="py_ops"):
        made.b.build()
    assert "link" in made.ran and os.path.exists(made.b.LIB)


def test_extension_is_built_once_a_torch(made):
    made.b.build()
    assert made.ran.count("ops") == 1 and made.ran.count("link") == 1
    made.b.build()
    assert made.ran.count("ops") == 1 and made.ran.count("link") == 1
    (made.torch / "version.py").write_text("__version__ = '1.1'\n")
    made.b.build()
    assert made.ran.count("ops") == 2 and made.ran.count("link") == 1
    made.b.build(force=True)
    assert made.ran.count("ops") == 3 and made.ran.count("link") == 2


@pytest.mark.parametrize("lacks", ["torch", "cuda", "headers"])
def test_without_what_the_extension_needs(made, monkeypatch, capsys, lacks):
    """No torch, one without CUDA, or no Python headers: the library alone."""
    if lacks == "torch":
        monkeypatch.setattr(made.b.importlib.util, "find_spec", lambda name: None)
    elif lacks == "cuda":
        (made.torch / "lib" / "libc10_cuda.so").unlink()
    else:
        (made.headers / "Python.h").unlink()
    assert made.b.build() == made.b.LIB
    assert "ops" not in made.ran and "link" in made.ran and not os.path.exists(made.b.OPS)
    assert "vector_cuda.ops" in capsys.readouterr().err

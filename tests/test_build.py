"""What the build leaves behind when a step of it fails, and when the machine's torch changes (no compiler runs here)."""

import os
import subprocess
from types import SimpleNamespace

import pytest
import torch

from ajllm_b200 import build
from ajllm_b200.ops import native


@pytest.fixture
def tools(tmp_path, monkeypatch):
    """A source tree of two kernels and the extension, compilers that write down what they were given, and switches to fail."""
    csrc, out = tmp_path / "csrc", tmp_path / "_native"
    csrc.mkdir()
    for name in ("a.cu", "b.cu", "fast_calls.cpp", "serving_args.h"):
        (csrc / name).write_text("first")
    monkeypatch.setattr(build, "CSRC", csrc)
    monkeypatch.setattr(build, "OUT", out)
    monkeypatch.setattr(build, "LIB", out / "lib.so")
    monkeypatch.setattr(build, "find_nvcc", lambda: "/none/bin/nvcc")
    state = SimpleNamespace(csrc=csrc, out=out, lib=out / "lib.so", broken=set(), now=1e9, ran=[])

    def run(command, **_):
        name = "link" if "-shared" in command and "nvcc" in command[0] else "g++" if command[0] == "g++" else "nvcc"
        state.ran.append(name)
        state.now += 1
        if name in state.broken:
            return subprocess.CompletedProcess(command, 1, "", f"{name} is broken")
        target = command[command.index("-o") + 1]
        inputs = [c for c in command if c.startswith(str(tmp_path)) and c != target and os.path.isfile(c)]
        with open(target, "w") as f:
            f.write(" ".join(open(c).read() for c in inputs))
        os.utime(target, (state.now, state.now))
        return subprocess.CompletedProcess(command, 0, "", "")

    monkeypatch.setattr(subprocess, "run", run)
    real = build._needs_build
    monkeypatch.setattr(build, "_needs_build", lambda source, obj, headers: real(source, obj, [h for h in headers if tmp_path in h.parents]))

    def write(name, text):
        state.now += 1
        (csrc / name).write_text(text)
        os.utime(csrc / name, (state.now, state.now))

    for name in ("a.cu", "b.cu", "fast_calls.cpp", "serving_args.h"):
        write(name, "first")
    state.write = write
    state.extensions = lambda: sorted(path.read_text() for path in out.glob("fast_calls*.so"))
    return state


def test_everything_is_built_once(tools):
    assert build.build() == tools.lib and tools.lib.read_text() == "first first" and tools.extensions() == ["first"]
    tools.ran.clear()
    build.build()
    assert tools.ran == []


def test_an_extension_that_cannot_be_built_leaves_the_library_and_no_older_extension(tools):
    build.build()
    tools.write("a.cu", "second")
    tools.write("serving_args.h", "other arguments")
    tools.broken.add("g++")
    with pytest.warns(UserWarning, match="g\\+\\+ is broken"):
        build.build()
    assert tools.lib.read_text() == "second first" and tools.extensions() == []
    tools.broken.clear()
    build.build()
    assert tools.extensions() == ["first"]


def test_a_compiler_that_is_not_there_is_a_warning_too(tools, monkeypatch):
    run = subprocess.run
    def without(command, **kw):
        if command[0] == "g++":
            raise FileNotFoundError("no g++ here")
        return run(command, **kw)
    monkeypatch.setattr(subprocess, "run", without)
    with pytest.warns(UserWarning, match="no g"):
        assert build.build() == tools.lib
    assert tools.lib.read_text() == "first first"


@pytest.mark.parametrize("broken", ["link", "nvcc"])
def test_a_library_older_than_its_objects_is_linked_again(tools, broken):
    build.build()
    tools.write("b.cu", "second")
    tools.broken.add(broken)
    with pytest.raises(RuntimeError, match="broken"):
        build.build()
    assert tools.lib.read_text() == "first first"           # still the older one, whole
    tools.broken.clear()
    build.build()
    assert tools.lib.read_text() == "first second"


def test_an_extension_built_for_another_torch_is_neither_kept_nor_loaded(tools, monkeypatch):
    build.build()
    monkeypatch.setattr(torch, "__version__", "99.0+cu999")
    monkeypatch.setattr(native, "_LIB_DIR", tools.out)
    with pytest.warns(UserWarning, match="could not be loaded"):
        assert native._load_fast_calls(None) is None
    tools.ran.clear()
    build.build()
    assert tools.ran == ["g++"] and len(tools.extensions()) == 1 and "99.0" in next(tools.out.glob("fast_calls*.so")).name

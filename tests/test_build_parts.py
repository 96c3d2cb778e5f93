"""The two parts of the build: the kernels' library, and the dense layer's autograd node, which needs a host compiler and torch's headers besides."""
import os

import pytest

from speech2lip_amd import autograd, build


@pytest.fixture
def parts(tmp_path, monkeypatch):
    """build_library on stand-ins: the library's compilation is noted, the node's output lies in tmp_path."""
    done = []
    for name in ("LIB", "REF_LIB", "RESOURCES"):
        monkeypatch.setattr(build, name, str(tmp_path / name))
    monkeypatch.setattr(build, "TORCH_OPS", str(tmp_path / "_linear_ops.so"))

    def hip(verbose):
        done.append("hip")
        for name in ("LIB", "REF_LIB", "RESOURCES"):
            open(getattr(build, name), "w").close()
    monkeypatch.setattr(build, "_build_hip", hip)
    return done


def command(text, monkeypatch):
    monkeypatch.setattr(build, "_torch_ops_command", lambda: ["sh", "-c", text])


def test_the_library_is_built_where_the_node_cannot_be(parts, monkeypatch):
    command("echo no headers; exit 1", monkeypatch)
    with pytest.warns(UserWarning, match="no headers"):
        assert build.build_library() == build.LIB
    assert parts == ["hip"] and not os.path.exists(build.TORCH_OPS)
    with pytest.warns(UserWarning):      # the library stands; the node is tried again
        build.build_library()
    assert parts == ["hip"]

    def no_compiler():
        raise FileNotFoundError("g++")
    monkeypatch.setattr(build, "_torch_ops_command", no_compiler)
    open(build.TORCH_OPS, "w").close()      # an old one does not stay
    with pytest.warns(UserWarning, match="g\\+\\+"):
        build.build_library(force=True)
    assert parts == ["hip", "hip"] and not os.path.exists(build.TORCH_OPS)


def test_a_node_of_another_torch_is_built_again(parts, monkeypatch):
    import torch
    write = lambda version: f"printf 'x built for torch {version}; y' > {build.TORCH_OPS}.tmp"  # noqa: E731
    command(write("0.1"), monkeypatch)
    build.build_library()
    assert parts == ["hip"] and build.needs_build()
    command(write(torch.__version__), monkeypatch)
    build.build_library()
    assert parts == ["hip"] and not build.needs_build()
    os.utime(build.TORCH_OPS, (1, 1))
    assert build.needs_build()


def test_a_node_of_another_torch_is_not_loaded(monkeypatch):
    ops = autograd._linear_ops()
    monkeypatch.setattr(autograd, "_linear_native", (None, None))
    monkeypatch.setattr(ops, "built_for", "built for torch 0.1;")
    with pytest.raises(RuntimeError, match="0.1"):
        autograd._linear_ops()

"""The build step with stand-ins for the compilers: what is built, and what is left when something fails."""

from __future__ import annotations

import subprocess
import sys

import pytest

from chroma_b200 import build
from tests.conftest import ROOT

TAG = "torch 9.9, cpython-test"


def compiler(name, target, code, text="x"):  # type: ignore[no-untyped-def]
    script = f"import sys, time; time.sleep(0.2); open({str(target)!r}, 'w').write({text!r}); print('{name} says', file=sys.stderr); sys.exit({code})"
    return [sys.executable, "-c", script]


@pytest.fixture
def place(tmp_path, monkeypatch):  # type: ignore[no-untyped-def]
    library, binding = tmp_path / "library.so", tmp_path / "binding.so"
    monkeypatch.setattr(build, "TARGET", library)
    monkeypatch.setattr(build, "TENSORS", binding)

    def use(library_code=0, binding_code=0, tag=TAG):  # type: ignore[no-untyped-def]
        monkeypatch.setattr(build, "command", lambda target: compiler("nvcc", target, library_code))
        monkeypatch.setattr(build, "tensors_command", lambda target: compiler("g++", target, binding_code, f"x {tag} x"))
        monkeypatch.setattr(build, "built_for", lambda: tag)
        return library, binding

    return use


def files(library):  # type: ignore[no-untyped-def]
    return sorted(p.name for p in library.parent.iterdir())


def test_both_are_built_once(place) -> None:  # type: ignore[no-untyped-def]
    library, binding = place()
    assert build.build() == library and files(library) == ["binding.so", "library.so"]
    before = [p.stat().st_mtime_ns for p in (library, binding)]
    build.build()
    assert before == [p.stat().st_mtime_ns for p in (library, binding)]


def test_without_torch_the_library_is_built(place) -> None:  # type: ignore[no-untyped-def]
    library, _ = place(tag=None)
    build.build(force=True)
    assert files(library) == ["library.so"]


def test_a_binding_that_fails_leaves_the_library(place) -> None:  # type: ignore[no-untyped-def]
    library, _ = place(binding_code=1)
    with pytest.raises(RuntimeError, match=r"g\+\+ says"):
        build.build()
    assert files(library) == ["library.so"]


def test_a_library_that_fails_waits_for_the_binding(place) -> None:  # type: ignore[no-untyped-def]
    library, _ = place(library_code=1)
    with pytest.raises(RuntimeError, match="nvcc says"):
        build.build()
    assert files(library) == ["binding.so"]


def test_no_compiler_starts_before_all_commands_are_there(place, monkeypatch) -> None:  # type: ignore[no-untyped-def]
    library, _ = place()

    def broken(target):  # type: ignore[no-untyped-def]
        raise ImportError("no Torch after all")

    monkeypatch.setattr(build, "tensors_command", broken)
    with pytest.raises(ImportError):
        build.build()
    assert files(library) == []


def test_a_binding_for_another_torch_is_built_again(place) -> None:  # type: ignore[no-untyped-def]
    library, binding = place(tag="torch 1.0, cpython-test")
    build.build()
    place()
    build.build()
    assert TAG in binding.read_text()


def test_tags() -> None:
    import torch

    from chroma_b200._src import paged

    assert build.built_for() == paged.ops.built_for and torch.__version__ in paged.ops.built_for
    code = "import sys; sys.modules['torch'] = None\nfrom chroma_b200 import build; print(build.built_for())"
    assert subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True).stdout == "None\n"

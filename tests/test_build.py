"""When the native libraries are rebuilt: their keys, and that loading one looks at its key."""

from __future__ import annotations

import shutil
import subprocess
import sys
from pathlib import Path

import pytest

from mgc_cuda import build, native
from mgc_cuda._errors import CodegenError

KEYS = ("import sys; sys.path.insert(0, {!r}); from mgc_cuda import build; "
        "print(build.source_key(build.nvcc_flags()), build.binding_key())")


def keys(root: Path) -> list[str]:
    run = subprocess.run([sys.executable, "-c", KEYS.format(str(root))], capture_output=True, text=True, check=True)
    return run.stdout.split()


def test_keys_go_by_the_sources_and_not_by_their_place(tmp_path: Path) -> None:
    here = build.PACKAGE_DIR.parent
    there = tmp_path / "elsewhere" / here.name
    shutil.copytree(here / "csrc", there / "csrc")
    shutil.copytree(build.PACKAGE_DIR, there / "mgc_cuda", ignore=shutil.ignore_patterns("lib", "__pycache__"))
    shutil.copytree(build.INCLUDE_DIR, tmp_path / "elsewhere" / "include")
    assert keys(there) == keys(here)
    header = tmp_path / "elsewhere" / "include" / "mgc_cuda.h"
    header.write_text(header.read_text().replace("int64_t batch, tokens;", "int64_t batch, tokens, more;"))
    assert all(a != b for a, b in zip(keys(there), keys(here)))


def test_loading_builds_what_is_out_of_date(monkeypatch: pytest.MonkeyPatch) -> None:
    """A library of an older header would read the new structs wrongly."""
    def stale(*_args: object, **_kw: object) -> Path:
        raise CodegenError("out of date")

    monkeypatch.setattr(native, "_LIB", None)
    monkeypatch.setattr(build, "build", stale)
    with pytest.raises(CodegenError, match="out of date"):
        native.library()


def test_loading_the_binding_builds_what_is_out_of_date(monkeypatch: pytest.MonkeyPatch) -> None:
    pytest.importorskip("torch")
    from mgc_cuda import paged

    def stale(*_args: object, **_kw: object) -> Path:
        raise CodegenError("out of date")

    monkeypatch.setattr(paged, "_EXT", None)
    monkeypatch.setattr(build, "build_binding", stale)
    with pytest.raises(CodegenError, match="out of date"):
        paged._binding()


def test_a_current_build_needs_no_compiler(monkeypatch: pytest.MonkeyPatch) -> None:
    pytest.importorskip("torch")
    build.build()
    build.build_binding()
    monkeypatch.setenv("MGC_NVCC", "/nowhere/nvcc")
    monkeypatch.setenv("PATH", "")
    monkeypatch.setattr(build, "find_nvcc", lambda: (_ for _ in ()).throw(CodegenError("nvcc not found")))
    assert build.build() == build.library_path() and build.build_binding() == build.binding_path()

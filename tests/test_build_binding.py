"""The build of the binding beside the library's: the library does without it."""

import os

import pytest

from recap_b200 import build as b


@pytest.fixture
def place(tmp_path, monkeypatch):
    """A binding of this test's own, compiled by a script that counts its calls."""
    calls = tmp_path / "calls"
    compiler = tmp_path / "cxx"
    compiler.write_text(f'#!/bin/sh\necho x >> {calls}\nwhile [ "$1" != -o ]; do shift; done\necho built > "$2"\n')
    compiler.chmod(0o755)
    monkeypatch.setattr(b, "BINDING_PATH", tmp_path / "_native.so")
    monkeypatch.setattr(b, "_build_library", lambda force, verbose: b.LIB_PATH)  # as if it were up to date
    monkeypatch.setenv("CXX", str(compiler))
    return lambda: len(calls.read_text().split()) if calls.exists() else 0


@pytest.mark.parametrize("compiler", ["false", "/nowhere/a-compiler"])
def test_the_library_is_built_where_the_binding_is_not(place, compiler, monkeypatch, capfd):
    monkeypatch.setenv("CXX", compiler)
    assert b.build() == b.LIB_PATH
    assert "was not built" in capfd.readouterr().err
    assert not b.BINDING_PATH.exists()


def test_a_binding_of_older_sources_does_not_outlive_a_failed_build(place, monkeypatch):
    b.build()
    assert b.BINDING_PATH.exists()
    os.utime(b.BINDING_PATH, (0, 0))
    monkeypatch.setenv("CXX", "false")
    b.build()
    assert not b.BINDING_PATH.exists()


def test_a_binding_of_another_torch_is_built_again(place, monkeypatch):
    import torch

    b.build()
    b.build()
    assert place() == 1
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    b.build()
    b.build()
    assert place() == 2

"""The build's own promises: build() compiles also where a library is there, and an object follows the flags it is built with."""
import os
import subprocess

import pytest

import __graft_entry__ as entry
from oracle import oracle as orc
from rtlamr_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Stop(Exception):
    pass


def make_lines(monkeypatch, call):
    lines = []

    def record(cmd, *args, **kwargs):
        lines.append(cmd)
        raise Stop

    monkeypatch.setattr(subprocess, "check_call", record)
    with pytest.raises(Stop):
        call()
    return lines


def test_entry_compiles_although_the_library_is_newer_than_its_sources(monkeypatch):
    monkeypatch.setattr(_lib.os.path, "getmtime", lambda path: 2.0 if path in (_lib.SO_PATH, orc._SO) else 1.0)
    monkeypatch.setattr(_lib.os.path, "exists", lambda path: True)
    (line,) = make_lines(monkeypatch, entry.build)
    assert line[0] == "make" and _lib.CSRC in line and "-B" in line


def test_oracle_is_compiled_anew_when_asked(monkeypatch):
    (line,) = make_lines(monkeypatch, lambda: orc.build(force=True))
    assert line[0] == "make" and "-B" in line


def test_objects_depend_on_the_flags():
    r = subprocess.run(["make", "-C", _lib.CSRC, "-n", "-W", "Makefile", "libamrdemod.so"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    objects = [f for f in os.listdir(_lib.CSRC) if f.endswith(".hip")]
    assert len(objects) > 10
    for f in objects:
        assert f" {f}" in r.stdout, f"{f} would keep its old object after a change of the flags"

"""The build's own promises: build() compiles also where a library is there, an object follows the flags it is built with, and
the device code of the built library holds no packed FP32 arithmetic."""
import os
import re
import shutil
import struct
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


def test_built_library_has_no_packed_fp32(tmp_path):
    objdump = "/opt/rocm/lib/llvm/bin/llvm-objdump"
    if not (os.path.exists(_lib.SO_PATH) and shutil.which("objcopy") and os.path.exists(objdump)):
        pytest.skip("library not built, or no binutils / llvm-objdump here")
    fat = tmp_path / "fat.bin"
    subprocess.check_call(["objcopy", "-O", "binary", "--only-section=.hip_fatbin", _lib.SO_PATH, str(fat)])
    blob, magic, found, seen = fat.read_bytes(), b"__CLANG_OFFLOAD_BUNDLE__", set(), 0
    for bundle in re.finditer(magic, blob):
        p = bundle.start() + len(magic)
        (count,) = struct.unpack_from("<Q", blob, p)
        p += 8
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", blob, p)
            triple = blob[p + 24:p + 24 + length].decode()
            p += 24 + length
            if "gfx950" not in triple or size == 0:
                continue
            code = tmp_path / "code.o"
            code.write_bytes(blob[bundle.start() + offset:bundle.start() + offset + size])
            text = subprocess.run([objdump, "-d", "--no-show-raw-insn", str(code)], capture_output=True, text=True, check=True).stdout
            assert "s_endpgm" in text
            found |= set(re.findall(r"\bv_pk_(?:add|mul|fma)_f32\b", text))
            seen += 1
    assert seen > 10 and not found

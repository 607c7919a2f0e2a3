"""Rules on the text of the sources, scripts and build files (no GPU, no compiler).

* Device code writes through the vector path only.  A write through the scalar data cache is not coherent with it and needs
  a write-back of its own before anything else can see it.  Comments and strings count: what is not written about is not
  copied from there into a kernel.
* A variant of the store microbenchmark that its main() does not launch has no figure that can be checked.
* No packed FP32 arithmetic: neither written by hand nor left to the compiler.
"""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TREES = ("rtlamr_amd", "include", "tests", "tools", "oracle", "go", "docs", "profiles")   # and the files at the top
SUFFIXES = (".hip", ".h", ".hpp", ".inc", ".c", ".cpp", ".s", ".S", ".ll", ".py", ".sh", ".go", ".mk", ".cmake")

# Scalar stores, scalar atomics, and the scalar cache's write-back and discard; the names are put together here so that
# this file itself holds none.  In a string of assembly a name may follow an escape (\n, \t) without a space.
S = "s_"
SCALAR_WRITE = re.compile(rf"(?:(?<!\w)|(?<=\\[nt])){S}(?:(?:(?:buffer|scratch)_)?(?:store|atomic)_\w+|dcache_(?:wb|discard)\w*)")


def source_files():
    walks = [(ROOT, [], os.listdir(ROOT))]
    for tree in TREES:
        walks += os.walk(os.path.join(ROOT, tree))
    for top, _, names in walks:
        for name in names:
            if name.endswith(SUFFIXES) or name == "Makefile":
                yield os.path.join(top, name)


def scalar_writes(text):
    return [(i, m.group(0)) for i, line in enumerate(text.splitlines(), 1) for m in SCALAR_WRITE.finditer(line)]


def test_no_source_writes_through_the_scalar_cache():
    files = list(source_files())
    assert any(f.endswith(".hip") for f in files) and any(f.endswith("Makefile") for f in files)
    found = []
    for path in files:
        with open(path, encoding="utf-8", errors="replace") as f:
            found += [f"{os.path.relpath(path, ROOT)}:{i}: {what}" for i, what in scalar_writes(f.read())]
    assert not found, found


@pytest.mark.parametrize("tail", ["store_dword", "store_dwordx4", "buffer_store_dwordx2", "scratch_store_dword", "atomic_add",
                                  "buffer_atomic_cmpswap_x2", "dcache_wb", "dcache_wb_vol", "dcache_discard_x2"])
def test_the_pattern_sees_every_form(tail):
    assert scalar_writes(f'asm volatile("{S}{tail} %0, %1, 0x0\\n\\t{S}{tail}");  // and {S}{tail}\n') == [(1, S + tail)] * 3


@pytest.mark.parametrize("line", [S + "load_dwordx4 s[0:3], s[4:5], 0x0", S + "dcache_inv", "global_store_dword v0, v1, s[0:1]",
                                  "buffer_store_dwordx4 v[0:3], v4, s[0:3], 0 offen", "ds_write_b32 v0, v1", "words_store_x"])
def test_the_pattern_leaves_other_code_alone(line):
    assert scalar_writes(line) == []


def test_every_store_variant_of_the_microbenchmark_is_launched():
    with open(os.path.join(ROOT, "tools", "sst_bench.hip"), encoding="utf-8") as f:
        kernel, main = f.read().split("int main()")
    launched = {int(st) for st in re.findall(r"run<(\d+), \d+>\(d, o\)", main)}
    single = {int(st) for st in re.findall(r"ST == (\d+)", kernel)}
    assert single == {st for st in launched if st < 10}
    assert "ST >= 10" in kernel and any(st >= 10 for st in launched)


PACKED_OFF = "-Xclang -target-feature -Xclang -packed-fp32-ops"


def test_device_code_is_compiled_without_packed_fp32():
    """hipcc -O3 forms packed float operations from scalar code by itself; every compile line of device code rules them out."""
    lines = []
    for path in source_files():
        if os.path.dirname(path) == os.path.join(ROOT, "tests"):
            continue                                     # host programs only
        with open(path, encoding="utf-8", errors="replace") as f:
            lines += [(path, line) for line in f if "--offload-arch" in line and "-shared" not in line]
    with open(os.path.join(ROOT, "tools", "README.md"), encoding="utf-8") as f:
        lines += [(f.name, line) for line in f if "--offload-arch" in line]
    assert any(path.endswith("csrc/Makefile") for path, _ in lines)
    assert [(path, line) for path, line in lines if PACKED_OFF not in line] == []


def test_no_packed_fp32_by_hand():
    packed = re.compile(r"\bv_pk_(?:add|mul|fma)_f32\b")
    for path in source_files():
        if path.endswith((".hip", ".h", ".inc")):
            with open(path, encoding="utf-8", errors="replace") as f:
                assert not packed.search(f.read()), path

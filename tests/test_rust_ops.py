"""rust/src/ops.rs's view of the C ABI, checked on the CPU through tests/csrc/rust_ops_abi.c (as
tests/test_rust_binding.py does for ffi.rs): the same functions, the header's types, the library's
symbols."""
import os
import re
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_ops_rs_and_its_mirror_agree_with_the_header_and_the_library(built_lib, tmp_path):
    src = open(os.path.join(REPO, "rust", "src", "ops.rs")).read()
    block = src[src.index('extern "C" {'):]
    rust = set(re.findall(r"\bpub fn (lrs_[a-z0-9_]+)\s*\(", block))
    mirror = os.path.join(REPO, "tests", "csrc", "rust_ops_abi.c")
    assert rust == set(re.findall(r"typedef [^;]*?\(\*rs_(lrs_[a-z0-9_]+)\)", open(mirror).read())) and len(rust) == 4
    exe = str(tmp_path / "rust_ops_abi")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", mirror, "-o", exe, "-ldl"], check=True)
    out = subprocess.run([exe, built_lib], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, (out.returncode, out.stderr)


def test_the_crate_builds_every_source_of_the_library():
    from lrs import build
    text = open(os.path.join(REPO, "rust", "build.rs")).read()
    assert not [s for s in build.SOURCES + build.HEADERS if f'"{s}"' not in text]

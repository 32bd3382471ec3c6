"""How lists of tensors are laid out as the argument tables of launches (csrc/hpx_tables.h): no launch of 2^32 lanes or more, however
large the list or one tensor of it.  The header has no GPU dependency; the test compiles tests/host_tables.cpp with the host
compiler and runs it."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_tables_cover_lists_of_any_size(tmp_path):
    exe = str(tmp_path / "host_tables")
    src = os.path.join(ROOT, "tests", "host_tables.cpp")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined",
                           "-I" + os.path.join(ROOT, "torch-hipress-extension_amd", "csrc"), "-I" + os.path.join(ROOT, "include"),
                           src, "-o", exe])
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "OK", (r.stdout, r.stderr)

"""The host layer of the microscaled operators under AddressSanitizer and UndefinedBehaviorSanitizer, driven by
tests/mx_host_fuzz.c; built as tests/test_host_sanitizers.py builds the rest of it."""
import os
import shutil
import subprocess
from pathlib import Path

import pytest

from gemm_zoo_b200 import build as b

ROOT = Path(__file__).resolve().parent.parent


def test_microscale_host_layer_is_clean_under_asan_and_ubsan(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not installed")
    b.build_lib()  # makes sure the kernel objects exist
    kernel_objs = sorted((b.CSRC / "build").glob("k_*.o"))
    san = "-fsanitize=address,-fsanitize=undefined,-fno-omit-frame-pointer"

    def run(*cmd, **kw):
        r = subprocess.run([str(c) for c in cmd], capture_output=True, text=True, **kw)
        assert r.returncode == 0, (r.stdout[-1500:], r.stderr[-3000:])
        return r

    obj, lib, exe = tmp_path / "gemm_api_san.o", tmp_path / "libgemmzoo_san.so", tmp_path / "mx_host_fuzz"
    run(b.nvcc_path(), *b.ARCH, "-O1", "-g", "-std=c++17", "-Xcompiler", f"-fPIC,{san}", "-c", f"-I{b.INCLUDE}", f"-I{b.CSRC}",
        "-o", obj, b.CSRC / "gemm_api.cu")
    run(b.nvcc_path(), *b.ARCH, "-shared", "-Xcompiler", "-fPIC", "-Xlinker", "-lasan", "-Xlinker", "-lubsan", "-o", lib, obj,
        *kernel_objs)
    run(gcc, "-O1", "-g", "-fsanitize=address,undefined", f"-I{b.INCLUDE}", "-o", exe, ROOT / "tests" / "mx_host_fuzz.c",
        f"-L{tmp_path}", "-lgemmzoo_san", f"-Wl,-rpath,{tmp_path}", "-lm")
    env = dict(os.environ, ASAN_OPTIONS="protect_shadow_gap=0:detect_leaks=0:abort_on_error=0",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    r = run(exe, env=env, timeout=600)
    assert "MX HOST FUZZ OK" in r.stdout
    assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr, r.stderr[-3000:]

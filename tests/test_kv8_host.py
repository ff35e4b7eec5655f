"""What of the 8-bit K/V entries needs no GPU: a state's size and its refusals, calls without a handle, the C++ wrappers' build (their program,
tests/cpp/kv8_host.cpp, runs on a B200)."""
import os
import subprocess

import pytest

from kv8_util import state_bytes
from straydog_b200 import _lib, build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BUILD = os.path.join(ROOT, "tests", "cpp", "_build")


@pytest.mark.parametrize("context,kv_heads,dim", [(32, 1, 64), (64, 3, 128), (32768, 2, 256), (1 << 24, 8, 128)])
def test_the_size_of_a_state(context, kv_heads, dim):
    assert _lib.load().sdx_kv8_bytes(context, kv_heads, dim) == state_bytes(context, kv_heads, dim)


@pytest.mark.parametrize("context,kv_heads,dim", [(0, 1, 64), (33, 1, 64), (1 << 25, 1, 64), (32, 0, 64), (32, 1025, 64), (32, 1, 96), (32, 1, 0)])
def test_sizes_that_are_none(context, kv_heads, dim):
    lib = _lib.load()
    assert lib.sdx_kv8_bytes(context, kv_heads, dim) == 0
    assert lib.sd_error()


def test_a_null_handle_is_an_error():
    lib = _lib.load()
    assert lib.sdx_kv8_write(None, None, None, None, None, 1, 1, 64, 0, None, None, 0, 0) == -1
    assert lib.sdx_kv8_attention(None, None, None, None, None, 1, 1, 1, 64, 0, 1.0, 0.0, None, 0, None, None, 0, None, None, 0, 1) == -1
    assert lib.sdx_masked_attention(None, None, 0, None, 0, None, 0, None, None, 1, 1, 1, 64, 1, 1.0, 0.0, None, 0, None, None, 0) == -1
    assert lib.sdx_kv8_evict(None, None, None, None, None, 1, 1, 0, 0, 1, 64, 0, None, None, None, None) == -1
    assert b"handle" in lib.sd_error()


def compile_program():
    library_dir = os.path.dirname(build.build())
    os.makedirs(BUILD, exist_ok=True)
    program, cuda = os.path.join(BUILD, "kv8_host"), os.environ.get("CUDA_HOME", "/usr/local/cuda")
    done = subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "cpp", "kv8_host.cpp"),
                           "-o", program, "-L", library_dir, "-lstraydog_gpu_b200", f"-Wl,-rpath,{library_dir}", f"-Wl,-rpath-link,{cuda}/lib64"],
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    return program


def test_the_cpp_wrappers_compile_and_link():
    assert os.path.exists(compile_program())


@pytest.mark.gpu
def test_the_cpp_wrappers_on_the_gpu():
    done = subprocess.run([compile_program()], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip().startswith("ok"), done.stdout + done.stderr

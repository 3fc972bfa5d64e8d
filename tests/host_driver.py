"""Runs Python code on the stand-in driver of fake_driver/ in a process of its own (no test
functions here): the library's host side without a GPU."""
from __future__ import annotations

import os
import pathlib
import shutil
import subprocess
import sys

import pytest

TESTS = pathlib.Path(__file__).resolve().parent
INCLUDE = pathlib.Path("/usr/local/cuda/include")

needs_compiler = pytest.mark.skipif(shutil.which("g++") is None or not (INCLUDE / "cuda.h").exists(),
                                    reason="no C++ compiler or no cuda.h on this machine")

PROLOGUE = """
import ctypes, threading
import numpy as np
import titan_rs_b200 as tb
from titan_rs_b200.kernel_abi import DType

fake = ctypes.CDLL("libcuda.so.1")

def lines():
    text = ctypes.create_string_buffer(1 << 22)
    assert fake.fake_log(text, len(text)) >= 0
    return text.value.decode().splitlines()

def in_threads(*work):
    failures = []
    def guarded(w):
        try:
            w()
        except Exception as e:
            failures.append(e)
    threads = [threading.Thread(target=guarded, args=(w,)) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures

def spec_of(t):
    return tb.TensorSpec(t.dtype, t.shape, t.strides)

session = tb.Session(0)
assert session.fingerprint()["model"] == "stand-in"
rt = tb.Runtime(session)
"""


def build_driver(folder: pathlib.Path) -> pathlib.Path:
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wall", "-Werror", "-I", str(INCLUDE),
                    str(TESTS / "fake_driver" / "fake_cuda.cpp"), "-o", str(folder / "libcuda.so.1"),
                    "-Wl,-soname,libcuda.so.1", "-pthread"], check=True, capture_output=True, text=True)
    return folder


def run(folder: pathlib.Path, script: str) -> str:
    env = dict(os.environ, LD_LIBRARY_PATH=f"{folder}:{os.environ.get('LD_LIBRARY_PATH', '')}",
               PYTHONPATH=str(TESTS.parent))
    done = subprocess.run([sys.executable, "-c", PROLOGUE + script], env=env, capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr
    return done.stdout

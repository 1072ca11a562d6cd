"""Calls on cache pages that need no GPU: refusals and book-keeping on the host, by a program that links the library (native/cache_host.cpp)."""
import os
import subprocess

import pytest

from juno_b200 import _lib, build

HERE = os.path.dirname(os.path.abspath(__file__))
SRC, EXE = os.path.join(HERE, "native", "cache_host.cpp"), os.path.join(HERE, "native", "build", "cache_host")


@pytest.fixture(scope="module")
def host():
    lib = build.build()
    os.makedirs(os.path.dirname(EXE), exist_ok=True)
    headers = [os.path.join(build.CSRC, f) for f in os.listdir(build.CSRC) if f.endswith(".cuh")]
    if not os.path.exists(EXE) or os.path.getmtime(EXE) < max(os.path.getmtime(f) for f in (SRC, *headers)):
        subprocess.check_call(["g++", "-O1", "-std=c++17", "-I/usr/local/cuda/include", "-o", EXE, SRC, lib, f"-Wl,-rpath,{os.path.dirname(lib)}"])
    assert lib == _lib.LIB_PATH

    def run(name):
        r = subprocess.run([EXE, name], capture_output=True, text=True, timeout=120, env=os.environ | {"CUDA_VISIBLE_DEVICES": ""})
        assert r.returncode == 0, r.stdout + r.stderr
    return run


def test_rows_of_one_sequence_do_not_share_weights(host):
    host("twice")


def test_sequences_without_weights_may_be_named_beside_one_with_weights(host):
    host("beside")


def test_sequences_of_a_closed_pool_or_context_are_refused(host):
    host("closed")


def test_positions_beyond_32_bits_are_refused(host):
    host("far")


def test_host_memory_that_runs_out_is_an_error_and_changes_nothing(host):
    host("memory")


def test_a_freed_sequence_gives_its_list_of_pages_back(host):
    host("freed")


def test_a_pool_that_is_far_too_large_costs_the_host_nothing(host):
    host("huge")

"""Shared by the tests of 4-bit cache pages."""
import ctypes as C
import os
import subprocess

import numpy as np

from oracle import q4_cache_oracle as q4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def host_library():
    src, so = (os.path.join(ROOT, "tests", "native", f) for f in ("q4_host.cpp", "libq4_host.so"))
    header = os.path.join(ROOT, "juno_b200", "csrc", "q4_pages.cuh")
    if not os.path.exists(so) or os.path.getmtime(so) < max(os.path.getmtime(src), os.path.getmtime(header)):
        subprocess.check_call(["g++", "-O2", "-std=c++17", "-ffp-contract=off", "-shared", "-fPIC", "-o", so, src])
    L = C.CDLL(so)
    L.q4_host_number.argtypes = L.q4_host_number_exact.argtypes = [C.c_float] * 3
    return L


def rows(rng, n, kv, dim):
    """Keys with channels of different spread and mean."""
    return (rng.standard_normal((n, kv, dim)) * np.exp(0.5 * rng.standard_normal((kv, dim))) + 0.5 * rng.standard_normal((kv, dim))).astype(np.float32)


def attention_tolerance(q, k, v, dim):
    """How far decode attention may be off, per element: a score is a sum of dim products with both factors exact to 2^-22 (two FP16 limbs of the query,
    FP32 otherwise) and at most dim roundings of 2^-24, so off by delta <= S (2^-22 + dim 2^-24) with S = max |q| |k| / sqrt(dim); a softmax weight is
    then off by 2 delta relative (its own exponential and the sum), the weighted sum by as much times max |v|; roundings of the weights' limbs (2^-22) and of the sums
    in FP32 (one per 16 positions in an MMA, splits merged pairwise: 2^-17 covers 128 roundings) come on top."""
    s = float(np.linalg.norm(q, axis=-1).max() * np.linalg.norm(k, axis=-1).max() / np.sqrt(dim)) if len(k) else 0.0
    delta = s * (2.0 ** -22 + dim * 2.0 ** -24)
    return 2 * delta + 2.0 ** -17, float(np.abs(v).max()) if len(v) else 1.0

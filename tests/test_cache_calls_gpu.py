"""Calls on 4-bit cache pages in the forms that one operator's tests do not have: from host memory, beyond usual sizes, after failures, with pages shared in part."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

from juno_b200._lib import JunoError
from juno_b200.matvec import GpuContext, PagedKvCache
from oracle import q4_cache_oracle as q4
from q4util import rows
from test_q4_cache_gpu import attend, check_attention, check_weights, dev, expected, f32, fill, read, settle, some_weights, weights
from test_readme_cpu import cache_example

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def words():
    src, so = (os.path.join(HERE, "native", f) for f in ("cache_words.cpp", "libcache_words.so"))
    header = os.path.join(HERE, "..", "juno_b200", "csrc", "common.cuh")
    if not os.path.exists(so) or os.path.getmtime(so) < max(os.path.getmtime(src), os.path.getmtime(header)):
        subprocess.check_call(["g++", "-O2", "-std=c++17", "-I/usr/local/cuda/include", "-shared", "-fPIC", "-o", so, src])
    L = C.CDLL(so)
    for f, t in (("cache_scratch_bytes", C.c_longlong), ("cache_gave_up", C.c_void_p), ("cache_calls", C.c_ulonglong)):
        getattr(L, f).restype, getattr(L, f).argtypes = t, [C.c_void_p]
    return L


def test_host_attention_names_a_sequence_with_weights_once(ctx):
    rng = np.random.default_rng(51)
    cache = PagedKvCache(ctx, 1, 2, 64, 16, "q4", track_seqs=1, track_tokens=64)
    a, b = cache.new_sequence(64, track=True), cache.new_sequence(64)
    k, v = rows(rng, 40, 2, 64), f32(rng.standard_normal((40, 2, 64)))
    fill(cache, 0, [a, b], [0, 0], [(k, v)] * 2)
    q = f32(rng.standard_normal((3, 8, 64)))
    for seqs in ([a, a], [b, a, a]):
        with pytest.raises(ValueError, match="there twice"):
            cache.attention(0, seqs, q[:len(seqs)].reshape(len(seqs), -1), 8)
    assert (weights(cache, 0, [a], [40]) == 0).all()  # a refused call adds nothing
    out = cache.attention(0, [b, a, b], q.reshape(3, -1), 8).reshape(q.shape)  # without weights a sequence may be there several times
    for i in range(3):
        w = check_attention(out[i], q[i], q4.held(k), q4.held(v))
        if i == 1:
            check_weights(weights(cache, 0, [a], [40])[0], w, q[i], k)
    cache.close()


# Queries so large that the softmax leaves one position: the result is that position's row.  What the kernel rounds of it: the two limbs of weight times step, 2^-22,
# and in FP32 the offset's product, the sum of both parts, the warps' merge and the division, four times 2^-24, of terms of up to 3 times the largest value
# (m and 15 d are up to twice it apart): 3 (2^-22 + 4 2^-24) < 2^-19.  No score comes near the largest: the gap is 1e-3 of it, the scores are off by some 1e-6 of it.
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (8, 2, 128), (16, 2, 128)])
def test_queries_of_any_size(ctx, heads, kv, dim):
    rng = np.random.default_rng(52)
    n = 70
    cache = PagedKvCache(ctx, 1, kv, dim, 8, "q4")
    s = cache.new_sequence(n)
    k, v = f32(rng.standard_normal((n, kv, dim))), f32(rng.standard_normal((n, kv, dim)))
    fill(cache, 0, [s], [0], [(k, v)])
    hk, hv = q4.held(k), q4.held(v)
    q = rng.standard_normal((1, heads, dim))
    scores = np.einsum("hgd,lhd->hgl", q[0].reshape(kv, -1, dim), hk).reshape(heads, n)
    first, second = np.sort(scores, -1)[:, -1], np.sort(scores, -1)[:, -2]
    assert (first - second > 1e-3 * np.abs(scores).max(-1)).all()
    best = scores.argmax(-1)
    want = hv[best, np.arange(heads) // (heads // kv)]
    for size in (1e8, 1e20, 1e30, 1e32, 1e34, 1e36):
        x = f32(size * q)
        assert np.isfinite(x).all()
        got = attend(cache, 0, [s], x)[0]
        assert np.abs(got - want).max() <= 2.0 ** -19 * np.abs(hv).max(), size
    for size in (1e-20, 1e-36, 1e-44, 0.0):
        x = f32(size * q)
        check_attention(attend(cache, 0, [s], x)[0], x[0], hk, hv)
    cache.close()


# Groups of a value whose sizes lie far apart keep their own digits.  What the kernel rounds relative to a group: the weights, which are off by some 2e-6 as in
# test_long_sums_are_not_biased, and weight times step in two limbs, 2^-22, both at random over the positions: about 2e-6 of the result's length in the group, and 1e-5 leaves
# a factor of five.
@pytest.mark.parametrize("ratio", [1e3, 1e6, 1e9])
@pytest.mark.parametrize("n,heads,kv,dim", [(300, 8, 2, 64), (300, 8, 2, 128), (5000, 16, 2, 128), (5000, 5, 1, 64)])
def test_groups_of_values_far_apart(ctx, n, heads, kv, dim, ratio):
    rng = np.random.default_rng(53)
    cache = PagedKvCache(ctx, 1, kv, dim, n // 16 + 1, "q4")
    s = cache.new_sequence(n)
    size = np.repeat(ratio ** np.linspace(0.5, -0.5, dim // 32), 32)
    for order in (size, size[::-1]):
        k, v = rows(rng, n, kv, dim), f32(rng.standard_normal((n, kv, dim)) * order)
        fill(cache, 0, [s], [0], [(k, v)])
        q = f32(rng.standard_normal((1, heads, dim)))
        got, (want, _) = attend(cache, 0, [s], q)[0], q4.attention(q[0], q4.held(k), q4.held(v))
        of_groups = lambda x: np.linalg.norm(x.reshape(heads, -1, 32), axis=-1)  # noqa: E731
        assert (of_groups(got - want) <= 1e-5 * of_groups(want)).all(), of_groups(got - want) / of_groups(want)
    cache.close()


def test_a_growing_sequence_with_weights_seldom_grows_the_working_memory(words):
    """Growing waits for the whole device: to twice the size each time, so that 400 steps do it a few times."""
    rng = np.random.default_rng(54)
    own = GpuContext(0)
    kv, dim, n = 2, 64, 16 * 400
    cache = PagedKvCache(own, 1, kv, dim, 400, "q4", track_seqs=1, track_tokens=n)
    s = cache.new_sequence(n, track=True)
    k, q, out = (torch.from_numpy(f32(rng.standard_normal((16, w)))).cuda() for w in (kv * dim, 16 * dim, 16 * dim))
    settle()
    sizes = []
    for at in range(0, n, 16):
        cache.append_device(0, [s], [at], [16], k, k)
        cache.attention_device(0, [s], q[:1], 16, out[:1])
        sizes.append(words.cache_scratch_bytes(own.handle))
    own.synchronize()
    need = n * 16 * 4  # the scores
    assert need <= sizes[-1] <= 4 * need + (1 << 20) and len(set(sizes)) <= 6, sorted(set(sizes))
    cache.close()
    own.close()


def test_a_call_that_gave_up_a_wait_adds_no_weights(ctx, words):
    """The word that such a call's kernel leaves is put there for the next call: its weights stay as they are, those of the call after it are added."""
    rng = np.random.default_rng(55)
    cache = PagedKvCache(ctx, 1, 2, 64, 200, "q4", track_seqs=2, track_tokens=1000)
    lens = [1000, 33]
    seqs, parts = [cache.new_sequence(1000, track=True) for _ in lens], [(rows(rng, n, 2, 64), rows(rng, n, 2, 64)) for n in lens]
    fill(cache, 0, seqs, [0, 0], parts)
    q = f32(rng.standard_normal((2, 8, 64)))
    want = [check_attention(o, x, q4.held(p[0]), q4.held(p[1])) for o, x, p in zip(attend(cache, 0, seqs, q), q, parts)]
    settle()
    number = C.c_ulonglong(words.cache_calls(ctx.handle) + 1)
    assert C.CDLL("libcuda.so.1").cuMemcpyHtoD_v2(C.c_ulonglong(words.cache_gave_up(ctx.handle)), C.byref(number), C.c_size_t(8)) == 0
    for times in (1, 2):  # the call that is marked, and the next one
        attend(cache, 0, seqs, q)
        w = weights(cache, 0, seqs, lens)
        for i, n in enumerate(lens):
            check_weights(w[i][:, :n], times * want[i], q[i], parts[i][0])
    cache.close()


def free_pages(cache, most):
    """How many pages of the pool are free: as many as a sequence of `most` pages can get."""
    s, wide = cache.new_sequence(16 * most), cache.n_kv_heads * cache.head_dim
    x, n = torch.zeros((16, wide), device="cuda"), 0
    settle()
    try:
        for n in range(most + 1):
            cache.append_device(0, [s], [16 * n], [16], x, x)
    except JunoError as e:
        assert "pages free" in str(e)
    except ValueError as e:
        assert "limit" in str(e)
    cache.ctx.synchronize()
    cache.free_sequence(s)
    return n


@pytest.mark.parametrize("both,free", [(False, 3), (False, 2), (True, 5), (True, 4)])
@pytest.mark.parametrize("kv,dim", [(2, 64), (3, 128)])
def test_eviction_with_room_for_shared_pages_alone(ctx, kv, dim, both, free):
    """A branch shares the first two of its pages, and the pool has room for those two but not for all that stay: some pages are fresh, the others are filled in place;
    alone, and together with the sequence that it came from.  With one page less the call is refused."""
    rng = np.random.default_rng(56)
    layers, lens, keep, recent = 2, [160, 140], 100, 17
    cache = PagedKvCache(ctx, layers, kv, dim, 10 + 7 + free, "q4", track_seqs=3, track_tokens=160)
    s = cache.new_sequence(160, track=True)
    have = [[(rows(rng, n, kv, dim), rows(rng, n, kv, dim)) for _ in range(layers)] for n in lens]
    for l in range(layers):
        fill(cache, l, [s], [0], [have[0][l]])
    b = cache.fork(s, 40)
    for l in range(layers):  # the third page is copied when the branch writes to it
        fill(cache, l, [b], [40], [tuple(x[40:] for x in have[1][l])])
        have[1][l] = tuple(np.concatenate([x[:40], y[40:]]) for x, y in zip(have[0][l], have[1][l]))
    w = [some_weights(rng, (layers, kv, n)) for n in lens]
    for l in range(layers):
        for seq, x in ((s, w[0]), (b, w[1])):
            t = dev(x[l][None])
            settle()
            cache.weights_device(l, [seq], [x.shape[-1]], t, store=True)
            settle()
    assert free_pages(cache, 12) == free
    cut = [s, b] if both else [b]
    if free in (2, 4):  # one page less
        other, x = cache.new_sequence(16), torch.zeros((1, kv * dim), device="cuda")
        settle()
        cache.append_device(0, [other], [0], [1], x, x)
        with pytest.raises(JunoError, match="pages free"):
            cache.evict(cut, keep, recent)
        assert [cache.length(q) for q in (s, b)] == lens
        cache.free_sequence(other)
    kept = torch.full((layers, len(cut), kv, keep), 99, dtype=torch.int32, device="cuda")
    settle()
    cache.evict(cut, keep, recent, kept=kept)
    settle()
    for i, seq in enumerate((s, b)):
        if seq in cut:
            want = expected(have[i], w[i], keep, recent)
        else:
            want = [(None, *have[i][l], w[i][l]) for l in range(layers)]
        for l, (at, k, v, wl) in enumerate(want):
            got = read(cache, l, [seq], [0], [len(k)])
            assert np.array_equal(got[0], f32(q4.held(k))) and np.array_equal(got[1], f32(q4.held(v)))
            assert np.array_equal(weights(cache, l, [seq], [len(k)])[0], wl, equal_nan=True)
            if at is not None:
                assert np.array_equal(kept[l, cut.index(seq)].cpu().numpy(), at)
    # the branch needs two fresh pages and gives its last two back; with its source, that gives its last three back and both leave the shared two
    assert free_pages(cache, 12) == free + (3 if both else 0)
    cache.close()


def test_the_example_of_the_readme_follows_the_tensors(ctx):
    """On a stream of its own, behind work that takes longer than the calls: the rows are not there yet when they are made."""
    rng = np.random.default_rng(57)
    k, v, q = f32(rng.standard_normal((5, 8, 128))), f32(rng.standard_normal((5, 8, 128))), f32(rng.standard_normal((1, 32, 128)))
    source = [dev(x.reshape(len(x), -1)) for x in (k, v, q)]
    names = dict(zip("kvq", (torch.full_like(x, 77.0) for x in source)), layer=3, pos=0, n=5, out=torch.full((1, 4096), 77.0, device="cuda"))
    busy = torch.randn((8192, 8192), device="cuda")
    settle()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(8):
            busy = busy @ busy * 1e-2
        for name, x in zip("kvq", source):
            names[name].copy_(x)
        exec(cache_example(), names)
        out = names["out"].clone()
    stream.synchronize()
    check_attention(out.cpu().numpy().reshape(32, 128), q[0], q4.held(k), q4.held(v))
    names["cache"].close()


# Scores beyond FP32 below zero weigh nothing: the result is the mean of the other positions' rows, whose keys are zero.  What the kernel rounds: weights of 2^11 each are
# exact, their products with steps in two limbs 2^-22, the sums of 16 positions a tile and of tiles, warps and parts 2^-24 each, fewer than 30 of them in a row:
# below 2^-18 of terms of up to 3 times the largest value.
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (4, 1, 128), (8, 1, 128)])
@pytest.mark.parametrize("n,bad", [(300, 64), (300, 299), (40, 33), (20000, 15000)])
def test_scores_that_overflow_below_zero(ctx, heads, kv, dim, n, bad):
    rng = np.random.default_rng(58)
    cache = PagedKvCache(ctx, 1, kv, dim, n // 16 + 1, "q4")
    s = cache.new_sequence(n)
    k, v = np.zeros((n, kv, dim), np.float32), f32(rng.standard_normal((n, kv, dim)))
    k[:bad] = -60000.0
    fill(cache, 0, [s], [0], [(k, v)])
    q = np.full((1, heads, dim), 1e37, np.float32)
    want = np.repeat(q4.held(v)[bad:].mean(0), heads // kv, 0)
    got = attend(cache, 0, [s], q)[0]
    assert np.abs(got - want).max() <= 3 * 2.0 ** -18 * np.abs(v).max()
    cache.close()


# Short contexts, every number of heads to a key/value head, rows whole and cut across, by the result's length in each group of a head's dimensions.  A score has up to nine
# sums and products in FP32, each off by 2^-24 of terms up to 30 in size: a weight by 1.6e-5 at most, the limbs of queries, weights and steps add 2^-22 each.  Over positions
# and dimensions that goes both ways; 2e-5 is ten times what such sums are off together.
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("kv,dim", [(2, 64), (2, 128)])
def test_digits_of_every_group_size(ctx, kv, dim, G):
    rng = np.random.default_rng(59 + G)
    lens = [1, 15, 16, 17, 33, 256, 300, 1000, 2500]
    heads = kv * G
    cache = PagedKvCache(ctx, 1, kv, dim, sum(n // 16 + 1 for n in lens), "q4")
    seqs = [cache.new_sequence(n) for n in lens]
    parts = [(rows(rng, n, kv, dim), f32(rng.standard_normal((n, kv, dim)))) for n in lens]
    fill(cache, 0, seqs, [0] * len(lens), parts)
    q = f32(1.5 * rng.standard_normal((len(lens), heads, dim)))
    whole = [attend(cache, 0, [s], q[i:i + 1])[0] for i, s in enumerate(seqs)]
    for out in (attend(cache, 0, seqs, q), whole):
        for i, (k, v) in enumerate(parts):
            want, _ = q4.attention(q[i], q4.held(k), q4.held(v))
            norm = lambda x: np.linalg.norm(x.reshape(heads, -1, 32), axis=-1)  # noqa: E731
            assert (norm(out[i] - want) <= 2e-5 * norm(want)).all(), (lens[i], (norm(out[i] - want) / norm(want)).max())
    cache.close()


def test_nothing_of_a_cache_goes_into_a_graph_of_the_contexts_stream(ctx):
    """Forks, tracking and the host-memory calls change page tables on that stream: refused while it is captured, and as usual afterwards."""
    rng = np.random.default_rng(60)
    handle = C.c_void_p()
    own = GpuContext(0)
    assert own._L.juno_ctx_stream(own.handle, C.byref(handle)) == 0
    stream = torch.cuda.ExternalStream(handle.value)
    cache = PagedKvCache(own, 1, 2, 64, 16, "q4", track_seqs=2, track_tokens=64)
    s, t = cache.new_sequence(64), cache.new_sequence(64, track=True)
    k = rows(rng, 40, 2, 64)
    cache.append(s, 0, 0, k.reshape(40, -1), k.reshape(40, -1))
    q = f32(rng.standard_normal((1, 8, 64)))
    x = torch.zeros(4, device="cuda")
    settle()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream, capture_error_mode="relaxed"):
        y = x + 1
        for call in (lambda: cache.fork(s, 20), lambda: cache.fork(t, 0), lambda: cache.new_sequence(64, track=True), lambda: cache.attention(0, [s], q.reshape(1, -1), 8),
                     lambda: cache.append(s, 0, 40, k[:8].reshape(8, -1), k[:8].reshape(8, -1)), lambda: cache.evict([t], 1)):
            with pytest.raises(ValueError, match="captured"):
                call()
    g.replay()
    settle()
    assert (y == 1).all() and cache.length(s) == 40
    b = cache.fork(s, 20)
    cache.append(b, 0, 20, k[:8].reshape(8, -1), k[:8].reshape(8, -1))
    both = np.concatenate([k[:20], k[:8]])
    check_attention(cache.attention(0, [b], q.reshape(1, -1), 8).reshape(8, 64), q[0], q4.held(both), q4.held(both))
    cache.free_sequence(cache.new_sequence(64, track=True))
    del g
    cache.close()
    own.close()

"""4-bit cache pages on the GPU against the oracle's 64 bits: append and read, decode attention, accumulated weights, eviction, and all of them in turn."""
import ctypes as C

import numpy as np
import pytest
import torch

from juno_b200 import _lib
from juno_b200._lib import JunoError
from juno_b200.matvec import GpuContext, PagedKvCache
from oracle import q4_cache_oracle as q4
from q4util import attention_tolerance, rows

pytestmark = pytest.mark.gpu


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def settle(*contexts):
    """Torch's work is on streams of its own: what it wrote is there before the context's stream reads it, and the other way round."""
    torch.cuda.synchronize()


def fill(cache, layer, seqs, positions, parts, **kw):
    """Appends parts[i] = (k, v) [n, kv, dim] to sequence i."""
    wide = cache.n_kv_heads * cache.head_dim
    k, v = (dev(np.concatenate([p[j].reshape(-1, wide) for p in parts])) for j in (0, 1))
    settle()
    cache.append_device(layer, seqs, positions, [len(p[0]) for p in parts], k, v, **kw)
    settle()


def read(cache, layer, seqs, positions, counts):
    wide = cache.n_kv_heads * cache.head_dim
    k, v = (torch.full((sum(counts), wide), 77.0, device="cuda") for _ in range(2))
    settle()
    cache.read_device(layer, seqs, positions, counts, k, v)
    settle()
    return k.cpu().numpy().reshape(-1, cache.n_kv_heads, cache.head_dim), v.cpu().numpy().reshape(-1, cache.n_kv_heads, cache.head_dim)


def attend(cache, layer, seqs, q, lens=None):
    """q [n, heads, dim]"""
    n, heads, dim = q.shape
    x, out = dev(q.reshape(n, -1)), torch.full((n, heads * dim), 77.0, device="cuda")
    settle()
    cache.attention_device(layer, seqs, x, heads, out, lens=lens)
    settle()
    return out.cpu().numpy().reshape(n, heads, dim)


def weights(cache, layer, seqs, counts):
    w = torch.zeros((len(seqs), cache.n_kv_heads, max(counts)), device="cuda")
    settle()
    cache.weights_device(layer, seqs, counts, w)
    settle()
    return w.cpu().numpy()


def f32(x):
    return x.astype(np.float32)


def check_attention(got, q, k, v):
    ref, w = q4.attention(q, k, v)
    rel, top = attention_tolerance(q, k, v, q.shape[-1])
    assert np.abs(got - ref).max() <= rel * top, (np.abs(got - ref).max() / top, rel)
    return w


# ── append and read ───────────────────────────────────────────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("kv,dim", [(1, 64), (4, 64), (8, 128), (3, 128)])
def test_rows_are_held_as_the_oracle_says(ctx, kv, dim):
    rng = np.random.default_rng(kv * dim)
    cache = PagedKvCache(ctx, 3, kv, dim, 64, "q4")
    seqs = [cache.new_sequence(300) for _ in range(4)]
    have = [(np.empty((0, kv, dim), np.float32),) * 2 for _ in seqs]
    for counts in ([1, 0, 15, 33], [16, 1, 2, 0], [0, 200, 1, 1], [3, 5, 7, 17]):  # odd starts, pages that end inside a part, nothing for some
        parts = [(rows(rng, n, kv, dim), f32(rng.standard_normal((n, kv, dim)))) for n in counts]
        fill(cache, 1, seqs, [len(h[0]) for h in have], parts)
        have = [tuple(np.concatenate([a, b]) for a, b in zip(h, p)) for h, p in zip(have, parts)]
    assert [cache.length(s) for s in seqs] == [len(h[0]) for h in have]
    k, v = read(cache, 1, seqs, [0] * 4, [len(h[0]) for h in have])
    assert np.array_equal(k, f32(q4.held(np.concatenate([h[0] for h in have]))))
    assert np.array_equal(v, f32(q4.held(np.concatenate([h[1] for h in have]))))
    k, v = read(cache, 1, [seqs[1], seqs[3], seqs[1]], [7, 0, 199], [30, 0, 2])  # parts, twice the same sequence
    assert np.array_equal(k, f32(q4.held(np.concatenate([have[1][0][7:37], have[1][0][199:201]]))))
    new = (rows(rng, 20, kv, dim), rows(rng, 20, kv, dim))  # written over: the rows behind stay
    fill(cache, 1, [seqs[1]], [9], [new])
    k, v = read(cache, 1, [seqs[1]], [0], [len(have[1][0])])
    want = have[1][0].copy()
    want[9:29] = new[0]
    assert np.array_equal(k, f32(q4.held(want))) and cache.length(seqs[1]) == len(want)
    cache.close()


@pytest.mark.parametrize("offset,extra", [(0, 0), (1, 3), (2, 5), (4, 4)])
def test_rows_of_other_strides_and_alignments(ctx, offset, extra):
    kv, dim, n = 2, 64, 21
    rng = np.random.default_rng(offset)
    x, y = rows(rng, n, kv, dim).reshape(n, -1), rows(rng, n, kv, dim).reshape(n, -1)
    wide = kv * dim + extra
    buf = [torch.full((n * wide + offset,), 3.0, device="cuda") for _ in range(4)]
    k, v, ko, vo = (b[offset:offset + n * wide].view(n, wide)[:, :kv * dim] for b in buf)
    k.copy_(dev(x)), v.copy_(dev(y))
    cache = PagedKvCache(ctx, 1, kv, dim, 8, "q4")
    s = cache.new_sequence(64)
    settle()
    cache.append_device(0, [s], [0], [n], k, v)
    cache.read_device(0, [s], [0], [n], ko, vo)
    settle()
    assert np.array_equal(ko.cpu().numpy(), f32(q4.held(x.reshape(n, kv, dim))).reshape(n, -1))
    assert np.array_equal(vo.cpu().numpy(), f32(q4.held(y.reshape(n, kv, dim))).reshape(n, -1))
    for b in buf[2:]:  # what lies beside the rows is left alone
        assert (b[:offset] == 3).all() and (extra == 0 or (b[offset:].view(n, wide)[:, kv * dim:] == 3).all())
    cache.close()


def special_rows(rng, kv, dim):
    x = rows(rng, 12, kv, dim)
    x[0, 0, 3] = np.nan
    x[1, 0, 5], x[1, 0, 6], x[1, 0, 40] = np.inf, -np.inf, 1e30
    x[2] = 7.25
    x[3] = 0.0
    x[4] = -0.0
    x[5] *= np.float32(1e-8)
    x[6] *= np.float32(1e-30)
    x[7] = 1000.0 + 1e-3 * x[7]
    x[8, :, ::2] = 65504.0
    x[9, :, 1::3] = -70000.0
    x[10] = np.float32(2.0) ** rng.integers(-24, 15, x[10].shape)
    x[11] = (np.arange(dim) % 31) * 0.5  # d = 1: every odd multiple lies half-way between two numbers
    return x


def test_special_values(ctx):
    rng = np.random.default_rng(3)
    cache = PagedKvCache(ctx, 1, 2, 128, 4, "q4")
    s = cache.new_sequence(32)
    x = special_rows(rng, 2, 128)
    fill(cache, 0, [s], [0], [(x, x[::-1].copy())])
    k, v = read(cache, 0, [s], [0], [12])
    assert np.array_equal(k, f32(q4.held(x)), equal_nan=True) and np.array_equal(v, f32(q4.held(x[::-1])), equal_nan=True)
    cache.close()


@pytest.mark.parametrize("kv_dtype,kind", [("f16", np.float16), ("f32", np.float32)])
def test_append_and_read_serve_the_other_pages_too(ctx, kv_dtype, kind):
    rng = np.random.default_rng(4)
    cache = PagedKvCache(ctx, 2, 4, 64, 32, kv_dtype)
    seqs = [cache.new_sequence(100) for _ in range(2)]
    parts = [(rows(rng, n, 4, 64), rows(rng, n, 4, 64)) for n in (37, 5)]
    fill(cache, 1, seqs, [0, 0], parts)
    k, v = read(cache, 1, seqs, [0, 0], [37, 5])
    assert np.array_equal(k, f32(np.concatenate([p[0] for p in parts]).astype(kind)))
    assert np.array_equal(v, f32(np.concatenate([p[1] for p in parts]).astype(kind)))
    q = rng.standard_normal((2, 16 * 64)).astype(np.float32)
    out = cache.attention(1, seqs, q, 16)
    for i, p in enumerate(parts):
        check_attention(out[i].reshape(16, 64), q[i].reshape(16, 64), p[0].astype(kind).astype(np.float64), p[1].astype(kind).astype(np.float64))
    cache.close()


def test_host_calls_on_4_bit_pages(ctx):
    rng = np.random.default_rng(9)
    cache = PagedKvCache(ctx, 1, 8, 128, 64, "q4")
    seqs, have = [cache.new_sequence(400) for _ in range(2)], []
    for s, n in zip(seqs, (301, 17)):
        k, v = rows(rng, n, 8, 128), rows(rng, n, 8, 128)
        cache.append(s, 0, 0, k[:5], v[:5])
        cache.append(s, 0, 5, k[5:], v[5:])
        have.append((k, v))
    k, v = read(cache, 0, seqs, [0, 0], [301, 17])
    assert np.array_equal(k, f32(q4.held(np.concatenate([h[0] for h in have]))))
    q = rng.standard_normal((2, 32, 128)).astype(np.float32)
    out = cache.attention(0, seqs, q.reshape(2, -1), 32).reshape(2, 32, 128)
    assert np.array_equal(out, attend(cache, 0, seqs, q))
    for i, h in enumerate(have):
        check_attention(out[i], q[i], q4.held(h[0]), q4.held(h[1]))
    with pytest.raises(ValueError, match="not behind"):
        cache.append(seqs[1], 0, 18, k[:1], v[:1])
    cache.close()


# ── attention ─────────────────────────────────────────────────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("kv,dim", [(2, 64), (3, 128)])
def test_attention_of_every_group_size(ctx, kv, dim, G):
    rng = np.random.default_rng(100 * G + dim)
    lens = [1, 15, 16, 17, 31, 33, 257, 1000]
    cache = PagedKvCache(ctx, 2, kv, dim, 120, "q4")
    seqs = [cache.new_sequence(1000) for _ in lens]
    parts = [(rows(rng, n, kv, dim), f32(rng.standard_normal((n, kv, dim)))) for n in lens]
    fill(cache, 1, seqs, [0] * len(lens), parts)
    q = f32(1.5 * rng.standard_normal((len(lens), G * kv, dim)))
    out = attend(cache, 1, seqs, q)
    for i, p in enumerate(parts):
        check_attention(out[i], q[i], q4.held(p[0]), q4.held(p[1]))
    cache.close()


@pytest.mark.parametrize("n,heads,kv,dim", [(20001, 32, 8, 128), (9999, 8, 4, 64), (33000, 8, 1, 128)])
def test_attention_of_long_contexts(ctx, n, heads, kv, dim):
    rng = np.random.default_rng(n)
    cache = PagedKvCache(ctx, 1, kv, dim, n // 16 + 1, "q4")
    s = cache.new_sequence(n)
    k, v = rows(rng, n, kv, dim), f32(rng.standard_normal((n, kv, dim)))
    k[n // 2, 0] *= 6  # one key that stands out
    fill(cache, 0, [s], [0], [(k, v)])
    q = f32(rng.standard_normal((1, heads, dim)))
    check_attention(attend(cache, 0, [s], q)[0], q[0], q4.held(k), q4.held(v))
    cache.close()


# Zero-mean values in a long context: the result is smaller than the sum of the weighted magnitudes by the root of the number of positions that count, so an error
# that goes one way (sums cut off instead of rounded) shows.  In 64 bits from the rows that the pages hold.  What the kernel rounds: a score's 5 to 9 sums and products
# in FP32, each to 2^-24 of terms up to 30 in size, together about 2e-6 of a weight, at random over the positions; weights in limbs, 2^-22.  So about 2e-6 of the
# result's length; 1e-5 leaves a factor of five.  Sums cut off at 2^-24 give 1e-4 here.
@pytest.mark.parametrize("n,batch,heads,kv,dim", [(65536, 1, 32, 8, 128), (16384, 7, 32, 4, 128), (9001, 16, 16, 4, 64), (30000, 5, 24, 4, 64), (12000, 40, 2, 1, 64)])
def test_long_sums_are_not_biased(ctx, n, batch, heads, kv, dim):
    g = torch.Generator("cuda")
    g.manual_seed(n)
    draw = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    cache = PagedKvCache(ctx, 1, kv, dim, batch * (n // 16 + 1), "q4")
    try:
        seqs = [cache.new_sequence(n) for _ in range(batch)]
        k = draw(batch * n, kv, dim) * (0.5 * draw(kv, dim)).exp() + 0.5 * draw(kv, dim)
        v, q = 0.5 * draw(batch * n, kv * dim), 1.5 * draw(batch, heads * dim)
        held_k, held_v, out = torch.empty_like(v), torch.empty_like(v), torch.empty_like(q)
        settle()
        cache.append_device(0, seqs, [0] * batch, [n] * batch, k.flatten(1), v)
        cache.read_device(0, seqs, [0] * batch, [n] * batch, held_k, held_v)
        cache.attention_device(0, seqs, q, heads, out)
        ctx.synchronize()
        for i in range(batch):
            for h in range(kv):
                of = lambda x: x[i * n:(i + 1) * n, h * dim:(h + 1) * dim].double()  # noqa: E731
                mine = slice(h * heads // kv * dim, (h + 1) * heads // kv * dim)
                x = q[i, mine].double().view(-1, dim) @ of(held_k).T / dim ** 0.5
                ref = torch.softmax(x, -1) @ of(held_v)
                error = (out[i, mine].double().view(-1, dim) - ref).norm(dim=-1) / ref.norm(dim=-1)
                assert error.max() <= 1e-5, (i, h, error)
    finally:
        cache.close()


def test_attention_of_many_short_sequences_and_of_parts(ctx):
    """More sequences than travel with a launch; a prompt's rows: one sequence many times, each time one position more, none at first."""
    rng = np.random.default_rng(11)
    kv, dim, n = 2, 64, 130
    cache = PagedKvCache(ctx, 1, kv, dim, 600, "q4")
    lens = rng.integers(1, 60, n).tolist()
    seqs = [cache.new_sequence(64) for _ in lens]
    parts = [(rows(rng, m, kv, dim), f32(rng.standard_normal((m, kv, dim)))) for m in lens]
    fill(cache, 0, seqs, [0] * n, parts)
    q = f32(rng.standard_normal((n, 8, dim)))
    out = attend(cache, 0, seqs, q)
    for i, p in enumerate(parts):
        check_attention(out[i], q[i], q4.held(p[0]), q4.held(p[1]))
    m = lens[5]
    out = attend(cache, 0, [seqs[5]] * (m + 1), q[:m + 1], lens=list(range(m + 1)))
    assert (out[0] == 0).all()
    for j in range(1, m + 1):
        check_attention(out[j], q[j], q4.held(parts[5][0][:j]), q4.held(parts[5][1][:j]))
    cache.close()


def test_positions_behind_the_end_do_not_count_whatever_they_hold(ctx):
    rng = np.random.default_rng(12)
    for dim in (64, 128):
        cache = PagedKvCache(ctx, 1, 2, dim, 40, "q4")
        s = cache.new_sequence(500)
        k, v = rows(rng, 450, 2, dim), f32(rng.standard_normal((450, 2, dim)))
        bad = k.copy()
        bad[::2], bad[1::2] = np.nan, np.inf
        fill(cache, 0, [s], [0], [(bad, bad)])
        q = f32(rng.standard_normal((1, 8, dim)))
        assert np.isnan(attend(cache, 0, [s], q)).all()  # attended, a NaN is one
        for n in (1, 9, 16, 40, 300):
            fill(cache, 0, [s], [0], [(k[:n], v[:n])])
            check_attention(attend(cache, 0, [s], q, lens=[n])[0], q[0], q4.held(k[:n]), q4.held(v[:n]))
        cache.close()


def test_scores_far_apart(ctx):
    """Weights over hundreds of powers of two: the largest score last, first, and in the middle of a split."""
    rng = np.random.default_rng(13)
    cache = PagedKvCache(ctx, 1, 1, 128, 80, "q4")
    for place in (0, 77, 1199):
        s = cache.new_sequence(1200)
        k, v = f32(0.05 * rng.standard_normal((1200, 1, 128))), f32(rng.standard_normal((1200, 1, 128)))
        q = f32(4.0 * rng.standard_normal((1, 4, 128)))
        k[place, 0] = q[0, 1]
        k[(place + 600) % 1200, 0] = -q[0, 2]
        fill(cache, 0, [s], [0], [(k, v)])
        check_attention(attend(cache, 0, [s], q)[0], q[0], q4.held(k), q4.held(v))
        cache.free_sequence(s)
    cache.close()


def test_values_of_any_size_keep_their_digits(ctx):
    rng = np.random.default_rng(14)
    cache = PagedKvCache(ctx, 1, 1, 64, 20, "q4")
    for size in (1e-20, 1e-6, 1.0, 3e3):
        s = cache.new_sequence(200)
        k, v = rows(rng, 200, 1, 64), f32(size * rng.standard_normal((200, 1, 64)))
        q = f32(rng.standard_normal((1, 4, 64)))
        fill(cache, 0, [s], [0], [(k, v)])
        check_attention(attend(cache, 0, [s], q)[0], q[0], q4.held(k), q4.held(v))
        cache.free_sequence(s)
    cache.close()


def test_rows_of_queries_and_results_apart(ctx):
    rng = np.random.default_rng(15)
    cache = PagedKvCache(ctx, 1, 2, 64, 20, "q4")
    s = cache.new_sequence(200)
    k, v = rows(rng, 150, 2, 64), rows(rng, 150, 2, 64)
    fill(cache, 0, [s], [0], [(k, v)])
    q = f32(rng.standard_normal((3, 8, 64)))
    whole, out = torch.full((3, 8 * 64 + 301), 5.0, device="cuda"), torch.full((3, 8 * 64 + 7), 5.0, device="cuda")
    whole[:, 13:13 + 512] = dev(q.reshape(3, -1))
    settle()
    cache.attention_device(0, [s] * 3, whole[:, 13:13 + 512], 8, out[:, 3:3 + 512], lens=[150, 20, 1])
    settle()
    for i, n in enumerate((150, 20, 1)):
        check_attention(out[i, 3:3 + 512].cpu().numpy().reshape(8, 64), q[i], q4.held(k[:n]), q4.held(v[:n]))
    assert (out[:, :3] == 5).all() and (out[:, 515:] == 5).all()
    cache.close()


def test_the_same_call_gives_the_same_bits(ctx):
    rng = np.random.default_rng(16)
    cache = PagedKvCache(ctx, 1, 8, 128, 400, "q4", track_seqs=2, track_tokens=4000)
    seqs = [cache.new_sequence(4000, track=True) for _ in range(2)]
    parts = [(rows(rng, n, 8, 128), rows(rng, n, 8, 128)) for n in (3999, 1234)]
    q = f32(rng.standard_normal((2, 32, 128)))
    got = []
    for _ in range(3):
        fill(cache, 0, seqs, [0, 0], parts)  # the weights start again
        got.append((attend(cache, 0, seqs, q), weights(cache, 0, seqs, [3999, 1234])))
    assert all(np.array_equal(a, b) for g in got[1:] for a, b in zip(got[0], g))
    cache.close()


def test_a_cache_beyond_32_bit_offsets(ctx):
    """The last layer of a pool of 6 GB: its blocks lie behind 2^32 bytes."""
    kv, dim, layers, pages = 8, 128, 64, 4700
    cache = PagedKvCache(ctx, layers, kv, dim, pages, "q4")
    rng = np.random.default_rng(17)
    s = cache.new_sequence(3000)
    k, v = rows(rng, 2999, kv, dim), rows(rng, 2999, kv, dim)
    fill(cache, layers - 1, [s], [0], [(k, v)])
    got = read(cache, layers - 1, [s], [0], [2999])
    assert np.array_equal(got[0], f32(q4.held(k))) and np.array_equal(got[1], f32(q4.held(v)))
    q = f32(rng.standard_normal((1, 32, dim)))
    check_attention(attend(cache, layers - 1, [s], q)[0], q[0], q4.held(k), q4.held(v))
    cache.close()


# ── weights and eviction ──────────────────────────────────────────────────────────────────────────────────────────────────────

def check_weights(got, want, q, k):
    """A weight is a softmax weight summed over the heads of a group and over calls: off by what attention's weights are (attention_tolerance with values of
    1), and one rounding per addition."""
    rel, _ = attention_tolerance(q, k, np.ones(1), q.shape[-1])
    assert (np.abs(got - want) <= rel * np.abs(want) + 1e-30).all(), np.nanmax(np.abs(got - want) / want)


@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (6, 2, 64), (16, 2, 128)])
def test_weights_add_up(ctx, heads, kv, dim):
    rng = np.random.default_rng(heads)
    lens = [1, 16, 333, 2100]
    cache = PagedKvCache(ctx, 2, kv, dim, 200, "q4", track_seqs=3, track_tokens=2110)
    seqs = [cache.new_sequence(2110, track=i != 1) for i in range(4)]  # one of them keeps none
    parts = [(rows(rng, n, kv, dim), rows(rng, n, kv, dim)) for n in lens]
    fill(cache, 1, seqs, [0] * 4, parts)
    sums = [np.zeros((kv, n)) for n in lens]
    for step in range(3):
        q = f32(rng.standard_normal((4, heads, dim)))
        at = lens if step != 1 else [1, 9, 300, 2000]
        out = attend(cache, 1, seqs, q, lens=at)
        for i, p in enumerate(parts):
            sums[i][:, :at[i]] += check_attention(out[i], q[i], q4.held(p[0][:at[i]]), q4.held(p[1][:at[i]]))
    kept = [seqs[i] for i in (0, 2, 3)]
    w = weights(cache, 1, kept, [lens[i] for i in (0, 2, 3)])
    for j, i in enumerate((0, 2, 3)):
        check_weights(w[j][:, :lens[i]], sums[i], q, parts[i][0])
    assert (weights(cache, 0, kept, [1, 1, 1]) == 0).all()  # the other layer has none
    fill(cache, 1, [seqs[2]], [300], [(parts[2][0][:40], parts[2][1][:40])])  # positions that are written anew begin at zero
    w = weights(cache, 1, [seqs[2]], [340])[0]
    assert (w[:, 300:] == 0).all() and (w[:, :300] > 0).all()
    with pytest.raises(ValueError, match="keeps no weights"):
        weights(cache, 1, [seqs[1]], [1])
    cache.close()


def expected(have, w, keep, recent):
    """have: per layer (k, v) [n, kv, dim], w: [layers, kv, n] -> places and the rows that stay, per layer."""
    out = []
    for l, (k, v) in enumerate(have):
        at = np.stack([q4.kept(w[l, h], keep, recent) for h in range(k.shape[1])])
        out.append((at, np.stack([k[at[h], h] for h in range(len(at))], 1), np.stack([v[at[h], h] for h in range(len(at))], 1), np.take_along_axis(w[l], at, 1)))
    return out


def some_weights(rng, shape):
    """Many equal ones among them, zeros of both signs and a NaN."""
    w = np.round(np.exp(2 * rng.standard_normal(shape)) * 4).astype(np.float32) / 4
    w[rng.random(shape) < 0.1] = -0.0
    w[..., 0] = np.nan
    return w


@pytest.mark.parametrize("kv,dim,keep,recent", [(2, 64, 1, 0), (2, 64, 16, 16), (8, 128, 100, 17), (3, 128, 333, 0), (1, 64, 500, 499), (4, 64, 1000, 64)])
def test_eviction_keeps_what_the_oracle_keeps(ctx, kv, dim, keep, recent):
    rng = np.random.default_rng(keep)
    layers, lens = 2, [1100, 501, max(1, keep - 1), 64, keep, keep + 1]
    cache = PagedKvCache(ctx, layers, kv, dim, 400, "q4", track_seqs=6, track_tokens=1200)
    seqs = [cache.new_sequence(1200, track=True) for _ in lens]
    have = [[(rows(rng, n, kv, dim), rows(rng, n, kv, dim)) for _ in range(layers)] for n in lens]
    w = [some_weights(rng, (layers, kv, n)) for n in lens]
    for l in range(layers):
        fill(cache, l, seqs, [0] * len(lens), [h[l] for h in have])
        buf = np.zeros((len(lens), kv, max(lens)), np.float32)
        for i, n in enumerate(lens):
            buf[i, :, :n] = w[i][l]
        t = dev(buf)
        settle()
        cache.weights_device(l, seqs, lens, t, store=True)
        settle()
    kept = torch.full((layers, len(lens), kv, keep), 99, dtype=torch.int32, device="cuda")
    settle()
    cache.evict(seqs, keep, recent, kept=kept)
    settle()
    kept = kept.cpu().numpy()
    now = [min(n, keep) for n in lens]
    assert [cache.length(s) for s in seqs] == now
    for i, n in enumerate(now):
        for l, (at, k, v, wl) in enumerate(expected(have[i], w[i], keep, recent)):
            assert np.array_equal(kept[l, i, :, :n], at) and (kept[l, i, :, n:] == -1).all()
            got = read(cache, l, [seqs[i]], [0], [n])
            assert np.array_equal(got[0], f32(q4.held(k))) and np.array_equal(got[1], f32(q4.held(v)))
            assert np.array_equal(weights(cache, l, [seqs[i]], [n])[0], wl, equal_nan=True)
    cache.close()


@pytest.mark.parametrize("n,keep,recent", [(24576, 9000, 100), (24577, 24576, 0), (60001, 777, 77)])
def test_eviction_of_long_sequences(ctx, n, keep, recent):
    """More weights than shared memory holds, and exactly as many."""
    rng = np.random.default_rng(n)
    kv, dim = 2, 64
    cache = PagedKvCache(ctx, 1, kv, dim, (n + keep) // 16 + 2, "q4", track_seqs=1, track_tokens=n)
    s = cache.new_sequence(n, track=True)
    have = (rows(rng, n, kv, dim), rows(rng, n, kv, dim))
    fill(cache, 0, [s], [0], [have])
    w = some_weights(rng, (1, kv, n))
    t, kept = dev(w), torch.full((1, 1, kv, keep), 99, dtype=torch.int32, device="cuda")
    settle()
    cache.weights_device(0, [s], [n], t, store=True)
    cache.evict([s], keep, recent, kept=kept)
    settle()
    at, k, v, wl = expected([have], w, keep, recent)[0]
    assert np.array_equal(kept.cpu().numpy()[0, 0], at)
    got = read(cache, 0, [s], [0], [keep])
    assert np.array_equal(got[0], f32(q4.held(k))) and np.array_equal(got[1], f32(q4.held(v)))
    assert np.array_equal(weights(cache, 0, [s], [keep])[0], wl, equal_nan=True)
    cache.close()


@pytest.mark.parametrize("n,branches", [(40000, 1), (500, 60)])
def test_branches_are_cut_down_alone(ctx, n, branches):
    """A long branch, whose page table takes several launches, and many at once, whose rows and pages do not fit into one; the sequence they come from stays."""
    rng = np.random.default_rng(branches)
    kv, dim, keep, recent = 2, 64, 300, 40
    cache = PagedKvCache(ctx, 1, kv, dim, (n + 15) // 16 + branches * ((keep + 15) // 16), "q4", track_seqs=branches + 1, track_tokens=n)
    s = cache.new_sequence(n, track=True)
    have = (rows(rng, n, kv, dim), rows(rng, n, kv, dim))
    fill(cache, 0, [s], [0], [have])
    w = some_weights(rng, (1, kv, n))
    t = dev(w)
    settle()
    cache.weights_device(0, [s], [n], t, store=True)
    of = [n - i for i in range(branches)]
    cut = [cache.fork(s, m) for m in of]
    kept = torch.full((1, branches, kv, keep), 99, dtype=torch.int32, device="cuda")
    settle()
    cache.evict(cut, keep, recent, kept=kept)
    settle()
    got, got_w = read(cache, 0, cut, [0] * branches, [keep] * branches), weights(cache, 0, cut, [keep] * branches)
    for i, m in enumerate(of):
        at, k, v, wl = expected([(have[0][:m], have[1][:m])], w[..., :m], keep, recent)[0]
        assert np.array_equal(kept.cpu().numpy()[0, i], at)
        mine = slice(i * keep, (i + 1) * keep)
        assert np.array_equal(got[0][mine], f32(q4.held(k))) and np.array_equal(got[1][mine], f32(q4.held(v)))
        assert np.array_equal(got_w[i], wl, equal_nan=True)
    whole = read(cache, 0, [s], [0], [n])
    assert np.array_equal(whole[0], f32(q4.held(have[0]))) and np.array_equal(whole[1], f32(q4.held(have[1])))
    assert np.array_equal(weights(cache, 0, [s], [n])[0], w[0], equal_nan=True)
    cache.close()


@pytest.mark.parametrize("kv,dim", [(2, 64), (3, 128)])
def test_eviction_in_a_full_pool_moves_rows_in_place(ctx, kv, dim):
    """No page is free: sequences are cut down within their own pages, one of them shares its first pages with a shorter one and is refused."""
    rng = np.random.default_rng(dim)
    lens, keep, recent, layers = [333, 250, 90], 100, 20, 2
    cache = PagedKvCache(ctx, layers, kv, dim, sum((n + 15) // 16 for n in lens), "q4", track_seqs=4, track_tokens=336)
    seqs = [cache.new_sequence(336, track=True) for _ in lens]
    have = [[(rows(rng, n, kv, dim), rows(rng, n, kv, dim)) for _ in range(layers)] for n in lens]
    w = [some_weights(rng, (layers, kv, n)) for n in lens]
    for l in range(layers):
        fill(cache, l, seqs, [0] * 3, [h[l] for h in have])
        buf = np.zeros((3, kv, max(lens)), np.float32)
        for i, n in enumerate(lens):
            buf[i, :, :n] = w[i][l]
        t = dev(buf)
        settle()
        cache.weights_device(l, seqs, lens, t, store=True)
        settle()
    b = cache.fork(seqs[1], 30)
    with pytest.raises(JunoError, match="pages free"):
        cache.evict(seqs, keep, recent)
    assert [cache.length(s) for s in seqs] == lens
    cache.free_sequence(b)
    cache.evict(seqs, keep, recent)
    settle()
    for i, s in enumerate(seqs):
        for l, (_, k, v, wl) in enumerate(expected(have[i], w[i], keep, recent)):
            got = read(cache, l, [s], [0], [len(k)])
            assert np.array_equal(got[0], f32(q4.held(k))) and np.array_equal(got[1], f32(q4.held(v)))
            assert np.array_equal(weights(cache, l, [s], [len(k)])[0], wl, equal_nan=True)
    cache.close()


def test_eviction_gives_pages_back_and_leaves_shared_ones(ctx):
    """A pool that a branch and its source fill but for the branch's new pages; without room nothing changes."""
    rng = np.random.default_rng(21)
    kv, dim, n, keep = 2, 64, 160, 40
    cache = PagedKvCache(ctx, 1, kv, dim, 10 + 2, "q4", track_seqs=3, track_tokens=160)
    s = cache.new_sequence(160, track=True)
    have = (rows(rng, n, kv, dim), rows(rng, n, kv, dim))
    fill(cache, 0, [s], [0], [have])
    w = some_weights(rng, (1, kv, n))
    t = dev(w)
    settle()
    cache.weights_device(0, [s], [n], t, store=True)
    b = cache.fork(s, n)
    with pytest.raises(JunoError, match="pages free"):
        cache.evict([b], keep, 8)
    assert cache.length(b) == n
    cache.evict([b], 32, 8)
    settle()
    for seq, rest in ((s, [(np.arange(n)[None].repeat(kv, 0), *have, w[0])]), (b, expected([have], w, 32, 8))):
        _, k, v, wl = rest[0]
        got = read(cache, 0, [seq], [0], [len(k)])
        assert np.array_equal(got[0], f32(q4.held(k))) and np.array_equal(got[1], f32(q4.held(v)))
        assert np.array_equal(weights(cache, 0, [seq], [len(k)])[0], wl, equal_nan=True)
    cache.free_sequence(s)  # its ten pages are free again, and no others
    c = cache.new_sequence(160)
    fill(cache, 0, [c], [0], [have])
    d = cache.new_sequence(16)
    with pytest.raises(JunoError, match="pages free"):
        fill(cache, 0, [d], [0], [(have[0][:1], have[1][:1])])
    got = read(cache, 0, [b], [0], [32])
    assert np.array_equal(got[0], f32(q4.held(expected([have], w, 32, 8)[0][1])))
    cache.close()


def test_a_bounded_cache_step_by_step(ctx):
    """As it is used: prompts, then steps that append, attend and cut the cache down when it is over its budget, against the oracle that does the same;
    nothing waits between the calls."""
    rng = np.random.default_rng(22)
    kv, dim, heads, layers, keep, recent, most = 2, 128, 8, 2, 48, 12, 64
    cache = PagedKvCache(ctx, layers, kv, dim, 16, "q4", track_seqs=2, track_tokens=most)
    seqs = [cache.new_sequence(most, track=True) for _ in range(2)]
    b = cache.batch(seqs)
    have = [[[np.empty((0, kv, dim)), np.empty((0, kv, dim)), np.zeros((kv, 0))] for _ in range(layers)] for _ in seqs]
    new = [[(rows(rng, 30 + 9 * i, kv, dim), rows(rng, 30 + 9 * i, kv, dim)) for _ in range(layers)] for i in range(2)]
    calls, outs = [], []
    for step in range(60):
        if step:
            new = [[(rows(rng, 1, kv, dim), rows(rng, 1, kv, dim)) for _ in range(layers)] for _ in seqs]
        counts, at = [len(n[0][0]) for n in new], [h[0][0].shape[0] for h in have]
        for l in range(layers):
            k, v = (dev(np.concatenate([n[l][j].reshape(-1, kv * dim) for n in new])) for j in (0, 1))
            q = f32(rng.standard_normal((2, heads, dim)))
            calls.append((l, at, counts, k, v, q, dev(q.reshape(2, -1)), torch.zeros((2, heads * dim), device="cuda")))
            for i in range(2):
                h = have[i][l]
                h[0], h[1], h[2] = np.concatenate([h[0], q4.held(new[i][l][0])]), np.concatenate([h[1], q4.held(new[i][l][1])]), np.pad(h[2], ((0, 0), (0, counts[i])))
                ref, w = q4.attention(q[i], h[0], h[1])
                h[2] = h[2] + w
                outs.append((len(calls) - 1, i, ref, attention_tolerance(q[i], h[0], h[1], dim)))
        if any(h[0][0].shape[0] >= most for h in have):
            calls.append(None)
            for i in range(2):
                if have[i][0][0].shape[0] > keep:
                    for l in range(layers):
                        h = have[i][l]
                        places = np.stack([q4.kept(h[2][x], keep, recent) for x in range(kv)])
                        h[0], h[1] = (np.stack([h[j][places[x], x] for x in range(kv)], 1) for j in (0, 1))
                        h[2] = np.take_along_axis(h[2], places, 1)
    settle()
    for c in calls:
        if c is None:
            cache.evict(b, keep, recent)
        else:
            cache.append_device(c[0], b, c[1], c[2], c[3], c[4])
            cache.attention_device(c[0], b, c[6], heads, c[7])
    settle()
    assert sum(c is None for c in calls) >= 2
    for call, i, ref, (rel, top) in outs:
        got = calls[call][7][i].cpu().numpy().reshape(heads, dim)
        assert np.abs(got - ref).max() <= rel * top, call
    cache.close()


# ── streams and order ─────────────────────────────────────────────────────────────────────────────────────────────────────────

def test_calls_on_several_streams_take_effect_in_order(ctx):
    rng = np.random.default_rng(23)
    kv, dim = 8, 128
    cache = PagedKvCache(ctx, 1, kv, dim, 800, "q4", track_seqs=4, track_tokens=3000)
    k, v = rows(rng, 2800, kv, dim), rows(rng, 2800, kv, dim)
    kd, vd = dev(k.reshape(2800, -1)), dev(v.reshape(2800, -1))
    q = f32(rng.standard_normal((1, 32, dim)))
    qd = dev(q.reshape(1, -1))
    streams = [torch.cuda.Stream() for _ in range(3)] + [None, 0]
    settle()
    for r in range(5):
        s = cache.new_sequence(3000, track=True)
        out = [torch.zeros((1, 32 * dim), device="cuda") for _ in range(4)]
        settle()
        a, b, c = streams[r], streams[(r + 1) % 5], streams[(r + 2) % 5]
        cache.append_device(0, [s], [0], [2500], kd[:2500], vd[:2500], stream=a)
        cache.attention_device(0, [s], qd, 32, out[0], stream=b)
        cache.append_device(0, [s], [2500], [300], kd[2500:], vd[2500:], stream=c)
        f = cache.fork(s, 2800)
        cache.evict([f], 1000, 100, stream=a)
        cache.attention_device(0, [s], qd, 32, out[1], stream=b)
        cache.attention_device(0, [f], qd, 32, out[2], stream=c)
        cache.append_device(0, [f], [1000], [300], kd[:300], vd[:300], stream=b)
        cache.attention_device(0, [f], qd, 32, out[3], stream=a)
        settle()
        check_attention(out[0].cpu().numpy().reshape(32, dim), q[0], q4.held(k[:2500]), q4.held(v[:2500]))
        check_attention(out[1].cpu().numpy().reshape(32, dim), q[0], q4.held(k), q4.held(v))
        got = read(cache, 0, [f], [0], [1300])
        check_attention(out[2].cpu().numpy().reshape(32, dim), q[0], got[0][:1000].astype(np.float64), got[1][:1000].astype(np.float64))
        check_attention(out[3].cpu().numpy().reshape(32, dim), q[0], got[0].astype(np.float64), got[1].astype(np.float64))
        assert np.array_equal(got[0][1000:], f32(q4.held(k[:300])))
        cache.free_sequence(f)
        cache.free_sequence(s)
    cache.close()


def test_results_on_a_torch_stream_follow_its_work(ctx):
    """Queries that torch makes on its stream, results that it uses there: nothing else orders them."""
    rng = np.random.default_rng(24)
    cache = PagedKvCache(ctx, 1, 2, 64, 20, "q4")
    s = cache.new_sequence(200)
    k, v = rows(rng, 200, 2, 64), rows(rng, 200, 2, 64)
    fill(cache, 0, [s], [0], [(k, v)])
    for stream in (torch.cuda.Stream(), torch.cuda.current_stream()):
        with torch.cuda.stream(stream):
            big = torch.ones((4096, 4096), device="cuda")
            q = (big @ big)[:1, :512] / 4096 * torch.linspace(-1, 1, 512, device="cuda")
            out = torch.empty_like(q)
            cache.attention_device(0, [s], q, 8, out, stream=stream)
            twice = out * 2
        torch.cuda.synchronize()
        check_attention(twice.cpu().numpy().reshape(8, 64) / 2, q.cpu().numpy().reshape(8, 64), q4.held(k), q4.held(v))
    cache.close()


# ── refusals ──────────────────────────────────────────────────────────────────────────────────────────────────────────────────

def test_refusals(ctx):
    L = ctx._L
    cache = PagedKvCache(ctx, 2, 2, 64, 8, "q4", track_seqs=1, track_tokens=64)
    a, b = cache.new_sequence(64, track=True), cache.new_sequence(64)
    x, y = torch.zeros((4, 128), device="cuda"), torch.zeros((4, 128), device="cuda")
    q, out = torch.zeros((1, 512), device="cuda"), torch.zeros((1, 512), device="cuda")
    settle()
    cache.append_device(0, [a, b], [0, 0], [2, 2], x, y)
    for match, call in [
        ("layer 2", lambda: cache.append_device(2, [a], [0], [4], x, y)),
        ("there twice", lambda: cache.append_device(0, [a, a], [2, 2], [2, 2], x, y)),
        ("not behind", lambda: cache.append_device(0, [a], [3], [4], x, y)),
        ("bad position", lambda: cache.append_device(0, [a], [-1], [4], x, y)),
        ("limit of 64", lambda: cache.append_device(0, [a], [2], [63], torch.zeros((63, 128), device="cuda"), torch.zeros((63, 128), device="cuda"))),
        ("cached positions", lambda: cache.read_device(0, [a], [0], [4], x, y)),
        ("cached positions", lambda: cache.attention_device(0, [a], q, 8, out, lens=[3])),
        ("cached positions", lambda: cache.attention_device(0, [a], q, 8, out, lens=[-1])),
        ("not a multiple", lambda: cache.attention_device(0, [a], torch.zeros((1, 192), device="cuda"), 3, torch.zeros((1, 192), device="cuda"))),
        ("there twice", lambda: cache.attention_device(0, [a, a], torch.zeros((2, 512), device="cuda"), 8, torch.zeros((2, 512), device="cuda"))),
        ("shape", lambda: cache.attention_device(0, [a], q, 4, out)),
        ("keeps no weights", lambda: cache.evict([b], 1)),
        ("keeps no weights", lambda: cache.evict([a, b], 1)),
        ("there twice", lambda: cache.evict([a, a], 1)),
        ("keep 0", lambda: cache.evict([a], 0)),
        ("32 bits", lambda: cache.evict([a], 2 ** 32 + 1)),
        ("32 bits", lambda: cache.attention_device(0, [a], q, 8, out, lens=[1.5])),
        ("recent 3", lambda: cache.evict([a], 2, 3)),
        ("recent -1", lambda: cache.evict([a], 2, -1)),
        ("cached positions", lambda: cache.weights_device(0, [a], [3], torch.zeros((1, 2, 3), device="cuda"))),
        ("hold no", lambda: cache.weights_device(0, [a], [2], torch.zeros((1, 2, 1), device="cuda"))),
        ("keeps weights already", lambda: _lib.check(L.juno_kvpool_track(cache.handle, 1, 16), "track")),
        ("keeps its weights already", lambda: _lib.check(L.juno_seq_track(a), "track")),
        ("CUDA tensor", lambda: cache.append_device(0, [a], [2], [4], x.double(), y)),
        ("elements apart", lambda: cache.append_device(0, [a], [2], [4], torch.zeros((4, 130), device="cuda")[:, :128], y)),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(JunoError, match="query/kv head ratio 9"):
        cache.attention_device(0, [a], torch.zeros((1, 18 * 64), device="cuda"), 18, torch.zeros((1, 18 * 64), device="cuda"))
    with pytest.raises(JunoError, match="no free weights"):
        cache.new_sequence(64, track=True)
    with pytest.raises(JunoError, match="no free weights"):
        cache.fork(a, 1)
    assert [cache.length(s) for s in (a, b)] == [2, 2]
    # host memory, and addresses that are not those of a float, are seen before any kernel runs
    host = np.zeros((4, 128), np.float32)
    one, zero, four = (C.c_void_p * 1)(a.value), np.zeros(1, np.int32), np.full(1, 4, np.int32)
    for k in (host.ctypes.data, 0, x.data_ptr() + 2):
        assert L.juno_kv_append_device(ctx.handle, cache.handle, 0, 1, one, zero.ctypes.data, four.ctypes.data, k, y.data_ptr(), 128, None) == _lib.ERR_INVALID_ARG
    assert L.juno_attn_decode_device(ctx.handle, cache.handle, 0, 1, one, None, 8, q.data_ptr(), 512, host.ctypes.data, 512, None) == _lib.ERR_INVALID_ARG
    assert L.juno_attn_decode_device(ctx.handle, cache.handle, 0, 1, one, None, 8, q.data_ptr(), 511, out.data_ptr(), 512, None) == _lib.ERR_INVALID_ARG
    assert L.juno_attn_decode_static(ctx.handle, cache.handle, 0, 1, one, 8, q.data_ptr(), out.data_ptr()) == _lib.ERR_UNSUPPORTED
    cache.free_sequence(a)
    with pytest.raises(JunoError, match="closed"):
        cache.attention_device(0, [a], q, 8, out)
    c = cache.new_sequence(64, track=True)  # its weights are free again
    assert cache.length(c) == 0
    other = PagedKvCache(ctx, 1, 2, 64, 4, "f16")
    s = other.new_sequence(16)
    other.append_device(0, [s], [0], [4], x, y)
    with pytest.raises(JunoError, match="4-bit pages"):
        other.attention_device(0, [s], q, 8, out)
    with pytest.raises(JunoError, match="4-bit pages"):
        _lib.check(L.juno_kvpool_track(other.handle, 1, 16), "track")
    with pytest.raises(ValueError, match="another pool"):
        cache.read_device(0, [s], [0], [4], x, y)
    settle()
    other.close()
    cache.close()
    with pytest.raises(Exception):
        PagedKvCache(ctx, 1, 2, 96, 4, "q4")


def test_a_graph_is_refused_and_goes_on(ctx):
    cache = PagedKvCache(ctx, 1, 2, 64, 8, "q4")
    s = cache.new_sequence(64)
    x = torch.zeros((4, 128), device="cuda")
    settle()
    stream = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream, capture_error_mode="relaxed"):
        y = x + 1
        with pytest.raises(ValueError, match="captured"):
            cache.append_device(0, [s], [0], [4], x, x, stream=stream)
    g.replay()
    torch.cuda.synchronize()
    assert (y == 1).all() and cache.length(s) == 0
    cache.append_device(0, [s], [0], [4], x, x, stream=stream)
    torch.cuda.synchronize()
    assert cache.length(s) == 4
    cache.close()


def test_a_wait_that_was_given_up_is_reported_once(ctx, wait_words):
    rng = np.random.default_rng(31)
    cache = PagedKvCache(ctx, 1, 2, 64, 8, "q4")
    s = cache.new_sequence(100)
    k = rows(rng, 100, 2, 64)
    fill(cache, 0, [s], [0], [(k, k)])
    q = f32(rng.standard_normal((1, 8, 64)))
    want = attend(cache, 0, [s], q)
    page = 9 | 2 << 8 | 5 << 16  # a page that warp 2 of block 5 waited for
    wait_words[0] = page
    with pytest.raises(JunoError, match="page of the cache .warp 2 of block 5") as e:
        cache.attention(0, [s], q.reshape(1, -1), 8)
    assert e.value.rc == _lib.ERR_TIMEOUT and wait_words[0] == 0
    wait_words[1] = page
    assert np.array_equal(attend(cache, 0, [s], q), want)  # enqueued work is answered for by the synchronisation
    with pytest.raises(JunoError, match="page of the cache"):
        ctx.synchronize()
    ctx.synchronize()
    assert np.array_equal(cache.attention(0, [s], q.reshape(1, -1), 8).reshape(want.shape), want)
    cache.close()


def test_eviction_of_sequences_that_are_short_enough(ctx):
    """Whatever the budget is: nothing moves, and no room is asked for that the sequences do not have."""
    rng = np.random.default_rng(32)
    cache = PagedKvCache(ctx, 2, 2, 64, 8, "q4", track_seqs=2, track_tokens=64)
    a, b = cache.new_sequence(64, track=True), cache.new_sequence(64, track=True)  # b is empty
    k = rows(rng, 50, 2, 64)
    for l in range(2):
        fill(cache, l, [a], [0], [(k, k)])
    for keep, recent in ((50, 0), (51, 51), (2 ** 31 - 1, 7), (2 ** 31 - 1, 2 ** 31 - 1)):
        cache.evict([a, b], keep, recent)
    kept = torch.full((2, 2, 2, 60), 9, dtype=torch.int32, device="cuda")
    settle()
    cache.evict([b, a], 60, 60, kept=kept)
    settle()
    kept = kept.cpu().numpy()
    assert (kept[:, 0] == -1).all() and (kept[:, 1, :, :50] == np.arange(50)).all() and (kept[:, 1, :, 50:] == -1).all()
    assert cache.length(a) == 50 and cache.length(b) == 0
    assert np.array_equal(read(cache, 1, [a], [0], [50])[0], f32(q4.held(k)))
    cache.close()


def test_two_threads_share_a_pool(ctx):
    """Calls from two threads, each with sequences of its own: as if one had made them."""
    import threading
    rng = np.random.default_rng(33)
    cache = PagedKvCache(ctx, 1, 4, 64, 300, "q4", track_seqs=8, track_tokens=400)
    q = f32(rng.standard_normal((1, 16, 64)))
    qd = dev(q.reshape(1, -1))
    parts = [rows(rng, 390, 4, 64) for _ in range(2)]
    data = [dev(p.reshape(390, -1)) for p in parts]
    outs = [[torch.zeros((1, 1024), device="cuda") for _ in range(25)] for _ in range(2)]
    settle()
    errors = []

    def work(t):
        try:
            for r in range(25):
                s = cache.new_sequence(400, track=True)
                cache.append_device(0, [s], [0], [300], data[t][:300], data[t][:300])
                f = cache.fork(s, 290)
                cache.append_device(0, [f], [290], [90], data[t][290:380], data[t][290:380])
                cache.attention_device(0, [f], qd, 16, outs[t][r])
                cache.evict([f], 100, 10)
                cache.free_sequence(s)
                cache.free_sequence(f)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(t,)) for t in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    settle()
    assert not errors, errors
    for t in range(2):
        h = q4.held(parts[t][:380])
        for o in outs[t]:
            check_attention(o.cpu().numpy().reshape(16, 64), q[0], h, h)
    cache.close()


def test_results_may_take_the_place_of_the_queries(ctx):
    rng = np.random.default_rng(34)
    cache = PagedKvCache(ctx, 1, 2, 128, 300, "q4")
    seqs, parts = [cache.new_sequence(2500) for _ in range(2)], [(rows(rng, n, 2, 128), rows(rng, n, 2, 128)) for n in (2500, 40)]
    fill(cache, 0, seqs, [0, 0], parts)
    q = f32(rng.standard_normal((2, 16, 128)))
    x = dev(q.reshape(2, -1))
    settle()
    cache.attention_device(0, seqs, x, 16, x)
    settle()
    for i, p in enumerate(parts):
        check_attention(x[i].cpu().numpy().reshape(16, 128), q[i], q4.held(p[0]), q4.held(p[1]))
    cache.close()


@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 64), (8, 1, 128), (64, 64, 64), (5, 1, 128)])
def test_attention_of_few_and_of_many_heads(ctx, heads, kv, dim):
    """One key/value head, whose parts are more than travel with a launch; more heads than CTAs of a wave; batches cut across their rows."""
    rng = np.random.default_rng(heads * dim)
    lens = [9000, 1, 4000, 700] if kv == 1 else [300, 1, 77, 640]
    cache = PagedKvCache(ctx, 1, kv, dim, sum((n + 15) // 16 for n in lens), "q4", track_seqs=4, track_tokens=max(lens))
    seqs = [cache.new_sequence(max(lens), track=i % 2 == 0) for i in range(4)]
    parts = [(rows(rng, n, kv, dim), rows(rng, n, kv, dim)) for n in lens]
    fill(cache, 0, seqs, [0] * 4, parts)
    q = f32(rng.standard_normal((4, heads, dim)))
    out = attend(cache, 0, seqs, q)
    for i, p in enumerate(parts):
        w = check_attention(out[i], q[i], q4.held(p[0]), q4.held(p[1]))
        if i % 2 == 0:
            check_weights(weights(cache, 0, [seqs[i]], [lens[i]])[0], w, q[i], p[0])
    cache.close()


def test_rows_of_unequal_lengths_share_the_work(ctx):
    """Rows that are cut across: one very long, one in the middle, many short, empty ones between; and each again in another order."""
    rng = np.random.default_rng(35)
    kv, dim, heads = 8, 128, 64
    lens = [3000, 0, 17, 6000, 1, 333, 0, 2900, 16] + [int(n) for n in rng.integers(1, 900, 30)]
    cache = PagedKvCache(ctx, 1, kv, dim, sum((n + 15) // 16 for n in lens), "q4")
    seqs = [cache.new_sequence(max(n, 1)) for n in lens]
    parts = [(rows(rng, n, kv, dim), rows(rng, n, kv, dim)) for n in lens]
    fill(cache, 0, seqs, [0] * len(lens), parts)
    q = f32(rng.standard_normal((len(lens), heads, dim)))
    for order in (np.arange(len(lens)), np.argsort(lens), np.argsort(lens)[::-1]):
        out = attend(cache, 0, [seqs[i] for i in order], q[order], lens=[lens[i] for i in order])
        for j, i in enumerate(order):
            if lens[i] == 0:
                assert (out[j] == 0).all()
            else:
                check_attention(out[j], q[i], q4.held(parts[i][0]), q4.held(parts[i][1]))
    cache.close()


def test_closing_a_context_gives_its_working_memory_back(ctx):
    own = GpuContext(0)
    cache = PagedKvCache(own, 1, 2, 64, 8, "q4")
    s = cache.new_sequence(64)
    x = torch.ones((40, 128), device="cuda")
    q, out = torch.ones((1, 512), device="cuda"), torch.zeros((1, 512), device="cuda")
    settle()
    cache.append_device(0, [s], [0], [40], x, x, stream=torch.cuda.Stream())
    cache.attention_device(0, [s], q, 8, out)
    own.synchronize()
    assert torch.allclose(out, torch.ones_like(out))
    with pytest.raises(ValueError, match="another context"):
        _lib.check(ctx._L.juno_kv_read_device(ctx.handle, cache.handle, 0, 1, cache.batch([s]).handles, np.zeros(1, np.int32).ctypes.data, np.ones(1, np.int32).ctypes.data,
                                              x.data_ptr(), x.data_ptr(), 128, None), "read")
    cache.close()
    own.close()

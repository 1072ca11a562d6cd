"""The operators on 4-bit pages of the key/value cache, as cases that can be timed and checked.

  append   new keys and values of `batch` sequences go into the pages, `rows` positions each behind the cached ones, and what the
           pages hold for them is read back (`PagedKvCache.append_device`, `read_device`)
  attend   decode attention of `batch` sequences over their cached positions (`attention_device`)
  weigh    the same for sequences that keep the weight which every cached position has received (`weights_device`)
  evict    a branch of each sequence (`fork`) is cut down to the `keep` positions of most weight, the newest `recent` of them in any
           case (`evict`), its rows and weights are read, and it is freed: all layers

Cached positions lie between half of `ctx` and `ctx`, one sequence has all of them.  Heads are those of this repository's models:
32 over 8 of 128 (Llama-3-8B), 64 over 8 of 128 (Llama-3-70B), 32 over 4 of 64 (TinyLlama).

A group is 32 neighbouring dimensions of one position and key/value head.  Its values are held as m + d q: m its minimum in FP16, d a
fifteenth of its range in BF16, q whole numbers from 0 to 15.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

GROUP = 32
MOST = 65504.0       # values are held within the range of FP16
NOTHING = 2.0 ** -80  # a range below this counts as none


def listed():
    return [
        # one request's newest position: the smallest call
        {"name": "append-b1", "kind": "append", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 1, "ctx": 2047, "rows": 1},
        # a decode step of a loaded server
        {"name": "append-b64", "kind": "append", "heads": 32, "kv_heads": 4, "dim": 64, "batch": 64, "ctx": 1500, "rows": 1},
        # prompts of several requests, odd lengths behind odd starts
        {"name": "append-prompts-4x2039", "kind": "append", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 4, "ctx": 77, "rows": 2039},
        # a chat with the 8B model
        {"name": "attend-b1-2048", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 1, "ctx": 2048},
        # one very long document
        {"name": "attend-b1-131072", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 1, "ctx": 131072},
        # a few requests with long contexts
        {"name": "attend-b8-4096", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 8, "ctx": 4096},
        # many requests of the small model
        {"name": "attend-b64-2048-d64", "kind": "attend", "heads": 32, "kv_heads": 4, "dim": 64, "batch": 64, "ctx": 2048},
        # many requests with long contexts, the 70B model's heads: the largest case
        {"name": "attend-b48-8192-g8", "kind": "attend", "heads": 64, "kv_heads": 8, "dim": 128, "batch": 48, "ctx": 8192},
        # one request whose cache will be cut down
        {"name": "weigh-b1-4096", "kind": "weigh", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 1, "ctx": 4096},
        # many of them
        {"name": "weigh-b16-8192", "kind": "weigh", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 16, "ctx": 8192},
        # a cache over its budget by half a thousand positions
        {"name": "evict-b1-2600-2048", "kind": "evict", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 1, "ctx": 2600, "keep": 2048, "recent": 256, "layers": 4},
        # long sessions condensed to an eighth
        {"name": "evict-b6-8192-1001", "kind": "evict", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 6, "ctx": 8192, "keep": 1001, "recent": 100, "layers": 4},
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 8, 128), (64, 8, 128), (32, 4, 64), (16, 16, 64), (12, 2, 128), (24, 8, 128)])
    case = {"kind": rng.choice(["append", "attend", "attend", "weigh", "evict"]), "heads": heads, "kv_heads": kv_heads, "dim": dim}
    if case["kind"] == "append":
        batch = size(1, 128)
        return case | {"batch": batch, "ctx": size(1, 4096), "rows": size(1, max(2, 8192 // batch))}
    if case["kind"] == "evict":
        batch, ctx = size(1, 6), size(64, 8192)
        keep = size(8, max(9, ctx // 2 - 1))
        return case | {"batch": batch, "ctx": ctx, "keep": min(keep, 2048), "recent": rng.randrange(0, min(keep, 2048) + 1), "layers": rng.randrange(1, 5)}
    batch = size(1, 64 if case["kind"] == "attend" else 32)
    return case | {"batch": batch, "ctx": min(size(1, 131072), (262144 if case["kind"] == "attend" else 131072) // batch)}


# ── inputs ────────────────────────────────────────────────────────────────────────────────────────────────────────────────────

def _lengths(case, seed):
    """Cached positions of each sequence; a cache that is cut down has more than it keeps."""
    r = np.random.default_rng([seed, 1])
    n = r.integers(max(1, case["ctx"] // 2, case.get("keep", 0) + 1), case["ctx"] + 1, case["batch"])
    n[0] = case["ctx"]
    return n.astype(np.int32)


def _generator(seed, part):
    g = torch.Generator("cuda")
    g.manual_seed(int(np.random.SeedSequence([seed, part]).generate_state(1, np.uint64)[0] >> np.uint64(1)))
    return g


def _keys_values(case, rows, g):
    """Keys have channels of different spread and mean, values do not."""
    shape = (rows, case["kv_heads"], case["dim"])
    spread = (0.5 * torch.randn(shape[1:], generator=g, device="cuda")).exp()
    mean = 0.5 * torch.randn(shape[1:], generator=g, device="cuda")
    return torch.randn(shape, generator=g, device="cuda") * spread + mean, 0.5 * torch.randn(shape, generator=g, device="cuda")


def _weights(case, rows, g):
    """Weight that cached positions have received: a few have much of it, some none at all."""
    shape = (case["kv_heads"], rows)
    return (2.0 * torch.randn(shape, generator=g, device="cuda")).exp() * (torch.rand(shape, generator=g, device="cuda") > 0.2)


def _rows_of(case, seed):
    """Rows that the pages get in a pass of `append`: every sequence has `rows` of them."""
    return case["batch"] * case["rows"]


def _queries(case, seed):
    return 1.5 * torch.randn((case["batch"], case["heads"] * case["dim"]), generator=_generator(seed, 2), device="cuda")


# ── the plain form ────────────────────────────────────────────────────────────────────────────────────────────────────────────

def _quantise(x):
    """FP32 [..., dim] -> whole numbers two to a byte [..., dim / 2], d and m [..., dim / 32]."""
    g = x.clamp(-MOST, MOST).unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    m = lo.half()
    reach = hi - lo
    d = torch.where(reach < NOTHING, torch.zeros_like(reach), reach / torch.full_like(reach, 15.0)).bfloat16()
    q = torch.where(d > 0, (g.double() - m.double()) / d.double(), torch.zeros((), dtype=torch.float64, device=x.device))
    q = q.round().clamp(0, 15).to(torch.uint8).flatten(-2)
    return q[..., 0::2] | (q[..., 1::2] << 4), d.squeeze(-1), m.squeeze(-1)


def _values(codes, d, m):
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, GROUP)).float()
    return (m.float()[..., None] + d.float()[..., None] * q).flatten(-2)


def _plain_append(s):
    for_k, for_v = _quantise(s["k"]), _quantise(s["v"])
    for held, new in zip(s["held_k"] + s["held_v"], for_k + for_v):
        held[s["at"]] = new
    k, v = (_values(*(held[s["at"]] for held in s[name])).flatten(1) for name in ("held_k", "held_v"))
    return {"k": k, "v": v}


def _plain_attend(s):
    k, v = _values(*s["held_k"]), _values(*s["held_v"])  # [batch, kv heads, positions, dim]
    n, h, _, dim = k.shape
    q = s["q"].view(n, h, -1, dim)
    x = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    x = x.masked_fill(s["behind"][:, None, None], -math.inf)
    p = (x - x.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    out = (p @ v).flatten(1)
    if "weights" not in s:
        return out
    s["weights"] += p.sum(2)
    return {"out": out, "weights": s["weights"]}


def _plain_evict(s):
    w, keep = s["weights"], s["keep"]  # [layers, batch, kv heads, positions]
    rank = w.masked_fill(s["newest"][None, :, None], math.inf).masked_fill(s["behind"][None, :, None], -math.inf)
    kept = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    take = lambda x: x.gather(3, kept[..., None].expand(*kept.shape, x.shape[-1]))  # noqa: E731
    rows = lambda held: _values(*(take(x) for x in held)).transpose(2, 3).flatten(-2).flatten(1, 2)  # noqa: E731
    return {"kept": kept.int(), "k": rows(s["held_k"]), "v": rows(s["held_v"]), "weights": w.gather(3, kept)}


# ── the framework's operators ─────────────────────────────────────────────────────────────────────────────────────────────────

class _Cache:
    """A pool of 4-bit pages and its sequences, given back with the state that holds it."""

    def __init__(self, case, lengths, room, track):
        from juno_b200.matvec import GpuContext, PagedKvCache
        batch, most = case["batch"], int(lengths.max()) + room
        pages = int(((lengths + room + 15) // 16).sum()) + batch * ((case.get("keep", 0) + 15) // 16)
        self.pool = PagedKvCache(GpuContext.shared(0), case.get("layers", 1), case["kv_heads"], case["dim"], pages, "q4",
                                 track_seqs=2 * batch if track else 0, track_tokens=most if track else 0)
        self.seqs = [self.pool.new_sequence(most, track=track) for _ in range(batch)]
        self.batch = self.pool.batch(self.seqs)
        self.zeros = np.zeros(batch, dtype=np.int32)

    def __del__(self):
        if hasattr(self, "pool"):
            self.pool.close()


def _own_append(s):
    c, pool = s["cache"], s["cache"].pool
    pool.append_device(0, c.batch, s["lengths"], s["counts"], s["k"], s["v"])
    pool.read_device(0, c.batch, s["lengths"], s["counts"], s["k_out"], s["v_out"])
    return {"k": s["k_out"], "v": s["v_out"]}


def _own_attend(s):
    c, pool = s["cache"], s["cache"].pool
    pool.attention_device(0, c.batch, s["q"], s["heads"], s["out"], lens=s["lengths"])
    if "w" not in s:
        return s["out"]
    pool.weights_device(0, c.batch, s["lengths"], s["w"])
    return {"out": s["out"], "weights": s["w"]}


def _own_evict(s):
    c, pool = s["cache"], s["cache"].pool
    branches = [pool.fork(q, n) for q, n in zip(c.seqs, s["of"])]
    b = pool.batch(branches)
    pool.evict(b, s["keep"], s["recent"], kept=s["kept"])
    for l in range(s["layers"]):
        pool.read_device(l, b, c.zeros, s["counts"], s["k_out"][l], s["v_out"][l])
        pool.weights_device(l, b, s["counts"], s["w_out"][l])
    for q in branches:
        pool.free_sequence(q)
    return {"kept": s["kept"], "k": s["k_out"], "v": s["v_out"], "weights": s["w_out"]}


# ── what the tools call ───────────────────────────────────────────────────────────────────────────────────────────────────────

def _padded(rows, lengths):
    """Rows of all sequences behind one another -> [batch, kv heads, most positions, dim], and where a sequence has ended."""
    place = torch.arange(int(lengths.max()), device="cuda")[None]
    n = torch.from_numpy(lengths).cuda().long()[:, None]
    at = (n.cumsum(0) - n + place).clamp(max=rows.shape[0] - 1)
    return rows[at].transpose(1, 2), place >= n


def _empty_like(parts, rows):
    return tuple(torch.zeros((rows, *p.shape[1:]), dtype=p.dtype, device="cuda") for p in parts)


def prepare(case, seed):
    kind, lengths, kv, dim = case["kind"], _lengths(case, seed), case["kv_heads"], case["dim"]
    g, total, wide = _generator(seed, 3), int(lengths.sum()), case["kv_heads"] * case["dim"]
    if kind == "append":
        k, v = _keys_values(case, _rows_of(case, seed), g)
        counts = np.full(case["batch"], case["rows"], dtype=np.int32)
        if own:
            c = _Cache(case, lengths, case["rows"], False)
            before = torch.zeros((total, wide), device="cuda")
            torch.cuda.synchronize()
            c.pool.append_device(0, c.batch, c.zeros, lengths, before, before)
            c.pool.ctx.synchronize()
            return {"kind": kind, "cache": c, "lengths": lengths, "counts": counts, "k": k.flatten(1), "v": v.flatten(1),
                    "k_out": torch.empty_like(k).flatten(1), "v_out": torch.empty_like(v).flatten(1)}
        after = torch.from_numpy(np.cumsum(lengths + case["rows"]) - case["rows"]).cuda()
        at = (after[:, None] + torch.arange(case["rows"], device="cuda")[None]).flatten()
        held = _empty_like(_quantise(k[:1]), total + k.shape[0])
        return {"kind": kind, "k": k, "v": v, "at": at, "held_k": held, "held_v": _empty_like(held, total + k.shape[0])}
    if kind == "evict":
        layers, keep, batch = case["layers"], case["keep"], case["batch"]
        newest = torch.arange(case["ctx"], device="cuda")[None] >= torch.from_numpy(lengths).cuda()[:, None] - case["recent"]
        c = _Cache(case, lengths, 0, True) if own else None
        held = []
        for l in range(layers):
            k, v = _keys_values(case, total, g)
            w, behind = _padded(_weights(case, total, g).T.contiguous(), lengths)  # [batch, kv heads, positions]
            w = w.masked_fill(behind[:, None], 0.0).contiguous()
            if own:
                torch.cuda.synchronize()
                c.pool.append_device(l, c.batch, c.zeros, lengths, k.flatten(1), v.flatten(1))
                c.pool.weights_device(l, c.batch, lengths, w, store=True)
                c.pool.ctx.synchronize()
            else:
                held.append((*_quantise(_padded(k, lengths)[0]), *_quantise(_padded(v, lengths)[0]), w))
        if own:
            rows = (layers, batch * keep, wide)
            return {"kind": kind, "cache": c, "of": [int(n) for n in lengths], "keep": keep, "recent": case["recent"], "layers": layers,
                    "counts": np.full(batch, keep, dtype=np.int32), "kept": torch.empty((layers, batch, kv, keep), dtype=torch.int32, device="cuda"),
                    "k_out": torch.empty(rows, device="cuda"), "v_out": torch.empty(rows, device="cuda"),
                    "w_out": torch.empty((layers, batch, kv, keep), device="cuda")}
        held = [torch.stack(x) for x in zip(*held)]
        return {"kind": kind, "held_k": held[:3], "held_v": held[3:6], "weights": held[6], "newest": newest, "behind": behind, "keep": keep}
    q = _queries(case, seed)
    k, v = _keys_values(case, total, g)
    w = None
    if kind == "weigh":
        w, behind = _padded(_weights(case, total, g).T.contiguous(), lengths)
        w = w.masked_fill(behind[:, None], 0.0).contiguous()
    if own:
        c = _Cache(case, lengths, 0, w is not None)
        torch.cuda.synchronize()
        c.pool.append_device(0, c.batch, c.zeros, lengths, k.flatten(1), v.flatten(1))
        if w is not None:
            c.pool.weights_device(0, c.batch, lengths, w, store=True)
        c.pool.ctx.synchronize()
        return {"kind": kind, "cache": c, "lengths": lengths, "heads": case["heads"], "q": q, "out": torch.empty_like(q)} | ({} if w is None else {"w": w})
    (k, behind), (v, _) = _padded(k, lengths), _padded(v, lengths)
    return {"kind": kind, "q": q, "held_k": _quantise(k), "held_v": _quantise(v), "behind": behind} | ({} if w is None else {"weights": w})


def run(state):
    if own:
        return {"append": _own_append, "attend": _own_attend, "weigh": _own_attend, "evict": _own_evict}[state["kind"]](state)
    return {"append": _plain_append, "attend": _plain_attend, "weigh": _plain_attend, "evict": _plain_evict}[state["kind"]](state)


def work(case):
    """A cached position and key/value head has 5 bits for each element of its key and value: 4 of the number, 1 of d and m."""
    # the lengths' mean stands for them: they depend on the seed
    batch, ctx, kv, dim = case["batch"], case["ctx"], case["kv_heads"], case["dim"]
    total = ctx + (batch - 1) * (max(1, ctx // 2, case.get("keep", 0) + 1) + ctx) / 2
    row = kv * dim * 2 * 5 / 8
    if case["kind"] == "append":
        rows = batch * case["rows"]
        return {"bytes": rows * (2 * row + 2 * kv * dim * 2 * 4), "flops": rows * kv * dim * 2 * 8}
    if case["kind"] == "evict":
        rows = batch * case["keep"] * case["layers"]
        # weights read; kept rows and weights moved, and read; kept places and values written
        return {"bytes": case["layers"] * total * kv * 4 + rows * (3 * row + 4 * kv * 4 + kv * 4 + kv * dim * 2 * 4), "flops": case["layers"] * total * kv * 4}
    ends = 2 * batch * case["heads"] * dim * 4
    weights = total * kv * (4 * 4) if case["kind"] == "weigh" else 0  # read, written, and given out
    return {"bytes": total * row + ends + weights, "flops": 4 * total * case["heads"] * dim}


# ── in 64 bits ────────────────────────────────────────────────────────────────────────────────────────────────────────────────

def _held(x):
    """What the pages hold for x, in 64 bits: each group's numbers and the two factors as they are rounded."""
    x = torch.minimum(torch.maximum(x, x.new_tensor(-MOST)), x.new_tensor(MOST))
    parts = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    ordered = parts.sort(-1).values
    least, reach = ordered[..., :1], ordered[..., -1:] - ordered[..., :1]
    offset = least.to(torch.float16).to(torch.float64)
    step = (reach / reach.new_full(reach.shape, 15.0)).to(torch.bfloat16).to(torch.float64)
    step[reach < NOTHING] = 0.0
    ratio = (parts.to(torch.float64) - offset) / torch.where(step == 0, torch.ones_like(step), step)
    number = torch.round(ratio).clamp(min=0.0, max=15.0) * (step != 0)
    return (offset + step * number).reshape(x.shape)


def exact(case, seed):
    kind, lengths = case["kind"], _lengths(case, seed)
    g, total = _generator(seed, 3), int(lengths.sum())
    if kind == "append":
        k, v = _keys_values(case, _rows_of(case, seed), g)
        return {"k": _held(k).flatten(1), "v": _held(v).flatten(1)}
    ends = np.cumsum(lengths)
    spans = [slice(int(e - n), int(e)) for e, n in zip(ends, lengths)]
    if kind == "evict":
        keep, out = case["keep"], {"kept": None, "k": [], "v": [], "weights": []}
        for _ in range(case["layers"]):
            k, v = _keys_values(case, total, g)
            w = _weights(case, total, g)
            for a in spans:
                n = a.stop - a.start
                order = w[:, a].double()
                order[:, n - case["recent"]:] = math.inf
                # the rank of a position: how many have more weight, or as much and come before it
                at = torch.argsort(-order, dim=-1, stable=True)[:, :keep].sort(-1).values
                heads = torch.arange(case["kv_heads"], device="cuda")
                for name, x in (("k", k), ("v", v)):
                    out[name].append(_held(x[a][at.T, heads]).flatten(1))
                out["weights"].append(w[:, a].double().gather(1, at))
        shape = (case["layers"], case["batch"] * keep, case["kv_heads"] * case["dim"])
        return {"kept": None, "k": torch.cat(out["k"]).view(shape), "v": torch.cat(out["v"]).view(shape),
                "weights": torch.stack(out["weights"]).view(case["layers"], case["batch"], case["kv_heads"], keep)}
    q = _queries(case, seed).double()
    k, v = _keys_values(case, total, g)
    w0 = _weights(case, total, g).double() if kind == "weigh" else None
    out = torch.empty_like(q)
    weights = torch.zeros((case["batch"], case["kv_heads"], case["ctx"]), dtype=torch.float64, device="cuda")
    for i, a in enumerate(spans):
        heads = q[i].view(case["kv_heads"], -1, case["dim"])
        scores = torch.einsum("hgd,lhd->hgl", heads, _held(k[a])) / math.sqrt(case["dim"])
        p = torch.softmax(scores, -1)
        out[i] = torch.einsum("hgl,lhd->hgd", p, _held(v[a])).flatten()
        if w0 is not None:
            weights[i, :, :a.stop - a.start] = w0[:, a] + p.sum(1)
    return out if w0 is None else {"out": out, "weights": weights}

"""What is measured of the 8-bit KV cache and of attention over drafted token trees.

Four operators of the serving path, each reached the way a user's program reaches it:

* write  -- ``kv_scatter`` into an e4m3 pool: every (token, KV head) row of K and of V is scaled by a
  power of two and stored in 8 bits.  The pass reads the rows back, so that its output is what the
  cache holds.
* read   -- ``kv_gather``: rows of a pool by slot, as bf16 (accepted draft paths, sequences that are
  moved or handed to another program).
* attend -- ``attend`` through an e4m3 pool: decode rows, verify rows and prompt chunks.
* tree   -- ``attend`` for sequences whose new tokens are a tree of drafts (``SeqChunk.parents``): a
  token sees the cached context, its ancestors and itself.  bf16 and e4m3 pools.

An 8-bit row x (128 values) is held as e4m3 codes c and one exponent e: e is the smallest integer in
[-100, 120] with max|x| 2^-e <= 448, c = the nearest e4m3 value to x 2^-e (ties to even), and the row
stands for c 2^e.  A row with an infinity or a NaN stands for NaN.

Geometry: head_dim 128, 16-token blocks, two query heads per KV head, bf16 activations.  Contexts
and trees are drawn from the case alone; values and block tables from the seed.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

HEAD_DIM = 128
GROUP = 2
BLOCK = 16
SCALE = HEAD_DIM ** -0.5
EXP_MIN, EXP_MAX = -100, 120
PAD = -2  # parent of an unused draft position

# Most context tokens x KV heads an attention case holds, and most (query row, visible key) pairs.
MAX_KV = 640_000 * 8
MAX_PAIRS = 2.2e8


def listed() -> list[dict]:
    return [
        # The new rows of one decode step of 61 sequences: launch latency counts.
        {"name": "write-decode-61", "kind": "write", "tokens": 61, "kv_heads": 8},
        # The largest step a runner schedules (its profiler's 16384 tokens).
        {"name": "write-prefill-16384", "kind": "write", "tokens": 16384, "kv_heads": 8},
        # Accepted draft paths of 64 sequences, read from a bf16 pool before they are moved.
        {"name": "read-paths-203", "kind": "read", "pool": "bf16", "tokens": 203, "kv_heads": 4},
        # Sequences moved out of an 8-bit cache.
        {"name": "read-e4m3-65521", "kind": "read", "pool": "e4m3", "tokens": 65521, "kv_heads": 8},
        # 8 decode rows of at most 512 tokens: the small interactive batch.
        {"name": "attend-decode-8", "kind": "attend", "pool": "e4m3", "kv_heads": 8, "geometry": 1,
         "rows": 8, "new": 1, "ctx_lo": 1, "ctx_hi": 512, "chunks": 0, "chunk_new": 0, "chunk_ctx": 0},
        # 256 decode rows of 256 to 4096 tokens: the throughput batch.
        {"name": "attend-decode-256", "kind": "attend", "pool": "e4m3", "kv_heads": 8, "geometry": 2,
         "rows": 256, "new": 1, "ctx_lo": 256, "ctx_hi": 4096, "chunks": 0, "chunk_new": 0,
         "chunk_ctx": 0},
        # 48 decode rows beside two prompt chunks of 1000 tokens over 512 cached ones.
        {"name": "attend-mixed", "kind": "attend", "pool": "e4m3", "kv_heads": 8, "geometry": 3,
         "rows": 48, "new": 1, "ctx_lo": 128, "ctx_hi": 2048, "chunks": 2, "chunk_new": 1000,
         "chunk_ctx": 512},
        # One very long sequence, 3 tokens to verify: the work is split over the context.
        {"name": "attend-long-1", "kind": "attend", "pool": "e4m3", "kv_heads": 8, "geometry": 4,
         "rows": 1, "new": 3, "ctx_lo": 100_001, "ctx_hi": 100_001, "chunks": 0, "chunk_new": 0,
         "chunk_ctx": 0},
        # One interactive sequence with a tree of 8 drafts.
        {"name": "tree-1x8", "kind": "tree", "pool": "bf16", "kv_heads": 8, "geometry": 5,
         "rows": 1, "new": 8, "ctx_lo": 777, "ctx_hi": 777, "padded": 0},
        # 64 sequences with 16 drafts each.
        {"name": "tree-64x16", "kind": "tree", "pool": "bf16", "kv_heads": 8, "geometry": 6,
         "rows": 64, "new": 16, "ctx_lo": 256, "ctx_hi": 4096, "padded": 0},
        # 48 sequences with up to 32 drafts each (a fixed tree size, unused positions padded) over
        # an 8-bit cache.
        {"name": "tree-e4m3-48x32", "kind": "tree", "pool": "e4m3", "kv_heads": 8, "geometry": 7,
         "rows": 48, "new": 32, "ctx_lo": 256, "ctx_hi": 4096, "padded": 5},
        # Wide trees of 63 drafts over long contexts, heads sharded over two GPUs.
        {"name": "tree-16x63", "kind": "tree", "pool": "bf16", "kv_heads": 4, "geometry": 8,
         "rows": 16, "new": 63, "ctx_lo": 4000, "ctx_hi": 8100, "padded": 0},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["write", "read", "attend", "attend", "tree", "tree"])
    kv_heads = rng.choice([4, 8, 8])
    if kind == "write":
        return {"kind": kind, "tokens": _log_int(rng, 61, 16384), "kv_heads": 8}
    if kind == "read":
        return {"kind": kind, "pool": rng.choice(["bf16", "e4m3"]),
                "tokens": _log_int(rng, 203, 65521), "kv_heads": kv_heads}
    while True:
        if kind == "attend":
            rows = _log_int(rng, 1, 256)
            hi = _log_int(rng, 512, 100_001) if rows <= 4 else _log_int(rng, 512, 4096)
            chunks = rng.choice([0, 0, 1, 2])
            case = {"kind": kind, "pool": "e4m3", "kv_heads": 8,
                    "geometry": rng.randrange(1 << 30), "rows": rows,
                    "new": rng.choice([1, 1, 1, 2, 3]), "ctx_lo": max(1, hi // rng.choice([2, 16, 512])),
                    "ctx_hi": hi, "chunks": chunks,
                    "chunk_new": _log_int(rng, 33, 1000) if chunks else 0,
                    "chunk_ctx": rng.randrange(0, 700) if chunks else 0}
        else:
            new = _log_int(rng, 8, 63)
            hi = _log_int(rng, 777, 8100)
            case = {"kind": kind, "pool": rng.choice(["bf16", "e4m3"]), "kv_heads": kv_heads,
                    "geometry": rng.randrange(1 << 30), "rows": _log_int(rng, 1, 64), "new": new,
                    "ctx_lo": max(1, hi // rng.choice([1, 2, 16])), "ctx_hi": hi,
                    "padded": rng.choice([0, 0, new // 4])}
        seqs = geometry(case)
        kv = sum(n + c for n, c, _ in seqs) * case["kv_heads"]
        limit = MAX_KV if case["pool"] == "e4m3" else MAX_KV // 3
        if kv <= limit and _pairs(case, seqs) * GROUP * case["kv_heads"] <= MAX_PAIRS:
            return case


def geometry(case: dict) -> list[tuple[int, int, list[int] | None]]:
    """(new tokens, cached tokens, parents) of each sequence.  ``ctx_lo..ctx_hi`` bounds the context
    with the new tokens for decode and verify rows, and the cached context for trees."""
    rng = random.Random(case["geometry"])
    out: list[tuple[int, int, list[int] | None]] = []
    for _ in range(case["rows"]):
        ctx = rng.randint(case["ctx_lo"], case["ctx_hi"])
        new = case["new"]
        if case["kind"] == "attend":
            out.append((new, max(0, ctx - new), None))
            continue
        used = new - (rng.randint(0, case["padded"]) if case["padded"] else 0)
        parents = [rng.randint(max(-1, i - 9), i - 1) for i in range(used)] + [PAD] * (new - used)
        out.append((new, ctx, parents))
    if case["kind"] == "attend":
        for _ in range(case["chunks"]):
            out.append((case["chunk_new"], case["chunk_ctx"], None))
    return out


def _tree_mask(parents: list[int]) -> np.ndarray:
    """[n, n]: whether draft i sees draft j (its ancestors and itself)."""
    n = len(parents)
    m = np.zeros((n, n), dtype=bool)
    for i, p in enumerate(parents):
        if p == PAD:
            continue
        if p >= 0:
            m[i] = m[p]
        m[i, i] = True
    return m


def _pairs(case: dict, seqs) -> int:
    """(query token, visible key) pairs."""
    total = 0
    for n, c, parents in seqs:
        if parents is None:
            total += n * c + n * (n + 1) // 2
        else:
            m = _tree_mask(parents)
            total += int(m.any(1).sum()) * c + int(m.sum())
    return total


def work(case: dict) -> dict:
    kvh = case["kv_heads"]
    row16, row8 = HEAD_DIM * 2, HEAD_DIM + 1
    if case["kind"] == "write":  # bf16 rows in, 8-bit rows stored, bf16 rows out; slots
        return {"bytes": case["tokens"] * (kvh * 2 * (2 * row16 + row8) + 8), "flops": 0}
    held = row16 if case["pool"] == "bf16" else row8
    if case["kind"] == "read":
        return {"bytes": case["tokens"] * (kvh * 2 * (held + row16) + 8), "flops": 0}
    seqs = geometry(case)
    tokens = sum(n for n, _, _ in seqs)
    ctx = sum(n + c for n, c, _ in seqs)
    return {"bytes": ctx * kvh * 2 * held + tokens * kvh * GROUP * 2 * row16,
            "flops": 4 * HEAD_DIM * kvh * GROUP * _pairs(case, seqs)}


# ---- inputs ---------------------------------------------------------------------------------------


def _layout(case: dict, seed: int):
    """Pool size in blocks and, per sequence, (flat start, new, cached, table, parents)."""
    gen = torch.Generator().manual_seed(seed * 2 + 1)
    seqs = geometry(case)
    need = [-(-(n + c) // BLOCK) for n, c, _ in seqs]
    blocks = sum(need) + max(2, sum(need) // 16)
    perm = torch.randperm(blocks, generator=gen).tolist()
    out, at, flat = [], 0, 0
    for (n, c, parents), b in zip(seqs, need):
        out.append((flat, n, c, perm[at : at + b], parents))
        at += b
        flat += n
    return blocks, out


def _values(case: dict, seed: int, slots: int):
    """K and V for every slot: keys with a few strong channels (as after a norm with learned
    weights), values whose size differs from token to token."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kvh = case["kv_heads"]
    chan = torch.exp(0.6 * torch.randn(kvh, HEAD_DIM, device="cuda", generator=gen))
    chan[:, 5] *= 4.0
    k = torch.empty(slots, kvh, HEAD_DIM, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    for a in range(0, slots, 1 << 16):
        b = min(slots, a + (1 << 16))
        shape = (b - a, kvh, HEAD_DIM)
        k[a:b] = torch.randn(shape, device="cuda", generator=gen) * chan * 0.7
        size = torch.exp(0.5 * torch.randn(b - a, kvh, 1, device="cuda", generator=gen))
        v[a:b] = torch.randn(shape, device="cuda", generator=gen) * size
    return k, v, gen


def _inputs(case: dict, seed: int) -> dict:
    """The tensors of a case in plain layout: k, v per slot (or per token), and what indexes them."""
    kvh = case["kv_heads"]
    if case["kind"] in ("write", "read"):
        t = case["tokens"]
        blocks = -(-t // BLOCK) * 5 // 4 + 3
        n = t if case["kind"] == "write" else blocks * BLOCK
        k, v, gen = _values(case, seed, n)
        if case["kind"] == "write":
            slots = torch.randperm(blocks * BLOCK, device="cuda", generator=gen)[:t]
        else:
            slots = torch.randint(0, n, (t,), device="cuda", generator=gen)
        return {"blocks": blocks, "k": k, "v": v, "slots": slots}
    blocks, seqs = _layout(case, seed)
    k, v, gen = _values(case, seed, blocks * BLOCK)
    tokens = sum(s[1] for s in seqs)
    q = torch.randn(tokens, kvh * GROUP, HEAD_DIM, device="cuda", generator=gen).to(torch.bfloat16)
    return {"blocks": blocks, "k": k, "v": v, "q": q, "seqs": seqs}


def _context_slots(n: int, c: int, table: list[int]) -> torch.Tensor:
    t = torch.tensor(table, dtype=torch.int64)
    p = torch.arange(n + c)
    return t[p // BLOCK] * BLOCK + p % BLOCK


def prepare(case: dict, seed: int) -> dict:
    x = _inputs(case, seed)
    pool = case.get("pool", "e4m3")
    state = {"case": case}
    if own:
        from miniserve_b200 import (SeqChunk, allocate_kv_cache, build_attention_metadata,
                                    kv_scatter)

        dtype = torch.bfloat16 if pool == "bf16" else torch.float8_e4m3fn
        state["pool"], views = allocate_kv_cache(1, x["blocks"], case["kv_heads"],
                                                 torch.device("cuda"), dtype=dtype)
        state["k_cache"], state["v_cache"] = views[0]
        if case["kind"] == "write":
            return state | {n: x[n] for n in ("k", "v", "slots")}
        every = torch.arange(x["blocks"] * BLOCK, device="cuda")
        kv_scatter(x["k"], x["v"], every, state["k_cache"], state["v_cache"])
        if case["kind"] == "read":
            return state | {"slots": x["slots"]}
        chunks = [SeqChunk(f, n, c, table) if parents is None
                  else SeqChunk(f, n, c, table, parents=parents)
                  for f, n, c, table, parents in x["seqs"]]
        new = torch.cat([_context_slots(n, c, t)[c:] for _, n, c, t, _ in x["seqs"]]).cuda()
        return state | {"q": x["q"], "meta": build_attention_metadata(chunks, new, BLOCK)}
    if case["kind"] == "write":
        return state | {n: x[n] for n in ("k", "v", "slots")}
    for name in ("k", "v"):
        if pool == "bf16":
            state[name] = x[name]
        else:
            parts = [_quantise(p) for p in x[name].split(1 << 16)]
            state[name] = torch.cat([p[0] for p in parts])
            state[name + "_scale"] = torch.cat([p[1] for p in parts])
    if case["kind"] == "read":
        return state | {"slots": x["slots"]}
    seqs = []
    for f, n, c, table, parents in x["seqs"]:
        tree = None if parents is None else torch.from_numpy(_tree_mask(parents)).cuda()
        seqs.append((f, n, c, _context_slots(n, c, table).cuda(), tree))
    return state | {"q": x["q"], "seqs": seqs}


# ---- the operators in their plain form ---------------------------------------------------------------


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32, exactly (normal numbers): pow() may be an ulp off."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 codes and 2^exponent of each row (NaN for a row with a NaN or an infinity)."""
    y = x.float()
    top = y.abs().amax(-1, keepdim=True)
    mant, expo = torch.frexp(top)  # top = mant 2^expo, mant in [0.5, 1): 448 = 0.875 2^9
    e = (expo - 9 + (mant > 0.875).to(expo.dtype)).clamp(EXP_MIN, EXP_MAX)
    ok = torch.isfinite(y).all(-1, keepdim=True)
    limit = torch.where(e == EXP_MAX, 240.0, 448.0)  # what still is a bf16 value at 2^120
    z = torch.where(ok, y, 0.0) * _pow2(-e)
    codes = torch.minimum(torch.maximum(z, -limit), limit).to(torch.float8_e4m3fn)
    return codes, torch.where(ok, _pow2(e), math.nan)


def _held(state: dict, name: str, slots: torch.Tensor) -> torch.Tensor:
    """Rows of the cache as fp32."""
    rows = state[name].index_select(0, slots).float()
    if name + "_scale" in state:
        rows = rows * state[name + "_scale"].index_select(0, slots)
    return rows


def _attend_plain(state: dict) -> torch.Tensor:
    q = state["q"]
    heads = q.shape[1]
    out = torch.empty_like(q)
    for f, n, c, slots, tree in state["seqs"]:
        k = _held(state, "k", slots).permute(1, 0, 2)  # [KVH, L, 128]
        v = _held(state, "v", slots).permute(1, 0, 2)
        qs = q[f : f + n].float().reshape(n, heads // GROUP, GROUP, HEAD_DIM)
        qs = qs.permute(1, 0, 2, 3).reshape(heads // GROUP, n * GROUP, HEAD_DIM)
        s = torch.matmul(qs, k.transpose(1, 2)) * SCALE
        if tree is not None:
            sees = torch.cat([tree.any(1, keepdim=True).expand(n, c), tree], 1)
        else:
            at = torch.arange(n + c, device=q.device)
            sees = at[None, :] <= at[c:, None]
        if tree is not None or n > 1:
            s = s.masked_fill(~sees.repeat_interleave(GROUP, 0), -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
        o = o.reshape(heads // GROUP, n, GROUP, HEAD_DIM).permute(1, 0, 2, 3)
        out[f : f + n] = o.reshape(n, heads, HEAD_DIM).to(out.dtype)
    return out


def run(state: dict):
    kind = state["case"]["kind"]
    if own:
        from miniserve_b200 import attend, kv_gather, kv_scatter

        if kind == "write":
            kv_scatter(state["k"], state["v"], state["slots"], state["k_cache"], state["v_cache"])
        if kind in ("write", "read"):
            return kv_gather(state["slots"], state["k_cache"], state["v_cache"])
        return attend(state["q"], state["k_cache"], state["v_cache"], state["meta"], SCALE)
    if kind == "write":
        out = []
        for name in ("k", "v"):
            codes, scale = _quantise(state[name])
            out.append((codes.float() * scale).to(torch.bfloat16))
        return tuple(out)
    if kind == "read":
        return tuple(_held(state, n, state["slots"]).to(torch.bfloat16) for n in ("k", "v"))
    return _attend_plain(state)


# ---- the definition in 64 bits ------------------------------------------------------------------------


def _two(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp64, exactly."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _floor_log2(x: torch.Tensor) -> torch.Tensor:
    """floor(log2 x) of positive normal fp64 numbers, from their exponent field."""
    return (x.view(torch.int64) >> 52) - 1023


def _exact_held(x: torch.Tensor) -> torch.Tensor:
    """What an 8-bit row stands for, by the definition: the exponent by trial, the code from the
    spacing of e4m3 at its size (2^-9 below 2^-6, else an eighth of its power of two)."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    e = (_floor_log2(top.clamp_min(1e-300)) - 9).clamp(EXP_MIN, EXP_MAX)
    for _ in range(2):
        e = torch.where(top > 448.0 * _two(e), e + 1, e)
    e = e.clamp(EXP_MIN, EXP_MAX)
    y = x * _two(-e)
    step = _two(_floor_log2(y.abs().clamp_min(1e-300)).clamp_min(-6) - 3)
    return torch.round(y / step) * step * _two(e)


def exact(case: dict, seed: int):
    x = _inputs(case, seed)
    pool = case.get("pool", "e4m3")
    if case["kind"] == "write":
        return tuple(_exact_held(x[n]) for n in ("k", "v"))
    hold = (lambda r: r.double()) if pool == "bf16" else _exact_held
    if case["kind"] == "read":
        return tuple(hold(x[n][x["slots"]]) for n in ("k", "v"))
    q = x["q"].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for f, n, c, table, parents in x["seqs"]:
        slots = _context_slots(n, c, table).to(q.device)
        k, v = hold(x["k"][slots]), hold(x["v"][slots])
        sees = np.zeros((n, n + c), dtype=bool)
        for i in range(n):
            if parents is None:
                sees[i, : c + i + 1] = True
            elif parents[i] != PAD:
                sees[i, :c] = True
                j = i
                while j >= 0:
                    sees[i, c + j] = True
                    j = parents[j]
        live = torch.from_numpy(sees.any(1)).to(q.device)
        sees_t = torch.from_numpy(sees).to(q.device)
        for h in range(q.shape[1]):
            s = q[f : f + n, h] @ k[:, h // GROUP].T * SCALE
            s[~sees_t] = -math.inf
            s[~live] = 0.0
            o = torch.softmax(s, -1) @ v[:, h // GROUP]
            o[~live] = 0.0
            out[f : f + n, h] = o
    return out

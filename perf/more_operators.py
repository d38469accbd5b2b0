"""Timed calls of the operators that fill a target's paged cache and keep it bounded: the attention of
a chunk of new tokens over the cached ones, the attention weight that each cached key has received, and
the eviction of the keys that received least.

A serving engine takes a prompt in chunks (with requests that decode one token riding in the same
batch), adds up from the chunk's log-sum-exp what weight every cached key got, and, where a request's
cache outgrows its budget, keeps the heaviest keys of each head.  ``run`` computes each call in
elementary torch operations, or through the framework where ``own`` is set.

Lengths and page layouts come from the case itself (``lens`` seeds them); the seed given to
``prepare`` makes the tensors' values.
"""

import math
import random
import sys
import types
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
TOPIC = 64  # tokens over which attention moves together


def listed():
    return [
        # A short follow-up question of one request: launch latency counts.
        dict(name="chunk-37", kind="chunk", rows=1, qlo=37, qhi=37, single=0, before_lo=211, before_hi=211, window=0,
             lens=1, hq=32, hkv=4, d=128, block=16, dtype="bf16"),
        # A whole prompt in one chunk, which attends to itself: half of the score matrix is masked.
        dict(name="chunk-4096-self", kind="chunk", rows=1, qlo=4096, qhi=4096, single=0, before_lo=0, before_hi=0,
             window=0, lens=2, hq=32, hkv=8, d=128, block=16, dtype="bf16"),
        # A chunk deep inside a long prompt: few query tiles, many keys.
        dict(name="chunk-512-on-32k", kind="chunk", rows=1, qlo=512, qhi=512, single=0, before_lo=32251,
             before_hi=32251, window=0, lens=3, hq=32, hkv=4, d=128, block=128, dtype="bf16"),
        # A mixed batch: prompt chunks of some requests beside single tokens of others, heads of 64 in fp16.
        dict(name="chunk-mixed-11-d64", kind="chunk", rows=11, qlo=150, qhi=420, single=7, before_lo=300,
             before_hi=5000, window=0, lens=4, hq=64, hkv=8, d=64, block=16, dtype="fp16"),
        # A layer with a sliding window and wide heads, ragged chunks, pages that end inside a tile.
        dict(name="chunk-window-d256", kind="chunk", rows=3, qlo=1200, qhi=2500, single=0, before_lo=0, before_hi=2100,
             window=1024, lens=5, hq=16, hkv=2, d=256, block=48, dtype="bf16"),
        # Two requests' single tokens over short caches: launch latency counts.
        dict(name="mass-2x300", kind="mass", rows=2, qlo=1, qhi=1, single=0, before_lo=200, before_hi=400, window=0,
             lens=6, hq=32, hkv=4, d=128, block=16, dtype="bf16"),
        # One decoding step of a batch: bound by the keys' bytes.
        dict(name="mass-16x1-on-16k", kind="mass", rows=16, qlo=1, qhi=1, single=0, before_lo=4096, before_hi=16384,
             window=0, lens=7, hq=32, hkv=4, d=128, block=128, dtype="bf16"),
        # The last tokens of several prompts weigh their whole caches: an observation window.
        dict(name="mass-6x32-d64", kind="mass", rows=6, qlo=32, qhi=32, single=0, before_lo=3000, before_hi=24000,
             window=0, lens=8, hq=64, hkv=8, d=64, block=16, dtype="fp16"),
        # A prompt chunk weighs its cache with every token: bound by the matrix product.
        dict(name="mass-2048-on-8k", kind="mass", rows=1, qlo=2048, qhi=2048, single=0, before_lo=6150, before_hi=6150,
             window=0, lens=9, hq=32, hkv=8, d=128, block=16, dtype="bf16"),
        # A decoding step at the budget: one token too many in every row.
        dict(name="evict-step-16", kind="evict", rows=16, lo=2049, hi=2049, keep_lo=2048, keep_hi=2048, settled=2048,
             gone=1400, sinks=4, recent=64, lens=10, hkv=4, d=128, block=128, dtype="bf16"),
        # Requests of ragged lengths and budgets after their prompts, some below their budget.
        dict(name="evict-ragged-57-d64", kind="evict", rows=57, lo=90, hi=6000, keep_lo=300, keep_hi=2100, settled=0,
             gone=0, sinks=4, recent=32, lens=11, hkv=8, d=64, block=16, dtype="fp16"),
        # Long prompts cut to their budgets.
        dict(name="evict-4x32k", kind="evict", rows=4, lo=20000, hi=32768, keep_lo=4096, keep_hi=4096, settled=0, gone=0,
             sinks=4, recent=256, lens=12, hkv=8, d=128, block=16, dtype="bf16"),
    ]


HEADS = ((32, 4), (64, 8), (32, 8), (16, 2), (28, 4), (16, 16), (40, 8))


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("chunk", "mass", "evict"), (4, 3, 3))[0]
    dtype, lens = rng.choice(("bf16", "bf16", "fp16")), rng.randrange(1 << 30)
    hq, hkv = rng.choice(HEADS)
    d, block = rng.choice((64, 128, 128, 256)), rng.choice((16, 16, 48, 128))
    if kind == "evict":
        rows = _log_int(rng, 1, 64)
        hi = _log_int(rng, 64, max(100, min(32768, int(6.0e7 / (rows * hkv * d)))))
        settled = rng.choice((0, 0, hi // 2))
        keep = _log_int(rng, 24, max(32, settled or hi))
        return dict(kind="evict", rows=rows, lo=max(1, settled, int(hi * rng.random())), hi=hi,
                    keep_lo=max(24, int(keep * rng.random())), keep_hi=max(24, keep), settled=settled,
                    gone=rng.randint(1, 2000) if settled else 0, sinks=rng.choice((0, 4)), recent=rng.choice((0, 16)),
                    lens=lens, hkv=hkv, d=d, block=block, dtype=dtype)
    rows = _log_int(rng, 1, 20)
    # Padded scores and products stay below the largest listed case's.
    most = 1 if kind == "mass" and rng.random() < 0.4 else _log_int(rng, 1, 2048)
    pairs = int(min(4.0e8 / (rows * hq), 3.0e10 / (rows * hq * d), 6.0e7 / (rows * hkv * d) * most))
    most = max(1, min(most, int(math.sqrt(pairs))))
    before = _log_int(rng, 1, max(2, min(32768, pairs // most)))
    return dict(kind=kind, rows=rows, qlo=rng.randint(1, most), qhi=most, single=rng.randint(0, rows - 1),
                before_lo=int(before * rng.random()), before_hi=before, window=rng.choice((0, 0, 0, rng.randint(1, 2048))),
                lens=lens, hq=hq, hkv=hkv, d=d, block=block, dtype=dtype)


# ---- inputs --------------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cdiv(a, b):
    return -(-a // b)


def _rows(case):
    """(query counts, total lengths): `single` rows have one query token, rows that decode among chunks."""
    r = random.Random(case["lens"])
    qlens = [r.randint(case["qlo"], case["qhi"]) for _ in range(case["rows"])]
    for b in r.sample(range(case["rows"]), case["single"]):
        qlens[b] = 1
    return qlens, [n + r.randint(case["before_lo"], case["before_hi"]) for n in qlens]


def _table(case, lens, width):
    """Pages of each row in no order, and their number."""
    counts = [_cdiv(n, case["block"]) for n in lens]
    order = list(range(sum(counts)))
    random.Random(case["lens"] + 1).shuffle(order)
    table = []
    for n in counts:
        table.append([order.pop() for _ in range(n)] + [0] * (width - n))
    return table, sum(counts)


def _prepare_attend(case, seed):
    g = _generator(seed)
    dtype, hq, hkv, d, block = DTYPES[case["dtype"]], case["hq"], case["hkv"], case["d"], case["block"]
    qlens, tlens = _rows(case)
    width = max(_cdiv(t, block) for t in tlens)
    table, pages = _table(case, tlens, width)
    tokens = sum(qlens)
    # Attention is uneven in earnest: queries lean towards one direction a head, and stretches of keys
    # towards or away from it by amounts that move the logits by a few units.
    lean = torch.nn.functional.normalize(torch.randn((hkv, d), generator=g, device="cuda"), dim=-1)
    query = torch.randn((tokens, hkv, hq // hkv, d), generator=g, device="cuda") + 0.5 * math.sqrt(d) * lean[:, None]
    keys = torch.randn((pages * block, hkv, d), generator=g, device="cuda")
    much = torch.randn((_cdiv(pages * block, TOPIC), hkv, 1), generator=g, device="cuda").repeat_interleave(TOPIC, 0)
    keys += 3.0 * much[: pages * block] * lean
    values = torch.randn((pages, block, hkv, d), generator=g, device="cuda").to(dtype)
    starts = [sum(qlens[:i]) for i in range(len(qlens))]
    state = types.SimpleNamespace(
        kind=case["kind"], query=query.reshape(tokens, hq, d).to(dtype),
        key_cache=keys.reshape(pages, block, hkv, d).to(dtype), value_cache=values, table=_i32(table),
        query_start=_i32(starts), query_len=_i32(qlens), target_len=_i32(tlens), scale=1.0 / math.sqrt(d),
        window=case["window"] or None,
        # What a scheduler knows on the host: the longest row and the most query tokens of one.
        longest=max(tlens), most=max(qlens), workspace=None, reuse={})
    if case["kind"] == "chunk":
        state.output = torch.zeros((tokens, hq, d), dtype=dtype, device="cuda")
        state.lse = torch.zeros((tokens, hq), dtype=torch.float32, device="cuda")
    else:
        del state.value_cache
        # The log-sum-exp of the layer's attention, and what weight the keys received before.
        state.lse = torch.zeros((tokens, hq), dtype=torch.float32, device="cuda")
        _, at, top, total = _plain_scores(state)
        state.lse.index_copy_(0, at[at < tokens], (top + torch.log(total)).permute(1, 2, 0, 3).reshape(*at.shape, hq)[at < tokens])
        shape = (case["rows"], hkv, width * block)
        old = torch.arange(shape[2], device="cuda") < (state.target_len - state.query_len)[:, None, None]
        state.previous = torch.rand(shape, generator=g, device="cuda").square() * 4 * old
        state.decay = 0.97
        state.mass = torch.zeros(shape, device="cuda")
    if own:
        if case["kind"] == "chunk":
            from ds355 import chunk_attention

            state.workspace = chunk_attention.new_chunk_workspace(len(qlens), tokens, hq, hkv, d, "cuda:0")
        else:
            from ds355 import eviction

            state.workspace = eviction.new_mass_workspace("cuda:0")
    return state


def _evict_rows(case):
    """(lengths, kept lengths) of the rows."""
    r = random.Random(case["lens"])
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["rows"])]
    return lens, [r.randint(case["keep_lo"], case["keep_hi"]) for _ in lens]


def _prepare_evict(case, seed):
    g = _generator(seed)
    dtype, rows, hkv, d, block = DTYPES[case["dtype"]], case["rows"], case["hkv"], case["d"], case["block"]
    lens, keep = _evict_rows(case)
    width = max(_cdiv(n, block) for n in lens)
    table, pages = _table(case, lens, width)
    caches = [torch.randn((pages, block, hkv, d), generator=g, device="cuda").to(dtype) for _ in range(2)]
    shape = (rows, hkv, width * block)
    size = rows * hkv * width * block
    # Mass, positions and what is settled lie in one buffer, which every pass starts from again.
    book = torch.zeros((2 * size + 2 * rows,), dtype=torch.int32, device="cuda")
    mass, positions = book[:size].view(torch.float32).view(shape), book[size: 2 * size].view(shape)
    settled = book[2 * size:].view(rows, 2)
    inside = torch.arange(shape[2], device="cuda") < _i32(lens)[:, None, None]
    # A few keys hold most of the weight, and many hold none that fp16 would show.
    weight = torch.rand(shape, generator=g, device="cuda").pow(6) * 8
    mass.copy_((weight * 512).floor() / 512 * inside)
    if case["settled"]:
        total = case["settled"] + case["gone"]
        order = torch.rand((rows, hkv, total), generator=g, device="cuda").argsort(-1)[..., : case["settled"]]
        positions[..., : case["settled"]] = order.int()
        settled[:, 0], settled[:, 1] = case["settled"], case["gone"]
    state = types.SimpleNamespace(
        kind="evict", key_cache=caches[0], value_cache=caches[1], book=book, before=book.clone(), mass=mass,
        positions=positions, settled=settled, table=_i32(table), target_len=_i32(lens), keep_len=_i32(keep),
        kept_len=torch.zeros((rows,), dtype=torch.int32, device="cuda"), sinks=case["sinks"], recent=case["recent"],
        workspace=None, reuse={})
    if own:
        from ds355 import eviction

        state.workspace = eviction.new_evict_workspace(rows, hkv, shape[2], "cuda:0")
    return state


def prepare(case, seed):
    if own:
        package = str(Path.cwd() / "vllm-ascend-hust-diffspec_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
    return _prepare_evict(case, seed) if case["kind"] == "evict" else _prepare_attend(case, seed)


# ---- the plain forms -----------------------------------------------------------------------------


def _slots(s):
    """Cache slots of all rows' tokens, padded to the longest row: [rows, longest]."""
    block = s.key_cache.shape[1]
    t = torch.arange(s.longest, device="cuda")
    return s.table.long()[:, t // block] * block + t % block


def _plain_scores(s):
    """exp(logit - row maximum) of every row's query tokens, padded to the most of any row, over its keys, padded to the
    longest row: ([hkv, rows, most, group, longest], token of each, row maxima, row sums)."""
    tokens, hq, d = s.query.shape
    hkv = s.key_cache.shape[2]
    rows, most, group = s.table.shape[0], s.most, hq // hkv
    step, t = torch.arange(most, device="cuda"), torch.arange(s.longest, device="cuda")
    at = torch.where(step < s.query_len[:, None], s.query_start[:, None] + step, tokens)  # row `tokens` is none
    q = torch.cat((s.query.float(), torch.zeros((1, hq, d), device="cuda")))[at]
    q = q.reshape(rows, most, hkv, group, d).permute(2, 0, 1, 3, 4).reshape(hkv, rows, most * group, d)
    keys = s.key_cache.reshape(-1, hkv, d)[_slots(s)].float().permute(2, 0, 3, 1).contiguous()
    scores = torch.matmul(q, keys).mul_(s.scale).reshape(hkv, rows, most, group, -1)
    limit = ((s.target_len - s.query_len)[:, None] + step + 1)[..., None]  # keys that each query token sees
    hidden = t >= limit
    if s.window is not None:
        hidden |= t < limit - s.window
    scores.masked_fill_(hidden[None, :, :, None], -math.inf)
    top = scores.amax(-1).nan_to_num(neginf=0.0)
    scores.sub_(top[..., None]).exp_()
    return scores, at, top, scores.sum(-1)


def _plain_chunk(s):
    tokens, hq, d = s.query.shape
    hkv = s.key_cache.shape[2]
    weights, at, top, total = _plain_scores(s)
    rows, most, group = weights.shape[1:4]
    values = s.value_cache.reshape(-1, hkv, d)[_slots(s)].float().permute(2, 0, 1, 3).contiguous()
    out = torch.matmul(weights.reshape(hkv, rows, most * group, -1), values).reshape(hkv, rows, most, group, d)
    out = (out / total[..., None]).permute(1, 2, 0, 3, 4).reshape(rows, most, hq, d)
    output = torch.zeros((tokens + 1, hq, d), dtype=s.query.dtype, device="cuda")
    lse = torch.zeros((tokens + 1, hq), dtype=torch.float32, device="cuda")
    output[at], lse[at] = out.to(s.query.dtype), (top + torch.log(total)).permute(1, 2, 0, 3).reshape(rows, most, hq)
    return {"output": output[:tokens], "lse": lse[:tokens]}


def _plain_mass(s):
    tokens, hq, _ = s.query.shape
    hkv = s.key_cache.shape[2]
    weights, at, top, _ = _plain_scores(s)
    rows, most, group = weights.shape[1:4]
    lse = torch.cat((s.lse, torch.full((1, hq), math.inf, device="cuda")))[at]
    lse = lse.reshape(rows, most, hkv, group).permute(2, 0, 1, 3)
    weights.mul_(torch.exp(top - lse)[..., None])
    got = weights.sum((2, 3)).transpose(0, 1)  # [rows, hkv, longest]
    mass = torch.zeros_like(s.previous)
    mass[..., : s.longest] = s.previous[..., : s.longest] * s.decay + got
    inside = torch.arange(mass.shape[2], device="cuda") < s.target_len[:, None, None]
    return {"mass": mass * inside}


def _plain_evict(s):
    rows, hkv, capacity = s.mass.shape
    block = s.key_cache.shape[1]
    t = torch.arange(capacity, device="cuda")
    length, keep = s.target_len[:, None, None], s.keep_len[:, None, None]
    known, gone = s.settled[:, :1, None], s.settled[:, 1:, None]
    inside, full = t < length, length > keep
    position = torch.where(t < known, s.positions, t + gone)
    must = (position < s.sinks) | (position >= length + gone - s.recent)
    weight = torch.where(must, math.inf, s.mass).masked_fill(~inside, -math.inf)
    rank = torch.argsort(torch.argsort(weight, dim=-1, descending=True, stable=True), dim=-1)
    stays = inside & ((rank < keep) | ~full)
    source = (stays & (t >= keep) & full).nonzero(as_tuple=True)
    hole = (~stays & (t < keep) & full).nonzero(as_tuple=True)  # as many, in the same order of rows and heads
    table = s.table.long()

    def slot(where):
        return table[where[0], where[2] // block], where[2] % block, where[1]

    for cache in (s.key_cache, s.value_cache):
        cache[slot(hole)] = cache[slot(source)]
    mass, moved = s.mass.clone(), torch.where(full & (t < keep), position, s.positions).int()
    mass[hole], moved[hole] = mass[source], position[source].int()
    s.mass.copy_(torch.where(full & inside & (t >= keep), 0.0, mass))
    s.positions.copy_(moved)
    s.kept_len.copy_(torch.minimum(s.target_len, s.keep_len))
    s.settled.copy_(torch.where(full[:, 0], torch.stack((s.keep_len, s.settled[:, 1] + s.target_len - s.keep_len), -1),
                                s.settled))
    return _evict_outputs(s)


def _evict_outputs(s):
    return {"key_cache": s.key_cache, "value_cache": s.value_cache, "mass": s.mass, "positions": s.positions,
            "settled": s.settled, "kept_len": s.kept_len}


# ---- the framework's calls -----------------------------------------------------------------------


def _own_chunk(s):
    from ds355 import chunk_attention

    chunk_attention.chunk_attention(
        s.query, s.key_cache, s.value_cache, s.output, s.lse, s.table, s.query_start, s.query_len, s.target_len,
        scale=s.scale, window=s.window, workspace=s.workspace, reuse=s.reuse)
    return {"output": s.output, "lse": s.lse}


def _own_mass(s):
    from ds355 import eviction

    eviction.attention_mass(
        s.query, s.key_cache, s.lse, s.mass, s.table, s.query_start, s.query_len, s.target_len, scale=s.scale,
        previous=s.previous, decay=s.decay, window=s.window, workspace=s.workspace, reuse=s.reuse)
    return {"mass": s.mass}


def _own_evict(s):
    from ds355 import eviction

    eviction.evict_tokens(
        s.key_cache, s.value_cache, s.mass, s.positions, s.settled, s.table, s.target_len, s.keep_len, s.kept_len,
        sinks=s.sinks, recent=s.recent, workspace=s.workspace, reuse=s.reuse)
    return _evict_outputs(s)


_PLAIN = {"chunk": _plain_chunk, "mass": _plain_mass, "evict": _plain_evict}
_OWN = {"chunk": _own_chunk, "mass": _own_mass, "evict": _own_evict}


def run(state):
    if state.kind == "evict":
        # The weights and positions of the pass before come back; the caches still hold, behind the kept tokens, what
        # a pass moves, and what it overwrites it overwrites with the same bytes.
        state.book.copy_(state.before)
    return (_OWN if own else _PLAIN)[state.kind](state)


# ---- the definitions in 64 bits ------------------------------------------------------------------


def _exact_attend(case, seed):
    s = _prepare_attend(case, seed)
    qlens, tlens = _rows(case)
    tokens, hq, d = s.query.shape
    group = hq // case["hkv"]
    out = torch.zeros((tokens, hq, d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((tokens, hq), dtype=torch.float64, device="cuda")
    if case["kind"] == "mass":
        mass = torch.zeros_like(s.previous, dtype=torch.float64)
        for b, n in enumerate(tlens):
            mass[b, :, :n] = s.previous[b, :, :n].double() * s.decay
    at = 0
    for b, (n, length) in enumerate(zip(qlens, tlens)):
        pages = s.table[b, : _cdiv(length, case["block"])].long()
        last = torch.arange(length - n, length, device="cuda")[:, None] - torch.arange(length, device="cuda")
        hidden = last < 0
        if case["window"]:
            hidden |= last >= case["window"]
        for h in range(hq):
            k = s.key_cache[pages, :, h // group].reshape(-1, d)[:length].double()
            logits = torch.mm(s.query[at: at + n, h].double(), k.t().contiguous()) * s.scale
            logits[hidden] = -math.inf
            if case["kind"] == "mass":
                mass[b, h // group, :length] += torch.exp(logits - s.lse[at: at + n, h].double()[:, None]).sum(0)
                continue
            v = s.value_cache[pages, :, h // group].reshape(-1, d)[:length].double()
            out[at: at + n, h] = torch.mm(torch.softmax(logits, -1), v)
            lse[at: at + n, h] = torch.logsumexp(logits, -1)
        at += n
    return {"mass": mass} if case["kind"] == "mass" else {"output": out, "lse": lse}


def _exact_evict(case, seed):
    """The rule head by head on the host."""
    s = _prepare_evict(case, seed)
    lens, keep = _evict_rows(case)
    block, table = case["block"], s.table.cpu().numpy()
    mass, positions, settled = (x.cpu().numpy().copy() for x in (s.mass, s.positions, s.settled))
    moves = []
    for b, (n, k) in enumerate(zip(lens, keep)):
        if n <= k:
            continue
        known, gone = settled[b]
        for h in range(case["hkv"]):
            place = np.concatenate((positions[b, h, :known], np.arange(known, n) + gone))
            must = (place < case["sinks"]) | (place >= n + gone - case["recent"])
            best = np.lexsort((np.arange(n), -mass[b, h, :n].astype(np.float64), ~must))[:k]
            stays = np.zeros(n, dtype=bool)
            stays[best] = True
            holes, movers = np.flatnonzero(~stays[:k]), k + np.flatnonzero(stays[k:])
            moves.append(np.stack((table[b][movers // block], movers % block, table[b][holes // block], holes % block,
                                   np.full(len(holes), h)), -1))
            positions[b, h, :k] = place[:k]
            positions[b, h, holes], mass[b, h, holes] = place[movers], mass[b, h, movers]
            mass[b, h, k:n] = 0
        settled[b] = k, gone + n - k
    caches = [s.key_cache.double(), s.value_cache.double()]
    if moves:
        m = torch.tensor(np.concatenate(moves), device="cuda").long()
        for cache in caches:
            cache[m[:, 2], m[:, 3], m[:, 4]] = cache[m[:, 0], m[:, 1], m[:, 4]]
    return {"key_cache": caches[0], "value_cache": caches[1], "mass": torch.tensor(mass).double(),
            "positions": torch.tensor(positions), "settled": torch.tensor(settled),
            "kept_len": _i32([min(n, k) for n, k in zip(lens, keep)])}


def exact(case, seed):
    return _exact_evict(case, seed) if case["kind"] == "evict" else _exact_attend(case, seed)


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    hkv, d, size = case["hkv"], case["d"], DTYPES[case["dtype"]].itemsize
    if case["kind"] == "evict":
        moved = read = kept = 0
        for n, k in zip(*_evict_rows(case)):
            if n > k:  # the newest are behind the kept places, and a like part of the others
                newest = min(case["recent"], n - k)
                moved += newest + (n - k - newest) * max(0, k - case["recent"]) // n
                read += 4 * n + 4 * min(n, case["settled"])
                kept += 4 * (k - min(k, case["settled"])) + 4 * (n - k)
        return {"bytes": hkv * (moved * (4 * d * size + 16) + read + kept), "flops": 0}
    hq, window = case["hq"], case["window"]
    pairs = keys = 0
    qlens, tlens = _rows(case)
    for n, t in zip(qlens, tlens):
        first = t - n + 1  # keys that the first query token sees
        if window:
            capped = min(n, max(0, t - window))  # query tokens that see a whole window and more lies before it
            pairs += capped * window + sum(range(first, first + n - capped))
            keys += min(t, n + window - 1)
        else:
            pairs += n * first + n * (n - 1) // 2
            keys += t
    if case["kind"] == "mass":
        return {"bytes": keys * hkv * d * size + sum(qlens) * hq * (d * size + 4) + sum(tlens) * hkv * 8,
                "flops": 2 * pairs * hq * d}
    return {"bytes": 2 * keys * hkv * d * size + sum(qlens) * hq * (2 * d * size + 4), "flops": 4 * pairs * hq * d}

"""Timed calls of the verifier-side operators: page tables that share prompts, the per-head norm
and rotation that fills the pages, and the attention that reads a shared prefix once.

A verification step of a serving engine forks requests from a common prompt (their page tables
share its pages), grows the tables for the draft tokens and cuts them back after rejection, norms
and rotates the queries and keys of the new tokens into the pages, and attends over them; the
attention's log-sum-exp is what the chunk scoring of the draft context takes.  ``run`` computes
each call in elementary torch operations, or through the framework where ``own`` is set.

Page layouts and lengths come from the case itself (``lens`` seeds them); the seed given to
``prepare`` makes the tensors' values.
"""

import math
import random
import sys
import types
from pathlib import Path

import torch

own = False

ROPE_THETA = 1.0e6
EPS = 1.0e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
TOPIC = 64  # tokens over which attention moves together


def listed():
    return [
        # Two samples of one short prompt, decoding one token each: launch latency counts.
        dict(name="attend-2x1k", kind="attend", rows=2, prefix=1024, lo=40, hi=200, qlo=1, qhi=1, lens=1, hq=32,
             hkv=4, d=128, block=16, dtype="bf16", pad=0),
        # A batch of agents behind one system prompt and document set, one token each: bound by the
        # pages' bytes, of which the rows' own parts are the larger half.
        dict(name="attend-16x16k", kind="attend", rows=16, prefix=16384, lo=500, hi=4000, qlo=1, qhi=1, lens=2,
             hq=32, hkv=4, d=128, block=128, dtype="bf16", pad=0),
        # The same batch verifying four draft tokens and the root over a 32k prompt: 640 query
        # rows a KV head meet every prefix key, bound by the matrix products.
        dict(name="attend-16x32k-verify", kind="attend", rows=16, prefix=32768, lo=300, hi=4096, qlo=5, qhi=5,
             lens=3, hq=32, hkv=4, d=128, block=128, dtype="bf16", pad=0),
        # Many requests with ragged query counts, a prompt that ends inside a page, head_dim 64 in
        # fp16 and a graph bucket larger than the batch.
        dict(name="attend-57-ragged-d64", kind="attend", rows=57, prefix=5003, lo=17, hi=1500, qlo=1, qhi=6, lens=4,
             hq=64, hkv=8, d=64, block=16, dtype="fp16", pad=7),
        # Queries and keys of one decoding batch out of the fused projection, keys and values into the pages.
        dict(name="qk-decode-16", kind="qk", tokens=16, hq=32, hkv=4, d=128, rot=128, neox=True, dtype="bf16",
             block=16, normed=False, far=40960, lens=5),
        # A verified batch with interleaved rotation over half of each head, in fp16.
        dict(name="qk-verify-320-gptj", kind="qk", tokens=320, hq=64, hkv=8, d=64, rot=32, neox=False, dtype="fp16",
             block=48, normed=False, far=131072, lens=6),
        # A prompt batch's prefill, which also keeps the normed keys before rotation for the draft's raw cache.
        dict(name="qk-prefill-16k", kind="qk", tokens=16411, hq=32, hkv=8, d=128, rot=128, neox=True, dtype="bf16",
             block=128, normed=True, far=40960, lens=7),
        # Four samples forked from one prompt: each shares its full pages and copies the last one.
        dict(name="fork-4", kind="fork", parents=1, children=4, lo=500, hi=900, pages=512, width=64, caches=4,
             block=16, hkv=4, d=128, dtype="bf16", lens=8),
        # A wide batch re-forked from eight prompts (a search step that restarts its branches).
        dict(name="fork-248", kind="fork", parents=8, children=248, lo=1000, hi=4000, pages=4096, width=256,
             caches=8, block=16, hkv=8, d=128, dtype="bf16", lens=9),
        # After verification: 128 rows cut back to their committed lengths, then grown for the next
        # draft tokens (and some for a prompt chunk).
        dict(name="regrow-128", kind="regrow", rows=128, lo=200, hi=12000, grow=300, pages=65536, width=1280,
             caches=1, block=16, hkv=1, d=64, dtype="bf16", lens=10),
        # Pages of swapped-in requests copied to their new places over all layers' caches.
        dict(name="copy-200", kind="copy", pairs=200, pages=1024, width=1, caches=12, block=16, hkv=8, d=128,
             dtype="bf16", lens=11),
        # A pool left full of holes by finished requests, compacted for a resize.
        dict(name="compact-4096", kind="compact", rows=64, lo=100, hi=1700, pages=4096, width=64, caches=8, block=32,
             hkv=8, d=128, dtype="fp16", lens=12),
    ]


HEADS = ((32, 4), (64, 8), (32, 8), (16, 2), (28, 4), (16, 16), (40, 8))


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("attend", "qk", "fork", "regrow", "copy", "compact"), (6, 4, 2, 1, 1, 1))[0]
    lens = rng.randrange(1 << 30)
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    hq, hkv = rng.choice(HEADS)
    if kind == "attend":
        rows = _log_int(rng, 1, 64)
        qhi = rng.choice((1, 1, 2, 5, 8))
        d = rng.choice((64, 128, 128, 256))
        tokens = rows * qhi
        # Products and keys stay below the largest listed case's.
        prefix = _log_int(rng, 100, max(200, min(40000, int(7.0e7 / (tokens * hq)), int(1.0e10 / (tokens * hq * d)))))
        hi = _log_int(rng, 2 * qhi, max(3 * qhi, min(4096, int(3.0e7 / (rows * hkv * d)))))
        return dict(kind="attend", rows=rows, prefix=prefix, lo=max(qhi, int(hi * rng.random())), hi=hi,
                    qlo=rng.randint(1, qhi), qhi=qhi, lens=lens, hq=hq, hkv=hkv, d=d,
                    block=rng.choice((16, 16, 48, 128)), dtype=dtype, pad=rng.choice((0, 0, 3)))
    if kind == "qk":
        d = rng.choice((64, 96, 128, 128, 256))
        tokens = _log_int(rng, 1, max(2, min(16384, int(1.0e8 / ((hq + 2 * hkv) * d)))))
        return dict(kind="qk", tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rng.choice((d, d, d // 2)),
                    neox=rng.random() < 0.7, dtype=dtype, block=rng.choice((16, 48, 128)),
                    normed=rng.random() < 0.4, far=rng.choice((4096, 40960, 131072)), lens=lens)
    heads, d, block = rng.choice((1, 2, 4, 8)), rng.choice((64, 128)), rng.choice((16, 32))
    case = dict(kind=kind, caches=rng.choice((1, 2, 4, 8)), block=block, hkv=heads, d=d, dtype=dtype, lens=lens)
    if kind == "fork":
        case.update(parents=rng.randint(1, 8), children=_log_int(rng, 1, 248), pages=4096)
        hi = rng.randint(block, 128 * block)
        case.update(lo=rng.randint(1, hi), hi=hi, width=rng.choice((128, 160)))
    elif kind == "regrow":
        rows = _log_int(rng, 1, 128)
        hi = _log_int(rng, 2 * block, 400 * block)
        case.update(rows=rows, lo=rng.randint(1, hi), hi=hi, grow=rng.choice((5, 5, 300)), width=448, caches=1,
                    hkv=1, pages=rows * 448)
    elif kind == "copy":
        pages = _log_int(rng, 16, 1024)
        case.update(pairs=rng.randint(1, pages // 2), pages=pages, width=1)
    else:
        rows = _log_int(rng, 1, 64)
        hi = rng.randint(1, 48 * block)
        case.update(rows=rows, lo=rng.randint(1, hi), hi=hi, width=64, pages=64 * rows + rng.randint(0, 50))
    return case


# ---- inputs --------------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cdiv(a, b):
    return -(-a // b)


def _attend_rows(case):
    """(query counts, total lengths) of a case's rows; padding rows have no query and no length."""
    r = random.Random(case["lens"])
    qlens = [r.randint(case["qlo"], case["qhi"]) for _ in range(case["rows"])]
    tlens = [case["prefix"] + max(q, r.randint(case["lo"], case["hi"])) for q in qlens]
    return qlens + [0] * case["pad"], tlens + [0] * case["pad"]


def _attend_table(case):
    """Page table of rows forked from one prompt: its full pages shared, the rest each row's own.

    Returns (table rows, pages in all, (first row's, other rows') copies of a partial last prompt page).
    """
    block, prefix = case["block"], case["prefix"]
    qlens, tlens = _attend_rows(case)
    width = max(_cdiv(t, block) for t in tlens)
    shared = prefix // block
    own_pages = [max(0, _cdiv(t, block) - shared) if t else 0 for t in tlens]
    total = shared + sum(own_pages)
    order = list(range(total))
    random.Random(case["lens"] + 1).shuffle(order)
    table, at = [], shared
    for n in own_pages:
        table.append(order[:shared] + order[at: at + n] + [0] * (width - shared - n) if n else [0] * width)
        at += n
    partial = [t[shared] for t, n in zip(table, own_pages) if n] if prefix % block else []
    return table, total, (partial[:1], partial[1:])


def _prepare_attend(case, seed):
    g = _generator(seed)
    dtype, hq, hkv, d, block = DTYPES[case["dtype"]], case["hq"], case["hkv"], case["d"], case["block"]
    qlens, tlens = _attend_rows(case)
    table, pages, (first, others) = _attend_table(case)
    tokens = sum(qlens) + case["pad"]
    # Attention mass is uneven in earnest: queries lean towards one direction a head, and stretches
    # of keys towards or away from it by amounts that move the logits by a few units.
    lean = torch.nn.functional.normalize(torch.randn((hkv, d), generator=g, device="cuda"), dim=-1)
    query = torch.randn((tokens, hkv, hq // hkv, d), generator=g, device="cuda") + 0.5 * math.sqrt(d) * lean[:, None]
    keys = torch.randn((pages, block, hkv, d), generator=g, device="cuda")
    much = torch.randn((_cdiv(pages * block, TOPIC), hkv, 1), generator=g, device="cuda").repeat_interleave(TOPIC, 0)
    keys += 3.0 * much[: pages * block].reshape(pages, block, hkv, 1) * lean
    keys = keys.to(dtype)
    values = _randn((pages, block, hkv, d), g, dtype)
    if others:
        keys[others], values[others] = keys[first], values[first]
        own_part = case["prefix"] % block  # the rest of a copied page is the row's own
        keys[others, own_part:] = _randn((len(others), block - own_part, hkv, d), g, dtype)
        values[others, own_part:] = _randn((len(others), block - own_part, hkv, d), g, dtype)
    starts = [sum(qlens[:i]) for i in range(len(qlens))]
    state = types.SimpleNamespace(
        kind="attend", query=query.reshape(tokens, hq, d).to(dtype), key_cache=keys, value_cache=values,
        table=_i32(table), query_start=_i32(starts), query_len=_i32(qlens), target_len=_i32(tlens),
        prefix_len=_i32([case["prefix"]]), scale=1.0 / math.sqrt(d),
        # What a scheduler knows on the host: the prefix, the longest own part and the most query tokens.
        prefix=case["prefix"], longest=max(tlens) - case["prefix"], most=max(qlens),
        output=torch.zeros((tokens, hq, d), dtype=dtype, device="cuda"),
        lse=torch.zeros((tokens, hq), dtype=torch.float32, device="cuda"), workspace=None, reuse={})
    if own:
        from ds355 import prefix_attention

        state.workspace = prefix_attention.new_prefix_workspace(len(qlens), tokens, hq, hkv, d, "cuda:0")
    return state


def _qk_slots(case):
    """Cache slots of the tokens (distinct, in no order), and the number of pages."""
    r = random.Random(case["lens"])
    pages = _cdiv(case["tokens"], case["block"]) + 3
    return r.sample(range(pages * case["block"]), case["tokens"]), pages


def _prepare_qk(case, seed):
    g = _generator(seed)
    dtype, tokens, hq, hkv, d = DTYPES[case["dtype"]], case["tokens"], case["hq"], case["hkv"], case["d"]
    qkv = _randn((tokens, (hq + 2 * hkv) * d), g, dtype)
    slots, pages = _qk_slots(case)
    rot, far = case["rot"], case["far"]
    inv = 1.0 / (ROPE_THETA ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot))
    freqs = torch.outer(torch.arange(far, dtype=torch.float64), inv)
    state = types.SimpleNamespace(
        kind="qk", query=qkv[:, : hq * d].unflatten(1, (hq, d)), key=qkv[:, hq * d: (hq + hkv) * d].unflatten(1, (hkv, d)),
        value=qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d)),
        q_weight=(1 + 0.2 * torch.randn((d,), generator=g, device="cuda")).to(dtype),
        k_weight=(1 + 0.2 * torch.randn((d,), generator=g, device="cuda")).to(dtype),
        positions=torch.randint(0, far, (tokens,), generator=g, device="cuda"),
        cos_sin=torch.cat((freqs.cos(), freqs.sin()), -1).float().cuda(), rot=rot, neox=case["neox"],
        slots=torch.tensor(slots, device="cuda"),
        query_out=torch.zeros((tokens, hq, d), dtype=dtype, device="cuda"),
        normed=torch.zeros((tokens, hkv, d), dtype=dtype, device="cuda") if case["normed"] else None,
        key_cache=torch.zeros((pages, case["block"], hkv, d), dtype=dtype, device="cuda"),
        value_cache=torch.zeros((pages, case["block"], hkv, d), dtype=dtype, device="cuda"), reuse={})
    return state


def _pool_rows(case):
    """What a pool's rows hold, on the host: (table rows, reference counts, call's row lists, call's lengths)."""
    kind, block, width, pages = case["kind"], case["block"], case["width"], case["pages"]
    r = random.Random(case["lens"])
    order = list(range(pages))
    r.shuffle(order)
    refs = [0] * pages
    table = []

    def hold(n):
        row = [order.pop() for _ in range(min(n, width, len(order)))]
        for p in row:
            refs[p] += 1
        table.append(row + [-1] * (width - len(row)))
        return len(row)

    if kind == "fork":
        plens = [r.randint(case["lo"], case["hi"]) for _ in range(case["parents"])]
        plens = [min(hold(_cdiv(n, block)) * block, n) for n in plens]
        for _ in range(case["children"]):
            hold(r.randint(0, 3))  # what the branch before held
        parents = [r.randrange(case["parents"]) for _ in range(case["children"])]
        children = [case["parents"] + i for i in range(case["children"])]
        return table, refs, (parents, children), [r.randint(max(0, plens[p] - 2 * block), plens[p]) for p in parents]
    if kind == "copy":
        table.append([-1] * width)
        picked = r.sample(range(pages), 2 * case["pairs"])
        return table, refs, (picked[: case["pairs"]], picked[case["pairs"]:]), []
    held = [hold(_cdiv(r.randint(case["lo"], case["hi"]), block)) for _ in range(case["rows"])]
    if kind == "regrow":
        keep = [r.randint(max(0, n * block - 40), n * block) for n in held]
        grown = [min(k + (5 if r.random() < 0.7 else r.randint(0, case["grow"])), width * block) for k in keep]
        return table, refs, (r.sample(range(case["rows"]), case["rows"]),), (keep, grown)
    for row in range(case["rows"]):  # some rows share the first pages of the row before
        if row and r.random() < 0.4:
            n = r.randint(0, min(held[row], held[row - 1]))
            for c in range(n):
                refs[table[row][c]] -= 1
                table[row][c] = table[row - 1][c]
                refs[table[row][c]] += 1
    return table, refs, (), []


def _prepare_pool(case, seed):
    g = _generator(seed)
    shape = (case["caches"], case["pages"], case["block"], case["hkv"], case["d"])
    caches = torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda")
    for cache in caches:
        cache.copy_(torch.randn(shape[1:], generator=g, device="cuda", dtype=torch.float32))
    table, refs, rows, lens = _pool_rows(case)
    state = types.SimpleNamespace(
        kind=case["kind"], caches=caches, table=_i32(table), refs=_i32(refs), rows=[_i32(x) for x in rows],
        block=case["block"], pool=None)
    if case["kind"] == "regrow":
        state.keep, state.lens = _i32([lens[0][i] for i in rows[0]]), _i32([lens[1][i] for i in rows[0]])
    elif case["kind"] == "fork":
        state.lens = _i32(lens)
    if case["kind"] == "compact":
        state.table_before, state.refs_before = state.table.clone(), state.refs.clone()
    if own:
        from ds355 import pages

        state.pool = pages.PagePool(list(caches), ref_counts=state.refs)
    return state


def prepare(case, seed):
    if own:
        package = str(Path.cwd() / "vllm-ascend-hust-diffspec_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
    return {"attend": _prepare_attend, "qk": _prepare_qk}.get(case["kind"], _prepare_pool)(case, seed)


# ---- the plain forms -----------------------------------------------------------------------------


def _plain_attend(s):
    """Prefix logits of all query tokens at once, own logits row by row in a padded batch, one softmax."""
    tokens, hq, d = s.query.shape
    hkv, block = s.key_cache.shape[2], s.key_cache.shape[1]
    group, rows, most = hq // hkv, s.table.shape[0], s.most
    device = s.query.device
    flat_k, flat_v = s.key_cache.reshape(-1, hkv, d), s.value_cache.reshape(-1, hkv, d)
    table = s.table.long()

    # Every row's query tokens, padded to the most of any row; row `tokens` stands for none.
    step = torch.arange(most, device=device)
    at = torch.where(step < s.query_len[:, None], s.query_start[:, None] + step, tokens)
    q = torch.cat((s.query.float(), torch.zeros((1, hq, d), device=device)))[at]  # [rows, most, hq, d]
    q = q.reshape(rows, most, hkv, group, d).permute(2, 0, 1, 3, 4)  # [hkv, rows, most, group, d]
    limit = (s.target_len - s.query_len)[:, None] + step + 1  # keys that each query token sees

    t = torch.arange(s.prefix, device=device)
    where = table[0, t // block] * block + t % block
    k, v = flat_k[where].float().permute(1, 2, 0), flat_v[where].float().transpose(0, 1)  # [hkv, d, n], [hkv, n, d]
    before = torch.matmul(q.reshape(hkv, -1, d), k.contiguous()).reshape(hkv, rows, most, group, -1) * s.scale
    before = before.masked_fill((t >= limit[..., None])[None, :, :, None], -math.inf)

    u = torch.arange(s.longest, device=device)
    pos = (s.prefix + u).clamp(max=table.shape[1] * block - 1)
    where = table[:, pos // block] * block + pos % block  # [rows, longest]
    ok, ov = flat_k[where].float().permute(2, 0, 3, 1), flat_v[where].float().permute(2, 0, 1, 3)
    after = torch.matmul(q.reshape(hkv, rows, most * group, d), ok.contiguous()).reshape(hkv, rows, most, group, -1)
    seen = (s.prefix + u < limit[..., None])[None, :, :, None]
    after = (after * s.scale).masked_fill(~seen, -math.inf)

    top = torch.maximum(before.amax(-1), after.amax(-1))
    before, after = torch.exp(before - top[..., None]), torch.exp(after - top[..., None])
    total = before.sum(-1) + after.sum(-1)
    out = torch.matmul(before.reshape(hkv, -1, s.prefix), v.contiguous()).reshape(hkv, rows, most, group, d)
    out = out + torch.matmul(after.reshape(hkv, rows, most * group, -1), ov.contiguous()).reshape(out.shape)
    out = (out / total[..., None]).permute(1, 2, 0, 3, 4).reshape(rows, most, hq, d)
    lse = (top + torch.log(total)).permute(1, 2, 0, 3).reshape(rows, most, hq)
    output = torch.zeros((tokens + 1, hq, d), dtype=s.query.dtype, device=device)
    lses = torch.zeros((tokens + 1, hq), dtype=torch.float32, device=device)
    output[at], lses[at] = out.to(s.query.dtype), lse
    return {"output": output[:tokens], "lse": lses[:tokens]}


def _plain_norm(x, weight):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()


def _plain_rotate(x, cos_sin, positions, rot, neox):
    cs = cos_sin[positions]
    c, s = cs[:, None, : rot // 2], cs[:, None, rot // 2: rot]
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if neox else (slice(0, rot, 2), slice(1, rot, 2))
    out = x.clone()
    out[..., first] = x[..., first] * c - x[..., second] * s
    out[..., second] = x[..., second] * c + x[..., first] * s
    return out


def _plain_qk(s):
    q = _plain_rotate(_plain_norm(s.query, s.q_weight), s.cos_sin, s.positions, s.rot, s.neox)
    normed = _plain_norm(s.key, s.k_weight)
    k = _plain_rotate(normed, s.cos_sin, s.positions, s.rot, s.neox)
    s.query_out.copy_(q)
    s.key_cache.flatten(0, 1)[s.slots] = k.to(s.key_cache.dtype)
    s.value_cache.flatten(0, 1)[s.slots] = s.value
    if s.normed is not None:
        s.normed.copy_(normed)
    return _qk_outputs(s)


def _qk_outputs(s):
    out = {"query": s.query_out, "key_cache": s.key_cache, "value_cache": s.value_cache}
    if s.normed is not None:
        out["normed"] = s.normed
    return out


def _plain_release(refs, table, rows, first):
    """Entries of `rows` from column first[i] on give their pages back."""
    held = table[rows]
    gone = (torch.arange(table.shape[1], device=table.device) >= first[:, None]) & (held >= 0)
    refs.scatter_add_(0, held.clamp(min=0).long().reshape(-1), -gone.int().reshape(-1))
    table[rows] = torch.where(gone, -1, held)


def _plain_free_pages(refs):
    """All pages, the free ones first, in ascending order."""
    return torch.argsort((refs != 0).to(torch.int8), stable=True).to(torch.int32)


def _plain_take(refs, table, rows, held, need, fill):
    """`need` more pages for each row behind its `fill` entries, in the rows' order."""
    col = torch.arange(table.shape[1], device=table.device)
    new = (col >= fill[:, None]) & (col < (fill + need)[:, None])
    rank = (torch.cumsum(need, 0) - need)[:, None] + col - fill[:, None]
    picked = _plain_free_pages(refs)[rank.clamp(0, refs.numel() - 1)]
    table[rows] = torch.where(new, picked, held)
    refs.scatter_add_(0, picked.long().reshape(-1), new.int().reshape(-1))
    return picked, new


def _plain_fork(s):
    parents, children = s.rows[0].long(), s.rows[1].long()
    _plain_release(s.refs, s.table, children, torch.zeros_like(s.lens))
    full, part = s.lens // s.block, (s.lens % s.block > 0).int()
    col = torch.arange(s.table.shape[1], device=s.table.device)
    source = s.table[parents]
    shared = (col < full[:, None]) & (source >= 0)
    s.refs.scatter_add_(0, source.clamp(min=0).long().reshape(-1), shared.int().reshape(-1))
    picked, _ = _plain_take(s.refs, s.table, children, torch.where(shared, source, -1), part, full)
    last = full.clamp(max=s.table.shape[1] - 1).long()[:, None]
    src = torch.where(part > 0, source.gather(1, last)[:, 0], source[:, 0]).long()
    dst = torch.where(part > 0, picked.gather(1, last)[:, 0], source[:, 0]).long()  # else a page onto itself
    s.caches[:, dst] = s.caches[:, src]
    return _pool_outputs(s)


def _plain_regrow(s):
    rows = s.rows[0].long()
    _plain_release(s.refs, s.table, rows, (s.keep + s.block - 1) // s.block)
    held = s.table[rows]
    have = (held >= 0).sum(1, dtype=torch.int32)
    _plain_take(s.refs, s.table, rows, held, ((s.lens + s.block - 1) // s.block - have).clamp(min=0), have)
    return _pool_outputs(s)


def _plain_copy(s):
    s.caches[:, s.rows[1].long()] = s.caches[:, s.rows[0].long()]
    return _pool_outputs(s)


def _plain_compact(s):
    ids = torch.arange(s.refs.numel(), device=s.refs.device)
    live = s.refs > 0
    count = live.sum()
    mover = live & (ids >= count)
    holes = torch.argsort((live | (ids >= count)).to(torch.int8), stable=True)
    to = torch.where(mover, holes[(torch.cumsum(mover, 0) - 1).clamp(min=0)], ids)
    src = mover.nonzero()[:, 0]
    s.caches[:, to[src]] = s.caches[:, src]
    refs = torch.where(mover, 0, s.refs)
    refs[to[src]] = s.refs[src]
    s.refs.copy_(refs)
    s.table.copy_(torch.where(s.table >= 0, to[s.table.clamp(min=0).long()].int(), -1))
    return _pool_outputs(s)


def _pool_outputs(s):
    return {"caches": s.caches, "ref_counts": s.refs, "table": s.table}


# ---- the framework's calls -----------------------------------------------------------------------


def _own_attend(s):
    from ds355 import prefix_attention

    prefix_attention.shared_prefix_attention(
        s.query, s.key_cache, s.value_cache, s.output, s.lse, s.table, s.query_start, s.query_len, s.target_len,
        s.prefix_len, scale=s.scale, workspace=s.workspace, reuse=s.reuse)
    return {"output": s.output, "lse": s.lse}


def _own_qk(s):
    from ds355 import qk_rope

    qk_rope.qk_norm_rope(
        s.query, s.key, s.q_weight, s.k_weight, s.positions, s.cos_sin, eps=EPS, rotary_dim=s.rot,
        is_neox_style=s.neox, query_out=s.query_out, normed_key=s.normed, value=s.value, key_cache=s.key_cache,
        value_cache=s.value_cache, slot_mapping=s.slots, reuse=s.reuse)
    return _qk_outputs(s)


def _own_pool(s):
    if s.kind == "fork":
        s.pool.fork(s.table, s.rows[0], s.rows[1], s.lens)
    elif s.kind == "regrow":
        s.pool.free(s.table, s.rows[0], s.keep)
        s.pool.extend(s.table, s.rows[0], s.lens)
    elif s.kind == "copy":
        s.pool.copy(s.rows[0], s.rows[1])
    else:
        s.pool.compact(s.table)
    return _pool_outputs(s)


_PLAIN = {"attend": _plain_attend, "qk": _plain_qk, "fork": _plain_fork, "regrow": _plain_regrow,
          "copy": _plain_copy, "compact": _plain_compact}
_OWN = {"attend": _own_attend, "qk": _own_qk}


def run(state):
    if state.kind == "compact":  # the holes of the pass before come back; its pages still hold their bytes
        state.table.copy_(state.table_before)
        state.refs.copy_(state.refs_before)
    if own:
        return _OWN.get(state.kind, _own_pool)(state)
    return _PLAIN[state.kind](state)


# ---- the definitions in 64 bits ------------------------------------------------------------------


def _exact_attend(case, seed):
    s = _prepare_attend(case, seed)
    qlens, tlens = _attend_rows(case)
    table, _, _ = _attend_table(case)
    tokens, hq, d = s.query.shape
    group, block = hq // case["hkv"], case["block"]
    out = torch.zeros((tokens, hq, d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((tokens, hq), dtype=torch.float64, device="cuda")
    at = 0
    for row, n, length in zip(table, qlens, tlens):
        if not n:
            continue
        pages = torch.tensor(row[: _cdiv(length, block)], device="cuda")
        later = torch.arange(length, device="cuda") >= torch.arange(length - n + 1, length + 1, device="cuda")[:, None]
        for h in range(hq):
            k = s.key_cache[pages, :, h // group].reshape(-1, d)[:length].double()
            v = s.value_cache[pages, :, h // group].reshape(-1, d)[:length].double()
            logits = torch.mm(s.query[at: at + n, h].double(), k.t().contiguous()) * s.scale
            logits[later] = -math.inf
            out[at: at + n, h] = torch.mm(torch.softmax(logits, -1), v)
            lse[at: at + n, h] = torch.logsumexp(logits, -1)
        at += n
    return {"output": out, "lse": lse}


def _exact_qk(case, seed):
    s = _prepare_qk(case, seed)
    rot = case["rot"]
    cs = s.cos_sin.double()[s.positions].unsqueeze(1)
    turn = torch.complex(cs[..., : rot // 2], cs[..., rot // 2: rot])
    found = []
    for x, w in ((s.query, s.q_weight), (s.key, s.k_weight)):
        x = x.double()
        n = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()
        part = n[..., :rot]
        pairs = part.unflatten(-1, (2, rot // 2)).transpose(-1, -2) if case["neox"] else part.unflatten(-1, (rot // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = (z.transpose(-1, -2) if case["neox"] else z).flatten(-2)
        found += [n, torch.cat((z, n[..., rot:]), -1)]
    key_cache, value_cache = s.key_cache.double(), s.value_cache.double()
    key_cache.flatten(0, 1)[s.slots] = found[3]
    value_cache.flatten(0, 1)[s.slots] = s.value.double()
    out = {"query": found[1], "key_cache": key_cache, "value_cache": value_cache}
    if case["normed"]:
        out["normed"] = found[2]
    return out


def _exact_pool(case, seed):
    """The pool's rules row by row on the host; pages are copied at the end (no page is written twice)."""
    s = _prepare_pool(case, seed)
    table, refs, rows, lens = _pool_rows(case)
    kind, block = case["kind"], case["block"]
    moves = []

    def release(row, first):
        for c in range(first, case["width"]):
            if table[row][c] >= 0:
                refs[table[row][c]] -= 1
                table[row][c] = -1

    if kind == "fork":
        for child in rows[1]:
            release(child, 0)
        for parent, child, n in zip(*rows, lens):
            for c in range(n // block):
                table[child][c] = table[parent][c]
                refs[table[parent][c]] += 1
        free = [p for p in range(case["pages"]) if refs[p] == 0]
        for parent, child, n in zip(*rows, lens):
            if n % block:
                page = free.pop(0)
                refs[page], table[child][n // block] = 1, page
                moves.append((table[parent][n // block], page))
    elif kind == "regrow":
        for row in rows[0]:
            release(row, _cdiv(lens[0][row], block))
        free = [p for p in range(case["pages"]) if refs[p] == 0]
        for row in rows[0]:
            have = sum(p >= 0 for p in table[row])
            for c in range(have, _cdiv(lens[1][row], block)):
                table[row][c] = free.pop(0)
                refs[table[row][c]] = 1
    elif kind == "copy":
        moves = list(zip(*rows))
    else:
        live = [p for p in range(case["pages"]) if refs[p]]
        holes = [p for p in range(len(live)) if not refs[p]]
        moves = list(zip([p for p in live if p >= len(live)], holes))
        to = dict(moves)
        for src, dst in moves:
            refs[dst], refs[src] = refs[src], 0
        table = [[to.get(p, p) for p in row] for row in table]
    if moves:
        src, dst = (torch.tensor(x, device="cuda") for x in zip(*moves))
        s.caches[:, dst] = s.caches[:, src]
    return {"caches": s.caches.double(), "ref_counts": _i32(refs), "table": _i32(table)}


def exact(case, seed):
    return {"attend": _exact_attend, "qk": _exact_qk}.get(case["kind"], _exact_pool)(case, seed)


# ---- what a pass cannot do without ---------------------------------------------------------------


def _work_pool(case):
    table, _, rows, lens = _pool_rows(case)
    kind, block = case["kind"], case["block"]
    page = case["caches"] * block * case["hkv"] * case["d"] * DTYPES[case["dtype"]].itemsize
    if kind == "copy":
        return 2 * case["pairs"] * (page + 4)
    counts = 4 * case["pages"]  # the search for free (or live) pages reads every count
    if kind == "fork":
        # A pass frees what the pass before took: entries written twice and read once, a count up and down for each.
        entries = sum(_cdiv(n, block) for n in lens)
        return counts + 24 * entries + sum(1 for n in lens if n % block) * 2 * page + 12 * len(lens)
    if kind == "regrow":
        entries = sum(max(0, _cdiv(lens[1][r], block) - _cdiv(lens[0][r], block)) for r in rows[0])
        return counts + 24 * entries + 12 * case["rows"]
    live = len({p for row in table for p in row if p >= 0})
    moved = sum(1 for p in {p for row in table for p in row} if p >= live)
    return 2 * counts + 8 * case["rows"] * case["width"] + moved * 2 * page


def work(case):
    if case["kind"] not in ("attend", "qk"):
        return {"bytes": _work_pool(case), "flops": 0}
    hq, hkv, d, size = case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]].itemsize
    if case["kind"] == "qk":
        row = ((2 * hq + 4 * hkv) + (hkv if case["normed"] else 0)) * d * size
        return {"bytes": case["tokens"] * (row + 16 + 4 * case["rot"]),
                "flops": case["tokens"] * (hq + hkv) * (4 * d + 3 * case["rot"])}
    qlens, tlens = _attend_rows(case)
    rows = [(n, t) for n, t in zip(qlens, tlens) if n]
    keys = case["prefix"] + sum(t - case["prefix"] for _, t in rows)
    seen = sum(n * t - n * (n - 1) // 2 for n, t in rows)  # (query token, key) pairs
    return {"bytes": 2 * keys * hkv * d * size + sum(qlens) * hq * (2 * d * size + 4), "flops": 4 * seen * hq * d}

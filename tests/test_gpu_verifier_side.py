"""GPU: the verifier's side of a serving loop as one run.

A prompt is written once, rows are forked from it, decode and verify, are cut back to what was accepted,
grow again, the pool is compacted, and the retrieval scores take the attention's LSE.  The oracle keeps
every row's keys and values as plain lists, with no pages, so a wrong page, slot, count or prefix shows in
an attention output.  What each operator computes is checked by the bounds of its own tests.
"""

import pytest
import torch

import test_gpu_prefix_attention as attention
import test_gpu_qk_rope as heads
from helpers import gen, randn

pytestmark = pytest.mark.gpu


class Server:
    """Two layers of caches over one pool and block table, and the oracle's rows."""

    def __init__(self, cuda, *, rows, d, hq, hkv, block, dtype, rot, neox, seed, pages=64, width=24):
        from ds355 import prefix_attention
        from ds355.pages import PagePool

        self.cuda, self.block, self.d, self.hq, self.hkv, self.dtype = cuda, block, d, hq, hkv, dtype
        self.rot, self.neox, self.g, self.layers = rot, neox, gen(seed), 2
        # Free pages hold NaN, which no row may ever see.
        self.caches = [torch.full((pages, block, hkv, d), float("nan"), dtype=dtype, device=cuda)
                       for _ in range(2 * self.layers)]
        self.pool = PagePool(self.caches)
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=cuda)
        phase = torch.arange(width * block)[:, None] * torch.arange(1, rot // 2 + 1)[None] / 37
        self.cos_sin = torch.cat((phase.cos(), phase.sin()), -1)
        self.weights = [(randn((d,), dtype, self.g), randn((d,), dtype, self.g)) for _ in range(self.layers)]
        self.dense = [[[torch.zeros(0, hkv, d, dtype=dtype)] * 2 for _ in range(rows)] for _ in range(self.layers)]
        self.workspace = prefix_attention.new_prefix_workspace(rows, 64, hq, hkv, d, cuda)
        self.status = torch.zeros(1, dtype=torch.int32, device=cuda)
        self.reuse = {}

    def i32(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.cuda)

    def lens(self, row):
        return self.dense[0][row][0].shape[0]

    def slots(self, rows, positions):
        """Where tokens go, from the table on the device (-1 for padding rows)."""
        at = self.table[rows.clamp_min(0).long(), (positions // self.block).long()] * self.block + positions % self.block
        return torch.where(rows >= 0, at, torch.full_like(at, -1))

    def write(self, layer, rows, positions):
        """New tokens of a layer through the norm and rotation into the pages; checks and returns the queries."""
        from ds355 import qk_rope

        tokens, d, hq, hkv = len(rows), self.d, self.hq, self.hkv
        qkv = randn((tokens, (hq + 2 * hkv) * d), self.dtype, self.g) * 3
        part = lambda t, a, b: t[:, a * d: b * d].unflatten(1, (b - a, d))  # noqa: E731
        dev = qkv.to(self.cuda)
        out = torch.empty(tokens, hq, d, dtype=self.dtype, device=self.cuda)
        keys = torch.empty(tokens, hkv, d, dtype=self.dtype, device=self.cuda)
        r, p = self.i32(rows), self.i32(positions)
        qw, kw = self.weights[layer]
        qk_rope.qk_norm_rope(
            part(dev, 0, hq), part(dev, hq, hq + hkv), qw.to(self.cuda), kw.to(self.cuda), p, self.cos_sin.to(self.cuda),
            eps=1e-6, rotary_dim=self.rot, is_neox_style=self.neox, query_out=out, key_out=keys,
            value=part(dev, hq + hkv, hq + 2 * hkv), key_cache=self.caches[2 * layer],
            value_cache=self.caches[2 * layer + 1], slot_mapping=self.slots(r, p), status=self.status, reuse=self.reuse)
        torch.cuda.synchronize()
        case = dict(eps=1e-6, cos_sin=self.cos_sin, positions=torch.tensor(positions))
        for got, x, w in ((out, part(qkv, 0, hq), qw), (keys, part(qkv, hq, hq + hkv), kw)):
            _, want, size = heads.expect(x, w, case, self.rot, self.neox)
            heads.assert_close(got, want, size, d)
        keys, values = keys.cpu(), part(qkv, hq + hkv, hq + 2 * hkv)
        for t, (row, at) in enumerate(zip(rows, positions)):
            if row >= 0:
                kv = self.dense[layer][row]
                assert kv[0].shape[0] == at
                self.dense[layer][row] = [torch.cat((old, new[t: t + 1])) for old, new in zip(kv, (keys, values))]
        return out

    def attend(self, layer, query, starts, qlens, prefix):
        """A layer's attention over the pages, against the oracle's rows; returns the call's tensors."""
        lens = [self.lens(b) for b in range(len(qlens))]
        case = dict(query=query.cpu(), dense=self.dense[layer], starts=starts, qlens=qlens, lens=lens, prefix=prefix,
                    scale=self.d ** -0.5, hq=self.hq, hkv=self.hkv, d=self.d, tokens=query.shape[0],
                    cache=self.caches[2 * layer: 2 * layer + 2], table=self.table)
        args = attention.device_args(case, self.cuda, workspace=self.workspace, reuse=self.reuse)
        attention.run(args)
        attention.check(case, args)
        return args

    def step(self, counts, prefix, grow=True):
        """Every row takes `counts[b]` new tokens, in both layers; a padding token stands last."""
        rows = range(len(counts))
        lens = [self.lens(b) for b in rows]
        if grow:
            self.pool.extend(self.table, self.i32(list(rows)), self.i32([n + c for n, c in zip(lens, counts)]))
        owner = [b for b in rows for _ in range(counts[b])] + [-1]
        positions = [lens[b] + i for b in rows for i in range(counts[b])] + [0]
        starts = [sum(counts[:b]) for b in rows]
        results = []
        for layer in range(self.layers):
            query = self.write(layer, owner, positions)
            results.append((query, starts, counts, prefix))
        return [self.attend(layer, *x) for layer, x in enumerate(results)]

    def cut(self, lens):
        self.pool.free(self.table, self.i32(list(range(len(lens)))), self.i32(lens))
        for layer in self.dense:
            for row, n in enumerate(lens):
                layer[row] = [x[:n] for x in layer[row]]

    def check_pages(self):
        """Counts are the table's, and rows hold exactly the pages of their tokens."""
        torch.cuda.synchronize()
        table = self.table.cpu().tolist()
        counts = [0] * self.pool.num_pages
        for row, entries in enumerate(table):
            held = [p for p in entries if p >= 0]
            assert entries[: len(held)] == held and len(held) == -(-self.lens(row) // self.block)
            for p in held:
                counts[p] += 1
        assert self.pool.ref_counts.cpu().tolist() == counts
        assert int(self.pool.status.item()) == 0 and int(self.status.item()) == 0
        return table


CONFIGS = (
    dict(d=128, hq=8, hkv=2, block=16, dtype=torch.bfloat16, rot=128, neox=True, prompt=70),
    dict(d=64, hq=6, hkv=2, block=16, dtype=torch.float16, rot=32, neox=False, prompt=64),  # ends with a page
    dict(d=256, hq=4, hkv=1, block=24, dtype=torch.bfloat16, rot=64, neox=True, prompt=37),
)


@pytest.mark.parametrize("config", range(len(CONFIGS)))
def test_prompt_fork_verify_cut_back_compact(cuda, config):
    from ds355 import kernels

    c = dict(CONFIGS[config])
    prompt = c.pop("prompt")
    s = Server(cuda, rows=4, seed=40 + config, **c)
    # The prompt, by row 0 alone (nothing is shared yet), in two chunks.
    s.step([prompt - 9, 0, 0, 0], 0)
    s.step([9, 0, 0, 0], 0)
    s.check_pages()
    # Three rows more from it: full pages are shared, the partial one is a copy.
    s.pool.fork(s.table, [0, 0, 0], [1, 2, 3], [prompt] * 3)
    for layer in s.dense:
        for row in (1, 2, 3):
            layer[row] = list(layer[0])
    table = s.check_pages()
    shared = prompt // s.block
    assert all(table[b][:shared] == table[0][:shared] for b in (1, 2, 3))
    # Verification of ragged drafts, cut back to what was accepted, and again from there.
    s.step([5, 1, 3, 2], prompt)
    s.cut([prompt + 2, prompt + 1, prompt + 3, prompt + 1])
    s.check_pages()
    s.step([1, 4, 5, 20], prompt)
    s.check_pages()
    # Row 2 ends and begins again from row 3's longer text; what the rows share stays the prompt.
    s.pool.fork(s.table, s.i32([3]), s.i32([2]), s.i32([prompt + 15]))
    for layer in s.dense:
        layer[2] = [x[: prompt + 15] for x in layer[3]]
    s.check_pages()
    before = s.step([1, 1, 1, 1], prompt)
    s.check_pages()
    # Compaction moves pages, not results: the same queries again, to the last bit.
    s.pool.compact(s.table)
    table = s.check_pages()
    held = {p for row in table for p in row if p >= 0}
    assert held == set(range(len(held)))
    for layer, old in enumerate(before):
        new = s.attend(layer, old["query"], [0, 1, 2, 3], [1, 1, 1, 1], prompt)
        assert torch.equal(new["output"], old["output"]) and torch.equal(new["lse"], old["lse"])
        # The draft's side takes the last layer's LSE and pages.
        rows = torch.arange(4, device=cuda)
        kw = dict(chunk_size=16, max_seq_len=int(old["target_len"].max()), scale=old["scale"])
        table4 = s.table.clamp_min(0)
        with_lse = kernels.paged_chunk_attention_scores(old["query"][rows].contiguous(), new["key_cache"],
                                                        new["lse"][rows].contiguous(), table4, old["target_len"], **kw)
        own = kernels.paged_chunk_attention_scores(old["query"][rows].contiguous(), new["key_cache"], None, table4,
                                                   old["target_len"], **kw)
        assert ((with_lse - own).abs() <= 1e-4 * own.abs() + 1e-12).all()


def test_decode_steps_from_one_graph(cuda):
    """Growing, slots, norm, paged write and attention captured once; every replay is a step of its own."""
    from ds355 import prefix_attention, qk_rope

    hq, hkv, d, block, dtype, prompt = 8, 2, 128, 16, torch.bfloat16, 45
    s = Server(cuda, rows=3, d=d, hq=hq, hkv=hkv, block=block, dtype=dtype, rot=d, neox=True, seed=50)
    s.step([prompt, 0, 0], 0)
    s.pool.fork(s.table, [0, 0], [1, 2], [prompt] * 2)
    for layer in s.dense:
        layer[1], layer[2] = list(layer[0]), list(layer[0])
    rows, lens = s.i32([0, 1, 2]), s.i32([prompt] * 3)
    starts, ones, prefix = s.i32([0, 1, 2]), s.i32([1, 1, 1]), s.i32([prompt])
    qkv = torch.zeros(3, (hq + 2 * hkv) * d, dtype=dtype, device=cuda)
    query, out = (torch.zeros(3, hq, d, dtype=dtype, device=cuda) for _ in range(2))
    keys, lse = torch.zeros(3, hkv, d, dtype=dtype, device=cuda), torch.zeros(3, hq, device=cuda)
    qw, kw = (w.to(cuda) for w in s.weights[0])
    cos_sin, places = s.cos_sin.to(cuda), torch.zeros(3, dtype=torch.int32, device=cuda)
    part = lambda t, a, b: t[:, a * d: b * d].unflatten(1, (b - a, d))  # noqa: E731

    def body():
        places.copy_(lens)
        lens.add_(1)
        s.pool.extend(s.table, rows, lens)
        qk_rope.qk_norm_rope(part(qkv, 0, hq), part(qkv, hq, hq + hkv), qw, kw, places, cos_sin, eps=1e-6, rotary_dim=d,
                             is_neox_style=True, query_out=query, key_out=keys, value=part(qkv, hq + hkv, hq + 2 * hkv),
                             key_cache=s.caches[0], value_cache=s.caches[1], slot_mapping=s.slots(rows, places),
                             status=s.status)
        prefix_attention.shared_prefix_attention(query, s.caches[0], s.caches[1], out, lse, s.table, starts, ones, lens,
                                                 prefix, scale=d ** -0.5, workspace=s.workspace, status=s.status)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    kept = s.table.clone(), s.pool.ref_counts.clone(), [c.clone() for c in s.caches]
    with torch.cuda.stream(stream):
        body()  # warm-up; its step is taken back below
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body()
    s.table.copy_(kept[0])
    s.pool.ref_counts.copy_(kept[1])
    for c, old in zip(s.caches, kept[2]):
        c.copy_(old)
    lens.fill_(prompt)
    for step in range(20):  # over a page's end
        new = randn(qkv.shape, dtype, s.g) * 3
        qkv.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        values = part(new, hq + hkv, hq + 2 * hkv)
        for row in range(3):
            for layer in range(2):  # the second layer's rows only keep their lengths
                s.dense[layer][row] = [torch.cat((old, x[row: row + 1])) for old, x in
                                       zip(s.dense[layer][row], (keys.cpu(), values))]
        s.check_pages()
        case = dict(query=query.cpu(), dense=s.dense[0], starts=[0, 1, 2], qlens=[1, 1, 1], lens=[prompt + step + 1] * 3,
                    prefix=prompt, scale=d ** -0.5, hq=hq, hkv=hkv, d=d, tokens=3)
        attention.check(case, dict(output=out, lse=lse, status=s.status))


def test_places_past_32_bits(cuda):
    """Pages a GiB apart: the last one begins past 4 GiB, in elements of a view and in bytes of a copy."""
    from ds355 import qk_rope
    from ds355.pages import PagePool

    pages, block, hq, hkv, d, dtype, far = 5, 16, 8, 2, 128, torch.bfloat16, (1 << 29) + 64
    caches = []
    for _ in range(2):
        cache = torch.empty((pages - 1) * far + block * hkv * d, dtype=dtype, device=cuda).as_strided(
            (pages, block, hkv, d), (far, hkv * d, d, 1))
        cache.zero_()
        caches.append(cache)
    pool = PagePool(caches)
    g = gen(70)
    qkv = (randn((block, (hq + 2 * hkv) * d), dtype, g) * 3).to(cuda)
    part = lambda a, b: qkv[:, a * d: b * d].unflatten(1, (b - a, d))  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    phase = torch.arange(block)[:, None] * torch.arange(1, d // 2 + 1)[None] / 37
    query, keys = torch.empty(block, hq, d, dtype=dtype, device=cuda), torch.empty(block, hkv, d, dtype=dtype, device=cuda)
    weight = randn((d,), dtype, g).to(cuda)
    qk_rope.qk_norm_rope(part(0, hq), part(hq, hq + hkv), weight, weight, i32(list(range(block))),
                         torch.cat((phase.cos(), phase.sin()), -1).to(cuda), eps=1e-6, rotary_dim=d, is_neox_style=True,
                         query_out=query, key_out=keys, value=part(hq + hkv, hq + 2 * hkv), key_cache=caches[0],
                         value_cache=caches[1], slot_mapping=i32([4 * block + t for t in range(block)]))
    values = part(hq + hkv, hq + 2 * hkv)
    assert torch.equal(caches[0][4], keys) and torch.equal(caches[1][4], values)
    assert all(int(c[:4].count_nonzero()) == 0 for c in caches)
    pool.copy([4], [1])
    assert torch.equal(caches[0][1], keys) and torch.equal(caches[1][1], values)
    kv = [keys.cpu(), values.cpu()]
    case = dict(query=query.cpu(), dense=[kv, kv], starts=[0, 8], qlens=[8, 8], lens=[16, 16], prefix=0, scale=d ** -0.5,
                hq=hq, hkv=hkv, d=d, tokens=block, cache=[c[:1] for c in caches], table=torch.tensor([[4], [1]], dtype=torch.int32))
    args = attention.device_args(case, cuda, key_cache=caches[0], value_cache=caches[1])
    attention.run(args)
    attention.check(case, args)


@pytest.mark.parametrize("lse_free", (False, True), ids=("lse", "no_lse"))
@pytest.mark.parametrize("path", ("chain", "fused"))
def test_a_retrieval_step_on_a_pools_table(cuda, path, lse_free):
    """The step takes the pool's table as it is (-1 behind a row's last page, rows without any) and the
    attention's LSE; pages that no row holds are NaN."""
    import test_gpu_step as steps
    from ds355.pages import PagePool

    lens = [900, 333, 64, 65, 1700, 17, 1201, 512]
    case = steps.build_case(7, real_rows=8, pad_rows=2, target_lens=lens, query_len=4, counts=[1, 3, 0, 4, 2, 1, 4, 3],
                            hq=16, hkv=4, head_dim=128, chunk=64, token_budget=512, block_size=16, lmax=2048,
                            slots=[3, 0, 7, 9, 1, 4, 2, 8], num_slots=10)
    given_k, given_table, given_lse = case["key_cache"], case["table"], case["lse"]
    caches = [torch.full((400, 16, 4, 128), float("nan"), dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    pool = PagePool(caches)
    table = torch.full((10, 120), -1, dtype=torch.int32, device=cuda)
    pool.extend(table, [4, 1, 0, 3], [1700, 1000, 900, 65])
    pool.extend(table, [7, 5, 2, 6], [512, 17, 64, 1201])
    pool.free(table, [1], [333])
    pool.compact(table)
    held = table.cpu()
    for b, n in enumerate(lens):
        pages = -(-n // 16)
        assert (held[b, :pages] >= 0).all() and (held[b, pages:] == -1).all()
        caches[0][held[b, :pages].long().to(cuda)] = given_k[given_table[b, :pages].long()].to(cuda)
        caches[1][held[b, :pages].long().to(cuda)] = randn((pages, 16, 4, 128), torch.bfloat16, gen(b)).to(cuda)
    assert int(pool.status.item()) == 0 and (held[8:] == -1).all()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    from ds355 import prefix_attention

    query = case["query"].to(cuda)
    out, lse = torch.zeros_like(query), torch.zeros(query.shape[:2], device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    prefix_attention.shared_prefix_attention(
        query, *caches, out, lse, table, i32(case["starts"]), i32(case["qlens"]), i32(case["tlens"]), i32([0]),
        scale=case["scale"], workspace=prefix_attention.new_prefix_workspace(10, query.shape[0], 16, 4, 128, cuda),
        batch_size=8, status=status)
    assert int(status.item()) == 0 and bool(out.isfinite().all())
    # The LSE of each scored row's committed query, against the one that the case computed over its own pages.
    _, q_index, _ = steps.O.retrieval_rows(case["counts"], case["ends"], case["tlens"], 8)
    assert (lse.cpu()[q_index] - given_lse[q_index]).abs().max() < 1e-4
    case.update(key_cache=caches[0].cpu(), table=held, lse=lse.cpu())
    state = steps.run_gpu(case, cuda, path=path, lse_free=lse_free)
    case["table"] = held.clamp_min(0)  # the oracle's lookup
    steps.check_step(case, state)

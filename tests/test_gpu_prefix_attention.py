"""GPU: paged attention of a batch that shares a prefix, against a plain implementation in 64 bits.

Bounds, with u = eps / 2 of the type (half a step, relative) and T = sum_t softmax_t |v_t| the size of
the terms an output sums:
  - each probability is rounded to the cache's type once (u T in all) and the output once (u |out|);
  - a logit is an fp32 sum of D products, off by at most (D + 4) 2^-24 scale sum_d |q_d k_d| =: E over
    the keys, which moves every weight by at most 2 E relative, and the LSE by E;
  - fp32 sums over n keys and their pieces: (n / 16 + 64) 2^-24, the lane and piece sums being short;
    exp2 and the scaling of the logits by log2 e add 2^-22 (1 + |x|) with |x| the largest logit.
"""

import pytest
import torch

from helpers import gen, randn

pytestmark = pytest.mark.gpu

DTYPES = (torch.bfloat16, torch.float16)


def build(seed, *, prefix, own, qlens, hq, hkv, d, block, dtype, extra=3, fill=float("nan"), diverge=True):
    """A batch on the CPU: rows forked from one prompt of `prefix` tokens with `own[b]` tokens of their own.

    The prompt's full pages are shared; the partial one is a copy of each row's own.  Unused pages and
    the places past each row's end hold `fill`.
    """
    g = gen(seed)
    lens = [prefix + n if n is not None else 0 for n in own]
    shared = prefix // block
    pages = [max(0, -(-n // block) - shared) for n in lens]
    total = shared + sum(pages) + extra
    order = torch.randperm(total, generator=g).tolist()
    width = max([-(-n // block) for n in lens] + [1]) + 2
    table = torch.zeros((len(own), width), dtype=torch.int32)
    cache = [torch.full((total, block, hkv, d), fill, dtype=dtype) for _ in range(2)]
    prompt = [randn((max(prefix, 1), hkv, d), dtype, g) for _ in range(2)]
    at = shared
    dense = []
    for b, n in enumerate(lens):
        row = order[:shared] + order[at: at + pages[b]] if n else []
        at += pages[b]
        table[b, : len(row)] = torch.tensor(row, dtype=torch.int32)
        kv = []
        for c, p in zip(cache, prompt):
            x = torch.cat((p[: min(prefix, n)], randn((max(0, n - prefix), hkv, d), dtype, g)))
            for t0 in range(0, n, block):
                part = x[t0: t0 + block]
                c[row[t0 // block], : part.shape[0]] = part
            kv.append(x)
        dense.append(kv)
    starts, at = [], 1  # token 0 belongs to no row
    for q in qlens:
        starts.append(at)
        at += q + 1 if diverge else q  # gaps between the rows' tokens
    tokens = at + 2
    query = randn((tokens, hq, d), dtype, g) * 2
    return dict(query=query, cache=cache, table=table, starts=starts, qlens=qlens, lens=lens, prefix=prefix, dense=dense,
                scale=d ** -0.5, hq=hq, hkv=hkv, d=d, tokens=tokens)


def expect(case):
    """(output, lse, terms, logit error, largest logit) in 64 bits; rows of no token stay None (NaN-filled)."""
    t, hq, d = case["query"].shape
    group = hq // case["hkv"]
    out = torch.full((t, hq, d), float("nan"), dtype=torch.float64)
    lse = torch.full((t, hq), float("nan"), dtype=torch.float64)
    terms, err, top = torch.zeros((t, hq, d), dtype=torch.float64), torch.zeros((t, hq), dtype=torch.float64), \
        torch.zeros((t, hq), dtype=torch.float64)
    for b, (start, q, n) in enumerate(zip(case["starts"], case["qlens"], case["lens"])):
        k, v = (x.double() for x in case["dense"][b])
        for i in range(q):
            seen = min(n, n - q + i + 1)
            if seen <= 0:
                out[start + i], lse[start + i] = 0, -float("inf")
                continue
            for h in range(hq):
                x = case["query"][start + i, h].double()
                kk, vv = k[:seen, h // group], v[:seen, h // group]
                logits = (kk @ x) * case["scale"]
                w = torch.softmax(logits, 0)
                out[start + i, h] = w @ vv
                lse[start + i, h] = torch.logsumexp(logits, 0)
                terms[start + i, h] = w @ vv.abs()
                err[start + i, h] = (d + 4) * 2.0 ** -24 * case["scale"] * (kk.abs() @ x.abs()).max()
                top[start + i, h] = logits.abs().max()
    return out, lse, terms, err, top


def device_args(case, cuda, **over):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    from ds355 import prefix_attention as pa

    args = dict(
        query=case["query"].to(cuda), key_cache=case["cache"][0].to(cuda), value_cache=case["cache"][1].to(cuda),
        output=torch.full(case["query"].shape, 7.0, dtype=case["query"].dtype, device=cuda),
        lse=torch.full(case["query"].shape[:2], 7.0, device=cuda), block_table=case["table"].to(cuda),
        query_start=i32(case["starts"]), query_len=i32(case["qlens"]), target_len=i32(case["lens"]),
        prefix_len=i32([case["prefix"]]), scale=case["scale"],
        workspace=pa.new_prefix_workspace(len(case["qlens"]), case["tokens"], case["hq"], case["hkv"], case["d"], cuda),
        status=torch.zeros(1, dtype=torch.int32, device=cuda))
    args.update(over)
    return args


def run(args):
    from ds355 import prefix_attention as pa

    out = pa.shared_prefix_attention(**args)
    torch.cuda.synchronize()
    return out


def check(case, args, expected=None, status=0):
    out, lse, terms, err, top = expected if expected is not None else expect(case)
    got, got_lse = args["output"].cpu().double(), args["lse"].cpu().double()
    keys = max(case["lens"] + [1])
    u = torch.finfo(case["query"].dtype).eps / 2
    sums = (keys / 16 + 64) * 2.0 ** -24 + 2.0 ** -22 * (1 + top)
    mine = ~out.isnan().any(-1).any(-1)
    for b, (start, q) in enumerate(zip(case["starts"], case["qlens"])):
        assert mine[start: start + q].all()
    assert (got[~mine] == 7).all() and (got_lse[~mine] == 7).all(), "tokens of no row were written"
    bound = u * out.abs() + (u * (1 + u) + 2 * err[..., None] + 2 * sums[..., None]) * terms + 1e-30
    excess = ((got - out).abs() - bound)[mine]
    assert not got[mine].isnan().any() and excess.numel() and float(excess.max()) <= 0, float(excess.max())
    nothing = lse == -float("inf")
    assert (got_lse[nothing] == -float("inf")).all() and (got[nothing] == 0).all()
    some = mine[:, None] & ~nothing
    off = ((got_lse - lse).abs() - (err + sums + 2.0 ** -22 * lse.abs()))[some]
    assert not got_lse[some].isnan().any() and (not off.numel() or float(off.max()) <= 0), float(off.max())
    assert int(args["status"].item()) == status


SHAPES = [
    # prefix, own keys per row (None: no keys at all), query tokens per row, hq, hkv, d, block
    dict(prefix=256, own=[5, 40, 130], qlens=[1, 1, 1], hq=8, hkv=2, d=128, block=16),
    dict(prefix=1000, own=[17, 300, 1, 64], qlens=[3, 5, 1, 2], hq=32, hkv=4, d=128, block=16),
    dict(prefix=129, own=[9, 9], qlens=[4, 2], hq=10, hkv=2, d=128, block=48),
    dict(prefix=127, own=[3, 200, 31], qlens=[1, 7, 6], hq=16, hkv=16, d=64, block=128),
    dict(prefix=515, own=[70, 6, 1], qlens=[5, 5, 1], hq=28, hkv=4, d=64, block=1),
    dict(prefix=700, own=[33, 2, 260], qlens=[2, 2, 8], hq=16, hkv=1, d=256, block=16),
    dict(prefix=64, own=[8, 100], qlens=[8, 8], hq=12, hkv=4, d=256, block=200),
    dict(prefix=1, own=[1, 2, 3], qlens=[1, 1, 1], hq=4, hkv=4, d=128, block=16),
    dict(prefix=0, own=[1, 77, 400], qlens=[1, 2, 3], hq=8, hkv=1, d=128, block=16),
    dict(prefix=300, own=[40], qlens=[3], hq=8, hkv=2, d=64, block=16),  # one row shares with nobody
    dict(prefix=0, own=[1], qlens=[1], hq=1, hkv=1, d=64, block=16),
    dict(prefix=200, own=[10, 10, 10], qlens=[2, 0, 2], hq=8, hkv=2, d=128, block=32),  # graph padding
    dict(prefix=640, own=[330, 50], qlens=[300, 40], hq=8, hkv=2, d=128, block=64),  # a prompt chunk
    dict(prefix=384, own=[130, 50, 129, 3], qlens=[128, 40, 65, 3], hq=4, hkv=4, d=256, block=64),
    dict(prefix=2048, own=[i + 1 for i in range(40)], qlens=[1] * 40, hq=8, hkv=1, d=64, block=16),
    # Several tiles of query rows per row in 256 dimensions, most of which see none of the row's last keys;
    # the last tile has waves without rows.
    dict(prefix=96, own=[310, 40], qlens=[300, 33], hq=8, hkv=2, d=256, block=17),
    dict(prefix=0, own=[150, 2], qlens=[150, 1], hq=8, hkv=1, d=256, block=32),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=("bf16", "fp16"))
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_against_64_bits(cuda, i, dtype):
    case = build(100 + i, dtype=dtype, **SHAPES[i])
    print("prefix attention", i, SHAPES[i], flush=True)
    args = device_args(case, cuda)
    run(args)
    check(case, args)


def test_rows_that_see_nothing(cuda):
    # A row without keys, a row with fewer keys than query tokens, beside an ordinary one.
    case = build(7, prefix=0, own=[None, 2, 50], qlens=[2, 5, 3], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    args = device_args(case, cuda)
    run(args)
    check(case, args)


@pytest.mark.parametrize("claimed", (0, 5, 64, 300, 100000, -3))
def test_any_prefix_length_up_to_the_shared_one_gives_the_same(cuda, claimed):
    # The batch shares 300 keys; a smaller claim shares less work, a larger one ends at the shortest row.
    case = build(8, prefix=300, own=[0, 0, 0], qlens=[1, 3, 2], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    args = device_args(case, cuda, prefix_len=torch.tensor([claimed], dtype=torch.int32, device=cuda))
    run(args)
    check(case, args)


@pytest.mark.parametrize("bad", (float("nan"), float("inf"), -float("inf")))
@pytest.mark.parametrize("d,hkv", ((128, 2), (64, 8), (256, 1)))
def test_keys_a_token_does_not_see_have_no_effect(cuda, bad, d, hkv):
    # The last two tokens of each row hold `bad` in some dimensions of K and V: their own query tokens are
    # lost, the earlier ones see nothing of it.
    case = build(9, prefix=100, own=[40, 90, 4], qlens=[5, 5, 4], hq=8, hkv=hkv, d=d, block=16, dtype=torch.bfloat16)
    clean = expect(case)
    for b, n in enumerate(case["lens"]):
        for t in (n - 1, n - 2):
            page = int(case["table"][b, t // 16])
            case["cache"][1][page, t % 16, :, ::3] = bad
            case["cache"][0][page, t % 16, :, 1::5] = bad
    args = device_args(case, cuda)
    run(args)
    got = args["output"].cpu().double()
    u = 2.0 ** -8
    for b, (start, q) in enumerate(zip(case["starts"], case["qlens"])):
        upto = slice(start, start + q - 2)
        assert not got[upto].isnan().any()
        assert ((got[upto] - clean[0][upto]).abs() <= 1.01 * u * (clean[0][upto].abs() + clean[2][upto]) + 1e-5).all()
        assert (args["lse"].cpu().double()[upto] - clean[1][upto]).abs().max() < 1e-4
        assert not got[start + q - 1].isfinite().all()


def test_a_value_that_is_not_finite_reaches_the_tokens_that_see_it(cuda):
    # V alone: the sum over a seen infinity is that infinity, over NaN NaN, in the dimensions that hold it.
    case = build(10, prefix=64, own=[20, 20], qlens=[4, 4], hq=8, hkv=2, d=128, block=16, dtype=torch.float16)
    for b, (t, value) in enumerate(((case["lens"][0] - 2, float("inf")), (case["lens"][1] - 2, float("nan")))):
        case["cache"][1][int(case["table"][b, t // 16]), t % 16, 1, 7] = value
        case["dense"][b][1][t, 1, 7] = value
    args = device_args(case, cuda)
    run(args)
    got = args["output"].cpu()
    for b, start in enumerate(case["starts"]):
        assert got[start: start + 2].isfinite().all()
        mine = got[start + 2: start + 4, 4:, 7]
        assert mine.isnan().all() if b else (mine == float("inf")).all()
        rest = torch.ones(128, dtype=torch.bool)
        rest[7] = False
        assert got[start + 2: start + 4][..., rest].isfinite().all() and got[start + 2: start + 4, :4].isfinite().all()


def test_strided_tensors(cuda):
    # Queries out of a fused projection, a padded output, LSEs by head, caches that are views of one
    # buffer with heads before tokens, a table with padding columns.
    case = build(11, prefix=333, own=[60, 5, 128], qlens=[2, 4, 1], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    args = device_args(case, cuda)
    t = case["tokens"]
    fused = torch.zeros((t, 12 * 128), dtype=torch.bfloat16, device=cuda)
    fused[:, : 8 * 128] = args["query"].reshape(t, -1)
    args["query"] = fused[:, : 8 * 128].unflatten(1, (8, 128))
    args["output"] = torch.full((t, 9, 160), 7.0, dtype=torch.bfloat16, device=cuda)[:, :8, :128]
    args["lse"] = torch.full((8, t), 7.0, device=cuda).t()
    pages = case["cache"][0].shape[0]
    both = torch.zeros((pages, 2, 2, 16, 128), dtype=torch.bfloat16, device=cuda)
    both[:, 0], both[:, 1] = (x.transpose(1, 2) for x in (args["key_cache"], args["value_cache"]))
    args["key_cache"], args["value_cache"] = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    run(args)
    check(case, args)
    wide = args["output"].as_strided((t, 9, 160), (9 * 160, 160, 1))
    assert (wide[:, 8:] == 7).all() and (wide[:, :, 128:] == 7).all()


def test_batch_size_and_no_lse(cuda):
    case = build(12, prefix=100, own=[20, 30, 40], qlens=[2, 2, 2], hq=8, hkv=2, d=64, block=16, dtype=torch.float16)
    args = device_args(case, cuda, batch_size=2)
    run(args)
    got = args["output"].clone()
    args["output"].fill_(7)
    args["lse"] = None
    run(args)
    assert torch.equal(args["output"], got)
    start = case["starts"][2]
    assert (got[start: start + 2] == 7).all()
    case["qlens"] = [2, 2, 0]
    args["lse"] = torch.full(got.shape[:2], 7.0, device=cuda)
    run(args)
    check(case, args)


def test_a_launch_gives_the_same_bits_again(cuda):
    case = build(13, prefix=3001, own=[200, 3, 77, 900], qlens=[5, 1, 3, 2], hq=32, hkv=4, d=128, block=16,
                 dtype=torch.bfloat16)
    args = device_args(case, cuda)
    run(args)
    first = args["output"].clone(), args["lse"].clone()
    for _ in range(3):
        args["workspace"].fill_(255)  # nothing of the call before is used
        args["output"].fill_(7)
        args["lse"].fill_(7)
        run(args)
        assert torch.equal(args["output"], first[0]) and torch.equal(args["lse"], first[1])


def test_status_bits(cuda):
    base = dict(prefix=64, own=[20, 30, 40], qlens=[2, 2, 2], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    # A row whose tokens are out of range is left out; the others are computed.
    case = build(14, **base)
    args = device_args(case, cuda)
    args["query_start"][1] = case["tokens"] - 1
    run(args)
    assert int(args["status"].item()) == 1
    args["status"].zero_()
    whole = expect(case)
    for t in (case["starts"][1], case["starts"][1] + 1):
        whole[0][t], whole[1][t] = float("nan"), float("nan")
    case["qlens"] = [2, 0, 2]
    check(case, args, whole)
    # A row longer than its table ends there.
    case = build(15, **base)
    args = device_args(case, cuda)
    capacity = case["table"].shape[1] * 16
    args["target_len"][2] = capacity + 50
    run(args)
    assert int(args["status"].item()) == 2
    # A page id out of range reads as zeros.
    for page in (-1, 10 ** 6):
        case = build(16, **base)
        args = device_args(case, cuda)
        args["block_table"][1, 5] = page  # keys 80 .. 95 of the row's 94
        run(args)
        assert int(args["status"].item()) == 4
        for kv in case["dense"][1]:
            kv[80:] = 0
        args["status"].zero_()
        check(case, args)


def test_rows_that_overlap_are_cut_off(cuda):
    # More query tokens in all than the query holds: the rows that bring the sum over are left out.
    case = build(17, prefix=64, own=[9, 9, 9], qlens=[3, 3, 3], hq=4, hkv=2, d=64, block=16, dtype=torch.float16,
                 diverge=False)
    args = device_args(case, cuda)
    args["query"], args["output"], args["lse"] = (args[k][:8] for k in ("query", "output", "lse"))
    args["query_start"][2] = 2
    run(args)
    assert int(args["status"].item()) == 1
    expected = expect(case)
    got = args["output"].cpu().double()
    assert (got[0] == 7).all() and (got[7] == 7).all()
    assert (got[1:7] - expected[0][1:7]).abs().max() < 0.02


def test_graph_follows_changed_lengths_and_shares_a_workspace(cuda):
    from ds355 import prefix_attention as pa

    cases = [build(20 + i, prefix=p, own=own, qlens=q, hq=16, hkv=2, d=128, block=16, dtype=torch.bfloat16, extra=200)
             for i, (p, own, q) in enumerate(((500, [30, 7, 200], [3, 1, 2]), (80, [400, 2, 9], [1, 1, 4])))]
    width, pages = 60, 300
    args = device_args(cases[0], cuda)
    t = 16
    for k in ("query", "output"):
        args[k] = torch.zeros((t, 16, 128), dtype=torch.bfloat16, device=cuda)
    args["lse"] = torch.zeros((t, 16), device=cuda)
    args["block_table"] = torch.zeros((3, width), dtype=torch.int32, device=cuda)
    args["key_cache"] = torch.zeros((pages, 16, 2, 128), dtype=torch.bfloat16, device=cuda)
    args["value_cache"] = torch.zeros_like(args["key_cache"])
    args["workspace"] = pa.new_prefix_workspace(3, t, 16, 2, 128, cuda)
    other = dict(args, output=torch.zeros_like(args["output"]), lse=torch.zeros_like(args["lse"]))

    def fill(case):
        n = case["cache"][0].shape[0]
        args["query"][: case["tokens"]].copy_(case["query"])
        args["key_cache"][:n].copy_(case["cache"][0])
        args["value_cache"][:n].copy_(case["cache"][1])
        args["block_table"].zero_()
        args["block_table"][:, : case["table"].shape[1]].copy_(case["table"])
        for name, key in (("query_start", "starts"), ("query_len", "qlens"), ("target_len", "lens")):
            args[name].copy_(torch.tensor(case[key], dtype=torch.int32))
        args["prefix_len"].fill_(case["prefix"])

    fill(cases[0])
    run(args)
    stream = torch.cuda.Stream()
    graphs = []
    for a in (args, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            pa.shared_prefix_attention(**a)
        graphs.append(graph)
    for case in (cases[0], cases[1], cases[0], cases[1]):
        fill(case)
        expected = expect(case)
        for graph, a in zip(graphs, (args, other)):
            a["output"].fill_(7)
            a["lse"].fill_(7)
            graph.replay()
            torch.cuda.synchronize()
            n = case["tokens"]
            check(case, dict(a, output=a["output"][:n], lse=a["lse"][:n]), expected)
            replayed = a["output"].clone(), a["lse"].clone()
            run(a)
            assert torch.equal(replayed[0], a["output"]) and torch.equal(replayed[1], a["lse"])


def test_on_another_stream_and_with_reuse(cuda):
    case = build(30, prefix=400, own=[33, 3], qlens=[2, 1], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    expected = expect(case)
    args = device_args(case, cuda, reuse={})
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(args)
    check(case, args, expected)
    # The same layout at other addresses, then another layout through the same dict.
    moved = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in args.items()}
    for k in ("output", "lse"):
        args[k].fill_(7)
        moved[k].fill_(7)
    run(moved)
    check(case, moved, expected)
    assert (args["output"] == 7).all()
    assert len(args["reuse"]) == 1
    other = build(31, prefix=30, own=[3, 90], qlens=[2, 5], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    more = device_args(other, cuda, reuse=args["reuse"])
    run(more)
    check(other, more)


def test_lse_feeds_the_chunk_scores(cuda):
    # The verified batch as a serving loop runs it: attention, then the scores of the committed queries
    # with its LSE, against the scores that compute their own over the same keys.
    from ds355 import kernels

    case = build(32, prefix=700, own=[100, 30, 260], qlens=[1, 1, 1], hq=32, hkv=4, d=128, block=16,
                 dtype=torch.bfloat16, fill=0.0)
    args = device_args(case, cuda)
    run(args)
    rows = torch.tensor(case["starts"], device=cuda)
    kw = dict(chunk_size=64, max_seq_len=max(case["lens"]), scale=case["scale"])
    lens = args["target_len"]
    got = kernels.paged_chunk_attention_scores(args["query"][rows], args["key_cache"], args["lse"][rows],
                                               args["block_table"], lens, **kw)
    own = kernels.paged_chunk_attention_scores(args["query"][rows], args["key_cache"], None, args["block_table"], lens,
                                               **kw)
    assert ((got - own).abs() <= 1e-4 * own.abs() + 1e-12).all()


@pytest.mark.parametrize("rows,d", ((1024, 64), (700, 128), (513, 256), (65, 128)))
def test_many_rows(cuda, rows, d):
    # Rows in several waves and rounds of the layout: some are padding, some without keys, lengths differ.
    own = [None if b % 97 == 5 else (b * 37) % 41 + (b % 4) for b in range(rows)]
    qlens = [0 if b % 11 == 3 else 1 + (b % 29 == 0) * 3 for b in range(rows)]
    case = build(60, prefix=48, own=own, qlens=qlens, hq=4, hkv=2, d=d, block=16, dtype=torch.bfloat16)
    args = device_args(case, cuda)
    run(args)
    check(case, args)


def test_many_rows_that_overlap_are_cut_off(cuda):
    # As many query tokens as the tensor holds belong to the first rows; the rows after them, of which the
    # first begins in the last round, are left out.
    rows, kept = 900, 800
    case = build(61, prefix=32, own=[b % 23 + 4 for b in range(rows)], qlens=[1] * rows, hq=2, hkv=1, d=128, block=16,
                 dtype=torch.bfloat16, diverge=False)
    expected = expect(case)
    args = device_args(case, cuda)
    case["tokens"] = kept
    for name in ("query", "output", "lse"):
        args[name] = args[name][:kept].contiguous()
    args["query_start"] = (args["query_start"] - 1) % kept  # row b has token b, those past the end token b - kept
    args["query"][: kept] = case["query"][1: kept + 1].to(cuda)
    run(args)
    out, lse, terms, err, top = (x[1: kept + 1] for x in expected)
    case.update(query=case["query"][1: kept + 1], starts=list(range(kept)), qlens=[1] * kept, lens=case["lens"][:kept])
    check(case, args, (out, lse, terms, err, top), status=1)


def test_a_long_tail_of_small_probabilities(cuda):
    # One key outweighs each of the others by e^14, near the smallest normal fp16, and has a value of 0: the
    # output is the others' sum, which would be percents off were they rounded at fp16's smallest step.
    n, d, block = 20000, 64, 16
    keys, values = torch.zeros(n, 1, d, dtype=torch.float16), torch.ones(n, 1, d, dtype=torch.float16)
    keys[0, 0, 0], values[0] = 1.75, 0
    query = torch.zeros(1, 1, d, dtype=torch.float16)
    query[0, 0, 0] = 8
    cache = [x.view(n // block, block, 1, d) for x in (keys, values)]
    case = dict(query=query, dense=[[keys, values]], starts=[0], qlens=[1], lens=[n], prefix=0, scale=1.0, hq=1, hkv=1, d=d,
                tokens=1, cache=cache, table=torch.arange(n // block, dtype=torch.int32)[None])
    args = device_args(case, cuda)
    run(args)
    check(case, args)


def test_a_share_longer_than_the_prefix(cuda):
    # A prompt batch of 1024 rows of 1024 tokens: 65536 tiles of query rows, whose own keys make a share of
    # 65536 key tiles, while the shared prefix is one.  (65536 + 3) 65536 places do not fit 32 bits.
    from ds355 import prefix_attention as pa

    rows, q, hq, d, block, prefix, own, pages = 1024, 1024, 8, 64, 16, 256, 64512, 64
    g = gen(62)
    cache = [randn((pages, block, 1, d), torch.bfloat16, g) for _ in range(2)]
    width = (prefix + own) // block
    order = torch.arange(width)[None] + torch.where(torch.arange(width) < prefix // block, 0, torch.arange(rows)[:, None])
    table = (order % pages).int()
    query = (torch.randn((rows * q, hq, d), generator=torch.Generator(device=cuda).manual_seed(62), device=cuda) * 2).bfloat16()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    output, lse = torch.full_like(query, float("nan")), torch.full((rows * q, hq), float("nan"), device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    pa.shared_prefix_attention(
        query, *(c.to(cuda) for c in cache), output, lse, table.to(cuda), i32([q * b for b in range(rows)]),
        i32([q] * rows), i32([prefix + own] * rows), i32([prefix]), scale=d ** -0.5,
        workspace=pa.new_prefix_workspace(rows, rows * q, hq, 1, d, cuda), status=status)
    torch.cuda.synchronize()
    assert int(status.item()) == 0 and bool(output.isfinite().all()) and bool(lse.isfinite().all())
    # A token from the first, a middle and the last row, and each at the other ends of its row.
    for b, i in ((0, 0), (0, 1023), (511, 300), (1023, 0), (1023, 1023)):
        dense = [c[table[b].long()].reshape(-1, 1, d)[: prefix + own - q + i + 1] for c in cache]
        n = dense[0].shape[0]
        case = dict(query=query[b * q + i][None].cpu(), dense=[dense], starts=[0], qlens=[1], lens=[n], hq=hq, hkv=1, d=d,
                    scale=d ** -0.5)
        args = dict(output=output[b * q + i][None], lse=lse[b * q + i][None], status=status)
        check(case, args)


@pytest.mark.parametrize("dtype", DTYPES, ids=("bf16", "fp16"))
@pytest.mark.parametrize("d,hkv", ((64, 2), (128, 2), (256, 1)))
@pytest.mark.parametrize("scale", (0.0, -0.0, -1.0, "negative"))
def test_zero_and_negative_scales(cuda, scale, d, hkv, dtype):
    # Scale 0 weighs all seen keys alike: the mean of their values, and the logarithm of their number.  The
    # prefix has tiles that every token sees whole, the rows end inside a tile; one row sees a single key.
    def run_and_check(case):
        case["scale"] = -(d ** -0.5) if scale == "negative" else scale
        args = device_args(case, cuda)
        run(args)
        out, lse, terms, err, top = expect(case)
        # A logit's error is |scale| times that of the product: E has the scale's sign here, a bound has none.
        check(case, args, (out, lse, terms, err.abs(), top))
        return args["lse"].cpu()

    case = build(63, prefix=600, own=[17, 300, 1, 64], qlens=[3, 5, 1, 2], hq=8, hkv=hkv, d=d, block=16, dtype=dtype)
    lse = run_and_check(case)
    if scale == 0:
        assert (lse[case["starts"][1] + 4] - torch.tensor(900.0).log()).abs().max() < 1e-5
    run_and_check(build(64, prefix=0, own=[1, None, 2], qlens=[1, 2, 4], hq=8, hkv=hkv, d=d, block=16, dtype=dtype))


def test_scale_zero_and_keys_a_token_does_not_see(cuda):
    case = build(65, prefix=100, own=[40, 90], qlens=[3, 3], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    case["scale"] = 0.0
    clean = expect(case)
    for b, n in enumerate(case["lens"]):
        page = int(case["table"][b, (n - 1) // 16])
        case["cache"][0][page, (n - 1) % 16, :, ::2] = float("inf")
        case["cache"][1][page, (n - 1) % 16, :, ::3] = float("nan")
    args = device_args(case, cuda)
    run(args)
    got, lse = args["output"].cpu().double(), args["lse"].cpu().double()
    u = 2.0 ** -8
    for start in case["starts"]:
        upto = slice(start, start + 2)
        assert ((got[upto] - clean[0][upto]).abs() <= 1.01 * u * (clean[0][upto].abs() + clean[2][upto])).all()
        assert (lse[upto] - clean[1][upto]).abs().max() < 1e-5


def test_a_row_longer_than_its_table_ends_there(cuda):
    # Row 2 fills its table's 11 pages; a length past them counts as 176, for its causal ends as well.
    case = build(66, prefix=64, own=[20, 30, 112], qlens=[2, 2, 5], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    expected = expect(case)
    for beyond in (0, 1, 50, 10 ** 9):
        args = device_args(case, cuda, block_table=case["table"][:, :11].contiguous().to(cuda))
        args["target_len"][2] = 176 + beyond
        run(args)
        check(case, args, expected, status=2 if beyond else 0)


def test_rows_in_any_order_of_their_tokens(cuda):
    # Rows' query tokens need not lie in the rows' order.
    case = build(67, prefix=300, own=[40, 5, 90, 17], qlens=[3, 1, 5, 2], hq=8, hkv=2, d=64, block=16, dtype=torch.float16)
    starts = [10, 8, 3, 1]
    query = case["query"].clone()
    for old, new, n in zip(case["starts"], starts, case["qlens"]):
        query[new: new + n] = case["query"][old: old + n]
    case.update(query=query, starts=starts)
    args = device_args(case, cuda)
    run(args)
    check(case, args)


@pytest.mark.parametrize("dtype", DTYPES, ids=("bf16", "fp16"))
@pytest.mark.parametrize("gap", (1.0, 40.0))
def test_a_value_that_is_not_finite_in_a_tile_that_all_see(cuda, gap, dtype):
    # Far from the rows' ends no mask applies: the infinity reaches every token of its row and KV head in its
    # dimension, whether its weight is an ordinary one or e^-40 of the largest, and nothing else.
    case = build(68, prefix=0, own=[700, 650], qlens=[2, 3], hq=8, hkv=2, d=64, block=16, dtype=dtype)
    case["query"][:] = 0
    case["query"][..., 0] = 8
    for b in range(2):
        for t in range(case["lens"][b]):
            page = int(case["table"][b, t // 16])
            for x in (case["cache"][0][page, t % 16], case["dense"][b][0][t]):
                x[:, 0] = 0 if t == 40 else gap
    case["scale"] = 1 / 8
    case["cache"][1][int(case["table"][0, 2]), 8, 1, 7] = float("inf")  # key 40
    args = device_args(case, cuda)
    run(args)
    got = args["output"].cpu()
    start = case["starts"][0]
    rest = torch.ones(64, dtype=torch.bool)
    rest[7] = False
    assert not got[start: start + 2, 4:, 7].isfinite().any()
    assert got[start: start + 2, 4:][..., rest].isfinite().all() and got[start: start + 2, :4].isfinite().all()
    start = case["starts"][1]
    assert got[start: start + 3].isfinite().all()
    if gap == 1:
        assert (got[case["starts"][0]: case["starts"][0] + 2, 4:, 7] == float("inf")).all()

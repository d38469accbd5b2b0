"""GPU: attention of a chunk of new tokens over a paged cache, against a plain implementation in 64 bits.

Bounds, with u = eps / 2 of the type (half a step, relative) and T = sum_t softmax_t |v_t| the size of
the terms an output sums:
  - each probability is rounded to the cache's type once (u T in all) and the output once (u |out|);
  - a logit is an fp32 sum of D products, off by at most (D + 4) 2^-24 |scale| sum_d |q_d k_d| =: E over
    the keys, which moves every weight by at most 2 E relative, and the LSE by E;
  - fp32 sums over n keys and their parts: (n / 16 + 64) 2^-24, the lane and part sums being short;
    exp2 and the scaling of the logits by log2 e add 2^-22 (1 + |x|) with |x| the largest logit.
"""

import pytest
import torch

from helpers import gen, randn

pytestmark = pytest.mark.gpu

DTYPES = (torch.bfloat16, torch.float16)
INF = float("inf")


def build(seed, *, lens, qlens, hq, hkv, d, block, dtype, window=None, extra=3, fill=float("nan"), gaps=True, scale=None):
    """Rows on the CPU.  Unused pages and the places past each row's end hold `fill`."""
    g = gen(seed)
    pages = [-(-n // block) for n in lens]
    order = torch.randperm(sum(pages) + extra, generator=g).tolist()
    table = torch.zeros((len(lens), max(pages + [1]) + 2), dtype=torch.int32)
    cache = [torch.full((len(order), block, hkv, d), fill, dtype=dtype) for _ in range(2)]
    dense, at = [], 0
    for b, n in enumerate(lens):
        row = order[at: at + pages[b]]
        at += pages[b]
        table[b, : len(row)] = torch.tensor(row, dtype=torch.int32)
        dense.append([randn((n, hkv, d), dtype, g) for _ in range(2)])
        for c, x in zip(cache, dense[b]):
            for t0 in range(0, n, block):
                part = x[t0: t0 + block]
                c[row[t0 // block], : part.shape[0]] = part
    starts, at = [], 1 if gaps else 0  # token 0 belongs to no row
    for q in qlens:
        starts.append(at)
        at += q + 1 if gaps else q  # gaps between the rows' tokens
    tokens = at + 2 if gaps else at
    query = randn((tokens, hq, d), dtype, g) * 2
    return dict(query=query, cache=cache, table=table, starts=starts, qlens=qlens, lens=lens, dense=dense, window=window,
                scale=d ** -0.5 if scale is None else scale, hq=hq, hkv=hkv, d=d, tokens=tokens)


def expect(case):
    """(output, lse, terms, logit error, largest logit) in 64 bits; rows of no token stay NaN."""
    t, hq, d = case["query"].shape
    group = hq // case["hkv"]
    out = torch.full((t, hq, d), float("nan"), dtype=torch.float64)
    lse = torch.full((t, hq), float("nan"), dtype=torch.float64)
    terms, err, top = torch.zeros((t, hq, d), dtype=torch.float64), torch.zeros((t, hq), dtype=torch.float64), \
        torch.zeros((t, hq), dtype=torch.float64)
    for b, (start, q, n) in enumerate(zip(case["starts"], case["qlens"], case["lens"])):
        if not q:
            continue
        ends = torch.arange(n - q + 1, n + 1)
        at = torch.arange(n)
        seen = at < ends[:, None]
        if case["window"]:
            seen &= at >= ends[:, None] - case["window"]
        some = seen.any(1)
        for h in range(hq):
            x = case["query"][start: start + q, h].double()
            k, v = (y[:, h // group].double() for y in case["dense"][b])
            logits = (x @ k.t() * case["scale"]).masked_fill(~seen, -INF)
            w = torch.where(some[:, None], torch.softmax(logits, -1), 0.0).nan_to_num(0.0)
            rows = slice(start, start + q)
            out[rows, h], terms[rows, h] = w @ v, w @ v.abs()
            lse[rows, h] = torch.logsumexp(logits, -1) if n else -INF
            e = abs(case["scale"]) * (d + 4) * 2.0 ** -24 * (x.abs() @ k.abs().t())
            if n:
                err[rows, h] = e.masked_fill(~seen, 0).amax(-1)
                top[rows, h] = logits.abs().masked_fill(~seen, 0).amax(-1)
    return out, lse, terms, err, top


def device_args(case, cuda, **over):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    from ds355 import chunk_attention as ca

    args = dict(
        query=case["query"].to(cuda), key_cache=case["cache"][0].to(cuda), value_cache=case["cache"][1].to(cuda),
        output=torch.full(case["query"].shape, 7.0, dtype=case["query"].dtype, device=cuda),
        lse=torch.full(case["query"].shape[:2], 7.0, device=cuda), block_table=case["table"].to(cuda),
        query_start=i32(case["starts"]), query_len=i32(case["qlens"]), target_len=i32(case["lens"]),
        scale=case["scale"], window=case["window"],
        workspace=ca.new_chunk_workspace(len(case["qlens"]), case["tokens"], case["hq"], case["hkv"], case["d"], cuda),
        status=torch.zeros(1, dtype=torch.int32, device=cuda))
    args.update(over)
    return args


def run(args):
    from ds355 import chunk_attention as ca

    out = ca.chunk_attention(**args)
    torch.cuda.synchronize()
    return out


def check(case, args, expected=None, status=0):
    out, lse, terms, err, top = expected if expected is not None else expect(case)
    got, got_lse = args["output"].cpu().double(), args["lse"].cpu().double()
    keys = max(case["lens"] + [1])
    u = torch.finfo(case["query"].dtype).eps / 2
    sums = (keys / 16 + 64) * 2.0 ** -24 + 2.0 ** -22 * (1 + top)
    mine = ~out.isnan().any(-1).any(-1)
    for start, q in zip(case["starts"], case["qlens"]):
        assert mine[start: start + q].all()
    assert (got[~mine] == 7).all() and (got_lse[~mine] == 7).all(), "tokens of no row were written"
    bound = u * out.abs() + (u * (1 + u) + 2 * err[..., None] + 2 * sums[..., None]) * terms + 1e-30
    excess = ((got - out).abs() - bound)[mine]
    assert not got[mine].isnan().any() and excess.numel() and float(excess.max()) <= 0, float(excess.max())
    nothing = lse == -INF
    assert (got_lse[nothing] == -INF).all() and (got[nothing] == 0).all()
    some = mine[:, None] & ~nothing
    off = ((got_lse - lse).abs() - (err + sums + 2.0 ** -22 * lse.abs()))[some]
    assert not got_lse[some].isnan().any() and (not off.numel() or float(off.max()) <= 0), float(off.max())
    assert int(args["status"].item()) == status


SHAPES = [
    dict(lens=[1], qlens=[1], hq=1, hkv=1, d=64, block=16),
    dict(lens=[37], qlens=[37], hq=8, hkv=2, d=128, block=16),
    dict(lens=[300], qlens=[300], hq=8, hkv=2, d=128, block=16),
    dict(lens=[301, 64, 65], qlens=[129, 64, 1], hq=4, hkv=4, d=128, block=48),
    dict(lens=[1000, 9, 700, 130], qlens=[3, 9, 1, 128], hq=32, hkv=4, d=128, block=128),
    dict(lens=[600, 31, 500], qlens=[100, 31, 7], hq=16, hkv=16, d=64, block=16),
    dict(lens=[515, 70, 1], qlens=[200, 5, 1], hq=28, hkv=4, d=64, block=1),  # groups of seven, pages of one token
    dict(lens=[333, 260], qlens=[70, 260], hq=10, hkv=2, d=128, block=7),  # pages that no load lies in
    dict(lens=[700, 33, 130], qlens=[20, 33, 65], hq=16, hkv=1, d=256, block=16),
    dict(lens=[310, 64], qlens=[300, 33], hq=8, hkv=2, d=256, block=200),
    dict(lens=[2000, 4500], qlens=[2, 33], hq=8, hkv=2, d=128, block=16),  # long rows in parts
    dict(lens=[3000], qlens=[128], hq=1, hkv=1, d=256, block=64),
    dict(lens=[5000], qlens=[1], hq=8, hkv=1, d=64, block=32),
    dict(lens=[100, 0, 50], qlens=[2, 0, 2], hq=8, hkv=2, d=128, block=32),  # graph padding
    # Windows: of one key, inside a tile, of a tile, longer than the row.
    dict(lens=[300, 40], qlens=[150, 3], hq=8, hkv=2, d=128, block=16, window=1),
    dict(lens=[700, 90], qlens=[333, 90], hq=8, hkv=2, d=128, block=16, window=50),
    dict(lens=[700, 1500], qlens=[400, 1], hq=4, hkv=2, d=64, block=16, window=128),
    dict(lens=[900, 130], qlens=[300, 130], hq=2, hkv=1, d=256, block=48, window=257),
    dict(lens=[260, 70], qlens=[260, 1], hq=8, hkv=8, d=128, block=16, window=100000),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=("bf16", "fp16"))
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_against_64_bits(cuda, i, dtype):
    case = build(100 + i, dtype=dtype, **SHAPES[i])
    print("chunk attention", i, SHAPES[i], flush=True)
    args = device_args(case, cuda)
    run(args)
    check(case, args)


def test_rows_that_see_nothing(cuda):
    # A row without keys, a row with fewer keys than query tokens, beside ordinary ones.
    for window in (None, 3):
        case = build(7, lens=[0, 2, 50, 10], qlens=[2, 5, 3, 200], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16,
                     window=window)
        args = device_args(case, cuda)
        run(args)
        check(case, args)


@pytest.mark.parametrize("bad", (float("nan"), INF, -INF))
@pytest.mark.parametrize("d,hkv", ((128, 2), (64, 8), (256, 1)))
@pytest.mark.parametrize("q", (5, 70))
def test_keys_a_token_does_not_see_have_no_effect(cuda, bad, d, hkv, q):
    # The last two tokens of each row hold `bad` in some dimensions of K and V: their own query tokens are
    # lost, the earlier ones see nothing of it.
    case = build(9, lens=[140, 190, 104], qlens=[q, q, 4], hq=8, hkv=hkv, d=d, block=16, dtype=torch.bfloat16)
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
    for start, n in zip(case["starts"], case["qlens"]):
        upto = slice(start, start + n - 2)
        assert not got[upto].isnan().any()
        assert ((got[upto] - clean[0][upto]).abs() <= 1.01 * u * (clean[0][upto].abs() + clean[2][upto]) + 1e-5).all()
        assert (args["lse"].cpu().double()[upto] - clean[1][upto]).abs().max() < 1e-4
        assert not got[start + n - 1].isfinite().all()


def test_keys_before_the_window_have_no_effect(cuda):
    case = build(10, lens=[400], qlens=[120], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16, window=100)
    expected = expect(case)
    for t in range(0, 181):  # the first query token, at 280, sees 181 .. 280
        page = int(case["table"][0, t // 16])
        case["cache"][0][page, t % 16] = float("nan")
        case["cache"][1][page, t % 16] = INF
    args = device_args(case, cuda)
    run(args)
    check(case, args, expected)


def test_a_value_that_is_not_finite_reaches_the_tokens_that_see_it(cuda):
    # V alone: the sum over a seen infinity is that infinity, over NaN NaN, in the dimensions that hold it.
    for q in (4, 40):
        case = build(11, lens=[84, 84], qlens=[q, q], hq=8, hkv=2, d=128, block=16, dtype=torch.float16)
        for b, value in enumerate((INF, float("nan"))):
            t = case["lens"][b] - 2
            case["cache"][1][int(case["table"][b, t // 16]), t % 16, 1, 7] = value
        args = device_args(case, cuda)
        run(args)
        got = args["output"].cpu()
        for b, start in enumerate(case["starts"]):
            assert got[start: start + q - 2].isfinite().all()
            mine = got[start + q - 2: start + q, 4:, 7]
            assert mine.isnan().all() if b else (mine == INF).all()
            rest = torch.ones(128, dtype=torch.bool)
            rest[7] = False
            assert got[start + q - 2: start + q][..., rest].isfinite().all() and got[start: start + q, :4].isfinite().all()


def test_strided_tensors(cuda):
    # Queries out of a fused projection, a padded output, LSEs by head, caches that are views of one
    # buffer with heads before tokens, a table with padding columns.
    case = build(12, lens=[393, 338, 461], qlens=[2, 104, 1], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
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
    case = build(13, lens=[120, 130, 140], qlens=[2, 90, 2], hq=8, hkv=2, d=64, block=16, dtype=torch.float16)
    args = device_args(case, cuda, batch_size=2)
    run(args)
    got = args["output"].clone()
    args["output"].fill_(7)
    args["lse"] = None
    run(args)
    assert torch.equal(args["output"], got)
    start = case["starts"][2]
    assert (got[start: start + 2] == 7).all()
    case["qlens"] = [2, 90, 0]
    args["lse"] = torch.full(got.shape[:2], 7.0, device=cuda)
    run(args)
    check(case, args)


def test_a_launch_gives_the_same_bits_again(cuda):
    case = build(14, lens=[3201, 300, 77, 4000], qlens=[50, 300, 3, 1], hq=32, hkv=4, d=128, block=16,
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
    base = dict(lens=[84, 94, 104], qlens=[2, 2, 60], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    # A row whose tokens are out of range is left out; the others are computed.
    case = build(15, **base)
    args = device_args(case, cuda)
    args["query_start"][1] = case["tokens"] - 1
    run(args)
    assert int(args["status"].item()) == 1
    args["status"].zero_()
    whole = expect(case)
    for t in (case["starts"][1], case["starts"][1] + 1):
        whole[0][t], whole[1][t] = float("nan"), float("nan")
    case["qlens"] = [2, 0, 60]
    check(case, args, whole)
    # A row longer than its table ends there, for its causal ends as well.
    case = build(16, lens=[84, 94, 176], qlens=[2, 2, 60], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    expected = expect(case)
    for beyond in (0, 1, 50, 10 ** 9):
        args = device_args(case, cuda, block_table=case["table"][:, :11].contiguous().to(cuda))
        args["target_len"][2] = 176 + beyond
        run(args)
        check(case, args, expected, status=2 if beyond else 0)
    # A page id out of range reads as zeros.
    for page in (-1, 10 ** 6):
        case = build(17, **base)
        args = device_args(case, cuda)
        args["block_table"][1, 5] = page  # keys 80 .. 95 of the row's 94
        args["block_table"][2, 2] = page  # keys 32 .. 47 of the row's 104, which all its tokens see
        run(args)
        assert int(args["status"].item()) == 4
        for kv in case["dense"][1]:
            kv[80:] = 0
        for kv in case["dense"][2]:
            kv[32:48] = 0
        args["status"].zero_()
        check(case, args)


def test_rows_that_overlap_are_cut_off(cuda):
    # More query tokens in all than the query holds: the rows that bring the sum over are left out.
    case = build(18, lens=[73, 73, 73], qlens=[3, 3, 3], hq=4, hkv=2, d=64, block=16, dtype=torch.float16, gaps=False)
    args = device_args(case, cuda)
    args["query"], args["output"], args["lse"] = (args[k][:7] for k in ("query", "output", "lse"))
    args["query_start"][2] = 1
    run(args)
    expected = expect(case)
    got = args["output"].cpu().double()
    assert int(args["status"].item()) == 1
    assert (got[6] == 7).all()
    assert (got[:6] - expected[0][:6]).abs().max() < 0.02


def test_rows_in_any_order_of_their_tokens(cuda):
    case = build(19, lens=[340, 305, 390, 317], qlens=[3, 1, 50, 2], hq=8, hkv=2, d=64, block=16, dtype=torch.float16)
    starts = [56, 54, 3, 0]
    query = case["query"].clone()
    for old, new, n in zip(case["starts"], starts, case["qlens"]):
        query[new: new + n] = case["query"][old: old + n]
    case.update(query=query, starts=starts)
    args = device_args(case, cuda)
    run(args)
    check(case, args)


@pytest.mark.parametrize("rows,d", ((1024, 64), (700, 128), (65, 256)))
def test_many_rows(cuda, rows, d):
    lens = [0 if b % 97 == 5 else 20 + (b * 37) % 41 + (b % 4) for b in range(rows)]
    qlens = [0 if b % 11 == 3 else 1 + (b % 29 == 0) * 3 for b in range(rows)]
    case = build(60, lens=lens, qlens=qlens, hq=4, hkv=2, d=d, block=16, dtype=torch.bfloat16)
    args = device_args(case, cuda)
    run(args)
    check(case, args)


@pytest.mark.parametrize("dtype", DTYPES, ids=("bf16", "fp16"))
@pytest.mark.parametrize("d,hkv", ((64, 2), (128, 2), (256, 1)))
@pytest.mark.parametrize("scale", (0.0, -0.0, -1.0))
def test_zero_and_negative_scales(cuda, scale, d, hkv, dtype):
    # Scale 0 weighs all seen keys alike: the mean of their values, and the logarithm of their number.
    case = build(63, lens=[617, 900, 1, 64], qlens=[30, 50, 1, 64], hq=8, hkv=hkv, d=d, block=16, dtype=dtype, scale=scale)
    args = device_args(case, cuda)
    run(args)
    check(case, args)
    if scale == 0:
        assert (args["lse"].cpu()[case["starts"][1] + 49] - torch.tensor(900.0).log()).abs().max() < 1e-5


def test_a_long_tail_of_small_probabilities(cuda):
    # One key outweighs each of the others by e^14, near the smallest normal fp16, and has a value of 0: the
    # output is the others' sum, which would be percents off were they rounded at fp16's smallest step.
    n, d, block = 20000, 64, 16
    keys, values = torch.zeros(n, 1, d, dtype=torch.float16), torch.ones(n, 1, d, dtype=torch.float16)
    keys[0, 0, 0], values[0] = 1.75, 0
    query = torch.zeros(1, 1, d, dtype=torch.float16)
    query[0, 0, 0] = 8
    cache = [x.view(n // block, block, 1, d) for x in (keys, values)]
    case = dict(query=query, dense=[[keys, values]], starts=[0], qlens=[1], lens=[n], window=None, scale=1.0, hq=1, hkv=1,
                d=d, tokens=1, cache=cache, table=torch.arange(n // block, dtype=torch.int32)[None])
    args = device_args(case, cuda)
    run(args)
    check(case, args)


def test_places_past_32_bits(cuda):
    # A cache of 5 GiB: the row's pages lie at both of its ends.
    block, hkv, d = 128, 8, 128
    pages = 20500
    key_cache = torch.zeros((pages, block, hkv, d), dtype=torch.bfloat16, device=cuda)
    value_cache = torch.zeros_like(key_cache)
    case = build(64, lens=[500], qlens=[90], hq=16, hkv=hkv, d=d, block=block, dtype=torch.bfloat16)
    spots = [pages - 1, 3, pages - 700, 16400]
    for i, page in enumerate(case["table"][0, :4].tolist()):
        key_cache[spots[i]], value_cache[spots[i]] = case["cache"][0][page].to(cuda), case["cache"][1][page].to(cuda)
    args = device_args(case, cuda, key_cache=key_cache, value_cache=value_cache)
    args["block_table"][0, :4] = torch.tensor(spots, dtype=torch.int32)
    run(args)
    check(case, args)


def test_graph_follows_changed_lengths_and_shares_a_workspace(cuda):
    from ds355 import chunk_attention as ca

    cases = [build(20 + i, lens=n, qlens=q, hq=16, hkv=2, d=128, block=16, dtype=torch.bfloat16, extra=200)
             for i, (n, q) in enumerate((([2530, 507, 700], [3, 100, 2]), ([480, 82, 89], [1, 1, 80])))]
    width, pages, t = 170, 500, 112
    args = device_args(cases[0], cuda)
    for k in ("query", "output"):
        args[k] = torch.zeros((t, 16, 128), dtype=torch.bfloat16, device=cuda)
    args["lse"] = torch.zeros((t, 16), device=cuda)
    args["block_table"] = torch.zeros((3, width), dtype=torch.int32, device=cuda)
    args["key_cache"] = torch.zeros((pages, 16, 2, 128), dtype=torch.bfloat16, device=cuda)
    args["value_cache"] = torch.zeros_like(args["key_cache"])
    args["workspace"] = ca.new_chunk_workspace(3, t, 16, 2, 128, cuda)
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

    fill(cases[0])
    run(args)
    stream = torch.cuda.Stream()
    graphs = []
    for a in (args, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ca.chunk_attention(**a)
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
    case = build(30, lens=[433, 403], qlens=[2, 100], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    expected = expect(case)
    args = device_args(case, cuda, reuse={})
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(args)
    check(case, args, expected)
    # The same layout at other addresses, then another window and another layout through the same dict.
    moved = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in args.items()}
    for k in ("output", "lse"):
        args[k].fill_(7)
        moved[k].fill_(7)
    run(moved)
    check(case, moved, expected)
    assert (args["output"] == 7).all()
    assert len(args["reuse"]) == 1
    case["window"] = args["window"] = 37
    run(args)
    check(case, args)
    other = build(31, lens=[33, 120], qlens=[2, 5], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    more = device_args(other, cuda, reuse=args["reuse"])
    run(more)
    check(other, more)


def test_shared_prefix_attention_gives_the_same(cuda):
    # The two attentions of the verifier's side on one batch, within both roundings of the output and of the
    # probabilities.
    from ds355 import prefix_attention as pa

    case = build(32, lens=[700, 260, 401], qlens=[60, 3, 1], hq=32, hkv=4, d=128, block=16, dtype=torch.bfloat16, fill=0.0)
    expected = expect(case)
    args = device_args(case, cuda)
    run(args)
    check(case, args, expected)
    other = dict(args, output=torch.full_like(args["output"], 7.0), lse=torch.full_like(args["lse"], 7.0),
                 prefix_len=torch.zeros(1, dtype=torch.int32, device=cuda),
                 workspace=pa.new_prefix_workspace(3, case["tokens"], 32, 4, 128, cuda))
    del other["window"]
    pa.shared_prefix_attention(**other)
    torch.cuda.synchronize()
    check(case, other, expected)


def test_two_calls_at_once_on_two_streams(cuda):
    from ds355 import chunk_attention as ca

    cases = [build(70 + i, lens=[900, 120], qlens=[300, 1], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
             for i in range(2)]
    args = [device_args(c, cuda) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for s, a in zip(streams, args):
        with torch.cuda.stream(s):
            ca.chunk_attention(**a)
    torch.cuda.synchronize()
    for c, a in zip(cases, args):
        check(c, a)


def test_output_in_place_of_the_query(cuda):
    case = build(72, lens=[3000, 200, 64], qlens=[3, 200, 64], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    args = device_args(case, cuda)
    run(args)
    again = dict(args, output=args["query"].clone())
    run(dict(again, query=again["output"]))
    # Tokens that no row has keep what was there, here the query.
    check(case, dict(again, output=torch.where((args["output"] == 7).all(-1, keepdim=True), args["output"], again["output"])))
    for start, q in zip(case["starts"], case["qlens"]):
        assert torch.equal(again["output"][start: start + q], args["output"][start: start + q])
    assert torch.equal(again["output"][:1], args["query"][:1])


@pytest.mark.parametrize("d,hkv,block", ((64, 1, 8), (64, 2, 24), (128, 1, 4), (128, 2, 20), (256, 1, 2), (256, 1, 6), (128, 1, 2)))
def test_runs_of_pages(cuda, d, hkv, block):
    # Long rows of small pages: their places are looked up for many tiles at a time.
    case = build(73, lens=[5003, 4096, 1033], qlens=[1, 200, 33], hq=4 * hkv, hkv=hkv, d=d, block=block, dtype=torch.bfloat16,
                 window=None)
    args = device_args(case, cuda)
    run(args)
    check(case, args)
    # A page that is not there, in the middle of a run, reads as zeros.
    page = 2500 // block
    for b, n in enumerate(case["lens"]):
        if page * block < n:
            args["block_table"][b, page] = 10 ** 6
            for kv in case["dense"][b][:2]:
                kv[page * block: (page + 1) * block] = 0
    args["output"].fill_(7)
    args["lse"].fill_(7)
    run(args)
    check(case, args, status=4)


# Tiles that a mask hides from some query rows of an item and that others, in another wave, see whole; where a row's or
# a window's first tile has the mask; parts that begin in one; pages that no load lies in.
NOT_FINITE = [
    dict(lens=[128], qlens=[128], hq=1, hkv=1, d=128, block=16),
    dict(lens=[84, 300], qlens=[40, 256], hq=8, hkv=2, d=128, block=16),
    dict(lens=[50, 63, 64, 65], qlens=[50, 63, 64, 65], hq=4, hkv=4, d=64, block=16),
    dict(lens=[300], qlens=[300], hq=8, hkv=2, d=128, block=16, window=200),
    dict(lens=[300, 90], qlens=[280, 90], hq=4, hkv=4, d=64, block=48, window=70),
    dict(lens=[200, 130], qlens=[150, 130], hq=2, hkv=1, d=256, block=16),
    dict(lens=[2000, 1500], qlens=[128, 70], hq=8, hkv=8, d=128, block=16),
    dict(lens=[190], qlens=[128], hq=4, hkv=2, d=128, block=7, window=100),
]


def not_finite_values(i, value, dtype, cuda):
    """(got, seen, rows): some values of head 0 are `value`, each in a dimension of its own; seen[token, head, dimension]
    says whether a query row sees the one of that dimension."""
    case = build(80 + i, dtype=dtype, **NOT_FINITE[i])
    block, hkv, d = NOT_FINITE[i]["block"], case["hkv"], case["d"]
    t, hq, _ = case["query"].shape
    seen, rows = torch.zeros((t, hq, d), dtype=torch.bool), torch.zeros(t, dtype=torch.bool)
    for b, (start, q, n) in enumerate(zip(case["starts"], case["qlens"], case["lens"])):
        rows[start: start + q] = True
        ends = torch.arange(n - q + 1, n + 1)
        at = sorted({0, 10, 31, 32, 63, 64, 70, n // 3, n // 2, n - q, n - 65, n - 64, n - 33, n - 10, n - 1})
        for dim, key in enumerate(k for k in at if 0 <= k < n):
            page = int(case["table"][b, key // block])
            case["cache"][1][page, key % block, 0, 3 * dim] = value
            sees = (key < ends) & (key >= ends - case["window"] if case["window"] else True)
            seen[start: start + q, : hq // hkv, 3 * dim] = sees[:, None]
    args = device_args(case, cuda)
    run(args)
    return args["output"].cpu(), seen, rows


@pytest.mark.parametrize("dtype", DTYPES, ids=("bf16", "fp16"))
@pytest.mark.parametrize("value", (float("nan"), INF, -INF))
@pytest.mark.parametrize("i", range(len(NOT_FINITE)))
def test_every_row_gets_the_values_that_are_not_finite_and_seen(cuda, i, value, dtype):
    got, seen, rows = not_finite_values(i, value, dtype, cuda)
    assert torch.equal(got[rows].isfinite(), ~seen[rows])


@pytest.mark.parametrize("dtype", DTYPES, ids=("bf16", "fp16"))
@pytest.mark.parametrize("value", (INF, -INF))
@pytest.mark.parametrize("i", range(len(NOT_FINITE)))
def test_a_seen_infinity_stays_one(cuda, i, value, dtype):
    # No weight here is below 2^-25 of its row's largest (2^-24.9 in 64 bits), and fp16 holds weights down to 2^-31 of it: none
    # rounds to 0.
    got, seen, _ = not_finite_values(i, value, dtype, cuda)
    assert (got[seen] == value).all()


@pytest.mark.parametrize("d", (64, 128, 256))
def test_an_infinity_behind_keys_of_no_weight_stays_one(cuda, d):
    # The keys of the first tile lie 2^-288 below those of the second, where the infinity is.
    case = build(95, lens=[100], qlens=[40], hq=1, hkv=1, d=d, block=16, dtype=torch.bfloat16, scale=1.0)
    case["query"].zero_()[..., 0] = 1
    k, v = case["dense"][0]
    k.zero_()[:64, :, 0] = -200
    exact = torch.stack([v[64: n].double().mean(0) if n > 64 else v[:n].double().mean(0) for n in range(61, 101)])
    terms = torch.stack([v[64: n].double().abs().mean(0) if n > 64 else v[:n].double().abs().mean(0) for n in range(61, 101)])
    v[70, 0, 5] = INF
    for t in range(100):
        for c, x in zip(case["cache"], (k, v)):
            c[int(case["table"][0, t // 16]), t % 16] = x[t]
    args = device_args(case, cuda)
    run(args)
    got = args["output"].cpu().double()[case["starts"][0]:][:40]
    assert (got[10:, 0, 5] == INF).all()  # query token 10 is the first that sees key 70
    rest = torch.ones((40, 1, d), dtype=torch.bool)
    rest[10:, 0, 5] = False
    # Weights are 1 each: the output rounds (2^-8), and fp32 sums.
    assert ((got - exact).abs()[rest] <= (2.0 ** -8 * exact.abs() + 2.0 ** -18 * terms)[rest]).all()


@pytest.mark.parametrize("shape", (
    dict(lens=[3000, 900], qlens=[5, 1], hq=8, hkv=1, d=128, block=16, window=2000),  # long rows in parts
    dict(lens=[2500], qlens=[200], hq=4, hkv=4, d=64, block=7, window=333),
    dict(lens=[1800, 300], qlens=[70, 300], hq=2, hkv=1, d=256, block=48, window=129),
))
def test_what_lies_before_every_window_has_no_effect(cuda, shape):
    case = build(96, dtype=torch.bfloat16, **shape)
    expected = expect(case)
    for b, (n, q) in enumerate(zip(case["lens"], case["qlens"])):
        for t in range(max(n - q + 1 - shape["window"], 0)):
            page = int(case["table"][b, t // shape["block"]])
            case["cache"][0][page, t % shape["block"]] = (float("nan"), INF, -INF)[t % 3]
            case["cache"][1][page, t % shape["block"]] = (INF, float("nan"))[t % 2]
    args = device_args(case, cuda)
    run(args)
    check(case, args, expected)

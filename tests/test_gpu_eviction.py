"""GPU: attention mass and eviction against plain implementations, and a request kept at its budget.

A weight exp(x - lse) has the relative error of its logit: x is an fp32 sum of D products, off by at most
(D + 4) 2^-24 |scale| sum_d |q_d k_d| =: E; scaling x and the LSE by log2 e and exp2 add 2^-22 (1 + |x| +
|lse|).  Sums over n weights, all positive: (n / 8 + 64) 2^-24 of the sum, lanes and parts adding up short
runs.  decay * previous adds two roundings of 2^-24.
"""

import pytest
import torch

from helpers import gen, randn
from test_gpu_chunk_attention import build, expect

pytestmark = pytest.mark.gpu

DTYPES = (torch.bfloat16, torch.float16)
INF = float("inf")


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


# ---- attention mass ------------------------------------------------------------------------------


def mass_case(seed, *, capacity=None, decay=0.9, previous=True, **shape):
    case = build(seed, **shape)
    rows = len(case["lens"])
    case["capacity"] = capacity or max(case["lens"] + [1]) + 5
    lse = expect(case)[1]
    case["lse"] = lse.nan_to_num(nan=3.0, neginf=-INF).float()
    g = gen(seed + 1000)
    case["decay"] = decay
    case["previous"] = torch.rand((rows, case["hkv"], case["capacity"]), generator=g) * 3 if previous else None
    return case


def expect_mass(case):
    """(mass, its error bound) in 64 bits; untouched entries are NaN."""
    rows, hkv, capacity = len(case["lens"]), case["hkv"], case["capacity"]
    group, d = case["hq"] // hkv, case["d"]
    mass = torch.full((rows, hkv, capacity), float("nan"), dtype=torch.float64)
    bound = torch.zeros_like(mass)
    for b, (start, q, n) in enumerate(zip(case["starts"], case["qlens"], case["lens"])):
        if not q:
            continue
        ends = torch.arange(n - q + 1, n + 1)
        at = torch.arange(n)
        seen = at < ends[:, None]
        if case["window"]:
            seen &= at >= ends[:, None] - case["window"]
        for h in range(hkv):
            old = 0 if case["previous"] is None else case["previous"][b, h, :n].double() * case["decay"]
            mass[b, h, :n], bound[b, h, :n] = old, 2.0 ** -23 * abs(old) if q else 0
            k = case["dense"][b][0][:, h].double()
            total = torch.zeros(n, dtype=torch.float64)
            for g in range(group):
                x = case["query"][start: start + q, h * group + g].double()
                lse = case["lse"][start: start + q, h * group + g].double()[:, None]
                logits = x @ k.t() * case["scale"]
                w = torch.where(seen & (lse != -INF), torch.exp(logits - lse), 0.0)
                e = (d + 4) * 2.0 ** -24 * abs(case["scale"]) * (x.abs() @ k.abs().t())
                e = e + 2.0 ** -22 * (1 + logits.abs() + torch.where(lse == -INF, 0.0, lse).abs())
                total += w.sum(0)
                bound[b, h, :n] += (w * torch.expm1(e)).sum(0)
            mass[b, h, :n] += total
            bound[b, h, :n] += (q * group / 8 + 64) * 2.0 ** -24 * mass[b, h, :n].abs() + 1e-37
    return mass, bound


def mass_args(case, cuda, **over):
    from ds355 import eviction

    args = dict(
        query=case["query"].to(cuda), key_cache=case["cache"][0].to(cuda), lse=case["lse"].to(cuda),
        mass=torch.full((len(case["lens"]), case["hkv"], case["capacity"]), 7.0, device=cuda),
        block_table=case["table"].to(cuda), query_start=i32(case["starts"], cuda), query_len=i32(case["qlens"], cuda),
        target_len=i32(case["lens"], cuda), scale=case["scale"], window=case["window"], decay=case["decay"],
        previous=None if case["previous"] is None else case["previous"].to(cuda),
        workspace=eviction.new_mass_workspace(cuda), status=torch.zeros(1, dtype=torch.int32, device=cuda))
    args.update(over)
    return args


def run_mass(args):
    from ds355 import eviction

    out = eviction.attention_mass(**args)
    torch.cuda.synchronize()
    return out


def check_mass(case, args, expected=None, status=0):
    mass, bound = expected if expected is not None else expect_mass(case)
    got = args["mass"].cpu().double()
    mine = ~mass.isnan()
    assert (got[~mine] == 7).all(), "entries of no key were written"
    assert not got[mine].isnan().any()
    if mine.any():
        excess = ((got - mass).abs() - bound)[mine]
        assert float(excess.max()) <= 0, float(excess.max())
    assert int(args["status"].item()) == status


MASS_SHAPES = [
    dict(lens=[1], qlens=[1], hq=1, hkv=1, d=64, block=16),
    dict(lens=[300], qlens=[300], hq=8, hkv=2, d=128, block=16),
    dict(lens=[37, 600], qlens=[37, 1], hq=32, hkv=4, d=128, block=128),
    dict(lens=[1000, 9, 700], qlens=[1, 1, 1], hq=32, hkv=4, d=128, block=48, previous=False),
    dict(lens=[515, 70, 1], qlens=[200, 5, 1], hq=28, hkv=4, d=64, block=1),
    dict(lens=[333, 260], qlens=[70, 260], hq=10, hkv=2, d=128, block=7),
    dict(lens=[700, 33, 130], qlens=[20, 33, 65], hq=16, hkv=1, d=256, block=16),
    dict(lens=[310, 64], qlens=[300, 33], hq=8, hkv=2, d=256, block=200, previous=False),
    dict(lens=[900], qlens=[800], hq=16, hkv=2, d=64, block=16),  # query rows in parts
    dict(lens=[100, 0, 50], qlens=[2, 0, 2], hq=8, hkv=2, d=128, block=32),
    dict(lens=[100, 80, 50], qlens=[2, 0, 2], hq=8, hkv=2, d=128, block=32),  # a row without query tokens
    dict(lens=[300, 40], qlens=[150, 3], hq=8, hkv=2, d=128, block=16, window=1),
    dict(lens=[700, 90], qlens=[333, 90], hq=8, hkv=2, d=128, block=16, window=50),
    dict(lens=[900, 1500], qlens=[600, 1], hq=4, hkv=2, d=64, block=16, window=300),
    dict(lens=[50, 2, 10], qlens=[3, 5, 70], hq=8, hkv=2, d=128, block=16),  # query tokens that see nothing
    dict(lens=[260, 70], qlens=[260, 1], hq=8, hkv=8, d=128, block=16, window=100000),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=("bf16", "fp16"))
@pytest.mark.parametrize("i", range(len(MASS_SHAPES)))
def test_mass_against_64_bits(cuda, i, dtype):
    case = mass_case(200 + i, dtype=dtype, **MASS_SHAPES[i])
    print("attention mass", i, MASS_SHAPES[i], flush=True)
    args = mass_args(case, cuda)
    run_mass(args)
    check_mass(case, args)


@pytest.mark.parametrize("scale", (0.0, -0.5))
def test_mass_with_zero_and_negative_scales(cuda, scale):
    case = mass_case(220, lens=[400, 33], qlens=[60, 1], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16, scale=scale)
    args = mass_args(case, cuda)
    run_mass(args)
    check_mass(case, args)


def test_a_token_gives_one_in_all(cuda):
    # Every query head of every token spreads a weight of 1.
    case = mass_case(221, lens=[900, 77], qlens=[500, 1], hq=32, hkv=4, d=128, block=16, dtype=torch.bfloat16, previous=False)
    args = mass_args(case, cuda)
    run_mass(args)
    for b, n in enumerate(case["lens"]):
        total = args["mass"][b, :, :n].double().sum(-1).cpu()
        assert (total / (case["qlens"][b] * 8) - 1).abs().max() < 1e-5


def test_mass_is_added_in_place_and_gives_the_same_bits_again(cuda):
    case = mass_case(222, lens=[900, 77, 400], qlens=[500, 1, 60], hq=32, hkv=4, d=128, block=16, dtype=torch.bfloat16)
    args = mass_args(case, cuda)
    run_mass(args)
    first = args["mass"].clone()
    for _ in range(3):
        args["workspace"].fill_(255)
        args["mass"].copy_(args["previous"])
        run_mass(dict(args, previous=args["mass"]))
        for b, n in enumerate(case["lens"]):
            assert torch.equal(args["mass"][b, :, :n], first[b, :, :n])
            assert torch.equal(args["mass"][b, :, n:], args["previous"][b, :, n:])


def test_mass_of_the_last_tokens_only(cuda):
    # Rows that name the last 32 tokens of each request, out of a longer chunk.
    case = mass_case(223, lens=[300, 120], qlens=[200, 120], hq=8, hkv=2, d=128, block=16, dtype=torch.float16)
    case["starts"] = [s + q - 32 for s, q in zip(case["starts"], case["qlens"])]
    case["qlens"] = [32, 32]
    args = mass_args(case, cuda)
    run_mass(args)
    check_mass(case, args)


@pytest.mark.parametrize("bad", (float("nan"), INF))
def test_mass_of_other_keys_than_one_that_is_not_finite(cuda, bad):
    case = mass_case(224, lens=[200, 90], qlens=[70, 1], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    mass, bound = expect_mass(case)
    for b, t in ((0, 150), (1, 3)):
        case["cache"][0][int(case["table"][b, t // 16]), t % 16, :, ::5] = bad
    args = mass_args(case, cuda)
    run_mass(args)
    got = args["mass"].cpu().double()
    for b, t in ((0, 150), (1, 3)):
        got[b, :, t] = mass[b, :, t]
    check_mass(case, dict(args, mass=got), (mass, bound))


def test_strided_mass(cuda):
    case = mass_case(225, lens=[393, 338, 461], qlens=[2, 104, 1], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    args = mass_args(case, cuda)
    t, cap = case["tokens"], case["capacity"]
    fused = torch.zeros((t, 12 * 128), dtype=torch.bfloat16, device=cuda)
    fused[:, : 8 * 128] = args["query"].reshape(t, -1)
    lse = args["lse"].t().contiguous().t()
    keys = args["key_cache"].transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.full((2, 3, cap + 9), 7.0, device=cuda)  # heads before rows
    args.update(query=fused[:, : 8 * 128].unflatten(1, (8, 128)), lse=lse, key_cache=keys,
                mass=wide[..., :cap].transpose(0, 1))
    run_mass(args)
    check_mass(case, args)
    assert (wide[..., cap:] == 7).all()


def test_mass_status_bits(cuda):
    base = dict(lens=[84, 94, 104], qlens=[2, 2, 60], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
    case = mass_case(226, **base)
    args = mass_args(case, cuda)
    args["query_start"][1] = case["tokens"] - 1
    run_mass(args)
    case["qlens"] = [2, 0, 60]
    check_mass(case, args, status=1)
    # A row longer than its mass ends there, for its causal ends as well.
    case = mass_case(227, capacity=104, **base)
    expected = expect_mass(case)
    for beyond in (0, 1, 10 ** 9):
        args = mass_args(case, cuda)
        args["target_len"][2] = 104 + beyond
        run_mass(args)
        check_mass(case, args, expected, status=2 if beyond else 0)
    # A page id out of range reads as zeros.
    for page in (-1, 10 ** 6):
        case = mass_case(228, **base)
        args = mass_args(case, cuda)
        args["block_table"][1, 5] = page  # keys 80 .. 95 of the row's 94
        run_mass(args)
        case["dense"][1][0][80:] = 0
        check_mass(case, args, status=4)


def test_mass_of_many_rows(cuda):
    rows = 1000
    lens = [0 if b % 97 == 5 else 20 + (b * 37) % 41 for b in range(rows)]
    qlens = [0 if b % 11 == 3 else 1 + (b % 29 == 0) * 3 for b in range(rows)]
    case = mass_case(229, lens=lens, qlens=qlens, hq=4, hkv=2, d=64, block=16, dtype=torch.bfloat16)
    args = mass_args(case, cuda)
    run_mass(args)
    check_mass(case, args)
    # Rows at or beyond batch_size are padding.
    args["mass"].fill_(7)
    run_mass(dict(args, batch_size=10))
    case["qlens"] = qlens[:10] + [0] * (rows - 10)
    check_mass(case, args)


# ---- eviction ------------------------------------------------------------------------------------


def evict_case(seed, *, lens, keep, hkv, d, block, dtype=torch.bfloat16, sinks=0, recent=0, settled=None, spread=None,
               capacity=None):
    """Rows on the CPU.  settled[b]: (slots with written positions, tokens evicted so far)."""
    g = gen(seed)
    rows = len(lens)
    pages = [-(-max(n, 0) // block) for n in lens]
    order = torch.randperm(sum(pages) + 3, generator=g).tolist()
    width = max(pages + [1]) + 1
    table = torch.full((rows, width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = torch.tensor(order[at: at + n], dtype=torch.int32)
        at += n
    caches = [randn((len(order), block, hkv, d), dtype, g) for _ in range(2)]
    cap = capacity or width * block
    mass = torch.rand((rows, hkv, cap), generator=g)
    if spread:  # few distinct values: ties
        mass = (mass * spread).floor() / spread
    for b, n in enumerate(lens):
        mass[b, :, max(n, 0):] = -5.0
    positions = torch.randint(-9, 10 ** 6, (rows, hkv, cap), generator=g, dtype=torch.int32)
    known = torch.zeros((rows, 2), dtype=torch.int32)
    for b, s in enumerate(settled or []):
        if s is None:
            continue
        known[b] = torch.tensor(s, dtype=torch.int32)
        for h in range(hkv):
            positions[b, h, : s[0]] = torch.randperm(s[0] + s[1], generator=g)[: s[0]].int()
    return dict(lens=lens, keep=keep, table=table, caches=caches, mass=mass, positions=positions, settled=known, sinks=sinks,
                recent=recent, block=block, hkv=hkv, capacity=cap)


def expect_evict(case, left_alone=()):
    """The rule slot by slot."""
    key, value = (c.clone() for c in case["caches"])
    mass, positions, settled = case["mass"].clone(), case["positions"].clone(), case["settled"].clone()
    kept_len = [max(n, 0) for n in case["lens"]]
    block = case["block"]
    for b, (n, k) in enumerate(zip(case["lens"], case["keep"])):
        if n <= k or b in left_alone:
            continue
        known, gone = (int(x) for x in case["settled"][b])
        for h in range(case["hkv"]):
            place = [int(positions[b, h, t]) if t < known else t + gone for t in range(n)]

            def rank(t):
                w = float(mass[b, h, t])
                must = place[t] < case["sinks"] or place[t] >= n + gone - case["recent"]
                return not must, w != w, -w if w == w else 0.0, t

            kept = set(sorted(range(n), key=rank)[:k])
            holes = [t for t in range(k) if t not in kept]
            movers = [t for t in range(k, n) if t in kept]
            for t in range(k):
                positions[b, h, t] = place[t]
            for src, dst in zip(movers, holes):
                positions[b, h, dst], mass[b, h, dst] = place[src], mass[b, h, src]
                for c, old in ((key, case["caches"][0]), (value, case["caches"][1])):
                    c[int(case["table"][b, dst // block]), dst % block, h] = old[int(case["table"][b, src // block]), src % block, h]
            mass[b, h, k:n] = 0
        settled[b] = torch.tensor([k, gone + n - k])
        kept_len[b] = k
    return dict(key_cache=key, value_cache=value, mass=mass, positions=positions, settled=settled,
                kept_len=torch.tensor(kept_len, dtype=torch.int32))


def evict_args(case, cuda, **over):
    from ds355 import eviction

    args = dict(
        key_cache=case["caches"][0].to(cuda), value_cache=case["caches"][1].to(cuda), mass=case["mass"].to(cuda),
        positions=case["positions"].to(cuda), settled=case["settled"].to(cuda), block_table=case["table"].to(cuda),
        target_len=i32(case["lens"], cuda), keep_len=i32(case["keep"], cuda),
        kept_len=i32([-7] * len(case["lens"]), cuda), sinks=case["sinks"], recent=case["recent"],
        workspace=eviction.new_evict_workspace(len(case["lens"]), case["hkv"], case["capacity"], cuda),
        status=torch.zeros(1, dtype=torch.int32, device=cuda))
    args.update(over)
    return args


def run_evict(args):
    from ds355 import eviction

    out = eviction.evict_tokens(**args)
    torch.cuda.synchronize()
    return out


def same(x, y):
    return torch.equal(x.cpu().contiguous().view(torch.uint8), y.cpu().contiguous().view(torch.uint8))  # NaN included


def check_evict(case, args, expected=None, status=0):
    expected = expected if expected is not None else expect_evict(case)
    for name, x in expected.items():
        assert same(args[name], x), name
    assert int(args["status"].item()) == status


EVICT_SHAPES = [
    dict(lens=[2], keep=[1], hkv=1, d=64, block=16),
    dict(lens=[100], keep=[99], hkv=2, d=128, block=16),
    dict(lens=[100, 40, 0, 64], keep=[30, 64, 5, 64], hkv=4, d=128, block=16, sinks=4, recent=8),
    dict(lens=[700, 1300], keep=[256, 1000], hkv=2, d=128, block=48, sinks=4, recent=100),
    dict(lens=[500, 500], keep=[0, 499], hkv=2, d=64, block=1),
    dict(lens=[900], keep=[450], hkv=3, d=80, block=7, spread=4),  # many ties
    dict(lens=[2000, 1025], keep=[64, 1024], hkv=1, d=256, block=128, spread=1),  # all masses alike
    dict(lens=[257, 600], keep=[256, 256], hkv=2, d=128, block=16, settled=[(256, 31), (500, 1000)], sinks=3, recent=20),
    dict(lens=[300, 300], keep=[200, 24], hkv=2, d=128, block=16, settled=[(0, 0), (250, 7)], sinks=4, recent=20, spread=8),
    dict(lens=[5000], keep=[3001], hkv=2, d=64, block=64, recent=3001),  # only the newest
    dict(lens=[5000], keep=[600], hkv=2, d=64, block=64, sinks=600),  # only the first
    dict(lens=[40000], keep=[20000], hkv=1, d=64, block=128, sinks=4, recent=64),  # more than a register's share
    dict(lens=[300, 20], keep=[100, 20], hkv=2, d=128, block=16, dtype=torch.float32, recent=5),
]


@pytest.mark.parametrize("i", range(len(EVICT_SHAPES)))
def test_eviction_against_the_rule(cuda, i):
    case = evict_case(300 + i, **EVICT_SHAPES[i])
    print("eviction", i, EVICT_SHAPES[i], flush=True)
    args = evict_args(case, cuda)
    out = run_evict(args)
    assert out is args["kept_len"]
    check_evict(case, args)


def test_masses_that_are_not_finite_or_negative(cuda):
    case = evict_case(330, lens=[400, 300], keep=[200, 290], hkv=2, d=128, block=16, sinks=2, recent=3)
    g = gen(1)
    values = torch.tensor([float("nan"), INF, -INF, 0.0, -0.0, -1.5, 1e-42, -1e-42, 3.0])
    for b, n in enumerate(case["lens"]):
        case["mass"][b, :, :n] = values[torch.randint(0, len(values), (2, n), generator=g)]
    args = evict_args(case, cuda)
    run_evict(args)
    check_evict(case, args)


def test_a_step_by_step_budget(cuda):
    # Rows at their budget, one token more in each of several steps; the positions of what is kept follow.
    case = evict_case(331, lens=[129, 129], keep=[128, 128], hkv=2, d=64, block=16, sinks=2, recent=16)
    args = evict_args(case, cuda)
    g = gen(2)
    for step in range(6):
        expected = expect_evict(case)
        run_evict(args)
        check_evict(case, args, expected)
        for h in range(2):
            held = args["positions"][0, h, :128].tolist()
            newest = 128 + step
            assert len(set(held)) == 128 and set(range(newest - 15, newest + 1)) <= set(held) and {0, 1} <= set(held)
        # The next token of each row goes to slot 128.
        case.update(caches=[args["key_cache"].cpu(), args["value_cache"].cpu()], mass=args["mass"].cpu(),
                    positions=args["positions"].cpu(), settled=args["settled"].cpu())
        for b in range(2):
            page = int(case["table"][b, 8])
            for c in case["caches"]:
                c[page, 0] = randn((2, 64), torch.bfloat16, g)
            case["mass"][b, :, :129] += torch.rand((2, 129), generator=g)
        args = evict_args(case, cuda)


def test_strided_caches_and_batch_size(cuda):
    case = evict_case(332, lens=[200, 90, 150], keep=[60, 30, 10], hkv=2, d=128, block=16, recent=7)
    args = evict_args(case, cuda)
    pages = args["key_cache"].shape[0]
    both = torch.zeros((pages, 2, 2, 16, 144), dtype=torch.bfloat16, device=cuda)
    views = [both[:, i, :, :, :128].transpose(1, 2) for i in range(2)]
    for view, name in zip(views, ("key_cache", "value_cache")):
        view.copy_(args[name])
        args[name] = view
    cap = case["capacity"]
    book = torch.zeros((2, 3, cap + 3), device=cuda)
    places = torch.zeros((3, 2, cap + 5), dtype=torch.int32, device=cuda)
    book[..., :cap] = args["mass"].transpose(0, 1)
    places[..., :cap] = args["positions"]
    args.update(mass=book[..., :cap].transpose(0, 1), positions=places[..., :cap], batch_size=2)
    run_evict(args)
    expected = expect_evict(case, left_alone=(2,))
    expected["kept_len"][2] = -7
    check_evict(case, args, expected)
    assert (both[..., 128:] == 0).all()


def test_rows_that_cannot_be_cut_are_left_alone(cuda):
    base = dict(lens=[200, 90, 150], keep=[60, 30, 10], hkv=2, d=128, block=16, recent=7, sinks=2)
    case = evict_case(333, **base)
    args = evict_args(case, cuda)
    case["keep"] = [60, -1, 8]  # negative, and below the nine tokens that are always kept
    args["keep_len"] = i32(case["keep"], cuda)
    run_evict(args)
    check_evict(case, args, expect_evict(case, left_alone=(1, 2)), status=8)
    for page in (-1, 10 ** 6):
        case = evict_case(334, **base)
        args = evict_args(case, cuda)
        args["block_table"][1, 5] = page  # its last slots
        run_evict(args)
        check_evict(case, args, expect_evict(case, left_alone=(1,)), status=4)
    case = evict_case(335, **base)
    args = evict_args(case, cuda)
    args["target_len"][1] = case["capacity"] + 1
    run_evict(args)
    expected = expect_evict(case, left_alone=(1,))
    expected["kept_len"][1] = case["capacity"] + 1
    check_evict(case, args, expected, status=2)
    # A page that other rows hold: among the kept slots' pages, and behind them.
    for column, refused in ((1, True), (4, False)):
        case = evict_case(336, **base)
        counts = torch.ones(case["caches"][0].shape[0], dtype=torch.int32, device=cuda)
        counts[int(case["table"][1, column])] = 2
        args = evict_args(case, cuda, ref_counts=counts)
        run_evict(args)
        check_evict(case, args, expect_evict(case, left_alone=(1,) if refused else ()), status=16 if refused else 0)


def test_eviction_gives_the_same_again_and_from_a_graph(cuda):
    cases = [evict_case(340 + i, lens=n, keep=k, hkv=2, d=64, block=16, recent=5, capacity=640)
             for i, (n, k) in enumerate((([500, 300], [100, 299]), ([600, 3], [599, 2])))]
    for case in cases:
        case["table"] = torch.nn.functional.pad(case["table"], (0, 40 - case["table"].shape[1]), value=-1)
        case["recent"], case["sinks"] = 2, 0
        pages = 60 - case["caches"][0].shape[0]
        case["caches"] = [torch.cat((c, torch.zeros((pages, *c.shape[1:]), dtype=c.dtype))) for c in case["caches"]]
    args = evict_args(cases[0], cuda)
    names = dict(key_cache=0, value_cache=1)

    def fill(case):
        for name, i in names.items():
            args[name].copy_(case["caches"][i])
        for name in ("mass", "positions", "settled"):
            args[name].copy_(case[name])
        args["block_table"].copy_(case["table"])
        args["target_len"].copy_(i32(case["lens"], "cpu"))
        args["keep_len"].copy_(i32(case["keep"], "cpu"))
        args["kept_len"].fill_(-7)

    run_evict(args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        from ds355 import eviction

        eviction.evict_tokens(**args)
    for case in (cases[0], cases[1], cases[0], cases[1]):
        expected = expect_evict(case)
        fill(case)
        graph.replay()
        torch.cuda.synchronize()
        check_evict(case, args, expected)
        fill(case)
        args["workspace"].fill_(255)
        run_evict(args)
        check_evict(case, args, expected)


def test_reuse_and_another_stream(cuda):
    case = evict_case(350, lens=[300, 200], keep=[100, 150], hkv=2, d=128, block=16, recent=5)
    expected = expect_evict(case)
    args = evict_args(case, cuda, reuse={})
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run_evict(args)
    check_evict(case, args, expected)
    again = evict_args(case, cuda, reuse=args["reuse"])
    run_evict(again)
    check_evict(case, again, expected)
    assert len(args["reuse"]) == 1
    case["recent"] = 50
    other = evict_args(case, cuda, reuse=args["reuse"])
    run_evict(other)
    check_evict(case, other)


# ---- a run together ------------------------------------------------------------------------------


def test_a_request_kept_at_its_budget(cuda):
    """Prompt in chunks, mass, eviction, pages back to the pool, then decoding at the budget, all on the
    device; against the same run in 64 bits on what the kernels kept."""
    from ds355 import chunk_attention, eviction, pages, prefix_attention

    hq, hkv, d, block, rows, budget = 8, 2, 128, 16, 2, 96
    g = gen(360)
    prompt, steps = [250, 180], 5
    capacity = 320
    caches = [torch.zeros((64, block, hkv, d), dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    pool = pages.PagePool(caches)
    table = torch.full((rows, capacity // block), -1, dtype=torch.int32, device=cuda)
    mass = torch.zeros((rows, hkv, capacity), device=cuda)
    positions = torch.zeros((rows, hkv, capacity), dtype=torch.int32, device=cuda)
    settled = torch.zeros((rows, 2), dtype=torch.int32, device=cuda)
    row_ids, lens = i32([0, 1], cuda), i32([0, 0], cuda)
    kept = torch.zeros_like(lens)
    keep = i32([budget] * rows, cuda)
    work = chunk_attention.new_chunk_workspace(rows, 256, hq, hkv, d, cuda)
    mass_work, evict_work = eviction.new_mass_workspace(cuda), eviction.new_evict_workspace(rows, hkv, capacity, cuda)
    prefix_work = prefix_attention.new_prefix_workspace(rows, 256, hq, hkv, d, cuda)
    history = [randn((n + steps, 2, hkv, d), torch.bfloat16, g) for n in prompt]  # every token's key and value
    done = [0] * rows  # tokens of each request so far
    chunks = [[100, 64], [150, 116]] + [[1, 1]] * steps
    scale = d ** -0.5
    seen_positions = None
    for chunk in chunks:
        total = lens + i32(chunk, cuda)
        pool.extend(table, row_ids, total)
        host_table, host_lens = table.cpu(), lens.cpu().tolist()
        for b, n in enumerate(chunk):
            for i in range(n):
                slot = host_lens[b] + i
                for c in range(2):
                    caches[c][int(host_table[b, slot // block]), slot % block] = history[b][done[b] + i, c].to(cuda)
        query = (randn((sum(chunk), hq, d), torch.bfloat16, g) * 2).to(cuda)
        starts, counts = i32([0, chunk[0]], cuda), i32(chunk, cuda)
        out, lse = torch.zeros_like(query), torch.zeros((sum(chunk), hq), device=cuda)
        chunk_attention.chunk_attention(query, *caches, out, lse, table, starts, counts, total, scale=scale, workspace=work)
        if chunk[0] == 1:  # the other attention of the verifier's side reads the same rows
            again, lse2 = torch.zeros_like(out), torch.zeros_like(lse)
            prefix_attention.shared_prefix_attention(query, *caches, again, lse2, table, starts, counts, total,
                                                     torch.zeros(1, dtype=torch.int32, device=cuda), scale=scale,
                                                     workspace=prefix_work)
            # The output's rounding and that of the probabilities, twice (terms of at most 4 each).
            assert (again.float() - out.float()).abs().max() < 4 * 2.0 ** -8 * 4 and (lse - lse2).abs().max() < 1e-4
        eviction.attention_mass(query, caches[0], lse, mass, table, starts, counts, total, scale=scale, previous=mass,
                                workspace=mass_work)
        # Attention in 64 bits over the tokens that the slots hold.
        host = positions.cpu()
        at = 0
        for b, n in enumerate(chunk):
            have = host_lens[b]
            for h in range(hkv):
                held = (host[b, h, :have].tolist() if seen_positions else list(range(have))) + \
                    list(range(done[b], done[b] + n))
                kv = history[b][held, :, h].double()
                for g0 in range(hq // hkv):
                    q = query[at: at + n, h * (hq // hkv) + g0].cpu().double()
                    x = q @ kv[:, 0].t() * scale
                    x.masked_fill_(torch.arange(len(held)) > have + torch.arange(n)[:, None], -INF)
                    w = torch.softmax(x, -1)
                    exact, terms = w @ kv[:, 1], w @ kv[:, 1].abs()
                    got = out[at: at + n, h * (hq // hkv) + g0].cpu().double()
                    assert ((got - exact).abs() <= 1.01 * 2.0 ** -8 * (exact.abs() + terms) + 1e-5).all()
            at += n
        eviction.evict_tokens(*caches, mass, positions, settled, table, total, keep, kept, sinks=4, recent=16,
                              ref_counts=pool.ref_counts, workspace=evict_work)
        pool.free(table, row_ids, kept)
        lens = kept.clone()
        done = [a + b for a, b in zip(done, chunk)]
        torch.cuda.synchronize()
        seen_positions = chunk is not chunks[0] or max(done) > budget
        if done[1] <= budget:  # the second row has not been cut yet: its slots hold its tokens in order
            positions[1, :, : done[1]] = torch.arange(done[1], dtype=torch.int32, device=cuda)
        for b in range(rows):
            n = int(lens[b])
            assert n == min(budget, done[b])
            assert int((table[b] >= 0).sum()) == -(-n // block)
            if done[b] > budget:
                for h in range(hkv):
                    held = set(positions[b, h, :n].tolist())
                    assert len(held) == n and set(range(4)) <= held and set(range(done[b] - 16, done[b])) <= held
    assert int(pool.status.item()) == 0


# ---- sizes, graphs and streams -------------------------------------------------------------------


@pytest.mark.parametrize("d,hq,hkv,most", ((256, 16, 1, 2), (128, 32, 2, 3), (128, 4, 4, 5), (64, 8, 1, 4)))
def test_mass_of_as_many_rows_as_there_may_be(cuda, d, hq, hkv, most):
    lens = [1 + (b * 37) % 90 for b in range(1024)]
    case = mass_case(400, lens=lens, qlens=[min(n, 1 + b % most) for b, n in enumerate(lens)], hq=hq, hkv=hkv, d=d, block=16,
                     dtype=torch.bfloat16)
    args = mass_args(case, cuda)
    run_mass(args)
    check_mass(case, args)


def test_mass_of_one_long_row_beside_short_ones(cuda):
    lens = [3000, 1, 17, 64, 65, 2] + [5] * 20
    case = mass_case(401, lens=lens, qlens=[700, 1, 17, 1, 65, 2] + [1] * 20, hq=8, hkv=2, d=64, block=16,
                     dtype=torch.float16, window=900)
    args = mass_args(case, cuda)
    run_mass(args)
    check_mass(case, args)


def test_mass_graphs_share_a_workspace(cuda):
    from ds355 import eviction

    shape = dict(hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16, capacity=640)
    cases = [mass_case(410 + i, lens=n, qlens=q, **shape)
             for i, (n, q) in enumerate((([600, 31, 80], [100, 1, 19]), ([44, 620, 300], [1, 118, 1])))]
    args = [mass_args(c, cuda) for c in cases]
    for a in args:
        a["workspace"] = args[0]["workspace"]
        run_mass(a)
    stream, graphs = torch.cuda.Stream(), []
    for a in args:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            eviction.attention_mass(**a)
        graphs.append(graph)
    expected = [expect_mass(c) for c in cases]
    for i in (0, 1, 1, 0, 1):
        args[i]["mass"].fill_(7)
        args[i]["workspace"].fill_(255)
        graphs[i].replay()
        torch.cuda.synchronize()
        check_mass(cases[i], args[i], expected[i])
        replayed = args[i]["mass"].clone()
        run_mass(args[i])
        assert torch.equal(replayed, args[i]["mass"])
    # Other lengths at the same addresses.
    a = args[0]
    for n, q in (([300, 0, 79], [100, 0, 19]), ([1, 31, 5], [1, 1, 0])):
        case = dict(cases[0], lens=n, qlens=q)
        a["target_len"].copy_(i32(n, "cpu"))
        a["query_len"].copy_(i32(q, "cpu"))
        a["mass"].fill_(7)
        graphs[0].replay()
        torch.cuda.synchronize()
        case["dense"] = [tuple(x[:m] for x in kv) for kv, m in zip(cases[0]["dense"], n)]
        check_mass(case, a)


def test_mass_on_two_streams_and_with_reuse(cuda):
    cases = [mass_case(420 + i, lens=[500, 90], qlens=[60, 1], hq=8, hkv=2, d=128, block=16, dtype=torch.bfloat16)
             for i in range(2)]
    reuse = {}
    args = [mass_args(c, cuda, reuse=reuse) for c in cases]
    from ds355 import eviction

    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for s, a in zip(streams, args):
        with torch.cuda.stream(s):
            eviction.attention_mass(**a)
    torch.cuda.synchronize()
    for c, a in zip(cases, args):
        check_mass(c, a)
    assert len(reuse) == 1


def test_mass_places_past_32_bits(cuda):
    # A cache of 5 GiB: the row's pages lie at both of its ends.
    block, hkv, d = 128, 8, 128
    pages = 20500
    keys = torch.zeros((pages, block, hkv, d), dtype=torch.bfloat16, device=cuda)
    case = mass_case(430, lens=[500], qlens=[90], hq=16, hkv=hkv, d=d, block=block, dtype=torch.bfloat16)
    spots = [pages - 1, 3, pages - 700, 16400]
    for i, page in enumerate(case["table"][0, :4].tolist()):
        keys[spots[i]] = case["cache"][0][page].to(cuda)
    args = mass_args(case, cuda, key_cache=keys)
    args["block_table"][0, :4] = torch.tensor(spots, dtype=torch.int32)
    run_mass(args)
    check_mass(case, args)


def test_eviction_places_past_32_bits(cuda):
    block, hkv, d = 128, 8, 128
    pages = 20500
    case = evict_case(431, lens=[500], keep=[300], hkv=hkv, d=d, block=block, sinks=2, recent=9)
    expected = expect_evict(case)
    spots = [16400, pages - 1, 3, pages - 700]
    args = evict_args(case, cuda)
    mine = case["table"][0, :4].tolist()
    for i, name in enumerate(("key_cache", "value_cache")):
        big = torch.zeros((pages, block, hkv, d), dtype=torch.bfloat16, device=cuda)
        big[spots] = case["caches"][i][mine].to(cuda)
        args[name] = big
    args["block_table"][0, :4] = torch.tensor(spots, dtype=torch.int32)
    run_evict(args)
    for name in ("key_cache", "value_cache"):
        assert same(args[name][spots], expected.pop(name)[mine])
        assert int((args[name].flatten(1) != 0).any(1).sum()) == 4
    check_evict(case, args, expected)


@pytest.mark.parametrize("shape", (
    dict(lens=[70000], keep=[66000], spread=50),  # more slots than are held, ties on both sides of that many
    dict(lens=[32769, 32768], keep=[32768, 1], settled=[(32768, 5), (100, 3)], recent=0),
    dict(lens=[40000], keep=[33000], settled=[(39000, 12)], sinks=70, recent=500, spread=3),
    dict(lens=[8192, 8193, 4096, 4097], keep=[8000, 8192, 64, 4032], sinks=1, recent=2),
))
def test_eviction_of_long_rows(cuda, shape):
    case = evict_case(440, hkv=1, d=8, block=128, **shape)
    args = evict_args(case, cuda)
    run_evict(args)
    check_evict(case, args)


def test_evictions_graphs_share_a_workspace(cuda):
    from ds355 import eviction

    cases = [evict_case(450 + i, lens=n, keep=k, hkv=2, d=64, block=16, recent=5)
             for i, (n, k) in enumerate((([500, 300], [100, 299]), ([77, 400], [76, 33])))]
    args = [evict_args(c, cuda) for c in cases]
    work = eviction.new_evict_workspace(2, 2, max(c["capacity"] for c in cases), cuda)
    starts = []
    stream, graphs = torch.cuda.Stream(), []
    for a in args:
        a["workspace"] = work
        starts.append({k: v.clone() for k, v in a.items() if isinstance(v, torch.Tensor) and k != "workspace"})
        run_evict(a)
    for a in args:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            eviction.evict_tokens(**a)
        graphs.append(graph)
    for order in ((0, 1), (1, 0), (1, 1, 0, 0)):
        for i in order:
            for k, v in starts[i].items():
                args[i][k].copy_(v)
            graphs[i].replay()
            torch.cuda.synchronize()
            check_evict(cases[i], args[i])


def test_eviction_without_rows_and_of_padding_rows(cuda):
    case = evict_case(460, lens=[200, 300, 100], keep=[100, 100, 50], hkv=2, d=64, block=16)
    args = evict_args(case, cuda)
    before = {k: args[k].clone() for k in ("key_cache", "value_cache", "mass", "positions", "settled", "kept_len")}
    run_evict(dict(args, batch_size=0))
    for k, v in before.items():
        assert same(args[k], v), k
    # Rows of no length and of fewer slots than they may keep.
    case["lens"] = [0, 99, -3]
    args["target_len"].copy_(i32(case["lens"], "cpu"))
    run_evict(args)
    check_evict(case, args)


def test_the_same_eviction_twice_changes_nothing(cuda):
    case = evict_case(461, lens=[700, 90], keep=[128, 64], hkv=2, d=128, block=16, sinks=4, recent=32)
    args = evict_args(case, cuda)
    run_evict(args)
    check_evict(case, args)
    after = {k: args[k].clone() for k in ("key_cache", "value_cache", "mass", "positions", "settled", "kept_len")}
    args["target_len"].copy_(args["kept_len"])
    run_evict(args)
    for k, v in after.items():
        assert same(args[k], v), k


def _weights(query, lse, keys, ends, scale):
    """(weights [rows, keys], the errors of their logits) in 64 bits: row i sees the keys below ends[i]."""
    d = query.shape[1]
    x = query @ keys.t() * scale
    hidden = torch.arange(keys.shape[0]) >= ends[:, None]
    exact = torch.logsumexp(x.masked_fill(hidden, -INF), -1, keepdim=True)
    e = (d + 4) * 2.0 ** -24 * scale * (query.abs() @ keys.abs().t())
    own = (e + 2.0 ** -22 * (1 + x.abs())).masked_fill(hidden, 0).amax(-1, keepdim=True)
    # The LSE's own error, as the attention's tests have it, and that of the weight.
    error = own + (keys.shape[0] / 16 + 64) * 2.0 ** -24 + e + 2.0 ** -22 * (2 + x.abs() + 2 * exact.abs())
    assert ((lse[:, None].double() - exact).abs() <= error.amax(-1, keepdim=True)).all()
    return torch.exp(x - exact).masked_fill(hidden, 0.0), error


@pytest.mark.parametrize("dtype", DTYPES, ids=("bf16", "fp16"))
def test_rejected_drafts_leave_no_mass(cuda, dtype):
    """Prompts in chunks, then verified drafts of which some are rejected: mass and eviction of what was accepted, pages cut
    back, other tokens in the slots.  Masses are those of the accepted tokens alone, in 64 bits, and the kept slots
    those that the rule picks from the masses."""
    from ds355 import chunk_attention, eviction, pages, prefix_attention

    hq, hkv, d, block, rows, budget, capacity, decay = 8, 2, 128, 16, 2, 96, 320, 0.9
    group, scale, g = hq // hkv, d ** -0.5, gen(365)
    caches = [torch.zeros((64, block, hkv, d), dtype=dtype, device=cuda) for _ in range(2)]
    pool = pages.PagePool(caches)
    table = torch.full((rows, capacity // block), -1, dtype=torch.int32, device=cuda)
    mass = torch.zeros((rows, hkv, capacity), device=cuda)
    positions = torch.zeros((rows, hkv, capacity), dtype=torch.int32, device=cuda)
    settled, row_ids = torch.zeros((rows, 2), dtype=torch.int32, device=cuda), i32([0, 1], cuda)
    length, kept, keep = i32([0, 0], cuda), i32([0, 0], cuda), i32([budget] * rows, cuda)
    work = chunk_attention.new_chunk_workspace(rows, 256, hq, hkv, d, cuda)
    prefix_work = prefix_attention.new_prefix_workspace(rows, 256, hq, hkv, d, cuda)
    mass_work, evict_work = eviction.new_mass_workspace(cuda), eviction.new_evict_workspace(rows, hkv, capacity, cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    held = [[[] for _ in range(hkv)] for _ in range(rows)]  # by slot: [key, mass, its error] of a head
    for new, taken in [([100, 64], [100, 64]), ([37, 20], [37, 20])] + [([5, 5], t) for t in ([2, 5], [1, 1], [4, 3], [5, 1], [1, 2])]:
        total, committed = length + i32(new, cuda), length + i32(taken, cuda)
        pool.extend(table, row_ids, total)
        host_table, lens = table.cpu(), length.cpu().tolist()
        tokens = [randn((n, 2, hkv, d), dtype, g) for n in new]
        for b, n in enumerate(new):
            for i in range(n):
                slot = lens[b] + i
                for c in range(2):
                    caches[c][int(host_table[b, slot // block]), slot % block] = tokens[b][i, c].to(cuda)
        query = (randn((sum(new), hq, d), dtype, g) * 2).to(cuda)
        out, lse = torch.zeros_like(query), torch.zeros((sum(new), hq), device=cuda)
        starts = i32([0, new[0]], cuda)
        if new[0] > 5:
            chunk_attention.chunk_attention(query, *caches, out, lse, table, starts, i32(new, cuda), total, scale=scale,
                                            workspace=work, status=status)
        else:
            prefix_attention.shared_prefix_attention(query, *caches, out, lse, table, starts, i32(new, cuda), total,
                                                     i32([0], cuda), scale=scale, workspace=prefix_work, status=status)
        # The accepted tokens are the first ones of each row.
        eviction.attention_mass(query, caches[0], lse, mass, table, starts, i32(taken, cuda), committed, scale=scale,
                                previous=mass, decay=decay, workspace=mass_work, status=status)
        torch.cuda.synchronize()
        got, host_q, host_lse = mass.cpu().double(), query.cpu().double(), lse.cpu()
        at = 0
        for b, n in enumerate(new):
            for h in range(hkv):
                slots = held[b][h]
                slots += [[tokens[b][i, 0, h].double(), 0.0, 0.0] for i in range(taken[b])]
                keys, ends = torch.stack([s[0] for s in slots]), lens[b] + 1 + torch.arange(taken[b])
                sums, errors = torch.zeros(len(slots), dtype=torch.float64), torch.zeros(len(slots), dtype=torch.float64)
                for j in range(h * group, (h + 1) * group):
                    w, e = _weights(host_q[at: at + taken[b], j], host_lse[at: at + taken[b], j], keys, ends, scale)
                    sums, errors = sums + w.sum(0), errors + (w * torch.expm1(e)).sum(0)
                for t, slot in enumerate(slots):
                    slot[1] = slot[1] * decay + float(sums[t])
                    slot[2] = slot[2] + float(errors[t]) + (taken[b] * group / 8 + 64) * 2.0 ** -24 * slot[1] + 2.0 ** -23
                    assert abs(float(got[b, h, t]) - slot[1]) <= slot[2], (b, h, t)
                assert (got[b, h, len(slots):] == 0).all()  # of rejected tokens, and of none
            at += n
        case = dict(lens=committed.cpu().tolist(), keep=[budget] * rows, table=host_table, caches=[c.cpu() for c in caches],
                    mass=mass.cpu(), positions=positions.cpu(), settled=settled.cpu(), sinks=4, recent=16, block=block, hkv=hkv)
        expected = expect_evict(case)
        args = dict(key_cache=caches[0], value_cache=caches[1], mass=mass, positions=positions, settled=settled,
                    block_table=table, target_len=committed, keep_len=keep, kept_len=kept, sinks=4, recent=16,
                    ref_counts=pool.ref_counts, workspace=evict_work, status=status)
        run_evict(args)
        check_evict(case, args, expected)
        for b, n in enumerate(case["lens"]):
            if n > budget:  # which slots the rule kept, and where
                for h in range(hkv):
                    page = lambda t: (int(host_table[b, t // block]), t % block, h)  # noqa: E731
                    slot_of = {tuple(case["caches"][0][page(t)].tolist()): t for t in range(n)}
                    held[b][h] = [held[b][h][slot_of[tuple(expected["key_cache"][page(t)].tolist())]] for t in range(budget)]
        pool.free(table, row_ids, kept)
        length = kept.clone()
    # 150 tokens were accepted in the first row, and 96, which is its budget, in the second.
    assert int(pool.status.item()) == 0 and settled[:, 1].tolist() == [54, 0]


def test_a_captured_step_of_all_calls(cuda):
    """Two layers, one set of workspaces and one `reuse` for all calls: attention, mass of what is accepted, eviction and pages
    given back, replayed with changed lengths, and the same calls eagerly on a state of their own."""
    from ds355 import chunk_attention, eviction, pages, prefix_attention

    hq, hkv, d, block, rows, budget, capacity, most = 8, 2, 64, 16, 3, 64, 160, 40
    g = gen(370)

    class State:
        def __init__(self):
            zeros = lambda *s, dtype=torch.int32: torch.zeros(s, dtype=dtype, device=cuda)  # noqa: E731
            self.caches = [[zeros(40, block, hkv, d, dtype=torch.float16) for _ in range(2)] for _ in range(2)]
            self.pool = pages.PagePool([c for layer in self.caches for c in layer])
            self.table = torch.full((rows, capacity // block), -1, dtype=torch.int32, device=cuda)
            self.mass = [zeros(rows, hkv, capacity, dtype=torch.float32) for _ in range(2)]
            self.positions = [zeros(rows, hkv, capacity) for _ in range(2)]
            self.settled = [zeros(rows, 2) for _ in range(2)]
            self.length, self.kept, self.total, self.committed = (zeros(rows) for _ in range(4))
            self.start, self.new, self.taken, self.row_ids = zeros(rows), zeros(rows), zeros(rows), i32([0, 1, 2], cuda)
            self.keep, self.status, self.prefix = i32([budget] * rows, cuda), zeros(1), zeros(1)
            self.query = [zeros(most, hq, d, dtype=torch.float16) for _ in range(2)]
            self.out = [[torch.zeros_like(q) for _ in range(2)] for q in self.query]
            self.lse = [[zeros(most, hq, dtype=torch.float32) for _ in range(2)] for _ in range(2)]
            self.work = chunk_attention.new_chunk_workspace(rows, most, hq, hkv, d, cuda)
            self.prefix_work = prefix_attention.new_prefix_workspace(rows, most, hq, hkv, d, cuda)
            self.mass_work = eviction.new_mass_workspace(cuda)
            self.evict_work = eviction.new_evict_workspace(rows, hkv, capacity, cuda)
            self.reuse = {}

        def step(self):
            for i, cache in enumerate(self.caches):
                rest = dict(scale=d ** -0.5, status=self.status, reuse=self.reuse)
                chunk_attention.chunk_attention(self.query[i], *cache, self.out[i][0], self.lse[i][0], self.table, self.start,
                                                self.new, self.total, workspace=self.work, **rest)
                prefix_attention.shared_prefix_attention(self.query[i], *cache, self.out[i][1], self.lse[i][1], self.table,
                                                         self.start, self.new, self.total, self.prefix,
                                                         workspace=self.prefix_work, **rest)
            for i, cache in enumerate(self.caches):
                eviction.attention_mass(self.query[i], cache[0], self.lse[i][0], self.mass[i], self.table, self.start, self.taken,
                                        self.committed, scale=d ** -0.5, previous=self.mass[i], decay=0.9,
                                        workspace=self.mass_work, status=self.status, reuse=self.reuse)
                eviction.evict_tokens(*cache, self.mass[i], self.positions[i], self.settled[i], self.table, self.committed,
                                      self.keep, self.kept, sinks=2, recent=8, ref_counts=self.pool.ref_counts,
                                      workspace=self.evict_work, status=self.status, reuse=self.reuse)
            self.pool.free(self.table, self.row_ids, self.kept)

        def prepare(self, new, taken, queries, tokens):
            self.new.copy_(i32(new, "cpu"))
            self.taken.copy_(i32(taken, "cpu"))
            self.start.copy_(i32([sum(new[:b]) for b in range(rows)], "cpu"))
            self.length.copy_(self.kept)
            torch.add(self.length, self.new, out=self.total)
            torch.add(self.length, self.taken, out=self.committed)
            self.pool.extend(self.table, self.row_ids, self.total)
            table, length = self.table.cpu(), self.length.cpu().tolist()
            for i, layer in enumerate(self.caches):
                self.query[i][: sum(new)].copy_(queries[i])
                at = 0
                for b, n in enumerate(new):
                    for slot in range(length[b], length[b] + n):
                        for c in range(2):
                            layer[c][int(table[b, slot // block]), slot % block] = tokens[i, at, c].to(cuda)
                        at += 1
            torch.cuda.synchronize()

        def tensors(self):
            return [*sum(self.caches, []), *self.mass, *self.positions, *self.settled, self.kept, self.table, *sum(self.out, []),
                    *sum(self.lse, []), self.pool.ref_counts, self.status]

    replayed, eager = State(), State()
    warm = State()  # the calls are captured from their second time on, on a state that is thrown away
    warm.step()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    replayed.reuse = warm.reuse
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        replayed.step()
    steps = [([30, 7, 1], [30, 7, 1]), ([4, 33, 3], [4, 33, 3]), ([30, 5, 5], [30, 2, 5]), ([1, 30, 5], [1, 30, 1]),
             ([5, 5, 30], [3, 1, 30]), ([5, 1, 5], [5, 1, 2]), ([2, 5, 33], [1, 5, 33]), ([0, 4, 5], [0, 2, 5])]
    for new, taken in steps:
        n = sum(new)
        queries = [randn((n, hq, d), torch.float16, g) * 2 for _ in range(2)]
        tokens = randn((2, n, 2, hkv, d), torch.float16, g)
        for state in (replayed, eager):
            state.prepare(new, taken, queries, tokens)
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        for x, y in zip(replayed.tensors(), eager.tensors()):
            assert same(x, y)
        for i in range(2):  # the two attentions: both roundings of the output and of the weights, terms of at most 5 each
            assert (eager.out[i][0][:n].float() - eager.out[i][1][:n].float()).abs().max() < 4 * 2.0 ** -11 * 5
    assert int(eager.status.item()) == 0 and int(eager.pool.status.item()) == 0 and int(replayed.pool.status.item()) == 0
    assert int(eager.settled[0][:, 1].min()) > 0 and len(eager.reuse) >= 4

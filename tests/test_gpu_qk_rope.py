"""GPU: the norm of query and key heads with the rotation and the paged write, against 64 bits.

Bounds, with u = eps / 2 of the type: the sum of D squares is off by at most D 2^-24 relative (half
of it after the root), the division, root, products and weights by 2^-24 each, so a normed element by
delta = (D / 2 + 8) 2^-24 relative and a rotated one by (delta + 4 * 2^-24) (|a c| + |b s|); the one
rounding adds u of the result.  Below the type's smallest normal the rounding is half of its smallest
step instead (``tiny * eps / 2``).
"""

import pytest
import torch

from helpers import gen, randn

pytestmark = pytest.mark.gpu


def build(seed, *, tokens, hq, hkv, d, rot, dtype, block=16, table_dtype=torch.float32, weight_dtype=None, index=torch.int64):
    g = gen(seed)
    qkv = randn((tokens, (hq + 2 * hkv) * d), dtype, g) * 3
    rows = 500
    phase = torch.arange(rows)[:, None] * torch.arange(1, rot // 2 + 1)[None] / 37
    pages = -(-tokens // block) + 2
    return dict(
        qkv=qkv, query=qkv[:, : hq * d].unflatten(1, (hq, d)), key=qkv[:, hq * d: (hq + hkv) * d].unflatten(1, (hkv, d)),
        value=qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d)), q_weight=randn((d,), weight_dtype or dtype, g),
        k_weight=randn((d,), weight_dtype or dtype, g), positions=torch.randint(0, rows, (tokens,), generator=g).to(index),
        cos_sin=torch.cat((phase.cos(), phase.sin()), -1).to(table_dtype),
        slots=torch.randperm(pages * block, generator=g)[:tokens].to(index), pages=pages, block=block, eps=1e-6)


def expect(x, w, case, rot, neox):
    """(normed, rotated, size of the rotated terms) in 64 bits."""
    x = x.double()
    n = x / (x.square().mean(-1, keepdim=True) + case["eps"]).sqrt() * w.double()
    cs = case["cos_sin"].double()[case["positions"].long()][:, None]
    c, s = cs[..., : rot // 2], cs[..., rot // 2: rot]
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if neox else (slice(0, rot, 2), slice(1, rot, 2))
    y, size = n.clone(), n.abs()
    a, b = n[..., first], n[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first], size[..., second] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return n, y, size


def assert_close(got, want, size, d):
    got = got.cpu()
    info = torch.finfo(got.dtype)
    bound = info.eps / 2 * want.abs() + (d / 2 + 12) * 2.0 ** -24 * size + info.tiny * info.eps / 2
    excess = (got.double() - want).abs() - bound
    assert not got.isnan().any() and (not excess.numel() or float(excess.max()) <= 0), float(excess.max())


def run(case, cuda, *, rot, neox, out=True, keys=True, paged=True, normed=True, **over):
    from ds355 import qk_rope

    tokens, hq, d = case["query"].shape
    hkv = case["key"].shape[1]
    dtype = case["query"].dtype
    dev = lambda shape: torch.full(shape, 7.0, dtype=dtype, device=cuda)  # noqa: E731
    qkv = case["qkv"].to(cuda)
    args = dict(
        query=qkv[:, : hq * d].unflatten(1, (hq, d)), key=qkv[:, hq * d: (hq + hkv) * d].unflatten(1, (hkv, d)),
        q_weight=case["q_weight"].to(cuda), k_weight=case["k_weight"].to(cuda), positions=case["positions"].to(cuda),
        cos_sin_cache=case["cos_sin"].to(cuda), eps=case["eps"], rotary_dim=rot, is_neox_style=neox,
        status=torch.zeros(1, dtype=torch.int32, device=cuda))
    if out:
        args["query_out"] = dev((tokens, hq, d))
    if keys:
        args["key_out"] = dev((tokens, hkv, d))
    if normed:
        args["normed_key"] = dev((tokens, hkv, d))
    if paged:
        shape = (case["pages"], case["block"], hkv, d)
        args.update(value=qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d)), key_cache=dev(shape), value_cache=dev(shape),
                    slot_mapping=case["slots"].to(cuda))
    args.update(over)
    result = qk_rope.qk_norm_rope(**args)
    torch.cuda.synchronize()
    return args, result


def check(case, args, rot, neox, skip=()):
    tokens, hq, d = case["query"].shape
    keep = [t for t in range(tokens) if t not in skip]
    _, qy, qs = expect(case["query"], case["q_weight"], case, rot, neox)
    kn, ky, ks = expect(case["key"], case["k_weight"], case, rot, neox)
    for name, want, size in (("query_out", qy, qs), ("key_out", ky, ks), ("normed_key", kn, kn.abs())):
        if args.get(name) is not None:
            got = args[name].cpu()
            assert_close(got[keep], want[keep], size[keep], d)
            assert (got[list(skip)] == 7).all()
    if args.get("key_cache") is not None:
        slots = args["slot_mapping"].cpu().long()
        written = [t for t in keep if 0 <= int(slots[t]) < case["pages"] * case["block"]]
        at = slots[written]
        flat_k, flat_v = args["key_cache"].cpu().flatten(0, 1), args["value_cache"].cpu().flatten(0, 1)
        assert_close(flat_k[at], ky[written], ks[written], d)
        assert torch.equal(flat_v[at], case["value"][written])
        rest = torch.ones(flat_k.shape[0], dtype=torch.bool)
        rest[at] = False
        assert (flat_k[rest] == 7).all() and (flat_v[rest] == 7).all()


SHAPES = [
    dict(tokens=1, hq=32, hkv=4, d=128, rot=128),
    dict(tokens=17, hq=28, hkv=4, d=128, rot=64),
    dict(tokens=5, hq=3, hkv=1, d=64, rot=64),
    dict(tokens=33, hq=16, hkv=16, d=96, rot=96),
    dict(tokens=9, hq=8, hkv=2, d=256, rot=128),
    dict(tokens=4, hq=5, hkv=5, d=80, rot=20),   # pairs not in whole vectors
    dict(tokens=3, hq=7, hkv=2, d=6, rot=2),     # heads of a few elements
    dict(tokens=6, hq=2, hkv=1, d=250, rot=250),
    dict(tokens=3, hq=4, hkv=2, d=64, rot=0),    # the norm alone
    dict(tokens=2500, hq=12, hkv=4, d=128, rot=128),
]


@pytest.mark.parametrize("neox", (True, False), ids=("halves", "pairs"))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32), ids=("bf16", "fp16", "fp32"))
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_against_64_bits(cuda, i, dtype, neox):
    shape = SHAPES[i]
    print("qk norm rope", i, shape, dtype, neox, flush=True)
    case = build(i, dtype=dtype, table_dtype=dtype if i % 2 else torch.float32,
                 weight_dtype=torch.float32 if i % 3 == 0 else None, index=torch.int32 if i % 2 else torch.int64, **shape)
    args, result = run(case, cuda, rot=shape["rot"], neox=neox)
    assert result[0] is args["query_out"] and result[1] is args["key_out"]
    check(case, args, shape["rot"], neox)
    assert int(args["status"].item()) == 0


def test_in_place(cuda):
    case = build(40, tokens=7, hq=8, hkv=2, d=128, rot=128, dtype=torch.bfloat16)
    args, result = run(case, cuda, rot=128, neox=True, out=False, keys=False, paged=False, normed=False)
    assert result[0] is args["query"] and result[1] is args["key"]
    whole = torch.cat([t.flatten(1) for t in (args["query"], args["key"])], 1)
    base = args["query"].as_strided((7, 12 * 128), (12 * 128, 1))
    assert torch.equal(base[:, : 10 * 128], whole) and torch.equal(base[:, 10 * 128:].cpu(), case["qkv"][:, 10 * 128:])
    check(case, dict(query_out=args["query"], key_out=args["key"]), 128, True)
    # With pages and no key_out the keys go to the pages alone.
    args, result = run(case, cuda, rot=128, neox=True, out=False, keys=False)
    assert result[1] is None and torch.equal(args["key"].cpu(), case["key"])
    check(case, dict(args, query_out=args["query"]), 128, True)


@pytest.mark.parametrize("shift", (0, 1, 2))
def test_strides_and_alignment(cuda, shift):
    # Heads of a wider buffer, at addresses that are not whole vectors for shift 1 and 2; caches with
    # heads before tokens and keys and values in one buffer.
    case = build(41, tokens=5, hq=6, hkv=3, d=64, rot=32, dtype=torch.float16, block=4)
    wide = torch.zeros((5, 12, 68), dtype=torch.float16, device=cuda)
    parts = [wide[:, a:b, shift: shift + 64] for a, b in ((0, 6), (6, 9), (9, 12))]
    for p, name in zip(parts, ("query", "key", "value")):
        p.copy_(case[name])
    out = torch.full((5, 6, 70), 7.0, dtype=torch.float16, device=cuda)[:, :, shift: shift + 64]
    both = torch.full((case["pages"], 2, 3, 4, 64), 7.0, dtype=torch.float16, device=cuda)
    args, _ = run(case, cuda, rot=32, neox=True, query=parts[0], key=parts[1], value=parts[2], query_out=out,
                  key_cache=both[:, 0].transpose(1, 2), value_cache=both[:, 1].transpose(1, 2))
    check(case, args, 32, True)
    around = out.as_strided((5, 6, 70), (420, 70, 1), 0)
    assert (around[..., :shift] == 7).all() and (around[..., shift + 64:] == 7).all()


def test_padding_and_bad_tokens(cuda):
    case = build(42, tokens=6, hq=8, hkv=2, d=128, rot=128, dtype=torch.bfloat16)
    slots = case["slots"].clone()
    slots[1], slots[4] = -1, case["pages"] * case["block"] + 5
    positions = case["positions"].clone()
    positions[2], positions[3] = 500, -1
    case["positions"] = positions.clamp(0, 499)
    args, _ = run(case, cuda, rot=128, neox=True, slot_mapping=slots.to(cuda), positions=positions.to(cuda))
    check(case, args, 128, True, skip=(2, 3))
    assert int(args["status"].item()) == 3
    args, _ = run(case, cuda, rot=128, neox=True, slot_mapping=slots.to(cuda), positions=positions.to(cuda), status=None)


def test_extremes(cuda):
    # Zero heads, the largest values whose squares stay in fp32, and values that are not finite.
    case = build(43, tokens=4, hq=2, hkv=1, d=128, rot=64, dtype=torch.bfloat16)
    case["qkv"][0] = 0
    case["qkv"][1] = 1e18
    args, _ = run(case, cuda, rot=64, neox=True)
    check(case, args, 64, True)
    case["qkv"][2, 5] = float("inf")
    case["qkv"][3, 130] = float("nan")
    args, _ = run(case, cuda, rot=64, neox=True)
    got = args["query_out"].cpu()
    assert got[3, 1].isnan().all() and got[3, 0].isfinite().all() and got[2, 0, 5].isnan()
    assert got[2, 1].isfinite().all() and got[:2].isfinite().all()


def test_empty_and_reuse_and_streams(cuda):
    case = build(44, tokens=0, hq=4, hkv=2, d=64, rot=64, dtype=torch.float16)
    run(case, cuda, rot=64, neox=True)
    case = build(45, tokens=20, hq=4, hkv=2, d=64, rot=64, dtype=torch.float16)
    stream = torch.cuda.Stream()
    reuse = {}
    for _ in range(2):  # the second call takes the kept descriptor, at other addresses
        with torch.cuda.stream(stream):
            args, _ = run(case, cuda, rot=64, neox=True, reuse=reuse)
        check(case, args, 64, True)
    assert len(reuse) == 1
    args, _ = run(case, cuda, rot=32, neox=True, reuse=reuse)
    assert not torch.equal(args["query_out"].cpu(), torch.full_like(case["query"], 7.0))
    assert len(reuse) == 2


def test_from_a_graph(cuda):
    from ds355 import qk_rope

    case = build(46, tokens=20, hq=4, hkv=2, d=128, rot=128, dtype=torch.bfloat16)
    args, _ = run(case, cuda, rot=128, neox=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        qk_rope.qk_norm_rope(**args)
    for seed in (47, 48, 49):
        other = build(seed, tokens=20, hq=4, hkv=2, d=128, rot=128, dtype=torch.bfloat16)
        args["query"].copy_(other["query"])
        args["key"].copy_(other["key"])
        args["value"].copy_(other["value"])
        for k in ("q_weight", "k_weight", "positions"):
            args[k].copy_(other[k])
        args["slot_mapping"].copy_(other["slots"])
        for k in ("query_out", "key_out", "normed_key", "key_cache", "value_cache"):
            args[k].fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        check(other, args, 128, True)


@pytest.mark.parametrize("neox,dtype", ((True, torch.bfloat16), (False, torch.float16)))
def test_more_than_the_caches_hold(cuda, neox, dtype):
    # Over 32 MiB of heads: they go past the caches.
    case = build(47, tokens=3601, hq=36, hkv=2, d=128, rot=64, dtype=dtype)
    args, _ = run(case, cuda, rot=64, neox=neox)
    check(case, args, 64, neox)
    # In place, and no pages.
    args, _ = run(case, cuda, rot=64, neox=neox, out=False, keys=False, paged=False, normed=False)
    _, qy, qs = expect(case["query"], case["q_weight"], case, 64, neox)
    _, ky, ks = expect(case["key"], case["k_weight"], case, 64, neox)
    assert_close(args["query"], qy, qs, 128)
    assert_close(args["key"], ky, ks, 128)


@pytest.mark.parametrize("table", ("none", "short"))
@pytest.mark.parametrize("d,dtype", ((128, torch.bfloat16), (6, torch.float32)))
def test_the_norm_alone_needs_no_table(cuda, d, dtype, table):
    # Nothing is rotated, so no row of the table is read: positions past it are no fault.
    case = build(48, tokens=9, hq=4, hkv=2, d=d, rot=0, dtype=dtype)
    given = torch.zeros((0, 0) if table == "none" else (2, 64), device=cuda)
    positions = torch.tensor([0, 1, 2, 499, -1, 10 ** 6, 3, 4, 5], device=cuda)
    args, _ = run(case, cuda, rot=0, neox=True, cos_sin_cache=given, positions=positions)
    check(case, args, 0, True)
    assert int(args["status"].item()) == 0

"""CPU: the refusals and layouts of chunk attention, attention mass and eviction."""

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "ds355.h"
FAKE = 1 << 12  # a 4096-byte aligned address that is never dereferenced: every call fails its checks first


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
@pytest.mark.parametrize("struct,mirror", (("ds_chunk_attention_desc", "ChunkAttentionDesc"),
                                           ("ds_attention_mass_desc", "AttentionMassDesc"),
                                           ("ds_evict_desc", "EvictDesc")))
def test_descriptor_offsets_match_c_compiler(tmp_path, struct, mirror):
    from ds355 import _lib

    cls = getattr(_lib, mirror)
    names = [n for n, _ in cls._fields_]
    src = tmp_path / "layout.c"
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {",
             f'  printf("%zu\\n", sizeof({struct}));']
    lines += [f'  printf("%zu\\n", offsetof({struct}, {n}));' for n in names]
    lines += ["  return 0;", "}"]
    src.write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-O0", "-o", str(exe), str(src)], check=True)
    values = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert values[0] == ctypes.sizeof(cls)
    assert values[1:] == [getattr(cls, n).offset for n in names]
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), HEADER.read_text(), flags=re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    assert len(re.findall(r"[,;]", body)) == len(names)


def refuses(call, message):
    from ds355 import _lib

    rc = call()
    assert rc in (_lib.DS_ERR_INVALID, _lib.DS_ERR_UNSUPPORTED)
    assert message in _lib.load().ds_last_error().decode()


def chunk_desc(**over):
    from ds355 import _lib

    d = _lib.ChunkAttentionDesc()
    values = dict(dtype=_lib.DS_BF16, query=FAKE, q_row_stride=1024, q_head_stride=128, output=FAKE, o_row_stride=1024,
                  o_head_stride=128, key_cache=FAKE, k_block_stride=4096, k_token_stride=256, k_head_stride=128,
                  value_cache=FAKE, v_block_stride=4096, v_token_stride=256, v_head_stride=128, block_table=FAKE,
                  bt_stride=4, max_blocks=4, num_blocks=8, block_size=16, query_start=FAKE, query_len=FAKE,
                  target_len=FAKE, rows=2, tokens=3, num_q_heads=8, num_kv_heads=2, head_dim=128, scale=1.0,
                  workspace=FAKE, workspace_bytes=0)
    values.update(over)
    for k, v in values.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over,message", (
    (dict(dtype=2), "BF16 or FP16"), (dict(num_q_heads=7), "divisible"), (dict(head_dim=96), "64, 128 or 256"),
    (dict(rows=1025), "1024 rows"), (dict(rows=-1), "non-negative"), (dict(block_size=0), "positive"),
    (dict(num_blocks=0), "positive"), (dict(block_size=(1 << 20) + 1), "2^20"), (dict(query=None), "null"),
    (dict(window=-1), "window"), (dict(q_row_stride=1028), "multiples of 8"), (dict(v_token_stride=12), "multiples of 8"),
    (dict(k_block_stride=1 << 30), "2^30"), (dict(k_token_stride=1 << 26), "2^30"),
    (dict(key_cache=FAKE + 8), "16-byte aligned"), (dict(), "ds_chunk_attention_workspace_bytes"),
    (dict(workspace=FAKE + 16, workspace_bytes=1 << 40), "256-byte aligned"),
    (dict(tokens=(1 << 20) + 1, workspace_bytes=1 << 60), "2^20 query tokens"),
    (dict(tokens=1 << 20, num_q_heads=4096, num_kv_heads=2, workspace_bytes=1 << 60), "too many"),
))
def test_chunk_attention_refuses(over, message):
    from ds355 import _lib

    d = chunk_desc(**over)
    refuses(lambda: _lib.load().ds_chunk_attention(None, ctypes.byref(d)), message)
    assert _lib.load().ds_chunk_attention(None, None) == _lib.DS_ERR_INVALID


def test_chunk_attention_without_work_and_workspace_sizes():
    from ds355 import _lib, chunk_attention

    lib = _lib.load()
    assert lib.ds_chunk_attention(None, ctypes.byref(chunk_desc(rows=0))) == 0
    assert lib.ds_chunk_attention(None, ctypes.byref(chunk_desc(tokens=0, query=None))) == 0
    size = chunk_attention.chunk_workspace_bytes
    assert 0 < size(1, 1, 8, 2, 128) < size(64, 5000, 8, 2, 128)
    assert size(64, 1 << 20, 8, 2, 128) < 100 << 20
    for bad in ((0, 1, 8, 2, 128), (1, 0, 8, 2, 128), (1, 1, 8, 3, 128), (1, 1, 8, 2, 80)):
        assert size(*bad) == 0
    with pytest.raises(ValueError, match="workspace sizes"):
        chunk_attention.new_chunk_workspace(1, 1, 8, 2, 80, "cpu")


def chunk_args(**over):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    args = dict(query=bf(3, 8, 128), key_cache=bf(4, 16, 2, 128), value_cache=bf(4, 16, 2, 128), output=bf(3, 8, 128),
                lse=torch.zeros(3, 8), block_table=torch.zeros((2, 2), dtype=torch.int32), query_start=i32(0, 1),
                query_len=i32(1, 2), target_len=i32(9, 9), scale=1.0, workspace=torch.zeros(16, dtype=torch.uint8))
    args.update(over)
    return args


@pytest.mark.parametrize("over,message", (
    (dict(query=torch.zeros(3, 8, 64, dtype=torch.bfloat16)), "query and output"),
    (dict(value_cache=torch.zeros(4, 8, 2, 128, dtype=torch.bfloat16)), "value caches"),
    (dict(key_cache=torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16),
          value_cache=torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)), "head dimensions"),
    (dict(key_cache=torch.zeros(4, 16, 3, 128, dtype=torch.bfloat16),
          value_cache=torch.zeros(4, 16, 3, 128, dtype=torch.bfloat16)), "divisible"),
    (dict(output=torch.zeros(3, 8, 128, dtype=torch.float16)), "share a dtype"),
    (dict(output=torch.zeros(3, 128, 8, dtype=torch.bfloat16).transpose(1, 2)), "contiguous in head_dim"),
    (dict(lse=torch.zeros(3, 7)), "lse"), (dict(query_len=torch.zeros(2, dtype=torch.int64)), "int32"),
    (dict(target_len=torch.zeros(3, dtype=torch.int32)), "one entry per row"), (dict(window=0), "window"),
    (dict(batch_size=3), "batch_size"), (dict(block_table=torch.zeros((1, 4), dtype=torch.int32)), "block_table"),
    (dict(workspace=torch.zeros(16)), "workspace"), (dict(status=torch.zeros(1)), "status"), (dict(), "GPU only"),
))
def test_chunk_attention_checks_its_arguments(over, message):
    from ds355.chunk_attention import chunk_attention

    with pytest.raises(ValueError, match=message):
        chunk_attention(**chunk_args(**over), reuse={})


def mass_desc(**over):
    from ds355 import _lib

    d = _lib.AttentionMassDesc()
    values = dict(dtype=_lib.DS_BF16, query=FAKE, q_row_stride=1024, q_head_stride=128, key_cache=FAKE, k_block_stride=4096,
                  k_token_stride=256, k_head_stride=128, lse=FAKE, lse_token_stride=8, lse_head_stride=1, mass=FAKE,
                  mass_row_stride=128, mass_head_stride=64, capacity=64, block_table=FAKE, bt_stride=4, max_blocks=4,
                  num_blocks=8, block_size=16, query_start=FAKE, query_len=FAKE, target_len=FAKE, rows=2, tokens=3,
                  num_q_heads=8, num_kv_heads=2, head_dim=128, scale=1.0, decay=1.0, workspace=FAKE, workspace_bytes=0)
    values.update(over)
    for k, v in values.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over,message", (
    (dict(dtype=2), "BF16 or FP16"), (dict(num_q_heads=7), "divisible"), (dict(head_dim=96), "64, 128 or 256"),
    (dict(rows=1025), "1024 rows"), (dict(tokens=-1), "non-negative"), (dict(block_size=0), "positive"),
    (dict(capacity=0), "capacity"), (dict(window=-1), "window"), (dict(lse=None), "null"), (dict(mass=None), "null"),
    (dict(q_head_stride=4), "multiples of 8"), (dict(k_block_stride=1 << 30), "2^30"),
    (dict(query=FAKE + 2), "16-byte aligned"), (dict(), "ds_attention_mass_workspace_bytes"),
    (dict(workspace=FAKE + 16, workspace_bytes=1 << 40), "256-byte aligned"),
    (dict(max_blocks=1 << 30, capacity=1 << 30, workspace_bytes=1 << 60), "2^29"),
    (dict(tokens=(1 << 20) + 1, workspace_bytes=1 << 60), "2^20 query tokens"),
    (dict(max_blocks=1 << 25, capacity=1 << 29, rows=1024, workspace_bytes=1 << 60), "too many"),
))
def test_attention_mass_refuses(over, message):
    from ds355 import _lib

    d = mass_desc(**over)
    refuses(lambda: _lib.load().ds_attention_mass(None, ctypes.byref(d)), message)
    assert _lib.load().ds_attention_mass(None, None) == _lib.DS_ERR_INVALID
    assert _lib.load().ds_attention_mass(None, ctypes.byref(mass_desc(rows=0))) == 0


def mass_args(**over):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    args = dict(query=bf(3, 8, 128), key_cache=bf(4, 16, 2, 128), lse=torch.zeros(3, 8), mass=torch.zeros(2, 2, 32),
                block_table=torch.zeros((2, 2), dtype=torch.int32), query_start=i32(0, 1), query_len=i32(1, 2),
                target_len=i32(9, 9), scale=1.0, workspace=torch.zeros(16, dtype=torch.uint8))
    args.update(over)
    return args


@pytest.mark.parametrize("over,message", (
    (dict(query=torch.zeros(3, 8, 64, dtype=torch.bfloat16)), "head dimensions"),
    (dict(query=torch.zeros(3, 8, dtype=torch.bfloat16)), "query must be"),
    (dict(key_cache=torch.zeros(4, 16, 3, 128, dtype=torch.bfloat16)), "divisible"),
    (dict(key_cache=torch.zeros(4, 16, 2, 128, dtype=torch.float16)), "share a dtype"), (dict(lse=torch.zeros(3, 7)), "lse"),
    (dict(lse=torch.zeros(3, 8, dtype=torch.float64)), "lse"), (dict(mass=torch.zeros(2, 3, 32)), "mass"),
    (dict(mass=torch.zeros(1, 2, 32)), "mass"), (dict(mass=torch.zeros(2, 2, 32, dtype=torch.float16)), "mass"),
    (dict(mass=torch.zeros(2, 1, 32).expand(2, 2, 32)), "overlap"), (dict(previous=torch.zeros(2, 2, 31)), "capacity"),
    (dict(query_start=torch.zeros(2)), "int32"), (dict(target_len=torch.zeros(3, dtype=torch.int32)), "one entry per row"),
    (dict(window=0), "window"), (dict(batch_size=-1), "batch_size"), (dict(workspace=torch.zeros(16)), "workspace"),
    (dict(status=torch.zeros(1)), "status"), (dict(), "GPU only"),
))
def test_attention_mass_checks_its_arguments(over, message):
    from ds355.eviction import attention_mass

    with pytest.raises(ValueError, match=message):
        attention_mass(**mass_args(**over), reuse={})


def evict_desc(**over):
    from ds355 import _lib

    d = _lib.EvictDesc()
    values = dict(dtype=_lib.DS_BF16, key_cache=FAKE, k_block_stride=4096, k_token_stride=256, k_head_stride=128,
                  value_cache=FAKE, v_block_stride=4096, v_token_stride=256, v_head_stride=128, mass=FAKE,
                  mass_row_stride=128, mass_head_stride=64, positions=FAKE, positions_row_stride=128,
                  positions_head_stride=64, capacity=64, settled=FAKE, block_table=FAKE, bt_stride=4, max_blocks=4,
                  num_blocks=8, block_size=16, target_len=FAKE, keep_len=2 * FAKE, kept_len=3 * FAKE, rows=2,
                  num_kv_heads=2, head_dim=128, workspace=FAKE, workspace_bytes=0)
    values.update(over)
    for k, v in values.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over,message", (
    (dict(dtype=7), "BF16, FP16 or FP32"), (dict(rows=-1), "non-negative"), (dict(num_kv_heads=0), "positive"),
    (dict(head_dim=4), "16 bytes"), (dict(rows=1025), "1024 rows"), (dict(block_size=0), "positive"),
    (dict(capacity=0), "capacity"), (dict(sinks=-1), "sinks"), (dict(recent=-1), "recent"),
    (dict(sinks=1 << 29, recent=1), "always kept"), (dict(settled=None), "null"), (dict(kept_len=FAKE), "memory of its own"),
    (dict(kept_len=2 * FAKE), "memory of its own"), (dict(v_head_stride=4), "16 bytes"),
    (dict(value_cache=FAKE + 8), "16-byte aligned"), (dict(max_blocks=1 << 30, capacity=1 << 30), "2^29"),
    (dict(rows=1024, num_kv_heads=64), "65535"), (dict(), "ds_evict_workspace_bytes"),
    (dict(workspace=FAKE + 16, workspace_bytes=1 << 40), "256-byte aligned"),
))
def test_evict_refuses(over, message):
    from ds355 import _lib

    d = evict_desc(**over)
    refuses(lambda: _lib.load().ds_evict(None, ctypes.byref(d)), message)
    assert _lib.load().ds_evict(None, None) == _lib.DS_ERR_INVALID
    assert _lib.load().ds_evict(None, ctypes.byref(evict_desc(rows=0))) == 0


def test_eviction_workspace_sizes():
    from ds355 import eviction

    assert eviction.mass_workspace_bytes() > 0
    assert 0 < eviction.evict_workspace_bytes(1, 1, 1) < eviction.evict_workspace_bytes(4, 8, 32768)
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        assert eviction.evict_workspace_bytes(*bad) == 0
    with pytest.raises(ValueError, match="workspace sizes"):
        eviction.new_evict_workspace(1, 1, 0, "cpu")


def evict_args(**over):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    args = dict(key_cache=bf(4, 16, 2, 128), value_cache=bf(4, 16, 2, 128), mass=torch.zeros(2, 2, 32),
                positions=torch.zeros((2, 2, 32), dtype=torch.int32), settled=torch.zeros((2, 2), dtype=torch.int32),
                block_table=torch.zeros((2, 2), dtype=torch.int32), target_len=i32(9, 9), keep_len=i32(5, 5),
                kept_len=i32(0, 0), workspace=torch.zeros(16, dtype=torch.uint8))
    args.update(over)
    return args


@pytest.mark.parametrize("over,message", (
    (dict(value_cache=torch.zeros(4, 8, 2, 128, dtype=torch.bfloat16)), "value caches"),
    (dict(value_cache=torch.zeros(4, 16, 2, 128, dtype=torch.float16)), "share a dtype"),
    (dict(key_cache=torch.zeros(4, 16, 128, 2, dtype=torch.bfloat16).transpose(2, 3)), "contiguous in head_dim"),
    (dict(sinks=-1), "negative"), (dict(recent=-1), "negative"), (dict(mass=torch.zeros(2, 2)), "mass"),
    (dict(positions=torch.zeros(2, 2, 32)), "positions"), (dict(positions=torch.zeros((2, 2, 31), dtype=torch.int32)), "capacity"),
    (dict(settled=torch.zeros((2, 1), dtype=torch.int32)), "settled"), (dict(keep_len=torch.zeros(2)), "keep_len"),
    (dict(kept_len=torch.zeros(1, dtype=torch.int32)), "one entry per row"),
    (dict(ref_counts=torch.zeros(3, dtype=torch.int32)), "ref_counts"), (dict(batch_size=3), "batch_size"),
    (dict(block_table=torch.zeros((1, 4), dtype=torch.int32)), "block_table"), (dict(workspace=torch.zeros(16)), "workspace"),
    (dict(status=torch.zeros(1)), "status"), (dict(), "GPU only"),
))
def test_evict_tokens_checks_its_arguments(over, message):
    from ds355.eviction import evict_tokens

    with pytest.raises(ValueError, match=message):
        evict_tokens(**evict_args(**over), reuse={})


@pytest.mark.parametrize("name", ("target_len", "keep_len"))
@pytest.mark.parametrize("words", (-1, 1))
def test_evict_refuses_a_new_length_that_overlaps_an_old_one(name, words):
    from ds355 import _lib

    d = evict_desc(**{name: 3 * FAKE + 4 * words})
    refuses(lambda: _lib.load().ds_evict(None, ctypes.byref(d)), "memory of its own")
    d = evict_desc(**{name: 3 * FAKE + 8 * words})  # the two rows' words are apart
    refuses(lambda: _lib.load().ds_evict(None, ctypes.byref(d)), "ds_evict_workspace_bytes")


@pytest.mark.parametrize("over,message", (
    (dict(num_q_heads=1 << 17, num_kv_heads=1), "query heads for a KV head"),
    (dict(q_row_stride=1 << 29), "strides"), (dict(lse_token_stride=-8), "strides"), (dict(lse_head_stride=1 << 29), "strides"),
    (dict(num_q_heads=1 << 16, num_kv_heads=1, tokens=1 << 14, q_head_stride=8, q_row_stride=8), "too many"),
))
def test_attention_mass_refuses_places_past_32_bits(over, message):
    from ds355 import _lib

    d = mass_desc(workspace_bytes=1 << 60, **over)
    refuses(lambda: _lib.load().ds_attention_mass(None, ctypes.byref(d)), message)


OVERLAPPING = (((2, 2), (32, 32)), ((2, 3), (32, 63)), ((3, 2), (63, 32)), ((2, 4), (64, 32)), ((4, 2), (32, 96)),
               ((3, 3), (40, 70)))
APART = (((2, 2), (64, 32)), ((2, 2), (32, 64)), ((2, 3), (32, 70)), ((1, 3), (0, 32)), ((3, 1), (40, 7)), ((2, 2), (96, 64)))


@pytest.mark.parametrize("name", ("mass", "positions"))
@pytest.mark.parametrize("shape,strides", OVERLAPPING + APART)
def test_rows_and_heads_that_overlap_are_refused(name, shape, strides):
    # 32 slots each: rows and heads nested either way, equal strides, or the last of one inside the first of another.
    from ds355.eviction import attention_mass, evict_tokens

    rows, heads = shape
    places = sorted(strides[0] * b + strides[1] * h for b in range(rows) for h in range(heads))
    assert all(y - x >= 32 for x, y in zip(places, places[1:])) == ((shape, strides) in APART)
    lens = {k: torch.zeros(rows, dtype=torch.int32) for k in ("target_len", "keep_len", "kept_len")}
    tensors = dict(mass=torch.zeros(rows, heads, 32), positions=torch.zeros((rows, heads, 32), dtype=torch.int32))
    tensors[name] = torch.zeros(1000, dtype=tensors[name].dtype).as_strided((rows, heads, 32), (*strides, 1))
    cache = torch.zeros(4, 16, heads, 128, dtype=torch.bfloat16)
    table = torch.zeros((rows, 2), dtype=torch.int32)
    message = "GPU only" if (shape, strides) in APART else f"{name}'s rows and heads overlap"
    with pytest.raises(ValueError, match=message):
        evict_tokens(**evict_args(key_cache=cache, value_cache=cache, settled=torch.zeros((rows, 2), dtype=torch.int32),
                                  block_table=table, **lens, **tensors))
    if name == "mass":
        with pytest.raises(ValueError, match=message):
            attention_mass(**mass_args(query=torch.zeros(3, heads, 128, dtype=torch.bfloat16), key_cache=cache,
                                       lse=torch.zeros(3, heads), mass=tensors["mass"], block_table=table,
                                       query_start=lens["target_len"], query_len=lens["target_len"],
                                       target_len=lens["target_len"]))


@pytest.mark.parametrize("block_size", ((1 << 30) + 1, (1 << 31) - 1))
def test_evict_refuses_pages_whose_count_passes_32_bits(block_size):
    # A row's slots plus a page size past 2^31 made no pages of the row, and none of its page ids was checked.
    from ds355 import _lib

    d = evict_desc(block_size=block_size, max_blocks=1, workspace_bytes=1 << 40)
    d.workspace = FAKE + 16  # refused before a launch in any case
    refuses(lambda: _lib.load().ds_evict(None, ctypes.byref(d)), "2^30 tokens per page")


def test_sizes_past_32_bits_reach_the_library_as_its_largest(monkeypatch):
    # The descriptors' fields are 32-bit; 2^32 + 5 used to become 5.
    from ds355 import chunk_attention, eviction

    much, most = (1 << 32) + 5, (1 << 31) - 1
    meta = dict(device="meta")
    descs = []
    for module, name in ((chunk_attention, "_launch"), (eviction, "_launch_mass"), (eviction, "_launch_evict")):
        monkeypatch.setattr(module, name, lambda desc, *_: descs.append(desc))
    monkeypatch.setattr(chunk_attention._lib, "require_gpu", lambda *_: torch.device("cpu"))
    cache = torch.zeros((1, 16, 2, 128), dtype=torch.bfloat16, **meta).expand(much, 16, 2, 128)
    table = torch.zeros((2, much), dtype=torch.int32, **meta)
    chunk_attention.chunk_attention(**chunk_args(key_cache=cache, value_cache=cache, block_table=table))
    mass, positions = (torch.zeros((2, 2, much), dtype=t, **meta) for t in (torch.float32, torch.int32))
    eviction.attention_mass(**mass_args(key_cache=cache, block_table=table, mass=mass))
    eviction.evict_tokens(**evict_args(key_cache=cache, value_cache=cache, block_table=table, mass=mass, positions=positions),
                          sinks=much, recent=much)
    for desc in descs:
        assert (desc.num_blocks, desc.max_blocks) == (most, most)
    assert len(descs) == 3 and descs[1].capacity == descs[2].capacity == descs[2].sinks == descs[2].recent == most


def test_workspaces_are_sized_for_the_device_they_are_on(monkeypatch):
    # Both sizes follow the compute units of the device that is current while they are worked out.
    import contextlib

    from ds355 import chunk_attention, eviction

    current, asked = [None], []

    @contextlib.contextmanager
    def on_device(device):
        current.append(device)
        yield
        current.pop()

    monkeypatch.setattr(chunk_attention._lib, "on_device", on_device)
    monkeypatch.setattr(chunk_attention, "chunk_workspace_bytes", lambda *_: asked.append(current[-1]) or 256)
    monkeypatch.setattr(eviction, "mass_workspace_bytes", lambda: asked.append(current[-1]) or 256)
    assert chunk_attention.new_chunk_workspace(1, 1, 8, 2, 128, "cpu").numel() == 256
    assert eviction.new_mass_workspace("cpu").numel() == 256
    assert asked == [torch.device("cpu")] * 2

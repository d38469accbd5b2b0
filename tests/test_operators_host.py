"""CPU: the refusals and layouts of the shared-prefix attention, the query/key norm and the page pool."""

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "ds355.h"


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
@pytest.mark.parametrize("struct,mirror", (("ds_prefix_attention_desc", "PrefixAttentionDesc"),
                                           ("ds_qk_norm_rope_desc", "QkNormRopeDesc")))
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
    return rc


FAKE = 1 << 12  # a 4096-byte aligned address that is never dereferenced: every call fails its checks first


def prefix_desc(**over):
    from ds355 import _lib

    d = _lib.PrefixAttentionDesc()
    values = dict(dtype=_lib.DS_BF16, query=FAKE, q_row_stride=1024, q_head_stride=128, output=FAKE, o_row_stride=1024,
                  o_head_stride=128, key_cache=FAKE, k_block_stride=4096, k_token_stride=256, k_head_stride=128,
                  value_cache=FAKE, v_block_stride=4096, v_token_stride=256, v_head_stride=128, block_table=FAKE,
                  bt_stride=4, max_blocks=4, num_blocks=8, block_size=16, query_start=FAKE, query_len=FAKE,
                  target_len=FAKE, prefix_len=FAKE, rows=2, tokens=3, num_q_heads=8, num_kv_heads=2, head_dim=128,
                  scale=1.0, workspace=FAKE, workspace_bytes=0)
    values.update(over)
    for k, v in values.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over,message", (
    (dict(dtype=2), "BF16 or FP16"), (dict(num_q_heads=7), "divisible"), (dict(head_dim=96), "64, 128 or 256"),
    (dict(rows=1025), "1024 rows"), (dict(rows=-1), "non-negative"), (dict(block_size=0), "positive"),
    (dict(num_blocks=0), "positive"), (dict(block_size=(1 << 20) + 1), "2^20"), (dict(query=None), "null"),
    (dict(prefix_len=None), "null"), (dict(q_row_stride=1028), "multiples of 8"), (dict(v_token_stride=12), "multiples of 8"),
    (dict(key_cache=FAKE + 8), "16-byte aligned"), (dict(), "ds_prefix_attention_workspace_bytes"),
    (dict(workspace=FAKE + 16, workspace_bytes=1 << 30), "256-byte aligned"),
    (dict(tokens=(1 << 20) + 1, workspace_bytes=1 << 60), "2^20 query tokens"),
    (dict(tokens=1 << 20, max_blocks=1 << 26, workspace_bytes=1 << 60), "too many"),
))
def test_prefix_attention_refuses(over, message):
    from ds355 import _lib

    d = prefix_desc(**over)
    refuses(lambda: _lib.load().ds_prefix_attention(None, ctypes.byref(d)), message)
    assert _lib.load().ds_prefix_attention(None, None) == _lib.DS_ERR_INVALID


def test_prefix_attention_without_work_and_workspace_sizes():
    from ds355 import _lib, prefix_attention

    lib = _lib.load()
    assert lib.ds_prefix_attention(None, ctypes.byref(prefix_desc(rows=0))) == 0
    assert lib.ds_prefix_attention(None, ctypes.byref(prefix_desc(tokens=0, query=None))) == 0
    size = prefix_attention.prefix_workspace_bytes
    assert 0 < size(1, 1, 8, 2, 128) < size(64, 1, 8, 2, 128) < size(64, 5000, 8, 2, 128)
    for bad in ((0, 1, 8, 2, 128), (1, 0, 8, 2, 128), (1, 1, 8, 3, 128), (1, 1, 8, 2, 80)):
        assert size(*bad) == 0
    with pytest.raises(ValueError, match="workspace sizes"):
        prefix_attention.new_prefix_workspace(1, 1, 8, 2, 80, "cpu")


def prefix_args(**over):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    args = dict(query=bf(3, 8, 128), key_cache=bf(4, 16, 2, 128), value_cache=bf(4, 16, 2, 128), output=bf(3, 8, 128),
                lse=torch.zeros(3, 8), block_table=torch.zeros((2, 2), dtype=torch.int32), query_start=i32(0, 1),
                query_len=i32(1, 2), target_len=i32(9, 9), prefix_len=i32(4), scale=1.0,
                workspace=torch.zeros(16, dtype=torch.uint8))
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
    (dict(target_len=torch.zeros(3, dtype=torch.int32)), "one entry per row"),
    (dict(prefix_len=torch.zeros(2, dtype=torch.int32)), "one in all"), (dict(batch_size=3), "batch_size"),
    (dict(block_table=torch.zeros((1, 4), dtype=torch.int32)), "block_table"),
    (dict(workspace=torch.zeros(16)), "workspace"), (dict(status=torch.zeros(1)), "status"), (dict(), "GPU only"),
))
def test_shared_prefix_attention_refuses(over, message):
    from ds355.prefix_attention import shared_prefix_attention

    with pytest.raises(ValueError, match=message):
        shared_prefix_attention(**prefix_args(**over), reuse={})


def qk_desc(**over):
    from ds355 import _lib

    d = _lib.QkNormRopeDesc()
    values = dict(dtype=_lib.DS_BF16, weight_dtype=_lib.DS_BF16, cos_sin_dtype=_lib.DS_FP32, query=FAKE, q_row_stride=1024,
                  q_head_stride=128, key=FAKE, k_row_stride=256, k_head_stride=128, q_weight=FAKE, k_weight=FAKE,
                  positions=FAKE, cos_sin=FAKE, cs_stride=128, cs_rows=10, query_out=FAKE, qo_row_stride=1024,
                  qo_head_stride=128, tokens=2, num_q_heads=8, num_kv_heads=2, head_dim=128, rotary_dim=128, eps=1e-6)
    values.update(over)
    for k, v in values.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over,message", (
    (dict(dtype=9), "BF16, FP16 or FP32"), (dict(weight_dtype=1), "weights"), (dict(cos_sin_dtype=1), "cos/sin"),
    (dict(num_kv_heads=0), "positive"), (dict(head_dim=129), "even"), (dict(head_dim=258), "at most 256"),
    (dict(rotary_dim=130), "rotary_dim"), (dict(rotary_dim=63), "rotary_dim"), (dict(cs_stride=64), "rows must hold"),
    (dict(key_cache=FAKE), "together"), (dict(key_cache=FAKE, value_cache=FAKE, slot_mapping=FAKE), "together"),
    (dict(key_cache=FAKE, value_cache=FAKE, slot_mapping=FAKE, value=FAKE), "page sizes"),
    (dict(positions=None), "null"), (dict(query_out=None), "null"), (dict(cos_sin=None), "null"),
    (dict(tokens=-1), "positive"),
))
def test_qk_norm_rope_refuses(over, message):
    from ds355 import _lib

    d = qk_desc(**over)
    refuses(lambda: _lib.load().ds_qk_norm_rope(None, ctypes.byref(d)), message)


def qk_args(**over):
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    args = dict(query=bf(2, 8, 64), key=bf(2, 2, 64), q_weight=bf(64), k_weight=bf(64),
                positions=torch.zeros(2, dtype=torch.int64), cos_sin_cache=torch.zeros(10, 64), eps=1e-6, rotary_dim=64,
                is_neox_style=True)
    args.update(over)
    return args


BF = dict(dtype=torch.bfloat16)


@pytest.mark.parametrize("over,message", (
    (dict(query=torch.zeros(2, 512, **BF)), "tokens, heads"), (dict(key=torch.zeros(3, 2, 64, **BF)), "key must be"),
    (dict(query_out=torch.zeros(2, 8, 32, **BF)), "query_out"), (dict(normed_key=torch.zeros(2, 3, 64, **BF)), "normed_key"),
    (dict(key_out=torch.zeros(2, 2, 64)), "share a dtype"), (dict(value=torch.zeros(2, 2, 64, **BF)), "together"),
    (dict(q_weight=torch.zeros(32, **BF)), "q_weight"), (dict(k_weight=torch.zeros(64)), "weights must both"),
    (dict(cos_sin_cache=torch.zeros(10, 64, dtype=torch.float16)), "cos/sin"), (dict(rotary_dim=66), "rotary_dim"),
    (dict(cos_sin_cache=torch.zeros(10, 62)), "cos/sin"), (dict(positions=torch.zeros(2)), "positions"),
    (dict(value=torch.zeros(2, 2, 64, **BF), key_cache=torch.zeros(4, 16, 3, 64, **BF),
          value_cache=torch.zeros(4, 16, 3, 64, **BF), slot_mapping=torch.zeros(2, dtype=torch.int32)), "kv_heads"),
    (dict(value=torch.zeros(2, 2, 64, **BF), key_cache=torch.zeros(4, 16, 2, 64, **BF),
          value_cache=torch.zeros(4, 16, 2, 64, **BF), slot_mapping=torch.zeros(3, dtype=torch.int32)), "slot_mapping"),
    (dict(status=torch.zeros(1)), "status"), (dict(), "GPU only"),
))
def test_qk_rope_refuses(over, message):
    from ds355.qk_rope import qk_norm_rope

    with pytest.raises(ValueError, match=message):
        qk_norm_rope(**qk_args(**over), reuse={})


def test_page_entry_points_refuse():
    from ds355 import _lib

    lib = _lib.load()
    lst = [None, FAKE, 2, 4096, 100]
    table = [FAKE, FAKE, 8, 4, 8]
    work = [FAKE, 1 << 30]
    copy = lambda *a: refuses(lambda: lib.ds_pages_copy(*a), "")  # noqa: E731
    copy(None, None, 2, 4096, 100, FAKE, FAKE, 3, None)
    copy(None, FAKE, 2, 4096, 0, FAKE, FAKE, 3, None)
    copy(*lst, None, FAKE, 3, None)
    copy(*lst, FAKE, FAKE, -1, None)
    copy(None, FAKE, 2, 1 << 31, 100, FAKE, FAKE, 3, None)
    fork = lambda lst, table, lists, work, m: refuses(  # noqa: E731
        lambda: lib.ds_pages_fork(*lst, *table, *lists, *work, None), m)
    fork(lst, table, [FAKE, FAKE, FAKE, 4097, 16], work, "4096 rows")
    fork(lst, [FAKE, FAKE, 8, 4097, 8], [FAKE, FAKE, FAKE, 2, 16], work, "4096 block table rows")
    fork(lst, [FAKE, FAKE, 7, 4, 8], [FAKE, FAKE, FAKE, 2, 16], work, "overlap")
    fork(lst, [None, FAKE, 8, 4, 8], [FAKE, FAKE, FAKE, 2, 16], work, "null")
    fork(lst, table, [FAKE, None, FAKE, 2, 16], work, "null row list")
    fork(lst, table, [FAKE, FAKE, FAKE, 2, 0], work, "positive")
    fork(lst, table, [FAKE, FAKE, FAKE, 2, 16], [FAKE, 16], "workspace")
    assert lib.ds_pages_fork(*lst, *table, None, None, None, 0, 16, *work, None) == 0
    refuses(lambda: lib.ds_pages_extend(None, 100, *table, FAKE, None, 2, 16, None), "null row list")
    refuses(lambda: lib.ds_pages_extend(None, 0, *table, FAKE, FAKE, 2, 16, None), "positive")
    refuses(lambda: lib.ds_pages_free(None, 100, *table, None, None, 2, 16, None), "null row list")
    refuses(lambda: lib.ds_pages_free(None, 100, *table, FAKE, None, 2, -1, None), "positive")
    refuses(lambda: lib.ds_pages_compact(*lst, *table, None, *work, None), "null page map")
    refuses(lambda: lib.ds_pages_compact(*lst, *table, FAKE, None, 0, None), "workspace")
    assert lib.ds_pages_workspace_bytes(0) == 0 < lib.ds_pages_workspace_bytes(1) <= lib.ds_pages_workspace_bytes(10000)


def test_page_pool_refuses():
    from ds355.pages import PagePool

    with pytest.raises(ValueError, match="at least one"):
        PagePool([])
    with pytest.raises(ValueError, match="share"):
        PagePool([torch.zeros(4, 16, 8), torch.zeros(4, 8, 8)])
    with pytest.raises(ValueError, match="contiguous"):
        PagePool([torch.zeros(4, 8, 16).transpose(1, 2)])
    with pytest.raises(ValueError, match="overlap"):
        PagePool([torch.zeros(4, 16, 8)[:1].expand(4, 16, 8)])
    with pytest.raises(ValueError, match="positive"):
        PagePool([torch.zeros(0, 16, 8)])
    with pytest.raises(ValueError, match="GPU only"):
        PagePool([torch.zeros(4, 16, 8)])


class FakePool:
    """A pool whose device is the CPU, for the checks that come before any launch."""

    def __new__(cls):
        from ds355.pages import PagePool

        pool = object.__new__(PagePool)
        pool.device, pool.num_pages, pool.block_size = torch.device("cpu"), 10, 16
        pool.ref_counts = torch.zeros(10, dtype=torch.int32)
        return pool


def test_page_pool_calls_refuse():
    from ds355 import _lib

    pool, table = FakePool(), torch.full((4, 3), -1, dtype=torch.int32)
    for call, message in (
        (lambda: pool.copy([1, 2], [3]), "one entry per row"), (lambda: pool.copy([1, 2], [3, 3]), "distinct"),
        (lambda: pool.copy([1, 2], [2, 5]), "also a source"), (lambda: pool.copy([1], [10]), "between zero"),
        (lambda: pool.copy([-1], [1]), "between zero"), (lambda: pool.copy(torch.zeros(1), [1]), "int32"),
        (lambda: pool.fork(table, [0, 1], [2, 2], [1, 1]), "distinct"), (lambda: pool.fork(table, [0, 2], [1, 0], [1, 1]), "also a parent"),
        (lambda: pool.fork(table, [0], [1], [49]), "lens"), (lambda: pool.fork(table, [4], [1], [1]), "parents"),
        (lambda: pool.fork(table.long(), [0], [1], [1]), "block_table"), (lambda: pool.extend(table, [0, 0], [1, 1]), "distinct"),
        (lambda: pool.extend(table, [0], [1, 2]), "one entry per row"), (lambda: pool.extend(table, [0], [49]), "lens"),
        (lambda: pool.extend(table.t(), [0], [1]), "block_table"), (lambda: pool.free(table, [5]), "rows"),
        (lambda: pool.free(table, [1], [-1]), "keep_lens"), (lambda: pool.compact(table[0]), "block_table"),
    ):
        with pytest.raises(ValueError, match=message):
            call()
    with pytest.raises(_lib.UnsupportedShapeError, match="4096"):
        pool.compact(torch.zeros((4097, 1), dtype=torch.int32))


def test_page_entry_points_refuse_what_32_bits_do_not_count():
    from ds355 import _lib

    lib = _lib.load()
    lst, table, work = [None, FAKE, 2, 4096, 100], [FAKE, FAKE, 8, 4, 8], [FAKE, 1 << 62]
    many = (1 << 31) - (1 << 14)  # pages: the scans of the counts look ahead of the last one
    refuses(lambda: lib.ds_pages_copy(None, FAKE, 2, 4096, many, FAKE, FAKE, 3, None), "2^14 - 1 pages")
    refuses(lambda: lib.ds_pages_extend(None, many, *table, FAKE, FAKE, 2, 16, None), "2^14 - 1 pages")
    refuses(lambda: lib.ds_pages_free(None, many, *table, FAKE, None, 2, 16, None), "2^14 - 1 pages")
    refuses(lambda: lib.ds_pages_compact(None, FAKE, 2, 4096, many, *table, FAKE, *work, None), "2^14 - 1 pages")
    # Rows of 2^20 entries: 2048 of them may need 2^31 pages in one call.
    wide = [FAKE, FAKE, 1 << 20, 2048, 1 << 20]
    refuses(lambda: lib.ds_pages_extend(None, 100, *wide, FAKE, FAKE, 2, 16, None), "block table entries")
    refuses(lambda: lib.ds_pages_fork(*lst, *wide, FAKE, FAKE, FAKE, 2, 16, *work, None), "block table entries")
    # 65536 caches whose largest page has 2^18 pieces.
    refuses(lambda: lib.ds_pages_copy(None, FAKE, 65536, 1 << 30, 100, FAKE, FAKE, 3, None), "2^43")

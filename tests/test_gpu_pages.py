"""GPU: page pools (copy, fork, extend, free, compact) against a model of the pool on the host; all exact."""

import random

import pytest
import torch

from helpers import gen

pytestmark = pytest.mark.gpu


class Model:
    """The pool's rules, one entry after another, on the host."""

    def __init__(self, pages, rows, width, block):
        self.refs, self.table, self.block = [0] * pages, [[-1] * width for _ in range(rows)], block
        self.content = list(range(pages))  # what each page holds: the page it was first
        self.width = width

    def held(self, row):
        return [p for p in self.table[row] if p >= 0]

    def free_pages(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def release(self, row, first=0):
        for c in range(first, self.width):
            if self.table[row][c] >= 0:
                self.refs[self.table[row][c]] -= 1
                self.table[row][c] = -1

    def fork(self, parents, children, lens):
        ok = []
        for i, (p, c, n) in enumerate(zip(parents, children, lens)):
            rows = len(self.table)
            fine = 0 <= p < rows and 0 <= c < rows and p != c and n >= 0 and c not in children[:i] and c not in parents
            fine = fine and -(-n // self.block) <= min(self.width, len(self.held(p)) if 0 <= p < rows else 0)
            ok.append(fine)
        for c, fine in zip(children, ok):
            if fine:
                self.release(c)
        free, copies = self.free_pages(), []
        for p, c, n, fine in zip(parents, children, lens, ok):
            if not fine:
                continue
            full = n // self.block
            if n % self.block:
                if not free:
                    continue
                page = free.pop(0)
                self.refs[page], self.table[c][full] = 1, page
                copies.append((self.table[p][full], page))
            for k in range(full):
                self.table[c][k] = self.table[p][k]
                self.refs[self.table[p][k]] += 1
        for s, d in copies:
            self.content[d] = self.content[s]
        return (0 if all(ok) else 1)

    def extend(self, rows, lens):
        free, status = self.free_pages(), 0
        for i, (row, n) in enumerate(zip(rows, lens)):
            pages = -(-n // self.block) if n >= 0 else 0
            if not 0 <= row < len(self.table) or n < 0 or pages > self.width or row in rows[:i]:
                status |= 1
                continue
            have = len(self.held(row))
            if pages - have > len(free):
                return status | 2
            for c in range(have, pages):
                page = free.pop(0)
                self.refs[page], self.table[row][c] = 1, page
        return status

    def free(self, rows, keep=None):
        for i, row in enumerate(rows):
            self.release(row, -(-keep[i] // self.block) if keep else 0)

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r]
        moves = dict(zip([p for p in live if p >= len(live)], [p for p in range(len(live)) if not self.refs[p]]))
        page_map = [moves.get(p, p) if self.refs[p] else -1 for p in range(len(self.refs))]
        for s, d in moves.items():
            self.refs[d], self.refs[s], self.content[d] = self.refs[s], 0, self.content[s]
        self.table = [[moves.get(p, p) for p in row] for row in self.table]
        return page_map


class Pool:
    """A pool on the GPU beside its model."""

    def __init__(self, cuda, *, pages, rows, width, block, shapes=None, seed=0):
        from ds355.pages import PagePool

        g = gen(seed)
        shapes = shapes or [((2, 64), torch.bfloat16), ((3,), torch.float16), ((1, 5), torch.int8)]
        self.before = [torch.randint(-100, 100, (pages, block, *s), generator=g).to(t) for s, t in shapes]
        self.caches = [c.to(cuda) for c in self.before]
        self.model = Model(pages, rows, width, block)
        self.table = torch.full((rows, width + 3), -1, dtype=torch.int32, device=cuda)[:, :width]
        self.pool = PagePool(self.caches)
        self.cuda = cuda

    def i32(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.cuda)

    def check(self, status=0):
        torch.cuda.synchronize()
        assert self.table.cpu().tolist() == self.model.table
        assert self.pool.ref_counts.cpu().tolist() == self.model.refs
        for now, before in zip(self.caches, self.before):
            assert torch.equal(now.cpu(), before[self.model.content])
        assert int(self.pool.status.item()) == status
        self.pool.status.zero_()
        assert int(self.pool._workspace[:4].view(torch.int32).item()) == 0  # the counter between launches


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("block,pages,rows,width", ((16, 300, 12, 20), (1, 100, 5, 30), (7, 5000, 40, 100)))
def test_a_run_of_calls(cuda, seed, block, pages, rows, width):
    r = random.Random(1000 * seed + block)
    p = Pool(cuda, pages=pages, rows=rows, width=width, block=block, seed=seed)
    most = min(width, pages // rows) * block
    for step in range(25):
        kind = r.choice(("extend", "extend", "fork", "fork", "free", "compact"))
        some = r.sample(range(rows), r.randint(1, rows))
        print("pages", seed, step, kind, flush=True)
        if kind == "extend":
            lens = [r.randint(0, most) for _ in some]
            want = p.model.extend(some, lens)
            if step % 2:
                p.pool.extend(p.table, some, lens)
            else:
                p.pool.extend(p.table, p.i32(some), p.i32(lens))
            p.check(want)
        elif kind == "fork":
            parents = some[: max(1, len(some) // 3)]
            children = some[len(parents):]
            parents = [r.choice(parents) for _ in children]
            lens = [r.randint(0, len(p.model.held(x)) * block) for x in parents]
            free = len(p.model.free_pages())
            if free < len(children):
                continue
            assert p.model.fork(parents, children, lens) == 0
            p.pool.fork(p.table, p.i32(parents), p.i32(children), p.i32(lens))
            p.check()
        elif kind == "free":
            keep = [r.randint(0, most) for _ in some] if r.random() < 0.7 else None
            p.model.free(some, keep)
            p.pool.free(p.table, p.i32(some), None if keep is None else p.i32(keep))
            p.check()
        else:
            page_map = p.model.compact()
            assert p.pool.compact(p.table).cpu().tolist() == page_map
            p.check()


def test_fork_shares_and_copies(cuda):
    p = Pool(cuda, pages=40, rows=6, width=8, block=4)
    p.pool.extend(p.table, [0, 1], [13, 8])
    p.model.extend([0, 1], [13, 8])
    p.check()
    # Whole pages only, a partial page, no token at all, the parent's whole length.
    args = ([0, 0, 1, 0], [2, 3, 4, 5], [8, 6, 0, 13])
    assert p.model.fork(*args) == 0
    p.pool.fork(p.table, *args)
    p.check()
    assert p.model.held(4) == [] and p.model.refs[p.model.table[0][0]] == 4
    # The children again, from one of them: their pages come back first.
    args = ([3, 3], [2, 5], [6, 3])
    assert p.model.fork(*args) == 0
    p.pool.fork(p.table, *args)
    p.check()


def test_entries_that_are_left_out(cuda):
    p = Pool(cuda, pages=40, rows=6, width=5, block=4)
    p.model.extend([0, 1, 5], [18, 7, 9])
    p.pool.extend(p.table, [0, 1, 5], [18, 7, 9])
    p.check()
    for args in (([0, 0], [2, 2], [5, 9]),           # a child twice: the first counts
                 ([0, 1, 2], [2, 3, 4], [5, 3, 0]),  # a child that is a parent
                 ([0], [0], [4]), ([-1, 0], [3, 4], [2, 2]), ([9], [3], [2]), ([0], [6], [2]), ([0], [-2], [2]),
                 ([0, 1], [3, 4], [21, 1]),          # longer than the table
                 ([1, 0], [3, 4], [9, 5]),           # longer than the parent
                 ([0], [5], [-1]), ([0], [5], [19])):
        want = p.model.fork(*args)
        p.pool.fork(p.table, *(p.i32(x) for x in args))
        p.check(want)
    for args in (([0, 1, 1], [4, 9, 17]), ([2, 9], [5, 5]), ([-1, 3], [5, 5]), ([4, 3], [21, 6]), ([4], [-3])):
        want = p.model.extend(*args)
        assert want == 1
        p.pool.extend(p.table, *(p.i32(x) for x in args))
        p.check(want)
    # Freeing: rows out of range are left out, a row named twice gives its pages back once.
    p.pool.free(p.table, p.i32([0, 6, -1, 0]), p.i32([9, 0, 0, 5]))
    p.model.free([0], [5])
    p.check(1)
    p.pool.free(p.table, p.i32([1, 1, 1]))
    p.model.free([1])
    p.check()


def test_running_out_of_pages(cuda):
    p = Pool(cuda, pages=9, rows=6, width=5, block=4)
    p.model.extend([0, 1], [18, 7])
    p.pool.extend(p.table, [0, 1], [18, 7])
    p.check()  # 7 held, 2 free
    want = p.model.extend([2, 3, 4], [4, 12, 1])
    assert want == 2 and p.model.held(2) and not p.model.held(3)
    p.pool.extend(p.table, [2, 3, 4], [4, 12, 1])
    p.check(2)
    # One page free, three children want one: the first gets it, one with whole pages needs none.
    p.model.fork([0, 0, 0, 0], [3, 4, 5, 2], [5, 6, 8, 7])
    p.pool.fork(p.table, [0, 0, 0, 0], [3, 4, 5, 2], [5, 6, 8, 7])
    p.check(0 if p.model.held(4) and p.model.held(2) else 2)
    p.model.extend([1], [20])
    p.pool.extend(p.table, [1], [20])
    p.check(2)


def test_pages_out_of_the_pool_and_double_frees(cuda):
    p = Pool(cuda, pages=12, rows=3, width=4, block=4)
    p.pool.extend(p.table, [0, 1], [9, 5])
    p.model.extend([0, 1], [9, 5])
    p.check()
    p.table[2, 0] = 50  # no page of the pool
    p.table[2, 1] = 11  # a free page
    p.pool.free(p.table, [2])
    p.check(4)
    p.pool.copy(p.i32([0, 12, 3]), p.i32([8, 9, -1]))
    p.model.content[8] = p.model.content[0]
    p.check(4)


@pytest.mark.parametrize("device_lists", (False, True))
def test_copy(cuda, device_lists):
    p = Pool(cuda, pages=700, rows=1, width=1, block=16,
             shapes=[((8, 128), torch.bfloat16), ((8, 128), torch.bfloat16), ((65,), torch.float32), ((3,), torch.int8)])
    r = random.Random(3)
    picked = r.sample(range(700), 640)
    src, dst = picked[:320], picked[320:]
    src[7] = src[8]  # one source for two
    dst[9] = src[9]  # a page onto itself
    p.pool.copy(*((p.i32(src), p.i32(dst)) if device_lists else (src, dst)))
    for s, d in zip(src, dst):
        p.model.content[d] = p.model.content[s]
    p.check()
    p.pool.copy([], [])
    p.check()


def test_strided_caches(cuda):
    # Keys and values of one buffer: pages of a tensor lie a buffer page apart.
    from ds355.pages import PagePool

    both = torch.randn((30, 2, 16, 2, 64), generator=gen(4)).to(torch.bfloat16).to(cuda)
    before = both.clone()
    pool = PagePool([both[:, 0], both[:, 1]])
    pool.copy([3, 4], [10, 20])
    before[[10, 20]] = before[[3, 4]]
    assert torch.equal(both, before)


def test_large_pool_takes_the_lowest_pages(cuda):
    pages = 70001
    p = Pool(cuda, pages=pages, rows=8, width=9000, block=2, shapes=[((1,), torch.int8)])
    r = random.Random(5)
    refs = [1 if r.random() < 0.9 else 0 for _ in range(pages)]
    refs[-1] = 0
    p.pool.ref_counts.copy_(p.i32(refs))
    p.model.refs = refs
    free = refs.count(0)
    lens = [2 * (free // 4), 1, 0, 2 * (free // 4) + 1]
    assert p.model.extend([3, 1, 0, 7], lens) == 0
    p.pool.extend(p.table, [3, 1, 0, 7], lens)
    p.check()
    p.model.free([3])
    p.pool.free(p.table, [3])
    p.check()
    left = len(p.model.free_pages())
    want = p.model.extend([2, 5], [2 * (left - 1), 4])
    assert want == 2
    p.pool.extend(p.table, [2, 5], [2 * (left - 1), 4])
    p.check(2)
    p.model.compact()
    p.pool.compact(p.table)
    p.check()


def test_from_a_graph(cuda):
    # A verification cycle's bookkeeping as one graph: cut back, grow, fork; replayed with other lengths.
    p = Pool(cuda, pages=400, rows=8, width=16, block=4)
    rows, keep, lens = p.i32([0, 1, 2, 3]), p.i32([0] * 4), p.i32([0] * 4)
    parents, children, flens = p.i32([0, 1, 1]), p.i32([5, 6, 7]), p.i32([0] * 3)

    def cycle():
        p.pool.free(p.table, rows, keep)
        p.pool.extend(p.table, rows, lens)
        p.pool.fork(p.table, parents, children, flens)

    cycle()
    p.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        cycle()
    r = random.Random(6)
    for _ in range(5):
        k = [r.randint(0, 40) for _ in range(4)]
        n = [r.randint(1, 60) for _ in range(4)]
        p.model.free([0, 1, 2, 3], k)
        assert p.model.extend([0, 1, 2, 3], n) == 0
        f = [r.randint(0, 4 * len(p.model.held(x))) for x in (0, 1, 1)]
        assert p.model.fork([0, 1, 1], [5, 6, 7], f) == 0
        for t, v in ((keep, k), (lens, n), (flens, f)):
            t.copy_(p.i32(v))
        graph.replay()
        p.check()


def test_adopted_counts_and_empty_lists(cuda):
    from ds355.pages import PagePool

    cache = torch.zeros((6, 4, 8), dtype=torch.float16, device=cuda)
    refs = torch.tensor([1, 0, 2, 0, 0, 1], dtype=torch.int32, device=cuda)
    pool = PagePool([cache], ref_counts=refs)
    table = torch.tensor([[0, 2, -1], [2, 5, -1]], dtype=torch.int32, device=cuda)
    pool.extend(table, [], [])
    pool.free(table, [])
    pool.fork(table, [], [], [])
    assert pool.compact(table).tolist() == [0, -1, 2, -1, -1, 1]
    assert table.tolist() == [[0, 2, -1], [2, 1, -1]] and refs.tolist() == [1, 1, 2, 0, 0, 0]
    assert pool.ref_counts is refs


def test_forking_again_keeps_what_is_shared_and_may_run_out(cuda):
    p = Pool(cuda, pages=8, rows=5, width=6, block=4)
    p.model.extend([0], [18])
    p.pool.extend(p.table, [0], [18])
    for args in (([0, 0], [1, 2], [17, 10]),  # pages 5 and 6
                 ([0, 0], [1, 2], [16, 17]),  # row 1 whole pages only, row 2 two pages more
                 ([0, 0], [2, 1], [5, 18])):
        assert p.model.fork(*args) == 0
        p.pool.fork(p.table, *args)
        p.check()
    p.model.extend([3], [4])
    p.pool.extend(p.table, [3], [4])
    p.check()
    # No page is left but those that the children give back: row 4 takes the first, row 1 the second, row 2
    # none, and stays empty though it shared entries before.
    args = ([0, 0, 0], [4, 1, 2], [9, 18, 7])
    assert p.model.fork(*args) == 0 and p.model.held(2) == [] and len(p.model.held(1)) == 5
    p.pool.fork(p.table, *args)
    p.check(2)


def test_a_new_pool_serves_any_stream(cuda):
    # The pool's own buffers are filled on the stream it is made on; the first call may be on another.
    from ds355.pages import PagePool

    cache = torch.zeros((200, 4, 8), dtype=torch.float16, device=cuda)
    table = torch.full((9, 20), -1, dtype=torch.int32, device=cuda)
    lists = [torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0], [70], [0] * 8, list(range(1, 9)), [70] * 8)]
    dirty = [torch.full((1 << 15,), 255, dtype=torch.uint8, device=cuda) for _ in range(16)]
    torch.cuda.synchronize()
    del dirty
    made, used = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(made):
        pool = PagePool([cache])
        assert made.query()
    with torch.cuda.stream(used):
        pool.extend(table, *lists[:2])
        pool.fork(table, *lists[2:])
    used.synchronize()
    assert int(pool.status.item()) == 0 and pool.ref_counts.tolist() == [9] * 17 + [1] * 9 + [0] * 174
    assert table[:, :17].tolist() == [list(range(17))] * 9 and table[:, 17].tolist() == list(range(17, 26))

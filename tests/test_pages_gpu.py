"""Appending to a paged cache and handling its pages, on the GPU, against a plain model on the host (whole numbers and
moved values: equal)."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

f16, bf16, i32 = torch.float16, torch.bfloat16, torch.int32


@pytest.fixture(scope="module")
def P(built_libs, cuda_device):
    from triton_ext_b200 import paged
    return paged


class Model:
    """The record of pages as Python lists, and the pools on the CPU."""

    def __init__(self, cache):
        self.page = cache.page_size
        self.width = cache.table.shape[1]
        self.rows = [[p for p in r if p >= 0] for r in cache.table.tolist()]
        self.lens, self.refs = cache.lens.tolist(), cache.refs.tolist()
        self.k, self.v = cache.k.cpu().clone(), cache.v.cpu().clone()

    def same_as(self, cache):
        table = [r + [-1] * (self.width - len(r)) for r in self.rows]
        assert cache.table.tolist() == table
        assert cache.lens.tolist() == self.lens
        assert cache.refs.tolist() == self.refs
        assert torch.equal(cache.k.cpu().view(torch.int16), self.k.view(torch.int16))
        assert torch.equal(cache.v.cpu().view(torch.int16), self.v.view(torch.int16))

    def free(self, rows):
        for r in rows:
            for p in self.rows[r]:
                self.refs[p] -= 1
            self.rows[r], self.lens[r] = [], 0

    def fork(self, dst, src):
        old, old_lens = [list(r) for r in self.rows], list(self.lens)
        last = {d: s for d, s in zip(dst, src)}
        for d, s in last.items():
            for p in old[s]:
                self.refs[p] += 1
            for p in old[d]:
                self.refs[p] -= 1
            self.rows[d], self.lens[d] = list(old[s]), old_lens[s]

    def reserve(self, rows, counts):
        free = [p for p, r in enumerate(self.refs) if r == 0]   # as they are before the call
        for r, n in zip(rows, counts):
            if n == 0:
                continue
            if self.lens[r] % self.page:
                p = self.rows[r][-1]
                if self.refs[p] > 1:
                    new = free.pop(0)
                    self.k[:, new], self.v[:, new] = self.k[:, p], self.v[:, p]
                    self.refs[p] -= 1
                    self.refs[new] = 1
                    self.rows[r][-1] = new
            self.lens[r] += n
            while len(self.rows[r]) * self.page < self.lens[r]:
                new = free.pop(0)
                self.refs[new] = 1
                self.rows[r].append(new)

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        holes = [p for p in range(used) if self.refs[p] == 0]
        movers = [p for p in range(used, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.k[:, b], self.v[:, b] = self.k[:, a], self.v[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.rows = [[to.get(p, p) for p in r] for r in self.rows]


def make(P, pages=40, page=16, heads=2, d=64, rows=10, width=9, layers=2, dtype=bf16, seed=0):
    cache = P.PagedCache.create(pages, page, heads, d, rows=rows, width=width, layers=layers, dtype=dtype)
    g = torch.Generator().manual_seed(seed)
    for x in (cache.k, cache.v):
        x.copy_(torch.randn(x.shape, generator=g).to(dtype))
    return cache, Model(cache)


def ints(*x):
    return torch.tensor(x, dtype=i32, device="cuda")


@pytest.mark.parametrize("page,heads,d,layers,dtype", [(16, 2, 64, 2, bf16), (32, 1, 16, 1, f16), (128, 3, 128, 3, bf16)])
def test_a_history_of_calls(P, page, heads, d, layers, dtype):
    cache, model = make(P, pages=61, page=page, heads=heads, d=d, rows=12, width=11, layers=layers, dtype=dtype)
    rng = random.Random(5)
    for step in range(60):
        what = rng.choice(["reserve", "reserve", "fork", "free", "compact"])
        rows = rng.sample(range(12), rng.randint(1, 12))
        if what == "reserve":
            room = 61 - sum(r > 0 for r in model.refs) - len(rows)
            counts, keep = [], []
            for r in rows:
                n = rng.choice([0, 1, 1, page - 1, page, page + 1, 3 * page])
                n = max(0, min(n, model.width * page - model.lens[r]))
                need = -(-(model.lens[r] + n) // page) - len(model.rows[r])
                if need <= room:
                    room -= need
                    keep.append(r)
                    counts.append(n)
            if not keep:
                continue
            cache.reserve(ints(*keep), ints(*counts))
            model.reserve(keep, counts)
        elif what == "fork":
            src = [rng.randrange(12) for _ in rows]
            cache.fork(ints(*rows), ints(*src))
            model.fork(rows, src)
        elif what == "free":
            cache.free(ints(*rows[:4]))
            model.free(rows[:4])
        else:
            cache.compact()
            model.compact()
        model.same_as(cache)
    P.check()


def test_shared_last_pages(P):
    cache, model = make(P)
    for do in (lambda c, t: c.reserve(t(0), t(20)), lambda c, t: c.fork(t(1, 2, 3), t(0, 0, 0)),
               lambda c, t: c.reserve(t(2, 0, 1, 3), t(1, 1, 1, 1)),         # all four holders: the last keeps the page
               lambda c, t: c.fork(t(4, 5), t(3, 3)),
               lambda c, t: c.reserve(t(4), t(13)),                           # others hold it still: copied, and 1 new page
               lambda c, t: c.reserve(t(5, 3), t(0, 12)),                     # no tokens: nothing is copied for row 5
               lambda c, t: c.fork(t(0, 1, 2, 3), t(3, 2, 1, 0)),             # a reordering
               lambda c, t: c.fork(t(6, 6, 6), t(0, 1, 2)),                   # listed three times: the last holds
               lambda c, t: c.fork(t(6), t(6)),
               lambda c, t: c.free(t(1, 1, 2)), lambda c, t: c.compact()):
        do(cache, ints)
        do(model, lambda *x: list(x))
        model.same_as(cache)
    P.check()


def test_truncate(P):
    """Whole and part pages, shared ones, to nothing, to more than there is, a row twice; then the rows grow again."""
    from triton_ext_b200 import backend as B
    cache, model = make(P)

    def cut(rows, keep):
        for r, n in zip(rows, keep):
            while len(model.rows[r]) * model.page >= max(n, 0) + model.page:
                model.refs[model.rows[r].pop()] -= 1
            model.lens[r] = min(model.lens[r], n)
        cache.truncate(ints(*rows), ints(*keep))

    cache.reserve(ints(0, 1, 2), ints(100, 5, 64))
    model.reserve([0, 1, 2], [100, 5, 64])
    cache.fork(ints(3, 4, 5), ints(0, 0, 2))
    model.fork([3, 4, 5], [0, 0, 2])
    for rows, keep in (([0, 1], [97, 5]), ([2, 3], [49, 32]), ([4, 4, 4], [70, 33, 50]), ([5, 1, 0], [0, 9, 2 ** 31 - 1]), ([], [])):
        cut(rows, keep)
        model.same_as(cache)
        P.check()
    grow = [3, 2, 4, 0, 5, 1], [20, 1, 16, 1, 3, 40]                    # row 4 ends inside a page that row 0 holds
    cache.reserve(ints(*grow[0]), ints(*grow[1]))
    model.reserve(*grow)
    model.same_as(cache)
    for rows, keep, text in ((ints(10, -1, 0), ints(1, 1, 60), "outside the table"), (ints(1, 2), ints(-1, 50), "below zero")):
        cache.truncate(rows, keep)
        with pytest.raises(B.DotError, match=text):
            P.check()
    for r, n in ((0, 60), (2, 50)):
        while len(model.rows[r]) * model.page >= n + model.page:
            model.refs[model.rows[r].pop()] -= 1
        model.lens[r] = n
    model.same_as(cache)
    with pytest.raises(B.DotError, match="keep must be an int32 vector of 2"):
        cache.truncate(ints(1, 2), ints(1))


def test_many_pages_and_rows(P):
    """More pages than one step of the planning block (16384) looks at, a list longer than the block, and a full cache."""
    cache, model = make(P, pages=40000, page=16, heads=1, d=16, rows=2000, width=20, layers=1)
    rng = random.Random(6)
    rows = list(range(2000))
    rng.shuffle(rows)
    counts = [rng.randint(0, 300) for _ in rows]
    for do in (lambda c, t: c.reserve(t(*rows), t(*counts)), lambda c, t: c.free(t(*rows[::3])), lambda c, t: c.compact(),
               lambda c, t: c.reserve(t(*rows[::3]), t(*([320] * len(rows[::3])))),
               lambda c, t: c.fork(t(*rows[1::3]), t(*rows[::3][: len(rows[1::3])])), lambda c, t: c.compact()):
        do(cache, ints)
        do(model, lambda *x: list(x))
    model.same_as(cache)
    left = sum(r == 0 for r in model.refs)
    assert left > 4
    P.check()


def test_what_cannot_be_done_changes_nothing_and_is_reported(P):
    from triton_ext_b200 import backend as B
    cache, model = make(P, pages=6, rows=4, width=4)
    cache.reserve(ints(0, 1), ints(33, 5))
    model.reserve([0, 1], [33, 5])
    for rows, counts, text in ((ints(2), ints(16 * 3), "no free pages"), (ints(1, 1), ints(1, 1), "listed twice"),
                               (ints(0), ints(32), "width"), (ints(4), ints(1), "outside the table"),
                               (ints(2, -1), ints(1, 1), "outside the table"), (ints(2), ints(-1), "negative count"),
                               (ints(2), ints(2 ** 31 - 1), "width")):
        cache.reserve(rows, counts)
        with pytest.raises(B.DotError, match=text):
            P.check()
        P.check()                                       # reported once
        model.same_as(cache)
    cache.free(ints(9, 1))                              # the bad row is passed over
    model.free([1])
    cache.fork(ints(2, -3, 3), ints(0, 0, 7))
    model.fork([2], [0])
    with pytest.raises(B.DotError, match="outside the table"):
        P.check()
    model.same_as(cache)


def test_copy_pages(P):
    cache, model = make(P, pages=2500, page=16, heads=1, d=16, rows=2, width=4, layers=2)
    src, dst = list(range(0, 1200)), list(range(2400, 1200, -1))       # more pairs than one launch carries
    cache.copy_pages(src, dst)
    for a, b in zip(src, dst):
        model.k[:, b], model.v[:, b] = model.k[:, a], model.v[:, a]
    model.same_as(cache)
    cache.copy_pages([7, 7], [1, 2])                                    # one source, two destinations
    for b in (1, 2):
        model.k[:, b], model.v[:, b] = model.k[:, 7], model.v[:, 7]
    model.same_as(cache)
    cache.copy_pages([], [])
    from triton_ext_b200 import backend as B
    for a, b in (([1], [1]), ([1, 2], [3, 3]), ([1, 2], [2, 3]), ([2500], [0]), ([0], [-1]), ([0, 1], [2])):
        with pytest.raises(B.DotError):
            cache.copy_pages(a, b)
    model.same_as(cache)


def test_pages_in_a_graph(P):
    cache, model = make(P, pages=64, rows=6, width=12)
    rows, counts = ints(*range(6)), ints(5, 6, 7, 1, 2, 3)
    cache.reserve(rows, counts)
    model.reserve(range(6), counts.tolist())
    src = ints(1, 1, 0, 5, 4, 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.fork(rows, src)
        cache.reserve(rows, counts)
    for s in ([1, 1, 0, 5, 4, 4], [0, 1, 2, 3, 4, 5], [5, 5, 5, 5, 5, 5]):
        src.copy_(ints(*s))
        graph.replay()
        model.fork(range(6), s)
        model.reserve(range(6), counts.tolist())
        model.same_as(cache)
    P.check()


# ---- append --------------------------------------------------------------------------------------------------------------
def batch_of(q_lens, kv_lens, page, seed, spare=2):
    used = [-(-n // page) for n in kv_lens]
    pages, width = sum(used) + spare, max(max(used), 1) + 1
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = [], 0
    for n in used:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return pages, torch.tensor(table, dtype=i32, device="cuda"), ints(*kv_lens)


APPENDS = [
    # q lengths, kv lengths, q heads, kv heads, d, page, dtype, rotary_dim (0: none), interleaved
    ([1], [1], 2, 1, 64, 16, bf16, 64, False),
    ([1] * 40, list(range(1, 41)), 8, 2, 128, 16, bf16, 128, False),
    ([3, 0, 17, 1], [3, 9, 40, 33], 6, 3, 64, 32, f16, 32, True),
    ([300, 5], [300, 517], 4, 4, 256, 128, bf16, 0, False),
    ([70], [200], 2, 2, 16, 64, f16, 16, False),
    ([9, 9], [9, 30], 5, 1, 32, 256, bf16, 6, True),
]


@pytest.mark.parametrize("q_lens,kv_lens,h,hk,d,page,dtype,rd,inter", APPENDS)
@pytest.mark.parametrize("heads_first", [False, True])
def test_append(P, q_lens, kv_lens, h, hk, d, page, dtype, rd, inter, heads_first):
    from test_rotary_gpu import close, turned64
    from triton_ext_b200.rotary import Rope
    rope = Rope(rd, interleaved=inter) if rd else None
    pages, table, kv = batch_of(q_lens, kv_lens, page, 3)
    total, behind = sum(q_lens), 2 if max(q_lens) > 1 else 0
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(total + behind, h + 2 * hk, d, generator=g).to(dtype).cuda()
    q, k, v = qkv.split([h, hk, hk], dim=1)
    shape = (pages, hk, page, d) if heads_first else (pages, page, hk, d)
    pools = [torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(2)]
    views = [x.transpose(1, 2) if heads_first else x for x in pools]
    want = [x.clone() for x in views]
    cu = torch.tensor([0] + q_lens).cumsum(0).to(i32).cuda() if max(q_lens) > 1 else None
    out = torch.full((total + behind, h, d), 7.0, dtype=dtype, device="cuda")
    got = P.append(q, k, v, views[0], views[1], table, kv, rope=rope, cu_q=cu, out=out)
    P.check()
    assert got is out
    pos = torch.cat([torch.arange(m - n, m) for n, m in zip(q_lens, kv_lens)]).cuda()
    row = torch.cat([torch.full((n,), i) for i, n in enumerate(q_lens)]).cuda()
    page_of, slot = table[row, pos // page].long(), pos % page
    assert bool((out[total:] == 7.0).all())
    if rope is None:
        assert torch.equal(out[:total], q[:total])
        want[0][page_of, slot] = k[:total]
    else:
        tq, size = turned64(q[:total].transpose(0, 1)[None], pos, rope)
        close(out[:total], tq[0].transpose(0, 1), size[0].transpose(0, 1))
        tk, size = turned64(k[:total].transpose(0, 1)[None], pos, rope)
        written = views[0][page_of, slot]
        close(written, tk[0].transpose(0, 1), size[0].transpose(0, 1))
        want[0][page_of, slot] = written
    want[1][page_of, slot] = v[:total]
    assert torch.equal(views[0], want[0]) and torch.equal(views[1], want[1])   # and nothing else was written
    # without q, and in place
    P.append(None, k, v, views[0], views[1], table, kv, rope=rope, cu_q=cu)
    assert torch.equal(views[0], want[0])
    again = P.append(q, k, v, views[0], views[1], table, kv, rope=rope, cu_q=cu, out=q)
    assert again.data_ptr() == q.data_ptr() and torch.equal(q[:total], out[:total])


def test_append_of_overlapping_windows(P):
    """q rows that are windows of one vector, a column apart: empty_like lays such a tensor out with its columns not contiguous."""
    from triton_ext_b200.rotary import Rope
    q = torch.randn(200, device="cuda").bfloat16().unfold(0, 64, 1)[:10][None].transpose(0, 1)       # [10, 1, 64]
    pages, table, kv = batch_of([1] * 10, [3] * 10, 16, 7)
    pools = [torch.zeros(pages, 16, 1, 64, dtype=bf16, device="cuda") for _ in range(2)]
    got = P.append(q, q, q, *pools, table, kv, rope=Rope(64))
    want = P.append(q.clone(memory_format=torch.contiguous_format), q, q, *pools, table, kv, rope=Rope(64))
    P.check()
    assert torch.equal(got, want)


def test_append_with_bad_pages_and_lengths(P):
    """Entries outside the cache, positions past the table and lengths below the new tokens write nothing and are reported."""
    from triton_ext_b200 import backend as B
    pools = [torch.zeros(4, 16, 1, 64, dtype=bf16, device="cuda") for _ in range(2)]
    x = torch.ones(3, 1, 64, dtype=bf16, device="cuda")
    for table, lens, cu, text in (([[4], [-1], [2]], [1, 1, 1], None, "outside the cache"), ([[0], [1], [2]], [1, 17, 1], None, "width"),
                                  ([[0]], [2], [0, 3], "length below zero or below")):
        for p in pools:
            p.zero_()
        cu = ints(*cu) if cu else None
        P.append(None, x, x, *pools, torch.tensor(table, dtype=i32, device="cuda"), ints(*lens), cu_q=cu)
        with pytest.raises(B.DotError, match=text):
            P.check()
        good = {"outside the cache": [(2, 0)], "width": [(0, 0), (2, 0)], "length below zero or below": [(0, 0), (0, 1)]}[text]
        want = torch.zeros_like(pools[0])
        for page, slot in good:
            want[page, slot] = 1
        assert torch.equal(pools[0], want) and torch.equal(pools[1], want)

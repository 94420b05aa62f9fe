"""Steps over a paged cache in which something goes wrong: what must not be touched, and what `check` has to report."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

bf16, i32 = torch.bfloat16, torch.int32


@pytest.fixture(scope="module")
def P(built_libs, cuda_device):
    from triton_ext_b200 import paged
    return paged


def ints(*x):
    return torch.tensor(x, dtype=i32, device="cuda")


def everything(cache):
    """The cache's state as whole numbers (pools hold NaN)."""
    return [x.clone().view(torch.int16 if x.dtype == bf16 else i32) for x in (cache.k, cache.v, cache.table, cache.lens, cache.refs)]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


# ---- a reserve that cannot be done ---------------------------------------------------------------------------------------
DRAFTS = 3


def short_of_pages(P, page=16):
    """Rows 0 and 1 share their 20 tokens, row 2 holds every other page: no row can grow into a new page."""
    cache = P.PagedCache.create(6, page, 2, 64, rows=4, width=6, layers=2)
    cache.k.fill_(math.nan)
    cache.v.fill_(math.nan)
    lens = cache.reserve(ints(0), ints(20))
    g = torch.Generator().manual_seed(40)
    k, v = (torch.randn(20, 2, 64, generator=g).to(bf16).cuda() for _ in range(2))
    for layer in range(2):
        P.append(None, k, v, cache.k[layer], cache.v[layer], cache.table[:1], lens, cu_q=ints(0, 20))
    cache.fork(ints(1), ints(0))
    assert cache.reserve(ints(2), ints(64)).tolist() == [64]
    P.check()
    assert cache.refs.tolist() == [2, 2, 1, 1, 1, 1] and lens.tolist() == [20]
    return cache


def one_step(P, cache, rows, counts, kept, q, k, v, cu, causal=True):
    lens = cache.reserve(rows, counts)
    table, out = cache.table[rows.clamp(0, 3).long()], []
    for layer in range(2):
        P.append(None, k, v, cache.k[layer], cache.v[layer], table, lens, cu_q=cu)
        out.append(P.paged_attention(q, cache.k[layer], cache.v[layer], table, lens, 0.125, cu_q=cu, max_q=DRAFTS, causal=causal, return_m=True))
    cache.truncate(rows, lens - counts + kept)
    return lens, out


def step_tensors(tokens):
    g = torch.Generator().manual_seed(41)
    return [torch.randn(tokens, n, 64, generator=g).to(bf16).cuda() for n in (4, 2, 2)]


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("causal", [True, False])
def test_a_refused_reserve_stops_its_step(P, captured, causal):
    """No free page for a copy of the shared last page: reserve, append, attention and truncate leave pools, table, lengths and
    counts as they were, the sibling's tokens among them. With room made the same step goes through."""
    from triton_ext_b200 import backend as B
    cache = short_of_pages(P)
    rows, counts, kept, cu = ints(0), ints(DRAFTS), ints(1), ints(0, DRAFTS)
    q, k, v = step_tensors(DRAFTS)
    before = everything(cache)
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lens, out = one_step(P, cache, rows, counts, kept, q, k, v, cu, causal)
    for _ in range(2):
        if captured:
            graph.replay()
        else:
            lens, out = one_step(P, cache, rows, counts, kept, q, k, v, cu, causal)
        with pytest.raises(B.DotError, match="no free pages"):
            P.check()
        assert lens.tolist() == [-(1 << 30)]
        assert same(everything(cache), before)
        for o, m in out:
            assert bool((o == 0).all()) and bool((m == -math.inf).all())
    cache.free(ints(2))
    if captured:
        graph.replay()
    else:
        lens, out = one_step(P, cache, rows, counts, kept, q, k, v, cu, causal)
    P.check()
    assert lens.tolist() == [20 + DRAFTS] and cache.lens.tolist() == [21, 20, 0, 0]
    copied = int(cache.table[0, 1])
    assert cache.table[1, :2].tolist() == [0, 1] and copied == 2 and cache.refs.tolist() == [2, 1, 1, 0, 0, 0]
    for pool, old, new in ((cache.k, before[0], k), (cache.v, before[1], v)):
        assert torch.equal(pool.view(torch.int16)[:, :2], old[:, :2])                       # what row 1 sees
        assert torch.equal(pool.view(torch.int16)[:, copied, :4], old[:, 1, :4])
        assert torch.equal(pool[:, copied, 4:4 + DRAFTS], new[None].expand(2, -1, -1, -1))
    assert all(bool((o != 0).any()) and bool(m.isfinite().all()) for o, m in out)


@pytest.mark.parametrize("rows,counts,text", [((0, 3), (3, 90), "no free pages"), ((3, 0), (3, 96), "width"), ((0, 0), (3, 3), "listed twice"),
                                             ((3, 9), (3, 3), "outside the table"), ((3, 1), (3, -3), "negative count")])
def test_one_row_that_has_no_room_stops_the_batch(P, rows, counts, text):
    """Whatever row of a batch cannot be served, none of its rows are touched by the step."""
    from triton_ext_b200 import backend as B
    cache = short_of_pages(P)
    cache.free(ints(2))
    before = everything(cache)
    q, k, v = step_tensors(2 * DRAFTS)
    lens, out = one_step(P, cache, ints(*rows), ints(*counts), ints(1, 1), q, k, v, ints(0, DRAFTS, 2 * DRAFTS))
    with pytest.raises(B.DotError, match=text):
        P.check()
    assert lens.tolist() == [-(1 << 30)] * 2 and same(everything(cache), before)
    assert all(bool((o == 0).all()) for o, m in out)


def test_the_lengths_of_a_step(P):
    """Row by row of the list, rows that do not grow and an empty list among them; more rows than the planning block has threads."""
    cache = P.PagedCache.create(4000, 16, 1, 16, rows=3000, width=4)
    g = torch.Generator().manual_seed(42)
    rows = torch.randperm(3000, generator=g).to(i32).cuda()
    first, more = (torch.randint(0, 7, (3000,), generator=g).to(i32).cuda() for _ in range(2))
    assert torch.equal(cache.reserve(rows, first), first)
    assert torch.equal(cache.reserve(rows[:1500], more[:1500]), (first + more)[:1500])
    assert torch.equal(cache.lens[rows.long()][1500:], first[1500:])
    assert cache.reserve(rows[:0], more[:0]).shape == (0,)
    P.check()


# ---- what check reports ------------------------------------------------------------------------------------------------
def small_cache():
    g = torch.Generator().manual_seed(43)
    return [torch.randn(8, 16, 2, 64, generator=g).to(bf16).cuda() for _ in range(2)]


@pytest.mark.parametrize("q", [1, 100])
def test_a_wait_that_runs_out_is_reported_with_what_was_found_before(P, q, monkeypatch):
    """A page outside the cache is pending when the attention's wait runs out: both are in the report, as a time-out."""
    from triton_ext_b200 import backend as B
    pools = small_cache()
    x = torch.ones(1, 2, 64, dtype=bf16, device="cuda")
    P.append(None, x, x, *pools, ints(-1)[None], ints(1))
    monkeypatch.setenv("TXD_INJECT_STALL", "1")
    monkeypatch.setenv("TXD_WAIT_LIMIT_MS", "50")
    qs = torch.ones(q, 4, 64, dtype=bf16, device="cuda")
    P.paged_attention(qs, *pools, ints(0, 1, 2, 3, 4, 5, 6)[None], ints(112), 0.125, cu_q=ints(0, q), max_q=q)
    with pytest.raises(B.DotError, match="ran out.*outside the cache") as e:
        P.check()
    assert e.value.status == B.TXD_ERR_DEVICE_TIMEOUT
    P.check()


def test_no_finding_of_another_stream_is_lost(P):
    """A kernel on a side stream reports a bad page while the main stream checks over and over, each time with a finding of its
    own to clear: one of the checks has the page in its report, whenever the kernel ran."""
    from triton_ext_b200 import backend as B
    pools = small_cache()
    x, side = torch.ones(1, 2, 64, dtype=bf16, device="cuda"), torch.cuda.Stream()
    bad, good, one, short = ints(-1)[None], ints(0)[None], ints(1), ints(-3)
    torch.cuda.synchronize()

    def found():
        with pytest.raises(B.DotError) as e:
            P.append(None, x, x, *pools, good, short)
            P.check()
        return "outside the cache" in str(e.value)

    lost = 0
    for i in range(150):
        with torch.cuda.stream(side):
            torch.cuda._sleep(200000 + 7919 * i % 200000)
            P.append(None, x, x, *pools, bad, one)
            done = torch.cuda.Event()
            done.record()
        times = 0
        while not done.query():
            times += found()
        times += found()
        assert times <= 1                                         # and none is reported twice
        lost += times == 0
    assert lost == 0, f"{lost} of 150 findings lost"
    P.check()


def test_checks_of_two_threads_at_once(P):
    """Each finding is in exactly one report, whichever thread's."""
    import threading

    from triton_ext_b200 import backend as B
    pools, x, streams = small_cache(), torch.ones(1, 2, 64, dtype=bf16, device="cuda"), [torch.cuda.Stream() for _ in range(2)]
    bad, one, reports, wrong = ints(-1)[None], ints(1), [0, 0], []
    torch.cuda.synchronize()

    def run(i):
        try:
            with torch.cuda.stream(streams[i]):
                for _ in range(200):
                    if i == 0:
                        P.append(None, x, x, *pools, bad, one)
                    try:
                        P.check()
                    except B.DotError as e:
                        reports[i] += "outside the cache" in str(e)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and sum(reports) == 200
    P.check()


@pytest.mark.parametrize("tokens", [6, 300])
@pytest.mark.parametrize("what,cu,lens,text", [
    ("length", (0, 3, 6), (10, -1), "below zero"), ("length", None, (-5, 10), "below zero"),
    ("falling", (0, 4, 2), (10, 10), "cu_q that fall"), ("below", (-2, 3, 6), (10, 10), "outside the new tokens"),
    ("behind", (0, 3, 9), (10, 20), "outside the new tokens")])
def test_lengths_and_offsets_that_cannot_be_are_reported(P, tokens, what, cu, lens, text):
    """By append and by attention (both of its kernels), which stay inside their tensors."""
    from triton_ext_b200 import backend as B
    pools, table = small_cache(), torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=i32, device="cuda")
    rows = 2 if cu is None else tokens
    if cu is not None:
        cu, lens = ints(*(c * tokens // 6 for c in cu)), tuple(n if n < 0 else min(48, n * tokens // 6) for n in lens)
    q, out = (torch.full((rows + 2, 4, 64), x, dtype=bf16, device="cuda") for x in (1.0, 9.0))
    kw = dict(cu_q=cu, max_q=tokens) if cu is not None else {}
    P.paged_attention(q[:rows], *pools, table, ints(*lens), 0.125, out=out[:rows], **kw)
    with pytest.raises(B.DotError, match=text):
        P.check()
    assert bool((out[rows:] == 9.0).all()) and not bool(out.isnan().any())
    before = [x.clone() for x in pools]
    k = torch.ones(rows, 2, 64, dtype=bf16, device="cuda")
    P.append(None, k, k, *pools, table, ints(*lens), cu_q=cu)
    with pytest.raises(B.DotError, match=text):
        P.check()
    assert all(torch.equal(a[6:], b[6:]) for a, b in zip(pools, before))        # pages that are nobody's


def test_more_new_tokens_than_cached_ones_are_no_fault(P):
    """For attention: the first rows see nothing. And offsets that leave rows before, between none and behind are as they should be."""
    pools, table = small_cache(), torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=i32, device="cuda")
    q = torch.ones(40, 4, 64, dtype=bf16, device="cuda")
    for cu, lens in (((3, 20, 33), (5, 20)), ((0, 0, 40), (0, 40)), ((0, 0, 0), (0, 0)), ((40, 40, 40), (7, 7))):
        P.paged_attention(q, *pools, table, ints(*lens), 0.125, cu_q=ints(*cu), max_q=40)
        P.check()
        if lens[0] >= cu[1] - cu[0] and lens[1] >= cu[2] - cu[1]:
            P.append(None, q[:, :2], q[:, :2], *pools, table, ints(*lens), cu_q=ints(*cu))
            P.check()


# ---- lists that are parts of the cache's own state -------------------------------------------------------------------------
def test_lists_out_of_the_caches_lengths(P):
    """Rows cut to other rows' lengths, and grown by them: the lengths as they are before the call. More blocks and rows than run
    at once, in an order in which every length changes before it is read where the lists are not copied first."""
    n = 2000
    cache = P.PagedCache.create(3 * n, 16, 1, 16, rows=3 * n, width=4)
    every = torch.arange(3 * n, dtype=i32, device="cuda")
    sixteen = torch.full((n,), 16, dtype=i32, device="cuda")
    cache.reserve(every[n:2 * n], sixteen)
    cache.reserve(every[2 * n:], sixteen)
    cache.truncate(every[n:], cache.lens[:2 * n])                  # the second third to the first's 0, the last to the second's 16
    assert cache.lens.tolist() == [0] * (2 * n) + [16] * n and int(cache.refs.sum()) == n
    P.check()
    cache = P.PagedCache.create(3 * n, 16, 1, 16, rows=n, width=40)
    first = torch.arange(n, dtype=i32, device="cuda") % 7 + 1
    cache.reserve(every[:n], first)
    want = first + first.flip(0)
    lens = cache.reserve(every[:n].flip(0), cache.lens)
    assert torch.equal(cache.lens, want) and torch.equal(lens, want.flip(0))
    P.check()


def test_lists_out_of_the_caches_table(P):
    """Any of the state's arrays may be a list."""
    cache = P.PagedCache.create(8, 16, 1, 16, rows=4, width=3)
    assert cache.reserve(ints(0, 1, 3), ints(40, 20, 5)).tolist() == [40, 20, 5]   # pages 0 1 2, 3 4, 5
    cache.fork(cache.table[0], cache.table[1, :1].expand(3))        # rows 0, 1, 2 become row 3
    P.check()
    assert cache.lens.tolist() == [5, 5, 5, 5] and cache.table[:, 0].tolist() == [5] * 4 and cache.refs.tolist() == [0] * 5 + [4, 0, 0]
    cache.free(cache.refs[:2])                                      # row 0, twice
    P.check()
    assert cache.lens.tolist() == [0, 5, 5, 5] and cache.refs.tolist() == [0] * 5 + [3, 0, 0]


# ---- inputs that require a gradient ------------------------------------------------------------------------------------
@pytest.mark.parametrize("in_place", [False, True])
def test_a_backward_through_the_serving_operators_raises(P, in_place):
    """Neither operator has a gradient: whoever asks for one is told, instead of getting the other paths' alone."""
    from triton_ext_b200 import backend as B
    from triton_ext_b200.rotary import Rope
    pools, table, lens = small_cache(), ints(0, 1, 2)[None], ints(40)
    leaf = torch.randn(1, 4, 64, device="cuda").to(bf16).requires_grad_()
    k = torch.ones(1, 2, 64, dtype=bf16, device="cuda")

    def loss(step):
        return step(leaf * 2).float().sum() + (leaf * 3).float().sum()

    def attend(x):
        out, m = P.paged_attention(x, *pools, table, lens, 0.125, out=x if in_place else None, return_m=True)
        assert out.requires_grad and m.requires_grad
        return out

    def turn(x):
        return P.append(x, k, k, *pools, table, lens, rope=Rope(64), out=x if in_place else None)

    def keys(x):
        return P.append(leaf.detach(), x[:, :2], x[:, 2:], *pools, table, lens, rope=Rope(64))

    for step, name in ((attend, "paged_attention"), (turn, "append"), (keys, "append")):
        value = loss(step)
        with pytest.raises(B.DotError, match=f"{name} has no gradient"):
            value.backward()
        assert leaf.grad is None or bool((leaf.grad == 3).all())
        leaf.grad = None
    P.check()


def test_results_with_and_without_a_wanted_gradient_are_the_same(P):
    pools, table, lens = small_cache(), ints(0, 1, 2)[None], ints(40)
    q = torch.randn(1, 4, 64, device="cuda").to(bf16)
    want = P.paged_attention(q, *pools, table, lens, 0.125, return_m=True)
    got = P.paged_attention(q.clone().requires_grad_(), *pools, table, lens, 0.125, return_m=True)
    assert torch.equal(got[0].detach(), want[0]) and torch.equal(got[1].detach(), want[1])
    with torch.no_grad():
        got = P.paged_attention(q.clone().requires_grad_(), *pools, table, lens, 0.125)
    assert not got.requires_grad and torch.equal(got, want[0])
    x = q.clone().requires_grad_() * 1
    square = x * x                                                 # keeps x
    assert P.paged_attention(x, *pools, table, lens, 0.125, out=x).data_ptr() == x.data_ptr()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        square.sum().backward()
    P.check()


def test_outputs_that_overlap_themselves_are_refused(P):
    from triton_ext_b200 import backend as B
    pools, table = small_cache(), torch.zeros(10, 3, dtype=i32, device="cuda")
    lens, x = torch.ones(10, dtype=i32, device="cuda"), torch.zeros(10, 2, 64, dtype=bf16, device="cuda")
    memory = torch.full((4000,), 7.0, dtype=bf16, device="cuda")
    for strides in ((1, 64, 1), (64, 64, 1), (8, 128, 1)):
        out = memory.as_strided(x.shape, strides)
        for call in (lambda: P.paged_attention(x, *pools, table, lens, 0.125, out=out), lambda: P.append(x, x, x, *pools, table, lens, out=out)):
            with pytest.raises(B.DotError, match="overlap itself"):
                call()
    assert bool((memory == 7.0).all())
    P.check()


def test_a_list_that_reaches_into_the_lengths(P):
    """The lengths may be a part of the caller's vector, and a list begin before them in it."""
    n = 2000
    memory = torch.zeros(1 + 3 * n, dtype=i32, device="cuda")
    pools = [torch.zeros(1, 3 * n, 16, 1, 16, dtype=bf16, device="cuda") for _ in range(2)]
    cache = P.PagedCache(*pools, torch.full((3 * n, 4), -1, dtype=i32, device="cuda"), memory[1:], torch.zeros(3 * n, dtype=i32, device="cuda"))
    every = torch.arange(3 * n, dtype=i32, device="cuda")
    cache.reserve(every[n:2 * n], torch.full((n,), 16, dtype=i32, device="cuda"))
    cache.reserve(every[2 * n:], torch.full((n,), 16, dtype=i32, device="cuda"))
    cache.truncate(every[n - 1:], memory[:2 * n + 1])              # row n - 1 + i to memory[i], which is row i - 1's length
    P.check()
    assert cache.lens.tolist() == [0] * (2 * n) + [16] * n

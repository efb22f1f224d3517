"""Page operations on the GPU against a plain model on lists (tests/kv8_reference.py): equal entry for entry and byte for byte."""
import random

import pytest
import torch

import kv8_reference as ref
from omnikv_amd import ops
from omnikv_amd.pages import PagePool

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def make(seed, seqs, width, pages, page, lens, shapes=((16,), (3, 4), (5,))):
    """A pool with the given lengths on scattered pages and its model; shapes: of one page of each buffer, in floats."""
    r = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    buffers = [torch.randn((pages,) + s, generator=g).to(DEV) for s in shapes]
    table, refs = [[-1] * width for _ in range(seqs)], [0] * pages
    order = r.sample(range(pages), sum(-(-n // page) for n in lens))
    for s, n in enumerate(lens):
        for i in range(-(-n // page)):
            table[s][i] = order.pop()
            refs[table[s][i]] = 1
    table, refs, lens = i32(table), i32(refs), i32(list(lens) + [0] * (seqs - len(lens)))
    return table, lens, refs, buffers, ref.Pages(table.cpu(), lens.cpu(), refs.cpu(), page, [b.cpu() for b in buffers])


def same(table, lens, refs, buffers, model):
    assert table.tolist() == model.table
    assert lens.tolist() == model.lens
    assert refs.tolist() == model.refs
    for a, b in zip(buffers, model.buffers):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("page", [1, 4, 16, 48])
def test_fork_extend_free(page):
    lens = [1, page, page + 1, 5 * page - 1, 3 * page, 0]
    table, lt, refs, bufs, m = make(page, 14, 9, 70, page, lens)
    status = torch.full((2,), -5, dtype=torch.int32, device=DEV)
    parents, children = [0, 1, 2, 3, 3, 4, 5], [6, 7, 8, 9, 10, 11, 12]
    ops.pages_fork(table, lt, refs, i32(parents), i32(children), page, bufs, status)
    assert status.tolist() == m.fork(parents, children) == [0, 0]
    same(table, lt, refs, bufs, m)
    seqs, more = [9, 0, 10, 13, 8], [2, 3 * page, 0, 2 * page + 1, -4]
    ops.pages_extend(table, lt, refs, i32(seqs), i32(more), page, status)
    assert status.tolist() == m.extend(seqs, more) == [0, 0]
    same(table, lt, refs, bufs, m)
    ops.pages_free(table, lt, refs, i32([3, 9, 13, 5]), page, status)
    assert status.tolist() == m.free([3, 9, 13, 5]) == [0, 0]
    same(table, lt, refs, bufs, m)
    ops.pages_free(table, lt, refs, i32(list(range(14))), page)
    assert not refs.any() and not lt.any() and bool((table == -1).all())


def test_refused_entries_are_skipped():
    page = 4
    table, lt, refs, bufs, m = make(3, 8, 6, 40, page, [7, 9, 0, 5])
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    parents = [0, 1, 0, 1, 99, 0, 1, -1, 4, 2]
    children = [4, 4, 3, 1, 5, -2, 77, 5, 6, 7]  # again 4; 3 holds rows; itself; out of range; 4: a child of this very call
    ops.pages_fork(table, lt, refs, i32(parents), i32(children), page, bufs, status)
    assert status.tolist() == m.fork(parents, children)
    assert status[1] == 7
    same(table, lt, refs, bufs, m)
    seqs, more = [0, 0, 8, -1, 1, 2], [1, 1, 1, 1, 100, 24]
    ops.pages_extend(table, lt, refs, i32(seqs), i32(more), page, status)
    assert status.tolist() == m.extend(seqs, more) == [0, 4]
    same(table, lt, refs, bufs, m)
    ops.pages_free(table, lt, refs, i32([1, 1, 9, 1, -3, 7]), page, status)  # freed once, whoever comes first
    assert status.tolist() == m.free([1, 9, -3, 7])
    same(table, lt, refs, bufs, m)


def test_short_of_pages_changes_nothing():
    page = 4
    table, lt, refs, bufs, m = make(4, 8, 8, 9, page, [7, 9, 5])
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    ops.pages_fork(table, lt, refs, i32([0, 1, 2, 9]), i32([3, 4, 5, 6]), page, bufs, status)  # 7 of 9 in use, 3 wanted
    assert status.tolist() == m.fork([0, 1, 2, 9], [3, 4, 5, 6]) == [1, 1]
    same(table, lt, refs, bufs, m)
    ops.pages_extend(table, lt, refs, i32([0, 7]), i32([2, 12]), page, status)
    assert status.tolist() == m.extend([0, 7], [2, 12])
    assert status[0] == 2
    same(table, lt, refs, bufs, m)
    ops.pages_extend(table, lt, refs, i32([7]), i32([8]), page, status)
    assert status.tolist() == m.extend([7], [8]) == [0, 0]
    same(table, lt, refs, bufs, m)


def test_fork_copies_the_sequences_rows_of_served_pairs_only():
    page = 4
    table, lt, refs, bufs, m = make(5, 8, 6, 40, page, [7, 8, 0, 5])
    g = torch.Generator().manual_seed(5)
    rows = [torch.randn((8, 3, 4), generator=g).to(DEV), torch.randn((8, 500, 4), generator=g).to(DEV)]
    want = [r.clone() for r in rows]
    parents, children = [0, 1, 0, 99, 2, 3], [4, 5, 4, 6, 6, -1]  # again 4; out of range; an empty parent
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    ops.pages_fork(table, lt, refs, i32(parents), i32(children), page, bufs, status, ops.PageBuffers(rows))
    assert status.tolist() == m.fork(parents, children)
    same(table, lt, refs, bufs, m)
    for r, w in zip(rows, want):
        w[4], w[5] = w[0], w[1]
        assert torch.equal(r, w)


def test_the_largest_call_and_growth_over_many_trips_through_the_counts():
    """1024 entries at once; a pool of more pages than one trip through the counts covers."""
    page, seqs = 2, 2048
    r = random.Random(9)
    lens = [r.randint(0, 9) for _ in range(1024)]
    table, lt, refs, bufs, m = make(9, seqs, 12, 30000, page, lens, shapes=((2,),))
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    children = list(range(1024, 2048))
    r.shuffle(children)
    ops.pages_fork(table, lt, refs, i32(list(range(1024))), i32(children), page, bufs, status)
    assert status.tolist() == m.fork(list(range(1024)), children) == [0, 0]
    same(table, lt, refs, bufs, m)
    seqs_, more = r.sample(range(2048), 1024), [r.randint(-2, 12) for _ in range(1024)]
    ops.pages_extend(table, lt, refs, i32(seqs_), i32(more), page, status)
    assert status.tolist() == m.extend(seqs_, more)
    same(table, lt, refs, bufs, m)
    gone = r.sample(range(2048), 1500)
    ops.pages_free(table, lt, refs, i32(gone), page, status)
    m.free(gone)
    t, rf, n = ops.pages_compact(table, refs, bufs)
    assert int(n) == m.compact()
    same(t, lt, rf, bufs, m)


@pytest.mark.parametrize("pages, seqs", [(1, 1), (2, 1), (63, 4), (1024, 10), (1025, 40), (5000, 700)])
@pytest.mark.parametrize("used", [0.0, 0.3, 0.97, 1.0])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(pages, seqs, used, in_place):
    r = random.Random(pages)
    page, left, lens = 4, int(pages * used), []
    for s in range(seqs):
        n = left if s == seqs - 1 else min(left, r.randint(0, max(1, 2 * left // max(1, seqs - s))))
        left -= n
        lens.append(max(0, n * page - r.randrange(page)) if n else 0)
    table, lt, refs, bufs, m = make(pages, seqs + 3, pages + 1, pages, page, lens, shapes=((4,), (1,), (33,)))
    children, parents = list(range(seqs, seqs + 3)), [0, seqs - 1, seqs // 2]
    if m.fork(parents, children) == [0, 0]:  # shared pages move once
        ops.pages_fork(table, lt, refs, i32(parents), i32(children), page, bufs)
    before = table.clone(), refs.clone()
    t, rf, n = ops.pages_compact(table, refs, ops.PageBuffers(bufs), table_out=table if in_place else None,
                                 refs_out=refs if in_place else None)
    assert int(n) == m.compact()
    same(t, lt, rf, bufs, m)
    if not in_place:
        assert torch.equal(before[0], table) and torch.equal(before[1], refs)


@pytest.mark.parametrize("shape, dtype", [((16, 2, 128), torch.uint8), ((3,), torch.float32), ((2, 5), torch.float32),
                                          ((4096, 16), torch.float32), ((7, 4), torch.int8)])
def test_copy(shape, dtype):
    g = torch.Generator().manual_seed(6)
    bufs = [torch.randint(0, 100, (40,) + shape, generator=g).to(dtype).to(DEV) for _ in range(3)]
    want = [b.clone() for b in bufs]
    src, dst = [0, 3, 3, 39, 41, 5], [10, 11, 12, 13, 14, -2]
    for b in want:
        b[10:14] = b[[0, 3, 3, 39]]
    ops.pages_copy(bufs, i32(src), i32(dst))
    assert all(torch.equal(a, b) for a, b in zip(bufs, want))
    for b in want:
        b[20] = b[1]
    ops.pages_copy(bufs, i32([1, 2]), i32([20, 21]), count=i32([1]))
    assert all(torch.equal(a, b) for a, b in zip(bufs, want))


def test_many_buffers_and_an_unaligned_one():
    table, lt, refs, _, _ = make(7, 6, 8, 40, 4, [7, 9])
    g = torch.Generator().manual_seed(7)
    bufs = [torch.randn((40, 5 + i % 3), generator=g).to(DEV) for i in range(300)]
    off = torch.randn(40 * 4 + 1, generator=g).to(DEV)[1:].view(40, 4)  # 4-byte aligned only
    bufs.append(off)
    m = ref.Pages(table.cpu(), lt.cpu(), refs.cpu(), 4, [b.cpu() for b in bufs])
    ops.pages_fork(table, lt, refs, i32([0, 1]), i32([4, 5]), 4, bufs)
    m.fork([0, 1], [4, 5])
    same(table, lt, refs, bufs, m)
    t, rf, _ = ops.pages_compact(table, refs, bufs)
    m.compact()
    same(t, lt, rf, bufs, m)


def test_pool_of_an_8_bit_cache_in_a_replayed_graph():
    """PagePool over two layers of an 8-bit cache: prefill, fork, grow, append, attend, end the losers, compact -- the
    attention of every sequence as if it had a cache of its own; the page step is captured and replayed."""
    import test_gpu_kv8 as kv8

    g = torch.Generator().manual_seed(8)
    seqs, width, pages, page, hkv, block = 6, 12, 60, 32, 2, 16
    pool = PagePool(seqs, width, pages, page, DEV)
    layers = [ops.KV8.empty_paged(pool.table, pages, page, hkv, "int8", block, torch.bfloat16) for _ in range(2)]
    for c in layers:
        pool.add_cache(c)
    own = [[[], []] for _ in range(seqs)]  # per sequence: K rows, V rows of layer 0
    n0 = [70, 33, 0, 0, 0, 0]
    pool.extend([0, 1], n0[:2])
    x, y = kv8.rows(g, seqs, hkv, 70), kv8.rows(g, seqs, hkv, 70)
    for c in layers:
        ops.kv8_append(c, x.to(DEV), y.to(DEV), 0, i32(n0))
    for s in (0, 1):
        own[s] = [x[s, :, : n0[s]], y[s, :, : n0[s]]]
    assert pool.status() == (0, 0)
    parents, children = i32([0, 0, 1]), i32([2, 3, 4])
    before = [t.clone() for t in (pool.table, pool.lens, pool.refs)]
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        pool.free(children)
        pool.fork(parents, children)
    for t, b in zip((pool.table, pool.lens, pool.refs), before):
        assert torch.equal(t, b)  # nothing ran at capture
    graph.replay()
    first = [t.clone() for t in (pool.table, pool.lens, pool.refs)]
    for i in range(3):
        graph.replay()  # frees and forks again: the same pages, lowest first
        torch.cuda.synchronize()
        for t, b in zip((pool.table, pool.lens, pool.refs), first):
            assert torch.equal(t, b), i
    for p, c in ((0, 2), (0, 3), (1, 4)):
        own[c] = [t.clone() for t in own[p]]
    live, add = [0, 1, 2, 3, 4], 21
    lens = pool.lens.clone()
    x, y = kv8.rows(g, seqs, hkv, add), kv8.rows(g, seqs, hkv, add)
    pool.extend(live, [add] * 5)
    grow = i32([add] * 5 + [0])
    for c in layers:
        ops.kv8_append(c, x.to(DEV), y.to(DEV), lens, grow)
    for s in live:
        own[s] = [torch.cat([a, t[s]], 1) for a, t in zip(own[s], (x, y))]
    q = kv8.rows(g, seqs, hkv * 4)

    def attend():
        for c in layers:
            out = ops.kv8_dense_attn(q.to(DEV), c, seq_lens=pool.lens)
            kv8.check_attention(out, q, [kv8.held(own[s][0], "int8", block, True) if s in live else torch.zeros(hkv, 0, 128)
                                         for s in range(seqs)],
                                [kv8.held(own[s][1], "int8", block, True) if s in live else torch.zeros(hkv, 0, 128)
                                 for s in range(seqs)], 128 ** -0.5, torch.bfloat16)

    attend()
    pool.free([0, 3])
    live = [1, 2, 4]
    pool.compact()
    assert int((pool.refs > 0).sum()) == int(pool.used) and not pool.refs[int(pool.used):].any()
    attend()
    assert pool.status() == (0, 0)


def test_a_refused_array_leaves_the_pool_as_it_was():
    pool = PagePool(2, 4, 8, 16, DEV)
    pool.add(torch.zeros((8, 4), device=DEV))
    for bad in (torch.zeros((9, 4), device=DEV), torch.zeros((8, 8), device=DEV)[:, :4], torch.zeros((8, 4))):
        with pytest.raises(ValueError):
            pool.add(bad)
    part = ops.KV8.empty_paged(pool.table[:1], 8, 16, 2)  # the table's first row alone
    other = ops.KV8.empty_paged(pool.table.clone(), 8, 16, 2)
    for cache in (part, other):
        with pytest.raises(ValueError):
            pool.add_cache(cache)
    pool.extend([0], [20])
    pool.fork([0], [1])
    assert pool.status() == (0, 0) and pool.table.tolist() == [[0, 1, -1, -1], [0, 2, -1, -1]]


@pytest.mark.parametrize("want", [4095, 4096, 4097, 9000])
def test_growth_by_more_pages_than_a_plan_keeps(want):
    """Calls that take so many pages in all: one long sequence among short ones, then another of half a page more."""
    page, r = 4, random.Random(want)
    lens = [r.randint(0, 40) for _ in range(200)]
    table, lt, refs, bufs, m = make(10, 210, want, 2 * want + 2200, page, lens, shapes=((1,),))
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    for seqs, more in (([205, 206, 207, 208], [page * (want - 7), 1, 0, 6 * page]),
                       ([201, 202, 203], [2 * page, page * (want - 2) - 1, -5])):
        before = sum(refs.tolist())
        ops.pages_extend(table, lt, refs, i32(seqs), i32(more), page, status)
        assert status.tolist() == m.extend(seqs, more) == [0, 0]
        assert sum(refs.tolist()) - before == want
        same(table, lt, refs, bufs, m)


def test_pool_of_16_bit_pages_forks_grows_and_compacts():
    """PagePool under ops.PagedKV: attention through the table after every step is that of each sequence's own rows."""
    g = torch.Generator().manual_seed(11)
    seqs, width, pages, page, hkv = 5, 8, 40, 16, 2
    pool = PagePool(seqs, width, pages, page, DEV)
    pk, pv = (torch.zeros((pages, page, hkv, 128), dtype=torch.bfloat16, device=DEV) for _ in "kv")
    pool.add(pk, pv)
    kv = ops.PagedKV(pk, pv, pool.table, page)
    own = [[torch.zeros(hkv, 0, 128), torch.zeros(hkv, 0, 128)] for _ in range(seqs)]

    def write(s, n):  # n more rows of sequence s, through the table
        for t, mine in ((pk, 0), (pv, 1)):
            x = torch.randn(hkv, n, 128, generator=g).to(torch.bfloat16)
            at = torch.arange(own[s][mine].shape[1], own[s][mine].shape[1] + n, device=DEV)
            t[pool.table[s, at // page].long(), at % page] = x.transpose(0, 1).to(DEV)
            own[s][mine] = torch.cat([own[s][mine], x.float()], 1)

    def check(live):
        q = torch.randn(seqs, 2 * hkv, 128, generator=g).to(torch.bfloat16)
        out = ops.dense_attn(q.to(DEV), kv, seq_len=width * page, seq_lens=pool.lens)
        for s in live:
            k, v = (x.double() for x in own[s])
            assert int(pool.lens[s]) == k.shape[1]
            p = torch.softmax(torch.einsum("hgd,hnd->hgn", q[s].double().view(hkv, 2, 128), k) * 128 ** -0.5, -1)
            want = torch.einsum("hgn,hnd->hgd", p, v).reshape(2 * hkv, 128)
            assert float((out[s].cpu().double() - want).abs().max()) < 2e-2  # (the bar of 16-bit attention in these tests)

    pool.extend([0, 1], [37, 64])
    write(0, 37), write(1, 64)
    check([0, 1])
    pool.fork([0, 0, 1], [2, 3, 4])
    for c, p in ((2, 0), (3, 0), (4, 1)):
        own[c] = [x.clone() for x in own[p]]
    check(range(5))
    pool.extend(list(range(5)), [3, 20, 5, 0, 17])
    for s, n in enumerate([3, 20, 5, 0, 17]):
        write(s, n)
    check(range(5))
    pool.free([1, 3])
    pool.compact()
    assert int(pool.used) == int((pool.refs > 0).sum()) and bool((pool.refs[int(pool.used):] == 0).all())
    check([0, 2, 4])
    assert pool.status() == (0, 0)


def test_a_step_that_the_pool_refuses_leaves_the_caches_as_they_were():
    """Appending what extend granted (the difference of the lengths), not what was asked for: a pool that is short, and an
    entry that is refused, change neither codes nor open rows; the next step that fits goes on as if nothing had been asked."""
    import test_gpu_kv8 as kv8

    g = torch.Generator().manual_seed(12)
    seqs, page, hkv, block, bf = 3, 32, 2, 16, torch.bfloat16
    pool = PagePool(seqs, 4, 7, page, DEV)
    cache = ops.KV8.empty_paged(pool.table, 7, page, hkv, "int8", block, bf)
    pool.add_cache(cache)
    own = [[torch.zeros(hkv, 0, 128, dtype=bf)] * 2 for _ in range(seqs)]

    def step(more, granted):
        starts = pool.lens.clone()
        pool.extend(list(range(seqs)), more)
        x, y = (kv8.rows(g, seqs, hkv, max(more)) for _ in "kv")
        ops.kv8_append(cache, x.to(DEV), y.to(DEV), starts, pool.lens - starts)
        for s, n in enumerate(granted):
            own[s] = [torch.cat([a, t[s, :, :n]], 1) for a, t in zip(own[s], (x, y))]
        q = kv8.rows(g, seqs, 4 * hkv)
        out = ops.kv8_dense_attn(q.to(DEV), cache, seq_lens=pool.lens)
        kv8.check_attention(out, q, *([kv8.held(own[s][i], "int8", block, True) for s in range(seqs)] for i in (0, 1)), 128 ** -0.5, bf)

    step([45, 70, 20], [45, 70, 20])  # 2 + 3 + 1 of 7 pages
    state = [t.clone() for t in (cache.k.view(torch.uint8), cache.k_scale, cache.open_k, cache.open_v, pool.table, pool.lens)]
    step([30, 35, 10], [0, 0, 0])  # two more wanted, one left
    for t, was in zip((cache.k.view(torch.uint8), cache.k_scale, cache.open_k, cache.open_v, pool.table, pool.lens), state):
        assert torch.equal(t, was)
    assert pool.status() == (1, 0)
    step([100, 5, 3], [0, 5, 3])  # five pages for a sequence of at most four: that entry alone is refused
    assert pool.status() == (0, 1)
    step([19, 0, 30], [19, 0, 30])
    assert pool.status() == (0, 0)

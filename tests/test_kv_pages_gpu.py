"""Copying, freeing, forking and compacting pages against plain Python bookkeeping: tables, references
and every byte of the pools."""
import random

import pytest

import infb200 as I
from paged_ref import Cache

pytestmark = pytest.mark.gpu

SHAPES = [("bf16", 3, 2, 64, 16), ("bf16", 2, 8, 128, 16), ("fp32", 2, 6, 48, 16), ("bf16", 5, 1, 8, 4), ("fp32", 1, 3, 4, 1),
          ("bf16", 1, 4, 256, 64)]


def ints(torch, values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def filled(torch, shape, slots=6, pps=5, spare=7, seed=0):
    """A cache with random contents everywhere and nothing held."""
    dtype, layers, KV, hd, blk = shape
    c = Cache(torch, slots, pps, KV, hd, blk, dtype, layers, spare=spare, seed=seed)
    c.k.copy_(c.randn(*c.k.shape))
    c.v.copy_(c.randn(*c.v.shape))
    c.scratch = torch.full((I.kv_pages_scratch_bytes(c.kv),), 0xFF, dtype=torch.uint8, device="cuda")
    return c


def place(torch, c, lens, seed=0, share=()):
    """Sequences of the given lengths in pages taken at random; share: (slot, from, pages) shared prefixes."""
    r = random.Random(seed)
    free = list(range(c.n_pages))
    r.shuffle(free)
    table, refs = [[-1] * c.table.shape[1] for _ in range(c.table.shape[0])], [0] * c.n_pages
    for s, n in enumerate(lens):
        for i in range(-(-n // c.blk)):
            src = [f for (t, f, p) in share if t == s and i < p]
            page = table[src[0]][i] if src else free.pop()
            table[s][i] = page
            refs[page] += 1
    c.table.copy_(ints(torch, table))
    c.refs.copy_(ints(torch, refs))
    return table, refs


def code_of(c):
    try:
        c.check()
    except I.InfError as e:
        return e.code
    return 0


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("n", [1, 2, 13])
def test_copy(cuda, shape, n):
    torch = cuda
    c = filled(torch, shape)
    ids = torch.randperm(c.n_pages).tolist()
    src, dst = ids[:n], ids[n:2 * n]
    k, v = c.k.clone(), c.v.clone()
    k[:, dst], v[:, dst] = k[:, src], v[:, src]
    a, b = ints(torch, src), ints(torch, dst)
    I.kv_copy_pages(c.kv, a.data_ptr(), b.data_ptr(), n, c.status.data_ptr())
    c.check()
    assert torch.equal(c.k, k) and torch.equal(c.v, v)
    # one source copied to several pages is fine
    if n > 2:
        a.fill_(src[0])
        k[:, dst], v[:, dst] = k[:, [src[0]] * n], v[:, [src[0]] * n]
        I.kv_copy_pages(c.kv, a.data_ptr(), b.data_ptr(), n, c.status.data_ptr())
        c.check()
        assert torch.equal(c.k, k) and torch.equal(c.v, v)


def test_copy_pairs_that_meet_are_skipped(cuda):
    """An id outside the pool, a page written twice, a page written and read: reported, skipped; the first
    pair that writes a page is done."""
    torch = cuda
    c = filled(torch, SHAPES[0])
    src = [0, 1, 2, 3, -1, 5, c.n_pages]
    dst = [10, 10, 3, 11, 12, c.n_pages, 13]  # 3 is a source of the fourth pair
    k = c.k.clone()
    k[:, [10, 11]] = k[:, [0, 3]]
    a, b = ints(torch, src), ints(torch, dst)
    I.kv_copy_pages(c.kv, a.data_ptr(), b.data_ptr(), len(src), c.status.data_ptr())
    assert code_of(c) == 4
    assert torch.equal(c.k, k)
    a, b = ints(torch, [4]), ints(torch, [4])  # onto itself
    I.kv_copy_pages(c.kv, a.data_ptr(), b.data_ptr(), 1, c.status.data_ptr())
    assert code_of(c) == 4 and torch.equal(c.k, k)


def test_copy_past_4_gb_of_pool(cuda):
    """Byte offsets above 2^32 within a layer's pool."""
    torch = cuda
    c = Cache(torch, 1, 1, 8, 128, 16, "bf16", 1, n_pages=140_000)  # 32 KB pages: 4.6 GB per pool
    c.k[0, 3].copy_(c.randn(8, 16, 128))
    c.v[0, 139_000].copy_(c.randn(8, 16, 128))
    a, b = ints(torch, [3, 139_000]), ints(torch, [139_999, 7])
    I.kv_copy_pages(c.kv, a.data_ptr(), b.data_ptr(), 2, c.status.data_ptr())
    c.check()
    assert torch.equal(c.k[0, 139_999], c.k[0, 3]) and torch.equal(c.v[0, 7], c.v[0, 139_000])


def test_free(cuda):
    torch = cuda
    c = filled(torch, SHAPES[0])
    table, refs = place(torch, c, [70, 16, 33, 80, 0, 1], share=[(3, 0, 4)])
    slots, first, last = [0, 3, 0, 5, 2], [1, 0, 0, 0, 0], [3, 5, 2, 5, 0]  # entry (0, 1) is named twice

    def give_up(slots, first, last):
        for s, f, l in zip(slots, first, last):
            for e in range(f, l):
                if table[s][e] >= 0:
                    refs[table[s][e]] -= 1
                    table[s][e] = -1

    a, b, d = ints(torch, slots), ints(torch, first), ints(torch, last)
    I.kv_free(c.kv, a.data_ptr(), b.data_ptr(), d.data_ptr(), len(slots), c.status.data_ptr())
    c.check()
    give_up(slots, first, last)
    assert c.table.tolist() == table and c.refs.tolist() == refs
    # whole rows; a slot named twice and an empty one
    a = ints(torch, [1, 4, 1, 0])
    I.kv_free(c.kv, a.data_ptr(), 0, 0, 4, c.status.data_ptr())
    c.check()
    give_up([1, 4, 0], [0] * 3, [5] * 3)
    assert c.table.tolist() == table and c.refs.tolist() == refs
    # only the last bound, only the first one
    a, b = ints(torch, [2]), ints(torch, [1])
    I.kv_free(c.kv, a.data_ptr(), 0, b.data_ptr(), 1, c.status.data_ptr())
    give_up([2], [0], [1])
    I.kv_free(c.kv, a.data_ptr(), b.data_ptr(), 0, 1, c.status.data_ptr())
    give_up([2], [1], [5])
    c.check()
    assert c.table.tolist() == table and c.refs.tolist() == refs and sum(refs) == 0


def test_free_reports(cuda):
    torch = cuda
    c = filled(torch, SHAPES[0])
    table, refs = place(torch, c, [70, 16, 33])
    for slot, first, last in ((9, 0, 1), (-1, 0, 1), (0, -1, 1), (0, 0, 6)):
        a, b, d = ints(torch, [slot]), ints(torch, [first]), ints(torch, [last])
        I.kv_free(c.kv, a.data_ptr(), b.data_ptr(), d.data_ptr(), 1, c.status.data_ptr())
        assert code_of(c) == 4
        assert c.table.tolist() == table and c.refs.tolist() == refs
    a, b, d = ints(torch, [0]), ints(torch, [3]), ints(torch, [1])  # an empty range
    I.kv_free(c.kv, a.data_ptr(), b.data_ptr(), d.data_ptr(), 1, c.status.data_ptr())
    c.check()
    assert c.table.tolist() == table
    c.refs[table[1][0]] = 0  # a page without references
    c.table[2, 0] = c.n_pages + 4
    a = ints(torch, [1, 2])
    I.kv_free(c.kv, a.data_ptr(), 0, 0, 2, c.status.data_ptr())
    assert code_of(c) == 4
    assert bool((c.table[1:3] == -1).all()) and int(c.refs.min()) == 0


def plain_fork(c, table, refs, k, v, src, dst, lens):
    fresh = [p for p in range(c.n_pages) if refs[p] == 0]
    rows = [list(table[s]) for s in src]
    for i, n in enumerate(lens):
        s_row, row = rows[i], [-1] * len(table[0])
        full, rest = n // c.blk, n % c.blk
        row[:full] = s_row[:full]
        for p in row[:full]:
            if p >= 0:
                refs[p] += 1
        if rest and s_row[full] >= 0:
            p = fresh.pop(0)
            refs[p], row[full] = 1, p
            k[:, p, :, :rest], v[:, p, :, :rest] = k[:, s_row[full], :, :rest], v[:, s_row[full], :, :rest]
        table[dst[i]] = row


@pytest.mark.parametrize("shape", SHAPES)
def test_fork(cuda, shape):
    torch = cuda
    blk = shape[4]
    c = filled(torch, shape, slots=9, pps=6, spare=30)
    table, refs = place(torch, c, [6 * blk, 3 * blk + blk // 2, 1, blk])
    c.table[0, 1] = -1  # a page that left a window
    refs[table[0][1]] -= 1
    table[0][1] = -1
    c.refs.copy_(ints(torch, refs))
    src, dst = [1, 1, 0, 2, 3], [7, 4, 5, 8, 6]  # one sequence forks twice
    lens = [3 * blk + blk // 2, 2 * blk, 6 * blk - max(1, blk // 3), 1, 0]
    k, v = c.k.clone(), c.v.clone()
    plain_fork(c, table, refs, k, v, src, dst, lens)
    a, b, d = ints(torch, src), ints(torch, dst), ints(torch, lens)
    I.kv_fork(c.kv, a.data_ptr(), b.data_ptr(), d.data_ptr(), len(src), c.scratch.data_ptr(), c.scratch.numel(),
              c.status.data_ptr())
    c.check()
    assert c.table.tolist() == table and c.refs.tolist() == refs
    assert torch.equal(c.k, k) and torch.equal(c.v, v)


def test_fork_of_a_missing_last_page(cuda):
    torch = cuda
    c = filled(torch, SHAPES[0])
    table, refs = place(torch, c, [40])
    c.table[0, 2] = table[0][2] = -1
    a, b, d = ints(torch, [0]), ints(torch, [3]), ints(torch, [40])
    I.kv_fork(c.kv, a.data_ptr(), b.data_ptr(), d.data_ptr(), 1, c.scratch.data_ptr(), c.scratch.numel(), c.status.data_ptr())
    c.check()
    assert c.table[3].tolist() == table[0]


def test_fork_refusals_leave_the_rest(cuda):
    torch = cuda
    c = filled(torch, SHAPES[0], slots=12, spare=0)
    lens0 = [70, 16, 33]
    table, refs = place(torch, c, lens0)
    #       ok  dst held  dst twice  src range  dst range  len long  len < 0  dst is a source
    src = [0, 0, 1, 12, 1, 1, 1, 2]
    dst = [5, 1, 5, 6, -1, 7, 8, 0]
    lens = [70, 10, 16, 3, 3, 81, -1, 3]
    k, v = c.k.clone(), c.v.clone()
    plain_fork(c, table, refs, k, v, [0], [5], [70])
    a, b, d = ints(torch, src), ints(torch, dst), ints(torch, lens)
    I.kv_fork(c.kv, a.data_ptr(), b.data_ptr(), d.data_ptr(), len(src), c.scratch.data_ptr(), c.scratch.numel(),
              c.status.data_ptr())
    assert code_of(c) == 4
    assert c.table.tolist() == table and c.refs.tolist() == refs
    assert torch.equal(c.k, k) and torch.equal(c.v, v)


def test_fork_out_of_pages(cuda):
    """Two free pages, three partial ones wanted: the last fork is skipped whole."""
    torch = cuda
    c = filled(torch, SHAPES[0], slots=6, pps=3, spare=0)
    table, refs = place(torch, c, [33])
    for p in [p for p in range(c.n_pages) if refs[p] == 0][2:]:
        refs[p] = 9  # held elsewhere
    c.refs.copy_(ints(torch, refs))
    k, v = c.k.clone(), c.v.clone()
    plain_fork(c, table, refs, k, v, [0, 0, 0], [1, 2, 4], [33, 20, 16])
    a, b, d = ints(torch, [0, 0, 0, 0]), ints(torch, [1, 2, 3, 4]), ints(torch, [33, 20, 18, 16])
    I.kv_fork(c.kv, a.data_ptr(), b.data_ptr(), d.data_ptr(), 4, c.scratch.data_ptr(), c.scratch.numel(), c.status.data_ptr())
    assert code_of(c) == 2
    assert c.table.tolist() == table and c.refs.tolist() == refs
    assert torch.equal(c.k, k) and torch.equal(c.v, v)


def plain_compact(c, table, refs, k, v):
    live = [p for p in range(c.n_pages) if refs[p] > 0]
    L = len(live)
    moves = list(zip([p for p in live if p >= L], [p for p in range(L) if refs[p] <= 0]))
    where = {p: p for p in live}
    where.update(moves)
    new = [[where.get(p, p) for p in row] for row in table]
    for a, b in moves:
        k[:, b], v[:, b] = k[:, a], v[:, a]
        refs[b], refs[a] = refs[a], 0
    return new, [where.get(p, -1) for p in range(c.n_pages)], L


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("spare", [0, 1, 40, 2100])
def test_compact(cuda, shape, spare):
    torch = cuda
    blk = shape[4]
    c = filled(torch, shape, slots=7, pps=6, spare=spare, seed=spare)
    table, refs = place(torch, c, [6 * blk, 3 * blk + 1, 1, 0, 5 * blk, 6 * blk, 2 * blk], seed=spare, share=[(5, 0, 3), (6, 0, 2)])
    k, v = c.k.clone(), c.v.clone()
    table, where, L = plain_compact(c, table, refs, k, v)
    m, live = torch.empty(c.n_pages, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    for _ in range(2):  # the second time nothing moves
        I.kv_compact(c.kv, m.data_ptr(), live.data_ptr(), c.scratch.data_ptr(), c.scratch.numel(), c.status.data_ptr())
        c.check()
        assert int(live) == L and m.tolist() == where
        assert c.table.tolist() == table and c.refs.tolist() == refs
        assert torch.equal(c.k, k) and torch.equal(c.v, v)
        where = [p if p < L else -1 for p in range(c.n_pages)]


def test_compact_of_a_full_and_of_an_empty_pool(cuda):
    torch = cuda
    c = filled(torch, SHAPES[0], slots=2, pps=32, spare=0)  # 64 pages: whole words of the bit map
    m, live = torch.empty(c.n_pages, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    I.kv_compact(c.kv, m.data_ptr(), live.data_ptr(), c.scratch.data_ptr(), c.scratch.numel(), c.status.data_ptr())
    c.check()
    assert int(live) == 0 and bool((m == -1).all())
    table, refs = place(torch, c, [512, 512])
    I.kv_compact(c.kv, m.data_ptr(), live.data_ptr(), c.scratch.data_ptr(), c.scratch.numel(), c.status.data_ptr())
    c.check()
    assert int(live) == 64 and m.tolist() == list(range(64)) and c.table.tolist() == table and c.refs.tolist() == refs


def test_compact_reports_entries_without_a_page(cuda):
    torch = cuda
    c = filled(torch, SHAPES[0])
    place(torch, c, [70, 16])
    c.table[3, 0] = c.n_pages + 1
    m, live = torch.empty(c.n_pages, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    I.kv_compact(c.kv, m.data_ptr(), live.data_ptr(), c.scratch.data_ptr(), c.scratch.numel(), c.status.data_ptr())
    assert code_of(c) == 4
    assert int(c.table[3, 0]) == c.n_pages + 1


def test_a_scheduler_step_in_a_graph(cuda):
    """Free, fork and compact captured once and replayed on other contents."""
    torch = cuda
    c = filled(torch, SHAPES[1], slots=6, pps=5, spare=10)
    drop, src, lens = ints(torch, [1, 3]), ints(torch, [0, 2]), ints(torch, [70, 33])
    m, live = torch.empty(c.n_pages, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")

    def step(stream):
        I.kv_free(c.kv, drop.data_ptr(), 0, 0, 2, c.status.data_ptr(), stream)
        I.kv_fork(c.kv, src.data_ptr(), drop.data_ptr(), lens.data_ptr(), 2, c.scratch.data_ptr(), c.scratch.numel(),
                  c.status.data_ptr(), stream)
        I.kv_compact(c.kv, m.data_ptr(), live.data_ptr(), c.scratch.data_ptr(), c.scratch.numel(), c.status.data_ptr(), stream)

    place(torch, c, [70, 60, 40, 10, 20])
    step(0)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    for seed, cut in ((1, [70, 33]), (2, [16, 40])):
        table, refs = place(torch, c, [70, 60, 40, 10, 20], seed=seed)
        lens.copy_(torch.tensor(cut, dtype=torch.int32))
        k, v = c.k.clone(), c.v.clone()
        for s in (1, 3):
            for e in range(5):
                if table[s][e] >= 0:
                    refs[table[s][e]] -= 1
                    table[s][e] = -1
        plain_fork(c, table, refs, k, v, [0, 2], [1, 3], cut)
        table, where, L = plain_compact(c, table, refs, k, v)
        torch.cuda.synchronize()
        graph.replay()
        c.check()
        assert c.table.tolist() == table and c.refs.tolist() == refs and m.tolist() == where and int(live) == L
        assert torch.equal(c.k, k) and torch.equal(c.v, v)

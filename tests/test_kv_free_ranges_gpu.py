"""inf_kv_free with ranges at the ends of the integers: reported and skipped, the rest of the call done."""
import pytest

import infb200 as I
from test_kv_pages_gpu import SHAPES, code_of, filled, ints, place

pytestmark = pytest.mark.gpu

TOP = 2 ** 31 - 1


@pytest.mark.parametrize("first,last", [(6, 5), (6, None), (TOP, 5), (TOP, None), (TOP - 255, 5), (TOP - 16384, 5), (TOP, TOP), (2 ** 30, 0),
                                        (0, -1), (None, -1), (3, -TOP - 1), (0, TOP), (-TOP - 1, 5), (-TOP - 1, None)])
def test_ranges_outside_the_table(cuda, first, last):
    torch = cuda
    pps = 5
    c = filled(torch, SHAPES[0], pps=pps)
    table, refs = place(torch, c, [70, 16, 33, 80])
    # the bad range between two good ones
    a = ints(torch, [0, 1, 3])
    b = ints(torch, [1, first, 2]) if first is not None else None
    d = ints(torch, [2, last, 4]) if last is not None else None
    I.kv_free(c.kv, a.data_ptr(), b.data_ptr() if b is not None else 0, d.data_ptr() if d is not None else 0, 3, c.status.data_ptr())
    assert code_of(c) == 4
    for s, f, l in ((0, 1, 2), (3, 2, 4)):
        for e in range(f if first is not None else 0, l if last is not None else pps):
            if table[s][e] >= 0:
                refs[table[s][e]] -= 1
                table[s][e] = -1
    assert c.table.tolist() == table and c.refs.tolist() == refs


@pytest.mark.parametrize("first,last", [(5, 5), (5, 0), (0, 0), (5, None), (None, 0), (4, 1)])
def test_empty_ranges_are_no_fault(cuda, first, last):
    torch = cuda
    c = filled(torch, SHAPES[0], pps=5)
    table, refs = place(torch, c, [70, 16, 33, 80])
    a = ints(torch, [3])
    b = ints(torch, [first]) if first is not None else None
    d = ints(torch, [last]) if last is not None else None
    I.kv_free(c.kv, a.data_ptr(), b.data_ptr() if b is not None else 0, d.data_ptr() if d is not None else 0, 1, c.status.data_ptr())
    c.check()
    assert c.table.tolist() == table and c.refs.tolist() == refs


def test_window_eviction_of_long_tables(cuda):
    """Ranges that take more than one CTA and one trip of the grid: the pages that left a window, of a table of
    20001 entries, in every slot."""
    torch = cuda
    pps = 20001
    c = filled(torch, ("bf16", 1, 1, 8, 4), slots=3, pps=pps, spare=5)
    pages = torch.randperm(c.n_pages)[:3 * pps].to(torch.int32).view(3, pps)
    c.table.copy_(pages)
    c.refs.zero_()
    c.refs[c.table.flatten().long()] = 1
    first, last = [0, 19999, 300], [17001, 20001, 300]
    a, b, d = ints(torch, [0, 1, 2]), ints(torch, first), ints(torch, last)
    I.kv_free(c.kv, a.data_ptr(), b.data_ptr(), d.data_ptr(), 3, c.status.data_ptr())
    c.check()
    refs = torch.zeros(c.n_pages, dtype=torch.int32)
    refs[pages.flatten().long()] = 1
    for s in range(3):
        refs[pages[s, first[s]:last[s]].long()] = 0
        pages[s, first[s]:last[s]] = -1
    assert torch.equal(c.table.cpu(), pages) and torch.equal(c.refs.cpu(), refs)

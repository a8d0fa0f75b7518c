"""Page copies and forks by the thousand, against plain bookkeeping."""
import pytest

import infb200 as I
from test_kv_pages_gpu import code_of, filled, ints, place, plain_fork

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1000, 4097])
def test_thousands_of_copies(cuda, n):
    """Every pair of a long call is checked against every other: the last of them meet the first."""
    torch = cuda
    c = filled(torch, ("bf16", 2, 2, 64, 16), slots=1, pps=1, spare=2 * n + 20, seed=n)
    ids = torch.randperm(c.n_pages).tolist()
    src, dst = ids[:n], ids[n:2 * n]
    bad = {n - 1: (src[5], dst[0]),         # written by the first pair already
           n - 2: (src[6], src[1]),         # a source of the second
           n - 3: (c.n_pages, dst[n - 3]),
           n - 4: (src[n - 4], -1)}
    k, v = c.k.clone(), c.v.clone()
    good = [i for i in range(n) if i not in bad]
    k[:, [dst[i] for i in good]], v[:, [dst[i] for i in good]] = k[:, [src[i] for i in good]], v[:, [src[i] for i in good]]
    for i, (s, d) in bad.items():
        src[i], dst[i] = s, d
    a, b = ints(torch, src), ints(torch, dst)
    I.kv_copy_pages(c.kv, a.data_ptr(), b.data_ptr(), n, c.status.data_ptr())
    assert code_of(c) == 4
    assert torch.equal(c.k, k) and torch.equal(c.v, v)


def test_thousands_of_forks(cuda):
    """More forks than the plan has threads, each with a partial page of its own."""
    torch = cuda
    n, pps = 1500, 3
    c = filled(torch, ("bf16", 1, 1, 64, 16), slots=n + 4, pps=pps, spare=10, seed=1)
    table, refs = place(torch, c, [40, 33, 17, 48], seed=2)
    src, dst = [i % 4 for i in range(n)], list(range(n + 3, 3, -1))
    lens = [[40, 33, 17, 48][s] - i % 9 for i, s in enumerate(src)]
    k, v = c.k.clone(), c.v.clone()
    plain_fork(c, table, refs, k, v, src, dst, lens)
    a, b, d = ints(torch, src), ints(torch, dst), ints(torch, lens)
    I.kv_fork(c.kv, a.data_ptr(), b.data_ptr(), d.data_ptr(), n, c.scratch.data_ptr(), c.scratch.numel(), c.status.data_ptr())
    c.check()
    assert c.table.tolist() == table and c.refs.tolist() == refs
    assert torch.equal(c.k, k) and torch.equal(c.v, v)

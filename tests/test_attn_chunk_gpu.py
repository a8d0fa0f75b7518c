"""inf_attn_chunk against 64-bit attention: ragged lengths from one token on, every head layout, page
sizes, windows and sinks, with NaN in every position that no row sees and missing pages there."""
import pytest

import infb200 as I
from paged_ref import Cache, attention, visible

pytestmark = pytest.mark.gpu

SENTINEL = 7.0


class Call:
    """Buffers of one call; the rows behind the last sequence hold a sentinel."""

    def __init__(self, torch, seqs, H, KV, hd, dtype="bf16", blk=16, window=0, sinks=0, scale=0.0, seed=0, extra_rows=3,
                 pad=0, layers=1, layer=0, q_scale=1.5, max_new=None, slots=None, evict=True, spare=3):
        n = len(seqs)
        longest = max(max(ctx for _, ctx in seqs), 1)
        self.slots = slots or list(range(n))
        self.c = c = Cache(torch, max(self.slots) + 1, -(-longest // blk) + 1, KV, hd, blk, dtype, layers, spare=spare,
                           seed=seed)
        for (rows, ctx), s in zip(seqs, self.slots):
            keep = visible(rows, ctx, window, sinks) if evict else list(range(ctx))
            if rows:
                c.hold(s, keep, layer)
        self.torch, self.seqs, self.H, self.layer = torch, seqs, H, layer
        self.window, self.sinks, self.scale = window, sinks, scale
        self.tokens = sum(r for r, _ in seqs)
        total = self.tokens + extra_rows
        self.wide = (H + pad) * hd
        self.q_all = c.randn(total, self.wide, scale=q_scale)
        self.out_all = torch.full((total, self.wide), SENTINEL, dtype=c.dt, device="cuda")
        starts = [0]
        for r, _ in seqs:
            starts.append(starts[-1] + r)
        self.q_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.ctx = torch.tensor([x for _, x in seqs], dtype=torch.int32, device="cuda")
        self.slot_t = torch.tensor(self.slots, dtype=torch.int32, device="cuda")
        nb = I.attn_chunk_scratch_bytes(c.kv, n_heads=H, n_tokens=total, n_seqs=n)
        assert nb > 0
        self.scratch = torch.full((nb,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN partials, wild job records
        self.args = I.attn_chunk_args(
            d_q=self.q_all.data_ptr(), d_out=self.out_all.data_ptr(), d_q_start=self.q_start.data_ptr(),
            d_ctx_len=self.ctx.data_ptr(), d_seq_slot=self.slot_t.data_ptr(), n_seqs=n, n_tokens=total,
            max_new=max_new if max_new is not None else max(r for r, _ in seqs), n_heads=H, window=window, n_sink=sinks,
            scale=scale, q_stride=self.wide if pad else 0, out_stride=self.wide if pad else 0, layer=layer,
            d_scratch=self.scratch.data_ptr(), scratch_bytes=nb, d_status=c.status.data_ptr())

    @property
    def q(self):
        return self.q_all[:self.tokens].view(self.tokens, -1, self.c.hd)[:, :self.H]

    @property
    def out(self):
        return self.out_all[:self.tokens].view(self.tokens, -1, self.c.hd)[:, :self.H]

    def run(self, stream=0):
        I.attn_chunk(self.c.kv, self.args, stream)

    def verify(self):
        self.c.check()
        ref, tol = attention(self.c, self.q, self.seqs, self.slots, self.H, self.window, self.sinks, self.scale or None,
                             self.layer)
        err = (self.out.double() - ref).abs()
        bad = ~(err <= tol)
        assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} outputs off, first at "
                                     f"{bad.nonzero()[0].tolist()}, worst {float((err / (tol + 1e-30)).nan_to_num(9e9).max()):.2f} bounds")
        assert bool((self.out_all[self.tokens:] == SENTINEL).all()), "rows behind the last sequence were written"
        rest = self.out_all[:self.tokens].view(self.tokens, -1, self.c.hd)[:, self.H:]
        assert bool((rest == SENTINEL).all()), "padding between rows was written"


def check(torch, *a, **k):
    call = Call(torch, *a, **k)
    call.run()
    call.verify()
    return call


DECODE = [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 130), (1, 511), (1, 1000)]
MIXED = [(1, 40), (7, 7), (0, 33), (1, 1), (33, 300), (2, 129), (130, 131), (1, 700), (64, 64), (257, 900)]
LAYOUTS = [(8, 8, 64), (8, 4, 128), (32, 8, 128), (32, 4, 64), (6, 2, 128), (5, 1, 64), (14, 2, 128), (16, 1, 128), (24, 1, 64)]


@pytest.mark.parametrize("H,KV,hd", LAYOUTS)
@pytest.mark.parametrize("seqs", [DECODE, MIXED], ids=["decode", "mixed"])
def test_bf16_head_layouts(cuda, H, KV, hd, seqs):
    check(cuda, seqs, H, KV, hd, seed=H * hd)


@pytest.mark.parametrize("dtype,H,KV,hd,blk", [("fp32", 6, 6, 48, 16), ("fp32", 4, 2, 64, 16), ("fp32", 8, 1, 128, 4),
                                               ("fp32", 3, 1, 4, 1), ("fp32", 2, 2, 512, 16), ("bf16", 4, 2, 16, 16),
                                               ("bf16", 4, 1, 256, 16), ("bf16", 8, 2, 512, 16), ("bf16", 6, 3, 80, 16),
                                               ("bf16", 4, 2, 64, 8), ("bf16", 4, 2, 128, 5)])
def test_other_types_and_sizes(cuda, dtype, H, KV, hd, blk):
    check(cuda, [(1, 40), (7, 7), (0, 3), (20, 61), (1, 1), (3, 130)], H, KV, hd, dtype, blk, seed=hd + blk)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 4), (16, 0), (64, 4), (100, 20), (128, 130), (129, 1), (333, 4),
                                          (5000, 4)])
@pytest.mark.parametrize("shape", [("bf16", 8, 2, 128), ("bf16", 8, 1, 64), ("fp32", 6, 6, 48)], ids=["hd128", "hd64", "fp32"])
def test_window_and_sinks(cuda, shape, window, sinks):
    """Pages that left the window are missing, everything that no row sees is NaN."""
    dtype, H, KV, hd = shape
    seqs = [(1, 1), (1, 17), (1, 400), (1, 1000), (40, 40), (33, 500), (150, 777), (3, 64), (1, 129)]
    check(cuda, seqs, H, KV, hd, dtype, window=window, sinks=sinks, seed=window)


@pytest.mark.parametrize("blk", [16, 32, 64, 128])
def test_page_sizes(cuda, blk):
    check(cuda, MIXED, 8, 2, 128, blk=blk, seed=blk)
    check(cuda, MIXED, 8, 2, 64, blk=blk, seed=blk, window=70, sinks=3)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("seqs", [[(1, 20000)], [(16, 9000)], [(70, 12000)], [(1, 5), (1, 30000), (1, 9)], [(700, 8192)]],
                         ids=["one", "few", "some", "skewed", "chunk"])
def test_long_contexts_are_split(cuda, seqs, hd):
    check(cuda, seqs, 8, 2, hd, seed=3)
    check(cuda, seqs, 8, 2, hd, seed=4, window=2000, sinks=5)


def test_large_scores_and_a_growing_maximum(cuda):
    """Scores that reach hundreds: one key takes (almost) all weight, and the maximum keeps rising."""
    torch = cuda
    for hd, dtype in ((128, "bf16"), (64, "bf16"), (64, "fp32")):
        call = Call(torch, [(1, 700), (90, 400), (5, 30)], 8, 2, hd, dtype, q_scale=12.0, seed=9)
        ramp = torch.linspace(0.1, 3.0, 16, device="cuda").to(call.c.dt)
        call.c.k *= ramp[:, None]
        call.run()
        call.verify()


def test_rows_that_see_nothing_are_zero(cuda):
    """ctx < rows: the first rows are at negative positions."""
    torch = cuda
    for H, KV, hd, dtype in ((8, 2, 128, "bf16"), (8, 8, 64, "bf16"), (4, 4, 48, "fp32")):
        seqs = [(3, 1), (1, 0), (200, 50), (300, 0), (2, 2)]
        call = check(torch, seqs, H, KV, hd, dtype)
        assert bool((call.out[:2] == 0).all()) and bool((call.out[3] == 0).all())
        assert bool((call.out[4:4 + 150] == 0).all()) and bool((call.out[204:504] == 0).all())


def test_strides_layers_slots_and_scale(cuda):
    """Queries inside wider rows, the third layer of three, slots in another order than the sequences (one
    named twice), a scale of the caller's."""
    check(cuda, [(1, 40), (20, 60), (1, 33), (140, 200)], 8, 2, 128, pad=4, layers=3, layer=2, slots=[3, 0, 5, 1], scale=0.31)
    check(cuda, [(1, 40), (20, 60), (1, 33), (140, 200)], 8, 2, 64, pad=8, layers=2, layer=1, slots=[3, 0, 5, 1], scale=0.05)
    check(cuda, [(1, 40), (20, 60), (1, 33)], 6, 6, 48, "fp32", pad=2, layers=2, layer=1, slots=[2, 0, 1])
    torch = cuda
    call = Call(torch, [(1, 40), (30, 40)], 8, 2, 128, slots=[1, 1])
    call.run()
    call.verify()


def test_max_new_unknown_and_repeated_calls(cuda):
    """max_new 0 (the host does not know), and the same call again: bit for bit the same."""
    torch = cuda
    call = check(torch, MIXED, 8, 2, 128, max_new=0)
    first = call.out_all.clone()
    for _ in range(3):
        call.scratch.fill_(0x7F)
        call.out_all.fill_(SENTINEL)
        call.run()
        call.c.check()
        assert torch.equal(first, call.out_all)


def test_captured_and_replayed_with_new_lengths(cuda):
    """A captured call follows the lengths, tables and queries that the buffers hold at each replay."""
    torch = cuda
    H, KV, hd = 8, 2, 128
    call = Call(torch, [(40, 1000), (1, 900), (100, 300)], H, KV, hd, evict=False, max_new=140)
    call.run()  # warm-up outside the capture
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        call.run(torch.cuda.current_stream().cuda_stream)
    for seqs in ([(40, 1000), (1, 900), (100, 300)], [(1, 1), (140, 700), (0, 5)], [(2, 64), (1, 65), (138, 290)]):
        starts = [0]
        for r, _ in seqs:
            starts.append(starts[-1] + r)
        call.seqs, call.tokens = seqs, starts[-1]
        call.q_start.copy_(torch.tensor(starts, dtype=torch.int32))
        call.ctx.copy_(torch.tensor([x for _, x in seqs], dtype=torch.int32))
        call.out_all.fill_(SENTINEL)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        call.verify()


def test_on_a_stream_of_the_callers(cuda):
    torch = cuda
    s = torch.cuda.Stream()
    call = Call(torch, MIXED, 8, 2, 64)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        call.run(s.cuda_stream)
    s.synchronize()
    call.verify()


@pytest.mark.parametrize("H,KV,hd,dtype", [(8, 2, 128, "bf16"), (4, 4, 48, "fp32")])
def test_what_only_the_device_sees_is_reported(cuda, H, KV, hd, dtype):
    """A bad sequence is skipped and reported, the others are computed."""
    torch = cuda
    base = [(1, 40), (30, 60), (1, 33), (5, 50)]

    def broken(edit):
        call = Call(torch, base, H, KV, hd, dtype, seed=1)
        edit(call)
        call.run()
        with pytest.raises(I.InfError) as e:
            call.c.check()
        call.c.check()  # cleared
        return call, e.value.code

    def rest(call, skipped):
        ref, tol = attention(call.c, call.q, base, call.slots, H)
        row = 0
        for i, (n, _) in enumerate(base):
            got = call.out[row:row + n]
            if i == skipped:
                assert bool((got == SENTINEL).all())
            else:
                assert bool(((got.double() - ref[row:row + n]).abs() <= tol[row:row + n]).all())
            row += n

    call, code = broken(lambda c: c.ctx.__setitem__(1, 10_000))  # beyond the table
    assert code == 11
    rest(call, 1)
    call, code = broken(lambda c: c.ctx.__setitem__(2, -1))
    assert code == 11
    rest(call, 2)
    call, code = broken(lambda c: c.slot_t.__setitem__(0, 99))
    assert code == 11
    rest(call, 0)
    call, code = broken(lambda c: setattr(c.args, "max_new", 29))
    assert code == 4
    rest(call, 1)
    _, code = broken(lambda c: c.q_start.__setitem__(4, 10_000))  # rows outside q
    assert code == 4
    call, code = broken(lambda c: c.c.table.__setitem__((1, 0), -1))  # a page that rows see is missing
    assert code == 11
    call, code = broken(lambda c: c.c.table.__setitem__((3, 2), c.c.n_pages))
    assert code == 11


@pytest.mark.parametrize("H,KV,hd,dtype", [(8, 2, 128, "bf16"), (32, 1, 64, "bf16"), (4, 4, 48, "fp32")])
def test_starts_that_go_back_and_forth(cuda, H, KV, hd, dtype):
    """q_start 0, N, 0, N, ...: every second sequence is refused and the call reported; the rows hold what one
    of the sequences that name them computes, and the call ends."""
    torch = cuda
    n, pairs = 40, 30
    call = Call(torch, [(n, 60)] * pairs, H, KV, hd, dtype, extra_rows=0)
    call.q_start.copy_(torch.tensor([n * (i % 2) for i in range(pairs + 1)], dtype=torch.int32))
    call.run()
    with pytest.raises(I.InfError) as e:
        call.c.check()
    assert e.value.code == 4
    assert bool(call.out_all[:n].isfinite().all()) and bool((call.out_all[n:] == SENTINEL).all())


def test_costs_beyond_32_bits_are_refused(cuda):
    """The same with so many long sequences that the work would not fit 31 bits: reported, nothing written."""
    torch = cuda
    n_seqs, n, ctx = 4096, 8192, 1 << 20
    c = Cache(torch, 1, ctx // 16, 1, 64, n_pages=4)
    q = c.randn(n, 64 * 64)
    out = torch.full_like(q, SENTINEL)
    starts = torch.tensor([n * (i % 2) for i in range(n_seqs + 1)], dtype=torch.int32, device="cuda")
    lens = torch.full((n_seqs,), ctx, dtype=torch.int32, device="cuda")
    slot = torch.zeros(n_seqs, dtype=torch.int32, device="cuda")
    nb = I.attn_chunk_scratch_bytes(c.kv, n_heads=64, n_tokens=n, n_seqs=n_seqs)
    scratch = torch.empty(nb, dtype=torch.uint8, device="cuda")
    I.attn_chunk(c.kv, I.attn_chunk_args(
        d_q=q.data_ptr(), d_out=out.data_ptr(), d_q_start=starts.data_ptr(), d_ctx_len=lens.data_ptr(), d_seq_slot=slot.data_ptr(),
        n_seqs=n_seqs, n_tokens=n, n_heads=64, d_scratch=scratch.data_ptr(), scratch_bytes=nb, d_status=c.status.data_ptr()))
    with pytest.raises(I.InfError) as e:
        c.check()
    assert e.value.code == 4
    assert bool((out == SENTINEL).all())


@pytest.mark.parametrize("H,KV,hd,dtype,spare", [(32, 8, 128, "bf16", 270_000), (8, 8, 64, "fp32", 270_000)])
def test_pages_past_4_gb(cuda, H, KV, hd, dtype, spare):
    """Pools of 8.8 GB: half of the pages that a random draw takes lie beyond 32-bit byte offsets."""
    call = check(cuda, [(1, 300), (3, 40), (60, 200)], H, KV, hd, dtype, spare=spare, seed=6)
    assert int(call.c.table.max()) * KV * 16 * hd * call.c.k.element_size() > 1 << 32


@pytest.mark.parametrize("KV,hd", [(8, 128), (3, 64)])
def test_many_short_prompts_beside_a_long_one(cuda, KV, hd):
    """Items of one to three key tiles, whose own cost is as large: cuts that fall before an item's first tile."""
    check(cuda, [(69, 197)] * 10 + [(300, 1500)] + [(33, 40)] * 9 + [(1, 900), (130, 131)], 4 * KV, KV, hd, "bf16", seed=8)
    check(cuda, [(20, 20)], 4 * KV, KV, hd, "bf16", seed=9)

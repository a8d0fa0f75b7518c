"""inf_qk_norm_rope against a 64-bit norm, rotation and cache write; then, as a program uses them, the
cache's operators one after the other against 64-bit arithmetic on the same inputs."""
import pytest

import infb200 as I
from paged_ref import Cache, attention, dtype_of

pytestmark = pytest.mark.gpu

SENTINEL = 7.0


def tables(torch, n_pos, hd, theta=500000.0):
    inv = theta ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    a = torch.arange(n_pos, dtype=torch.float64)[:, None] * inv
    return a.cos().float().cuda(), a.sin().float().cuda()


class Call:
    def __init__(self, torch, tokens, H, KV, hd, dtype="bf16", blk=16, gains=(True, True), offset=0.0, eps=1e-6, pad=0,
                 layers=1, layer=0, in_place=False, slots=4, pps=8, seed=0, theta=500000.0, spare=3):
        self.torch, self.H, self.KV, self.hd, self.layer = torch, H, KV, hd, layer
        self.c = c = Cache(torch, slots, pps, KV, hd, blk, dtype, layers, spare=spare, seed=seed)
        self.tokens = tokens  # (slot, position)
        for s, p in tokens:
            if 0 <= s < slots and 0 <= p < pps * blk and int(c.table[s, p // blk]) < 0:
                c.table[s, p // blk] = c.ids.pop()
        n = len(tokens)
        self.cos, self.sin = tables(torch, pps * blk, hd, theta)
        self.wide = (H + 2 * KV + pad) * hd
        self.qkv = c.randn(n + 2, self.wide, scale=2.0)
        self.before = self.qkv.clone()
        self.q_out = self.qkv if in_place else torch.full((n + 2, (H + pad) * hd), SENTINEL, dtype=c.dt, device="cuda")
        self.gain = [(1.0 - offset + 0.3 * c.randn(hd)).to(c.dt) if g else None for g in gains]
        self.slot = torch.tensor([s for s, _ in tokens], dtype=torch.int32, device="cuda")
        self.pos = torch.tensor([p for _, p in tokens], dtype=torch.int32, device="cuda")
        self.eps, self.offset = eps, offset
        self.args = I.qk_norm_rope_args(
            d_qkv=self.qkv.data_ptr(), d_q_out=self.q_out.data_ptr(), d_cos=self.cos.data_ptr(), d_sin=self.sin.data_ptr(),
            n_pos=pps * blk, d_tok_slot=self.slot.data_ptr(), d_tok_pos=self.pos.data_ptr(), n_tokens=n, n_heads=H,
            d_q_gain=self.gain[0].data_ptr() if gains[0] else 0, d_k_gain=self.gain[1].data_ptr() if gains[1] else 0,
            eps=eps, gain_offset=offset, qkv_stride=self.wide if pad or in_place else 0,
            q_out_stride=self.q_out.shape[1] if pad or in_place else 0, layer=layer, d_status=c.status.data_ptr())

    def run(self, stream=0):
        I.qk_norm_rope(self.c.kv, self.args, stream)

    def turned(self, rows, gain):
        """(out, bound) of head rows [n][heads][hd] in 64 bits.

        fp32: the sum of squares and the root come to (hd / 2 + 4) roundings at most, the products and the
        rotation to 6 more, each of 2^-24 of |y_i cos| + |y_j sin|; cos and sin are the kernel's own inputs;
        then half a step of the output."""
        torch, hd = self.torch, self.hd
        x = rows.double()
        if gain is not None:
            x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + self.eps) * (gain.double() + self.offset)
        c, s = (t[self.pos.long()].double()[:, None] for t in (self.cos, self.sin))
        a, b = x[..., : hd // 2], x[..., hd // 2:]
        out = torch.cat((a * c - b * s, b * c + a * s), -1)
        mag = torch.cat(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()), -1)
        half = 2.0 ** -8 if self.c.name == "bf16" else 2.0 ** -24
        return out, half * out.abs() + (hd / 2 + 10) * 2.0 ** -24 * mag + 1e-40

    def verify(self):
        torch, H, KV, hd, c = self.torch, self.H, self.KV, self.hd, self.c
        c.check()
        n = len(self.tokens)
        rows = self.before[:n].view(n, -1, hd)
        q, tq = self.turned(rows[:, :H], self.gain[0])
        k, tk = self.turned(rows[:, H:H + KV], self.gain[1])
        got = self.q_out[:n].view(n, -1, hd)
        assert bool(((got[:, :H].double() - q).abs() <= tq).all())
        if self.q_out is self.qkv:
            assert torch.equal(got[:, H:], rows[:, H:]) and torch.equal(self.qkv[n:], self.before[n:])
        else:
            assert bool((got[:, H:] == SENTINEL).all()) and bool((self.q_out[n:] == SENTINEL).all())
            assert torch.equal(self.qkv, self.before)
        page, row = c.table[self.slot.long(), self.pos.long() // c.blk].long(), self.pos.long() % c.blk
        assert bool(((c.k[self.layer, page, :, row].double() - k).abs() <= tk).all())
        assert torch.equal(c.v[self.layer, page, :, row], rows[:, H + KV:H + 2 * KV])
        # nothing else in the pools was written
        c.k[self.layer, page, :, row] = float("nan")
        c.v[self.layer, page, :, row] = float("nan")
        assert bool(c.k.isnan().all()) and bool(c.v.isnan().all())


BATCH = [(0, 0), (1, 17), (2, 127), (3, 64), (0, 1), (0, 2), (1, 100)]


@pytest.mark.parametrize("H,KV,hd,dtype", [(32, 8, 128, "bf16"), (32, 4, 64, "bf16"), (6, 6, 48, "fp32"), (8, 2, 512, "bf16"),
                                           (8, 2, 512, "fp32"), (5, 1, 256, "bf16"), (3, 3, 16, "bf16"), (7, 1, 80, "bf16"),
                                           (2, 2, 8, "fp32"), (1, 1, 128, "fp32"), (9, 3, 384, "fp32")])
def test_head_layouts_and_types(cuda, H, KV, hd, dtype):
    for offset in (0.0, 1.0):
        call = Call(cuda, BATCH, H, KV, hd, dtype, offset=offset, seed=hd)
        call.run()
        call.verify()


@pytest.mark.parametrize("n", [1, 3, 500, 5000])
def test_token_counts(cuda, n):
    """From one token to enough for the kernel to keep cos and sin over several heads."""
    tokens = [(i % 3, i // 3) for i in range(n)]
    call = Call(cuda, tokens, 20, 4, 128, slots=3, pps=120, seed=n)
    call.run()
    call.verify()


@pytest.mark.parametrize("gains", [(False, False), (True, False), (False, True)])
def test_without_norms(cuda, gains):
    call = Call(cuda, BATCH, 8, 2, 128, gains=gains)
    call.run()
    call.verify()


def test_strides_in_place_layers_and_page_sizes(cuda):
    for kw in (dict(pad=2), dict(in_place=True), dict(in_place=True, pad=1), dict(layers=3, layer=2), dict(blk=1, pps=128),
               dict(blk=5, pps=30), dict(blk=64, pps=2)):
        call = Call(cuda, BATCH, 8, 2, 128, **kw)
        call.run()
        call.verify()


def test_pages_past_4_gb(cuda):
    call = Call(cuda, BATCH, 8, 8, 128, spare=270_000, seed=1)
    assert int(call.c.table.max()) * 8 * 16 * 128 * 2 > 1 << 32
    call.run()
    call.verify()


def test_rows_of_zeros_and_large_values(cuda):
    """eps 0 with ordinary rows, rows of zeros (0 / sqrt(eps)), rows of 1e15 (their squares stay finite)."""
    torch = cuda
    call = Call(torch, BATCH, 8, 2, 64, eps=1e-5, seed=2)
    call.qkv[0] = 0.0
    call.qkv[1] *= 1e15
    call.qkv[2] *= 1e-10
    call.before.copy_(call.qkv)
    call.run()
    call.verify()
    call = Call(torch, BATCH, 8, 2, 64, eps=0.0)
    call.run()
    call.verify()


def test_padding_tokens_are_left_alone(cuda):
    """Negative slots: not read, not written, not reported."""
    torch = cuda
    tokens = [(0, 3), (-1, 5), (1, 4), (-7, -3)]
    call = Call(torch, tokens, 8, 2, 128)
    call.qkv[1] = float("nan")
    call.run()
    call.c.check()
    assert bool((call.q_out[[1, 3]] == SENTINEL).all()) and not bool((call.q_out[[0, 2]] == SENTINEL).any())
    assert not bool(call.c.k[0, int(call.c.table[0, 0]), :, 3].isnan().any())
    assert int((~call.c.k.isnan()).sum()) == 2 * 2 * 128


@pytest.mark.parametrize("bad", [(4, 0), (0, 128), (0, -1), (1, 5)])
def test_what_only_the_device_sees_is_reported(cuda, bad):
    """A slot or position outside the tables, a missing page: reported; other tokens are done."""
    torch = cuda
    call = Call(torch, [(0, 3), (0, 4)], 8, 2, 128)
    call.slot[1], call.pos[1] = bad
    call.run()
    with pytest.raises(I.InfError) as e:
        call.c.check()
    assert e.value.code == 11
    assert bool((call.q_out[1] == SENTINEL).all()) == (bad != (1, 5))  # the query of a token without a page is written
    assert int((~call.c.k.isnan()).sum()) == 2 * 128


def test_captured_and_replayed(cuda):
    torch = cuda
    call = Call(torch, BATCH, 8, 2, 128)
    call.run()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call.run(torch.cuda.current_stream().cuda_stream)
    call.qkv.copy_(call.c.randn(*call.qkv.shape))
    call.before.copy_(call.qkv)
    torch.cuda.synchronize()
    graph.replay()
    call.verify()


@pytest.mark.parametrize("H,KV,hd,dtype,window,sinks", [(8, 2, 128, "bf16", 0, 0), (8, 4, 64, "bf16", 40, 4), (4, 4, 48, "fp32", 0, 0),
                                                        (6, 2, 128, "bf16", 64, 0)])
def test_a_serving_loop(cuda, H, KV, hd, dtype, window, sinks):
    """Prompts of ragged length are written and attended, then decode steps; a sequence forks and both
    copies go on; pages that left the window are freed; the pool is compacted.  At every step the
    attention over the cache equals 64-bit attention over the rows that the cache holds, and the two forks see
    the same past."""
    torch = cuda
    blk, slots, pps = 16, 4, 20
    c = Cache(torch, slots, pps, KV, hd, blk, dtype, seed=5, refs=True, spare=11)
    cos, sin = tables(torch, pps * blk, hd)
    gq, gk = c.randn(hd), c.randn(hd)
    scratch = torch.empty(I.kv_pages_scratch_bytes(c.kv), dtype=torch.uint8, device="cuda")
    m, live = torch.empty(c.n_pages, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    ctx = [0] * slots

    def grow(slot, n):
        for i in range(ctx[slot] // blk, -(-(ctx[slot] + n) // blk)):
            if int(c.table[slot, i]) < 0:
                page = int((c.refs == 0).nonzero()[0])
                c.table[slot, i], c.refs[page] = page, 1
        ctx[slot] += n

    def step(new):
        """new: {slot: tokens}; the rows of q in the order of the slots."""
        order = sorted(new)
        for s in order:
            grow(s, new[s])
        n = sum(new.values())
        qkv = c.randn(n, (H + 2 * KV) * hd)
        slot = torch.tensor([s for s in order for _ in range(new[s])], dtype=torch.int32, device="cuda")
        pos = torch.tensor([p for s in order for p in range(ctx[s] - new[s], ctx[s])], dtype=torch.int32, device="cuda")
        I.qk_norm_rope(c.kv, I.qk_norm_rope_args(
            d_qkv=qkv.data_ptr(), d_q_out=qkv.data_ptr(), qkv_stride=qkv.shape[1], q_out_stride=qkv.shape[1],
            d_cos=cos.data_ptr(), d_sin=sin.data_ptr(), n_pos=pps * blk, d_tok_slot=slot.data_ptr(), d_tok_pos=pos.data_ptr(),
            n_tokens=n, n_heads=H, d_q_gain=gq.data_ptr(), d_k_gain=gk.data_ptr(), gain_offset=1.0, d_status=c.status.data_ptr()))
        seqs = [(new[s], ctx[s]) for s in order]
        starts = [0]
        for r, _ in seqs:
            starts.append(starts[-1] + r)
        q_start, lens, which = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (starts, [x for _, x in seqs], order))
        out = torch.empty(n, H * hd, dtype=c.dt, device="cuda")
        nb = I.attn_chunk_scratch_bytes(c.kv, n_heads=H, n_tokens=n, n_seqs=len(seqs))
        ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
        I.attn_chunk(c.kv, I.attn_chunk_args(
            d_q=qkv.data_ptr(), q_stride=qkv.shape[1], d_out=out.data_ptr(), d_q_start=q_start.data_ptr(), d_ctx_len=lens.data_ptr(),
            d_seq_slot=which.data_ptr(), n_seqs=len(seqs), n_tokens=n, max_new=max(new.values()), n_heads=H, window=window,
            n_sink=sinks, d_scratch=ws.data_ptr(), scratch_bytes=nb, d_status=c.status.data_ptr()))
        c.check()
        q = qkv.view(n, -1, hd)[:, :H]
        ref, tol = attention(c, q, seqs, order, H, window, sinks)
        assert bool(((out.view(n, H, hd).double() - ref).abs() <= tol).all())

    def evict():
        """Pages wholly between the sinks and the window of the next token."""
        if not window:
            return
        rng = [(s, -(-sinks // blk), max(-(-sinks // blk), (ctx[s] + 1 - window) // blk)) for s in range(slots) if ctx[s]]
        a, b, d = (torch.tensor([r[i] for r in rng], dtype=torch.int32, device="cuda") for i in range(3))
        I.kv_free(c.kv, a.data_ptr(), b.data_ptr(), d.data_ptr(), len(rng), c.status.data_ptr())
        c.check()

    step({0: 37, 1: 150, 2: 1})
    step({0: 1, 1: 1, 2: 30})
    evict()
    step({0: 1, 1: 1, 2: 1})
    src, dst, n = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (1, 3, ctx[1]))
    I.kv_fork(c.kv, src.data_ptr(), dst.data_ptr(), n.data_ptr(), 1, scratch.data_ptr(), scratch.numel(), c.status.data_ptr())
    c.check()
    ctx[3] = ctx[1]
    past = c.k[0, c.table[3].long().clamp(min=0), :].clone()
    assert torch.equal(past[: ctx[1] // blk], c.k[0, c.table[1].long().clamp(min=0), :][: ctx[1] // blk])
    step({1: 1, 3: 2})
    first = torch.tensor([0], dtype=torch.int32, device="cuda")
    I.kv_free(c.kv, first.data_ptr(), 0, 0, 1, c.status.data_ptr())
    ctx[0] = 0
    I.kv_compact(c.kv, m.data_ptr(), live.data_ptr(), scratch.data_ptr(), scratch.numel(), c.status.data_ptr())
    c.check()
    assert int(live) == int((c.refs > 0).sum()) and bool((c.refs[int(live):] == 0).all())
    step({0: 20, 1: 1, 2: 17, 3: 1})
    evict()
    step({0: 1, 1: 1, 2: 1, 3: 1})

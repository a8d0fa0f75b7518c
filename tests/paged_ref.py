"""Plain 64-bit PyTorch forms of the paged-cache operators, and the buffers of their tests (a helper
module, not a test file)."""
import infb200 as I


def dtype_of(torch, name):
    return {"bf16": torch.bfloat16, "fp32": torch.float32}[name]


class Cache:
    """A paged cache of `layers` layers with one sequence per slot; the pools start as NaN, so whatever is
    read without having been written shows."""

    def __init__(self, torch, slots, pps, KV, hd, blk=16, dtype="bf16", layers=1, spare=3, seed=0, n_pages=None, refs=False):
        self.torch, self.KV, self.hd, self.blk, self.name = torch, KV, hd, blk, dtype
        self.dt = dtype_of(torch, dtype)
        self.n_pages = n_pages or slots * pps + spare
        self.layers = layers
        self.k = torch.full((layers, self.n_pages, KV, blk, hd), float("nan"), dtype=self.dt, device="cuda")
        self.v = torch.full_like(self.k, float("nan"))
        self.table = torch.full((slots, pps), -1, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(self.n_pages, dtype=torch.int32, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.ids = torch.randperm(self.n_pages, generator=self.g, device="cuda").tolist()
        self.kv = self.descriptor()

    def descriptor(self):
        return I.paged_kv(self.k.data_ptr(), self.v.data_ptr(), n_pages=self.n_pages, n_kv_heads=self.KV, head_dim=self.hd,
                          kv_block=self.blk, dtype=I.BF16 if self.name == "bf16" else I.F32,
                          d_block_table=self.table.data_ptr(), n_slots=self.table.shape[0],
                          pages_per_seq=self.table.shape[1], d_page_refs=self.refs.data_ptr(), n_layers=self.layers,
                          layer_stride=self.k.stride(0) * self.k.element_size())

    def randn(self, *shape, scale=1.0):
        return (self.torch.randn(*shape, generator=self.g, device="cuda") * scale).to(self.dt)

    def hold(self, slot, positions, layer=0):
        """Pages for `positions` (a sorted list) of the slot, filled at those positions."""
        torch = self.torch
        pos = torch.tensor(sorted(positions), device="cuda", dtype=torch.long)
        if pos.numel() == 0:
            return
        for i in torch.unique(pos // self.blk).tolist():
            if int(self.table[slot, i]) < 0:
                self.table[slot, i] = self.ids.pop()
        page = self.table[slot].long()[pos // self.blk]
        self.k[layer, page, :, pos % self.blk] = self.randn(pos.numel(), self.KV, self.hd)
        self.v[layer, page, :, pos % self.blk] = self.randn(pos.numel(), self.KV, self.hd)

    def check(self):
        I.check_status(self.status.data_ptr())


def visible(n, ctx, window, sinks):
    """Positions that some row of the sequence sees."""
    if ctx <= 0:
        return []
    lo = max(0, ctx - n - window + 1) if window else 0
    return [k for k in range(ctx) if k >= lo or k < sinks]


def attention(cache, q, seqs, slots, H, window=0, sinks=0, scale=None, layer=0):
    """(out, bound on each output's error) of the rows of q [tokens][H][hd] in 64 bits.  seqs: (rows, ctx).

    With A = sum p |V| / sum p, the bound counts, for a kernel that accumulates in fp32:
      scores   (hd + 8) roundings of 2^-24 of sum |q||k| scale, twice (numerator and denominator);
      sums     one rounding of 2^-24 per key, and 2^-20 for the exponentials;
      bf16     half a step (2^-8) of every weight for the second product on the tensor cores;
      output   half a step of the result."""
    torch = cache.torch
    hd, KV, blk = cache.hd, cache.KV, cache.blk
    G = H // KV
    scale = hd ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape[0], H, hd, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    half = 2.0 ** -8 if cache.name == "bf16" else 2.0 ** -24
    row = 0
    for (n, ctx), slot in zip(seqs, slots):
        seen = visible(n, ctx, window, sinks)
        if n and seen:
            pos = torch.tensor(seen, device="cuda")
            page = cache.table[slot].long()[pos // blk]
            k = cache.k[layer, page, :, pos % blk].double().transpose(0, 1)  # [KV][keys][hd]
            v = cache.v[layer, page, :, pos % blk].double().transpose(0, 1)
            p = torch.arange(ctx - n, ctx, device="cuda")[:, None]
            mask = pos <= p
            if window:
                mask &= (pos > p - window) | (pos < sinks)
            qq = q[row:row + n].double().reshape(n, KV, G, hd).permute(1, 2, 0, 3)  # [KV][G][n][hd]
            s = torch.einsum("kgnd,kcd->kgnc", qq, k) * scale
            s = s.masked_fill(~mask, float("-inf"))
            m = s.amax(-1, keepdim=True)
            w = torch.exp(s - torch.where(m.isinf(), torch.zeros_like(m), m))
            l = w.sum(-1, keepdim=True)
            l = torch.where(l == 0, torch.ones_like(l), l)
            o = torch.einsum("kgnc,kcd->kgnd", w, v) / l
            a = torch.einsum("kgnc,kcd->kgnd", w, v.abs()) / l
            mag = torch.einsum("kgnd,kcd->kgnc", qq.abs(), k.abs()).amax(-1, keepdim=True) * scale
            e = 2 * (hd + 8) * 2.0 ** -24 * mag + len(seen) * 2.0 ** -24 + 2.0 ** -20
            if cache.name == "bf16":
                e = e + 2.0 ** -8
            t = o.abs() * half + a * e
            out[row:row + n] = o.permute(2, 0, 1, 3).reshape(n, H, hd)
            tol[row:row + n] = t.permute(2, 0, 1, 3).reshape(n, H, hd)
        row += n
    return out, tol

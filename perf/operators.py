"""The paged-cache operators, case by case: what they are measured on.

Three operators of a serving step over the paged KV cache, in plain torch (`own` false) and as a
program calls them (`own` true):

  rope   the projected rows of new tokens: RMSNorm of every query and key head, rotation by the
         token's position, queries out, keys and values into the cache's pages
  attn   attention of every sequence's new tokens (one, a few, or a whole chunk) over its pages,
         causal, optionally with a sliding window and a few first tokens that stay visible
  pages  what a scheduler does to the cache between steps: copying pages, freeing sequences and
         forking others into their slots, compacting the pool

A cache is, per layer, K and V pools [pages][kv_heads][16][head_dim], one block table
[slots][pages per sequence] (-1: no page) and one reference count per page.
"""
import os
import random
import sys

import torch

own = False

BLOCK = 16  # positions per page, as in every configuration of this repository
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------ cases
def listed():
    # heads of the Llama-3-8B, TinyLlama-1.1B and tiny fp32 decoders of this repository
    big = dict(heads=32, kv_heads=8, head_dim=128, dtype="bf16")
    small = dict(heads=32, kv_heads=4, head_dim=64, dtype="bf16")
    tiny = dict(heads=6, kv_heads=6, head_dim=48, dtype="fp32")
    full = dict(window=0, sinks=0)
    return [
        # one sequence's next token: the latency a single user waits for in every layer
        dict(name="attn_decode_one", op="attn", **big, decodes=1, chunks=0, new_lo=1, new_hi=1, ctx_lo=513, ctx_hi=513,
             shape_seed=1, **full),
        # a full batch of decoding sequences with the contexts of the batched-decode workload
        dict(name="attn_decode_batch", op="attn", **big, decodes=64, chunks=0, new_lo=1, new_hi=1, ctx_lo=512,
             ctx_hi=4096, shape_seed=2, **full),
        # continuous batching: most sequences decode, a few prompts of ragged length are being read
        dict(name="attn_mixed", op="attn", **big, decodes=24, chunks=8, new_lo=2, new_hi=701, ctx_lo=90, ctx_hi=5003,
             shape_seed=3, **full),
        # the second prefill chunk of a long prompt
        dict(name="attn_chunk", op="attn", **big, decodes=0, chunks=1, new_lo=4096, new_hi=4096, ctx_lo=8192, ctx_hi=8192,
             shape_seed=4, **full),
        # long conversations held to a window, their early pages already freed, decoding
        dict(name="attn_window_decode", op="attn", **small, decodes=48, chunks=0, new_lo=1, new_hi=1, ctx_lo=700,
             ctx_hi=32768, shape_seed=5, window=1024, sinks=4),
        # two long prompts being read under a window
        dict(name="attn_window_chunk", op="attn", **big, decodes=0, chunks=2, new_lo=1801, new_hi=2300, ctx_lo=9001,
             ctx_hi=16384, shape_seed=6, window=2048, sinks=4),
        # the fp32 decoder: short prompts and decodes together
        dict(name="attn_fp32", op="attn", **tiny, decodes=12, chunks=6, new_lo=2, new_hi=40, ctx_lo=41, ctx_hi=256,
             shape_seed=7, **full),
        # one token of the fp32 decoder: the smallest call there is
        dict(name="rope_one_fp32", op="rope", **tiny, decodes=1, chunks=0, new_lo=1, new_hi=1, ctx_lo=77, ctx_hi=77,
             shape_seed=8, gain_offset=0),
        # a prefill chunk with a few decodes beside it
        dict(name="rope_chunk", op="rope", **big, decodes=7, chunks=1, new_lo=8192, new_hi=8192, ctx_lo=8192, ctx_hi=8300,
             shape_seed=9, gain_offset=1),
        # prompt pages copied for sequences about to diverge
        dict(name="pages_copy", op="copy", layers=22, kv_heads=4, head_dim=64, dtype="bf16", n_pages=600, n=37, shape_seed=10),
        # a beam step: half of the sequences are dropped, the others fork into their slots
        dict(name="pages_beam", op="beam", layers=22, kv_heads=4, head_dim=64, dtype="bf16", n_pages=2600, n_slots=64, n=32,
             ctx_lo=17, ctx_hi=1000, pages_per_seq=64, shape_seed=11),
        # a cache after hours of serving, half of its pool holes, brought together
        dict(name="pages_compact", op="compact", layers=22, kv_heads=4, head_dim=64, dtype="bf16", n_pages=3001, n_slots=48,
             ctx_lo=17, ctx_hi=1000, pages_per_seq=64, shape_seed=12),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _draw_attn(rng):
    c = dict(op="attn", shape_seed=rng.randrange(1 << 30))
    if rng.random() < 0.15:  # the fp32 decoder's kind
        kv = rng.choice([1, 2, 3, 6])
        c.update(heads=kv * rng.choice([1, 2, 4]), kv_heads=kv, head_dim=rng.choice([32, 48, 64]), dtype="fp32")
        c.update(decodes=rng.randint(0, 24), chunks=rng.randint(1, 8), new_lo=1, new_hi=_spread(rng, 2, 60))
        c.update(ctx_lo=c["new_hi"], ctx_hi=c["new_hi"] + _spread(rng, 1, 400))
    else:
        kv = rng.choice([1, 2, 4, 8])
        c.update(heads=kv * rng.choice([1, 2, 3, 4, 5, 7, 8]), kv_heads=kv, head_dim=rng.choice([64, 128, 128]), dtype="bf16")
        kind = rng.choice(["decode", "decode", "mixed", "chunk"])
        if kind == "decode":
            c.update(decodes=_spread(rng, 1, 128), chunks=0, new_lo=1, new_hi=1, ctx_lo=1)
            c["ctx_hi"] = _spread(rng, 40, 16384 if c["decodes"] < 32 else 5000)
        elif kind == "mixed":
            c.update(decodes=rng.randint(1, 40), chunks=rng.randint(1, 12), new_lo=1, new_hi=_spread(rng, 2, 900))
            c.update(ctx_lo=c["new_hi"], ctx_hi=c["new_hi"] + _spread(rng, 16, 6000))
        else:
            c.update(decodes=0, chunks=rng.randint(1, 2), new_lo=_spread(rng, 100, 1500))
            c["new_hi"] = c["new_lo"] + rng.randint(0, 1500)
            c.update(ctx_lo=c["new_hi"], ctx_hi=c["new_hi"] + _spread(rng, 16, 8000))
    c.update(window=0, sinks=0)
    if rng.random() < 0.35:
        c.update(window=_spread(rng, 16, 3500), sinks=rng.choice([0, 1, 4, 4, 20]))
    return c


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "attn", "rope", "rope", "copy", "beam", "compact"])
    if kind == "attn":
        while True:
            c = _draw_attn(rng)
            if work(c)["flops"] <= 3e11 and work(c)["bytes"] <= 7e8:
                return c
    if kind == "rope":
        c = dict(op="rope", shape_seed=rng.randrange(1 << 30), gain_offset=rng.choice([0, 1]))
        if rng.random() < 0.2:
            kv = rng.choice([1, 3, 6])
            c.update(heads=kv * rng.choice([1, 2]), kv_heads=kv, head_dim=rng.choice([32, 48, 64]), dtype="fp32")
        else:
            kv = rng.choice([1, 2, 4, 8])
            c.update(heads=kv * rng.choice([1, 3, 4, 7, 8]), kv_heads=kv, head_dim=rng.choice([64, 128, 128, 256]), dtype="bf16")
        c.update(decodes=rng.randint(0, 64), chunks=rng.randint(1, 3), new_lo=1, new_hi=_spread(rng, 2, 1200))
        c.update(ctx_lo=c["new_hi"], ctx_hi=c["new_hi"] + _spread(rng, 16, 5000))
        return c
    c = dict(op=kind, shape_seed=rng.randrange(1 << 30), layers=rng.randint(1, 24), kv_heads=rng.choice([1, 2, 4, 8]),
             head_dim=rng.choice([48, 64, 128]), dtype=rng.choice(["bf16", "bf16", "fp32"]))
    if kind == "copy":
        c.update(n=_spread(rng, 1, 60))
        c.update(n_pages=2 * c["n"] + rng.randint(0, 100))
    else:
        c.update(n_slots=_spread(rng, 2, 64), ctx_lo=1, ctx_hi=_spread(rng, 30, 700))
        c.update(pages_per_seq=-(-c["ctx_hi"] // BLOCK) + rng.randint(0, 9))
        c.update(n_pages=c["n_slots"] * (-(-c["ctx_hi"] // BLOCK) + 1))
        if kind == "beam":
            c["n"] = c["n_slots"] // 2
    if c["layers"] * c["n_pages"] * _page_bytes(c) * 2 > 1_000_000_000:
        c["layers"] = max(1, 500_000_000 // (c["n_pages"] * _page_bytes(c)))
    return c


# ------------------------------------------------------------------------------ shapes
def _page_bytes(c):
    return c["kv_heads"] * BLOCK * c["head_dim"] * (2 if c["dtype"] == "bf16" else 4)


def _sequences(c):
    """(new tokens, context with them) of every sequence, decodes and chunks shuffled together."""
    r = random.Random(c["shape_seed"])
    out = []
    for i in range(c["decodes"] + c["chunks"]):
        new = 1 if i < c["decodes"] else r.randint(c["new_lo"], c["new_hi"])
        out.append((new, max(new, r.randint(c["ctx_lo"], c["ctx_hi"]))))
    r.shuffle(out)
    return out


def _first_visible(c, new, ctx):
    """The first position past the sinks that some new token of the sequence sees."""
    return max(0, ctx - new - c["window"] + 1) if c["window"] else 0


def _lengths(c):
    """Context lengths of a page case's sequences."""
    r = random.Random(c["shape_seed"])
    return [r.randint(c["ctx_lo"], c["ctx_hi"]) for _ in range(c["n_slots"])]


def _beam(c):
    """(slots dropped, slots that fork, the length each fork keeps) of a beam step."""
    lens, r = _lengths(c), random.Random(c["shape_seed"] + 1)
    order = list(range(c["n_slots"]))
    r.shuffle(order)
    drop, stay = order[: c["n"]], order[c["n"]:]
    src = [stay[r.randrange(len(stay))] for _ in drop]  # one sequence may fork more than once
    return drop, src, [lens[s] for s in src]


def work(case):
    """Bytes and floating-point operations of one pass."""
    c, op = case, case["op"]
    if op in ("attn", "rope"):
        size = 2 if c["dtype"] == "bf16" else 4
        seqs = _sequences(c)
        tokens = sum(n for n, _ in seqs)
        row = c["head_dim"] * size
        if op == "rope":
            heads = c["heads"] + 2 * c["kv_heads"]
            rotated = tokens * (c["heads"] + c["kv_heads"]) * c["head_dim"]
            return {"bytes": 2 * tokens * heads * row + tokens * c["head_dim"] * 4 + tokens * 8, "flops": 8 * rotated}
        seen = keys = 0
        for new, ctx in seqs:
            first = _first_visible(c, new, ctx)
            keys += ctx - first + min(c["sinks"], first)
            for p in range(ctx - new, ctx):
                lo = max(0, p - c["window"] + 1) if c["window"] else 0
                seen += p + 1 - lo + min(c["sinks"], lo)
        return {"bytes": 2 * tokens * c["heads"] * row + 2 * keys * c["kv_heads"] * row,
                "flops": 4 * seen * c["heads"] * c["head_dim"]}
    page = 2 * c["layers"] * _page_bytes(c)
    if op == "copy":
        return {"bytes": 2 * c["n"] * page + 8 * c["n"], "flops": 0}
    if op == "beam":
        rows = sum(n % BLOCK for n in _beam(c)[2])
        table = sum(-(-n // BLOCK) for n in _beam(c)[2]) * 4
        return {"bytes": 2 * rows * page // BLOCK + 3 * table + c["n_pages"] * 4, "flops": 0}
    table, refs = _pool_state(c)
    live = sum(r > 0 for r in refs)
    moved = sum(r > 0 for r in refs[live:])
    return {"bytes": 2 * moved * page + 4 * c["n_pages"] + 8 * sum(p >= live for row in table for p in row), "flops": 0}


def _pool_state(c):
    """Block table and reference counts of a page case: sequences placed at random in the pool, and in a
    compaction some that share their first pages."""
    r = random.Random(c["shape_seed"] + 2)
    free = list(range(c["n_pages"]))
    r.shuffle(free)
    table = [[-1] * c["pages_per_seq"] for _ in range(c["n_slots"])]
    refs = [0] * c["n_pages"]
    for s, n in enumerate(_lengths(c)):
        shared = 0
        if c["op"] == "compact" and s % 3 == 2:
            shared = min(n, _lengths(c)[s - 1]) // BLOCK // 2
        for i in range(-(-n // BLOCK)):
            page = table[s - 1][i] if i < shared else free.pop()
            table[s][i] = page
            refs[page] += 1
    return table, refs


# ------------------------------------------------------------------------------ inputs
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pool(g, shape, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": c}
    if c["op"] in ("attn", "rope"):
        _prepare_tokens(c, g, s, int(seed))
    else:
        _prepare_pages(c, g, s, int(seed))
    if own:
        _prepare_own(c, s)
    return s


def _prepare_tokens(c, g, s, seed):
    dt = DTYPES[c["dtype"]]
    H, KV, hd = c["heads"], c["kv_heads"], c["head_dim"]
    seqs = _sequences(c)
    tokens, longest = sum(n for n, _ in seqs), max(ctx for _, ctx in seqs)
    per_seq = -(-longest // BLOCK) + 1
    held = []  # the pages each sequence still holds: those of the sinks and of the window
    for new, ctx in seqs:
        first = _first_visible(c, new, ctx) if c["op"] == "attn" else 0
        sinks = c.get("sinks", 0)
        held.append([i for i in range(-(-ctx // BLOCK)) if (i + 1) * BLOCK > first or i * BLOCK < sinks])
    n_pages = sum(map(len, held)) + 3
    ids = list(range(n_pages))
    random.Random(seed).shuffle(ids)
    table = torch.full((len(seqs), per_seq), -1, dtype=torch.int32)
    for i, idx in enumerate(held):
        table[i, idx] = torch.tensor([ids.pop() for _ in idx], dtype=torch.int32)
    starts = [0]
    for new, _ in seqs:
        starts.append(starts[-1] + new)
    if c["op"] == "attn":
        s["at"] = [(_ints(idx)[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")).flatten() for idx in held]
        s["pages"] = [table[i, idx].cuda().long() for i, idx in enumerate(held)]
    s.update(seqs=seqs, starts=starts, tokens=tokens, n_pages=n_pages, per_seq=per_seq, table=table.cuda(),
             q_start=_ints(starts), ctx_len=_ints([ctx for _, ctx in seqs]), max_new=max(n for n, _ in seqs))
    s["k"] = _pool(g, (n_pages, KV, BLOCK, hd), dt)
    s["v"] = _pool(g, (n_pages, KV, BLOCK, hd), dt)
    s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if c["op"] == "attn":
        s["q"] = (torch.randn(tokens, H, hd, device="cuda", generator=g) * 1.5).to(dt)
        s["out"] = torch.empty_like(s["q"])
        return
    s["qkv"] = (torch.randn(tokens, H + 2 * KV, hd, device="cuda", generator=g) * 2).to(dt)
    gain = 1.0 - c["gain_offset"]
    s["q_gain"] = (gain + 0.2 * torch.randn(hd, device="cuda", generator=g)).to(dt)
    s["k_gain"] = (gain + 0.2 * torch.randn(hd, device="cuda", generator=g)).to(dt)
    inv = 500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    angle = torch.arange(longest, dtype=torch.float64)[:, None] * inv
    s["cos"], s["sin"] = angle.cos().float().cuda(), angle.sin().float().cuda()
    s["tok_slot"] = _ints([i for i, (new, _) in enumerate(seqs) for _ in range(new)])
    s["tok_pos"] = _ints([p for new, ctx in seqs for p in range(ctx - new, ctx)])
    s["q_out"] = torch.empty(tokens, H, hd, dtype=dt, device="cuda")


def _prepare_pages(c, g, s, seed):
    dt = DTYPES[c["dtype"]]
    shape = (c["layers"], c["n_pages"], c["kv_heads"], BLOCK, c["head_dim"])
    s["k"], s["v"] = _pool(g, shape, dt), _pool(g, shape, dt)
    s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if c["op"] == "copy":
        ids = list(range(c["n_pages"]))
        random.Random(seed).shuffle(ids)
        s["src"], s["dst"] = _ints(ids[: c["n"]]), _ints(ids[c["n"]: 2 * c["n"]])
        return
    table, refs = _pool_state(c)
    s["table_now"], s["refs_now"] = _ints(table), _ints(refs)  # the scheduler's copy, taken at every step
    s["table"], s["refs"] = torch.empty_like(s["table_now"]), torch.empty_like(s["refs_now"])
    if c["op"] == "beam":
        drop, src, keep = _beam(c)
        part = [i for i, n in enumerate(keep) if n % BLOCK]  # the forks that end inside a page: that one is copied
        s.update(drop=_ints(drop), src=_ints(src), keep=_ints(keep), part=_ints(part).long(),
                 part_last=_ints([keep[i] // BLOCK for i in part]).long(), part_rows=_ints([keep[i] % BLOCK for i in part]))
    else:
        s["map"] = torch.empty(c["n_pages"], dtype=torch.int32, device="cuda")
        s["n_live"] = torch.zeros(1, dtype=torch.int32, device="cuda")


def _library():
    folder = os.path.join(os.getcwd(), "inference-project_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import infb200
    return infb200


def _prepare_own(c, s):
    """The descriptors a program builds once beside its cache and buffers."""
    I = _library()
    s["lib"] = I
    layers = c.get("layers", 1)
    n_pages = s["k"].shape[-4]
    s["kv"] = kv = I.paged_kv(
        s["k"].data_ptr(), s["v"].data_ptr(), n_pages=n_pages, n_kv_heads=c["kv_heads"], head_dim=c["head_dim"],
        kv_block=BLOCK, dtype=I.BF16 if c["dtype"] == "bf16" else I.F32,
        d_block_table=s["table"].data_ptr() if "table" in s else 0, n_slots=s["table"].shape[0] if "table" in s else 0,
        pages_per_seq=s["table"].shape[1] if "table" in s else 0, d_page_refs=s["refs"].data_ptr() if "refs" in s else 0,
        n_layers=layers, layer_stride=s["k"].stride(0) * s["k"].element_size() if layers > 1 else 0)
    if c["op"] == "attn":
        nb = I.attn_chunk_scratch_bytes(kv, n_heads=c["heads"], n_tokens=s["tokens"], n_seqs=len(s["seqs"]))
        s["scratch"] = torch.empty(max(nb, 16), dtype=torch.uint8, device="cuda")
        s["args"] = I.attn_chunk_args(
            d_q=s["q"].data_ptr(), d_out=s["out"].data_ptr(), d_q_start=s["q_start"].data_ptr(),
            d_ctx_len=s["ctx_len"].data_ptr(), n_seqs=len(s["seqs"]), n_tokens=s["tokens"], max_new=s["max_new"],
            n_heads=c["heads"], window=c["window"], n_sink=c["sinks"], d_scratch=s["scratch"].data_ptr(),
            scratch_bytes=nb, d_status=s["status"].data_ptr())
    elif c["op"] == "rope":
        s["args"] = I.qk_norm_rope_args(
            d_qkv=s["qkv"].data_ptr(), d_q_out=s["q_out"].data_ptr(), d_q_gain=s["q_gain"].data_ptr(),
            d_k_gain=s["k_gain"].data_ptr(), eps=1e-6, gain_offset=float(c["gain_offset"]), d_cos=s["cos"].data_ptr(),
            d_sin=s["sin"].data_ptr(), n_pos=s["cos"].shape[0], d_tok_slot=s["tok_slot"].data_ptr(),
            d_tok_pos=s["tok_pos"].data_ptr(), n_tokens=s["tokens"], n_heads=c["heads"], d_status=s["status"].data_ptr())
    elif c["op"] != "copy":
        nb = I.kv_pages_scratch_bytes(kv)
        s["scratch"] = torch.empty(nb, dtype=torch.uint8, device="cuda")


# ------------------------------------------------------------------------------ one pass
def run(state):
    c, s = state["case"], state
    op = c["op"]
    if op in ("beam", "compact"):  # the scheduler's tables of this step
        s["table"].copy_(s["table_now"])
        s["refs"].copy_(s["refs_now"])
    if own:
        return _run_own(c, s)
    return {"attn": _plain_attn, "rope": _plain_rope, "copy": _plain_copy, "beam": _plain_beam,
            "compact": _plain_compact}[op](c, s)


def _run_own(c, s):
    I, op = s["lib"], c["op"]
    stream = torch.cuda.current_stream().cuda_stream
    status = s["status"].data_ptr()
    if op == "attn":
        I.attn_chunk(s["kv"], s["args"], stream)
        return s["out"]
    if op == "rope":
        I.qk_norm_rope(s["kv"], s["args"], stream)
        return s["q_out"], s["k"], s["v"]
    if op == "copy":
        I.kv_copy_pages(s["kv"], s["src"].data_ptr(), s["dst"].data_ptr(), c["n"], status, stream)
        return s["k"], s["v"]
    scratch, nb = s["scratch"].data_ptr(), s["scratch"].numel()
    if op == "beam":
        I.kv_free(s["kv"], s["drop"].data_ptr(), 0, 0, c["n"], status, stream)
        I.kv_fork(s["kv"], s["src"].data_ptr(), s["drop"].data_ptr(), s["keep"].data_ptr(), c["n"], scratch, nb, status,
                  stream)
        return s["table"], s["refs"], s["k"], s["v"]
    I.kv_compact(s["kv"], s["map"].data_ptr(), s["n_live"].data_ptr(), scratch, nb, status, stream)
    return s["table"], s["refs"], s["map"], s["n_live"], s["k"], s["v"]


def _plain_attn(c, s):
    H, KV, hd = c["heads"], c["kv_heads"], c["head_dim"]
    G, W, sinks = H // KV, c["window"], c["sinks"]
    for i, (new, ctx) in enumerate(s["seqs"]):
        at, pages = s["at"][i], s["pages"][i]  # the positions of the pages that the sequence still holds
        k = s["k"][pages].float().transpose(0, 1).reshape(KV, -1, hd)
        v = s["v"][pages].float().transpose(0, 1).reshape(KV, -1, hd)
        v = torch.where((at < ctx)[:, None], v, torch.zeros_like(v))
        pos = torch.arange(ctx - new, ctx, device="cuda")[:, None]
        seen = at <= pos
        if W:
            seen = seen & ((at > pos - W) | (at < sinks))
        q = s["q"][s["starts"][i]: s["starts"][i + 1]].float().view(new, KV, G, hd)
        out = s["out"][s["starts"][i]: s["starts"][i + 1]].view(new, KV, G, hd)
        step = KV if new * at.numel() * H < 1 << 26 else 1  # KV heads at a time
        for h in range(0, KV, step):
            score = torch.einsum("nkgd,kcd->kgnc", q[:, h:h + step], k[h:h + step]) * hd ** -0.5
            score = torch.where(seen, score, torch.full_like(score, float("-inf")))
            p = torch.exp(score - score.amax(-1, keepdim=True))
            o = torch.einsum("kgnc,kcd->nkgd", p, v[h:h + step])
            out[:, h:h + step] = (o / p.sum(-1).permute(2, 0, 1)[..., None]).to(out.dtype)
    return s["out"]


def _plain_rope(c, s):
    H, KV, hd = c["heads"], c["kv_heads"], c["head_dim"]
    x = s["qkv"].float()
    pos, slot = s["tok_pos"].long(), s["tok_slot"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turned(rows, gain):
        y = rows * torch.rsqrt(rows.square().mean(-1, keepdim=True) + 1e-6) * (gain.float() + c["gain_offset"])
        a, b = y[..., : hd // 2], y[..., hd // 2:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    s["q_out"].copy_(turned(x[:, :H], s["q_gain"]))
    page, row = s["table"][slot, pos // BLOCK].long(), pos % BLOCK
    s["k"][page, :, row] = turned(x[:, H: H + KV], s["k_gain"]).to(s["k"].dtype)
    s["v"][page, :, row] = s["qkv"][:, H + KV:]
    return s["q_out"], s["k"], s["v"]


def _plain_copy(c, s):
    for pool in (s["k"], s["v"]):
        pool[:, s["dst"].long()] = pool[:, s["src"].long()]
    return s["k"], s["v"]


def _plain_beam(c, s):
    table, refs = s["table"], s["refs"]
    drop, src = s["drop"].long(), s["src"].long()
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    gone = table[drop]
    refs.index_put_((gone.clamp(min=0).long(),), torch.where(gone >= 0, -one, 0 * one), accumulate=True)
    table[drop] = -1
    before = table[src]
    at = torch.arange(table.shape[1], device="cuda")
    full = (s["keep"] // BLOCK)[:, None]
    row = torch.where(at < full, before, -one)
    refs_was_free = refs == 0
    refs.index_put_((row.clamp(min=0).long(),), torch.where(row >= 0, one, 0 * one), accumulate=True)
    which, last = s["part"], s["part_last"]
    fresh = torch.argsort((~refs_was_free).to(torch.uint8), stable=True)[: which.numel()]
    old = before[which, last].long()
    row[which, last] = fresh.to(torch.int32)
    refs[fresh] = 1
    kept = (torch.arange(BLOCK, device="cuda") < s["part_rows"][:, None])[None, :, None, :, None]
    for pool in (s["k"], s["v"]):
        pool[:, fresh] = torch.where(kept, pool[:, old], pool[:, fresh])
    table[drop] = row
    return table, refs, s["k"], s["v"]


def _plain_compact(c, s):
    table, refs = s["table"], s["refs"]
    live = refs > 0
    at = torch.arange(c["n_pages"], device="cuda")
    n_live = live.sum()
    old = torch.nonzero(live & (at >= n_live)).flatten()
    new = torch.nonzero(~live & (at < n_live)).flatten()
    moved = at.to(torch.int32)
    moved[old] = new.to(torch.int32)
    s["map"].copy_(torch.where(live, moved, torch.full_like(moved, -1)))
    for pool in (s["k"], s["v"]):
        pool[:, new] = pool[:, old]
    table.copy_(torch.where(table >= 0, s["map"][table.clamp(min=0).long()], table))
    refs[new] = refs[old]
    refs[old] = 0
    s["n_live"].copy_(n_live)
    return table, refs, s["map"], s["n_live"], s["k"], s["v"]


# ------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The computed outputs from their definitions in 64 bits (nothing is computed by the page cases)."""
    c = dict(case)
    if c["op"] not in ("attn", "rope"):
        return None
    s = {}
    _prepare_tokens(c, torch.Generator(device="cuda").manual_seed(int(seed)), s, int(seed))
    return (_exact_attn if c["op"] == "attn" else _exact_rope)(c, s)


def _exact_attn(c, s):
    H, hd, group = c["heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    out = torch.zeros(s["tokens"], H, hd, dtype=torch.float64, device="cuda")
    for i, (new, ctx) in enumerate(s["seqs"]):
        first = _first_visible(c, new, ctx)
        where = torch.tensor(list(range(min(c["sinks"], first))) + list(range(first, ctx)), device="cuda")
        page = s["table"][i].long()[where // BLOCK]
        for h in range(H):
            keys = s["k"][page, h // group, where % BLOCK].double()
            values = s["v"][page, h // group, where % BLOCK].double()
            for t in range(0, new, 1024):
                u = min(new, t + 1024)
                query = s["q"][s["starts"][i] + t: s["starts"][i] + u, h].double()
                when = torch.arange(ctx - new + t, ctx - new + u, device="cuda").unsqueeze(1)
                hidden = where > when
                if c["window"]:
                    hidden |= (when - where >= c["window"]) & (where >= c["sinks"])
                logits = (query @ keys.T / hd ** 0.5).masked_fill_(hidden, float("-inf"))
                logits = (logits - logits.max(1, keepdim=True).values).exp_()
                out[s["starts"][i] + t: s["starts"][i] + u, h] = logits @ values / logits.sum(1, keepdim=True)
    return out


def _exact_rope(c, s):
    H, KV, half = c["heads"], c["kv_heads"], c["head_dim"] // 2
    out = torch.zeros(s["tokens"], H, 2 * half, dtype=torch.float64, device="cuda")
    k, v = s["k"].double(), s["v"].double()
    pos = s["tok_pos"].long()
    angle = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())
    page = s["table"][s["tok_slot"].long(), pos // BLOCK].long()
    for h in range(H + 2 * KV):
        x = s["qkv"][:, h].double()
        if h >= H + KV:
            v[page, h - H - KV, pos % BLOCK] = x
            continue
        gain = (s["q_gain"] if h < H else s["k_gain"]).double() + c["gain_offset"]
        x = x / (x.pow(2).sum(1, keepdim=True) / (2 * half) + 1e-6).sqrt() * gain
        z = torch.complex(x[:, :half], x[:, half:]) * angle
        x = torch.cat((z.real, z.imag), 1)
        if h < H:
            out[:, h] = x
        else:
            k[page, h - H, pos % BLOCK] = x
    return out, k, v

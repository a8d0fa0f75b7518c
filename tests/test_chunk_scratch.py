"""The scratch of inf_attn_chunk asked for once, for the most tokens and sequences."""
import itertools

import pytest

import infb200 as I

SEQS = (1, 2, 3, 64, 85, 86, 146, 147, 256, 512, 1000, 2048, 4096)
TOKENS = (1, 2, 64, 255, 1024, 8192)


@pytest.mark.parametrize("dtype", [I.BF16, I.F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("hd", [8, 16, 48, 64, 80, 96, 128, 256, 320, 512])
@pytest.mark.parametrize("H,KV,blk,pps", [(32, 8, 16, 256), (6, 6, 16, 8), (5, 1, 8, 1000)])
def test_no_smaller_call_asks_for_more(dtype, hd, H, KV, blk, pps):
    """Every type and head size, sequence counts around those where a kernel's shared memory admits a CTA less on an
    SM: more tokens or more sequences never need less."""
    kv = I.paged_kv(0, 0, n_pages=10, n_kv_heads=KV, head_dim=hd, kv_block=blk, dtype=dtype, n_slots=4096, pages_per_seq=pps)
    size = {(t, s): I.attn_chunk_scratch_bytes(kv, n_heads=H, n_tokens=t, n_seqs=s) for t, s in itertools.product(TOKENS, SEQS)}
    assert min(size.values()) > 0
    for i, t in enumerate(TOKENS):
        for j, s in enumerate(SEQS):
            if i:
                assert size[t, s] >= size[TOKENS[i - 1], s], (t, s)
            if j:
                assert size[t, s] >= size[t, SEQS[j - 1]], (t, s)

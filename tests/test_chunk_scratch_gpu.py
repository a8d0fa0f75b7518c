"""A scratch of inf_attn_chunk sized for the most sequences serves calls of fewer."""
import pytest

import infb200 as I
from test_attn_chunk_gpu import Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,H,KV,hd,most", [("bf16", 8, 2, 96, 256), ("bf16", 4, 2, 80, 4096), ("fp32", 8, 2, 64, 512)])
def test_sized_once_for_the_most_sequences(cuda, dtype, H, KV, hd, most):
    torch = cuda
    call = Call(torch, [(1, 900), (7, 7), (0, 33), (33, 300), (2, 129)] + [(1, 50 + 17 * i) for i in range(30)], H, KV, hd, dtype, seed=hd)
    nb = I.attn_chunk_scratch_bytes(call.c.kv, n_heads=H, n_tokens=8192, n_seqs=most)
    assert nb >= I.attn_chunk_scratch_bytes(call.c.kv, n_heads=H, n_tokens=8192, n_seqs=len(call.seqs))
    scratch = torch.full((nb + 4096,), 0xFF, dtype=torch.uint8, device="cuda")
    call.args.scratch, call.args.scratch_bytes = scratch.data_ptr(), nb
    call.run()
    call.verify()
    assert bool((scratch[nb:] == 0xFF).all())

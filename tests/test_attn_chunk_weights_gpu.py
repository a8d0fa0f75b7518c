"""How many bits of the softmax weights reach the second product of inf_attn_chunk where few rows attend."""
import math

import pytest

from paged_ref import attention
from test_attn_chunk_gpu import Call

pytestmark = pytest.mark.gpu


def worst_weights(torch):
    """Two scores x in [-1, 0), bf16 values, whose weights e^x lie furthest above and below their bf16 roundings."""
    x = (-torch.arange(1, 129, dtype=torch.float64) / 128).to(torch.bfloat16).double()
    w = torch.exp(x)
    off = (w.to(torch.bfloat16).double() - w) / w
    assert off.max() > 2.0 ** -10 and off.min() < -2.0 ** -10
    return float(x[off.argmax()]), float(x[off.argmin()])


@pytest.mark.parametrize("H,KV,hd", [(32, 8, 128), (32, 4, 64), (8, 8, 128), (16, 1, 64)])
@pytest.mark.parametrize("window", [0, 700])
def test_weights_of_few_rows_keep_16_bits(cuda, H, KV, hd, window):
    """Weights that round up belong to values of +1, weights that round down to values of about -1: the outputs
    nearly cancel, the roundings of the weights add up.

    The bound counts two bf16 parts of a weight (2^-8 of what 2^-8 left over: 2^-16), beside what the scores,
    the fp32 sums and the output's rounding can cost.  Weights of one part would be off by about 2^-9."""
    torch = cuda
    seqs = [(1, 40), (1, 600), (1, 2000), (1, 17), (max(1, 16 // (H // KV)), 300), (1, 1)]
    call = Call(torch, seqs, H, KV, hd, window=window, scale=1.0, seed=H + hd, evict=False)
    c = call.c
    up, down = worst_weights(torch)
    back = -math.exp(up) / math.exp(down)
    call.q_all.zero_()
    call.q.copy_(torch.zeros_like(call.q))
    call.q[..., 0] = 1.0
    for (_, ctx), slot in zip(seqs, call.slots):
        pos = torch.arange(ctx, device="cuda")
        page, row = c.table[slot].long()[pos // c.blk], pos % c.blk
        score = torch.where(pos % 2 == 0, up, down)
        value = torch.where(pos % 2 == 0, 1.0, back)
        every = pos % 64 == 63  # the row's maximum, with no say in the output
        k = torch.zeros(ctx, KV, hd, device="cuda")
        k[:, :, 0] = torch.where(every, 0.0, score)[:, None]
        c.k[0, page, :, row] = k.to(c.dt)
        c.v[0, page, :, row] = torch.where(every, 0.0, value)[:, None, None].expand(ctx, KV, hd).to(c.dt)
    call.run()
    call.c.check()
    got = call.out.double()
    ref, _ = attention(c, call.q, seqs, call.slots, H, window, 0, 1.0)
    c.v.abs_()
    size, _ = attention(c, call.q, seqs, call.slots, H, window, 0, 1.0)  # sum p |V| / sum p
    keys = max(ctx for _, ctx in seqs)
    bound = ref.abs() * 2.0 ** -8 + size * (2 * (hd + 8) * 2.0 ** -24 + keys * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -16)
    err = (got - ref).abs()
    assert bool((err <= bound).all()), f"worst {float((err / bound).max()):.2f} bounds"

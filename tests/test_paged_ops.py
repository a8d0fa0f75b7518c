"""What the paged-cache operators refuse on the host, without a GPU: every shape rule answers before a
pointer is looked at, and host pointers are refused before anything is launched."""
import ctypes as C

import pytest

import infb200 as I

BUF = C.create_string_buffer(4096)
HOST = (C.addressof(BUF) + 255) & ~255  # host memory, aligned: never device memory


def cache(**kw):
    d = dict(d_kpool=HOST, d_vpool=HOST, n_pages=10, n_kv_heads=2, head_dim=64, kv_block=16, dtype=I.BF16, d_block_table=HOST,
             n_slots=3, pages_per_seq=4, d_page_refs=HOST)
    d.update(kw)
    return I.paged_kv(d.pop("d_kpool"), d.pop("d_vpool"), **d)


def attn(kv, **kw):
    d = dict(d_q=HOST, d_out=HOST + 16, d_q_start=HOST, d_ctx_len=HOST, n_seqs=2, n_tokens=5, n_heads=4, d_scratch=HOST,
             scratch_bytes=1 << 40)
    d.update(kw)
    I.attn_chunk(kv, I.attn_chunk_args(**d))


def rope(kv, **kw):
    d = dict(d_qkv=HOST, d_q_out=HOST + 16, d_cos=HOST, d_sin=HOST, n_pos=64, d_tok_slot=HOST, d_tok_pos=HOST, n_tokens=5,
             n_heads=4, d_q_gain=HOST, d_k_gain=HOST)
    d.update(kw)
    I.qk_norm_rope(kv, I.qk_norm_rope_args(**d))


def refused(code, f, *a, **k):
    with pytest.raises(I.InfError) as e:
        f(*a, **k)
    assert e.value.code == code, str(e.value)


OPS = {
    "attn": attn,
    "rope": rope,
    "copy": lambda kv: I.kv_copy_pages(kv, HOST, HOST, 2),
    "free": lambda kv: I.kv_free(kv, HOST, 0, 0, 2),
    "fork": lambda kv: I.kv_fork(kv, HOST, HOST, HOST, 2, HOST, 1 << 30),
    "compact": lambda kv: I.kv_compact(kv, HOST, HOST, HOST, 1 << 30),
}


@pytest.mark.parametrize("op", OPS)
def test_cache_shapes(op):
    f = OPS[op]
    for bad in (dict(dtype=7), dict(n_pages=0), dict(n_kv_heads=0), dict(head_dim=0), dict(kv_block=0), dict(n_layers=0),
                dict(n_layers=2, layer_stride=24), dict(n_layers=2, layer_stride=16)):
        refused(4, f, cache(**bad))
    refused(15, f, cache(head_dim=60))   # rows of 120 bytes
    refused(15, f, cache(n_kv_heads=60000, kv_block=65536, head_dim=64))  # pages of 2 GB and more
    if op != "copy":
        for bad in (dict(n_slots=0), dict(pages_per_seq=0), dict(pages_per_seq=1 << 30)):
            refused(4, f, cache(**bad))
    refused(4, f, cache(d_kpool=HOST + 8))  # alignment
    refused(6, f, cache())                  # host memory


def test_null_arguments():
    L = I.lib()
    kv = cache()
    assert L.inf_attn_chunk(None, I.InfAttnChunk(n_heads=4), None) == 4
    assert L.inf_attn_chunk(kv, None, None) == 4
    assert L.inf_qk_norm_rope(None, I.InfQkNormRope(n_heads=4), None) == 4
    assert L.inf_qk_norm_rope(kv, None, None) == 4
    assert L.inf_kv_copy_pages(None, None, None, 1, None, None) == 4
    assert L.inf_kv_free(None, None, None, None, 1, None, None) == 4
    assert L.inf_kv_fork(None, None, None, None, 1, None, 0, None, None) == 4
    assert L.inf_kv_compact(None, None, None, None, 0, None, None) == 4
    assert L.inf_attn_chunk_scratch_bytes(None, 4, 5, 2) == 0
    assert L.inf_kv_pages_scratch_bytes(None) == 0
    assert L.inf_check_status(None, None) == 6


def test_attention_arguments():
    refused(4, attn, cache(), n_heads=0)
    refused(4, attn, cache(), n_heads=5)         # not a multiple of the KV heads
    refused(4, attn, cache(), n_seqs=4097)
    refused(15, attn, cache(head_dim=520))
    assert I.attn_chunk_scratch_bytes(cache(), n_heads=5, n_tokens=5, n_seqs=2) == 0
    assert I.attn_chunk_scratch_bytes(cache(), n_heads=4, n_tokens=5, n_seqs=2) > 0


def test_scratch_covers_every_smaller_call():
    """A scratch sized for the most tokens and sequences serves any call of fewer."""
    for H, hd, dtype in ((4, 64, I.BF16), (8, 128, I.BF16), (2, 48, I.F32)):
        kv = cache(head_dim=hd, dtype=dtype, pages_per_seq=100)
        sizes = [I.attn_chunk_scratch_bytes(kv, n_heads=H, n_tokens=t, n_seqs=s) for t, s in
                 ((1, 1), (5, 2), (64, 64), (65, 64), (700, 64), (8192, 64), (8192, 100))]
        assert sizes == sorted(sizes) and sizes[0] > 0

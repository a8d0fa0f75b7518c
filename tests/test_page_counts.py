"""Caches whose pages have more pieces than the page operators count: refused on the host, without a GPU."""
import pytest

import infb200 as I
from test_paged_ops import OPS, cache, refused


@pytest.mark.parametrize("op", ["copy", "fork", "compact"])
@pytest.mark.parametrize("shape", [dict(n_layers=1 << 31, n_kv_heads=1, kv_block=1, head_dim=8),     # 2 pieces a layer
                                   dict(n_layers=1 << 30, n_kv_heads=1, kv_block=1, head_dim=8),
                                   dict(n_layers=1 << 15, n_kv_heads=65535, kv_block=1, head_dim=8),  # a fork's pieces are heads
                                   dict(n_layers=1 << 13, n_kv_heads=1, kv_block=65536, head_dim=8192)])
def test_more_pieces_than_31_bits(op, shape):
    page = shape["n_kv_heads"] * shape["kv_block"] * shape["head_dim"] * 2
    refused(15, OPS[op], cache(dtype=I.BF16, n_pages=10, layer_stride=10 * page, **shape))


@pytest.mark.parametrize("op", ["copy", "fork", "compact"])
def test_one_layer_of_many_heads_is_taken(op):
    refused(6, OPS[op], cache(n_layers=2, n_kv_heads=65535, kv_block=1, head_dim=8, layer_stride=10 * 65535 * 16))  # (host memory)

"""A prompt that continues a cached prefix: the cache read back as the tree
attention's keys and values, against the attention over the cache itself."""
import pytest

from test_decode_gpu import _gen, _i32, _randn
from test_decode_limits_gpu import ROW

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prefix,new", [(1, 1), (37, 5), (300, 90), (2100, 40)])
@pytest.mark.parametrize("window", [2047, 50])
def test_tree_attention_over_a_cached_prefix(cuda, prefix, new, window):
    import torch

    from aps2026_b200 import decode, ops

    g, n, q_heads, kv_heads, dim, page = _gen(prefix), prefix + new, 16, 4, 128, 16
    width = -(-n // page)
    table = torch.randperm(width, generator=g, device="cuda").to(torch.int32).view(1, width)
    cache = decode.KVCache4(width, page, kv_heads, dim, "cuda")
    cos, sin = (t.to("cuda") for t in ops.rope_table_host(n, dim, ops.ROPE_THETA))
    seq, pos = _i32([0] * n), _i32(list(range(n)))
    q, k, v = _randn(g, new, q_heads, dim), _randn(g, n, kv_heads, dim), _randn(g, n, kv_heads, dim)
    decode.kv4_append_gpu(k[:prefix], v[:prefix], seq[:prefix], pos[:prefix], cache, table, cos=cos, sin=sin)
    decode.kv4_append_gpu(k[prefix:], v[prefix:], seq[prefix:], pos[prefix:], cache, table, q=q, q_out=q, cos=cos, sin=sin)
    over_cache = torch.empty_like(q)
    decode.attention_kv4_gpu(q, cache, table, _i32([n]), over_cache, q_offsets=_i32([0, new]), max_queries=new,
                             window=window)
    # the prefix's rows are rows of the tree, with queries of no interest
    held_k, held_v = torch.empty_like(k), torch.empty_like(v)
    decode.kv4_read_gpu(cache, table, seq, pos, held_k, held_v)
    rows = torch.cat([torch.zeros(prefix, q_heads, dim, device="cuda"), q])
    chains = torch.arange(n, device="cuda", dtype=torch.int32).repeat(n, 1)
    out = torch.empty_like(rows)
    ops.attention_tree_gpu(rows, held_k, held_v, out, pos, chains, n, n, q_heads, kv_heads, dim, window=window)
    # the tree attention is held to 1e-5
    off = (out[prefix:] - over_cache).double().norm() / over_cache.double().norm()
    assert float(off) < 1e-5 + ROW and ops.device_status() == 0

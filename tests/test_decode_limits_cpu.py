"""What the decode operators refuse or hold without a GPU: buffers smaller than
their objects say."""
import pytest

from aps2026_b200 import decode, ops


def _table():
    import torch

    return torch.zeros(1, 2, dtype=torch.int32)


@pytest.mark.parametrize("change", [dict(pages=3), dict(pages=2 ** 32 - 2), dict(page_size=16), dict(kv_heads=2), dict(head_dim=128),
                                    dict(data=slice(1)), dict(data=(slice(None), slice(0, None, 2)))])
def test_a_cache_smaller_than_it_says_is_refused(change):
    import torch

    cache = decode.KVCache4(2, 8, 1, 64, "cpu")
    if "data" in change:
        change = dict(data=cache.data[change["data"]])
    for name, value in change.items():
        setattr(cache, name, value)
    k, i = torch.zeros(1, cache.kv_heads, cache.head_dim), torch.zeros(1, dtype=torch.int32)
    ws = type("Workspace", (), dict(buf=torch.zeros(8), bytes=32))()
    for call in (lambda: decode.kv4_append_gpu(k, k, i, i, cache, _table()),
                 lambda: decode.kv4_read_gpu(cache, _table(), i, i, k, k),
                 lambda: decode.attention_kv4_gpu(k, cache, _table(), i, k, ws=ws)):
        with pytest.raises(ops.InvalidArgument, match="cache: expected"):
            call()

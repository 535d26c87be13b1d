"""Refusals of the decode operators' C entry points before any device work,
and the sizes they report."""
import ctypes as C

import pytest

from aps2026_b200 import _lib, decode, ops

BAD = _lib.B2_ERR_INVALID_ARGUMENT


def _cache(**kw):
    f = dict(data=None, pages=0, page_size=16, kv_heads=2, head_dim=128, page_table=None, seqs=0, max_pages=0)
    f.update(kw)
    return decode._CacheStruct(*f.values())


def _page_bytes(*a):
    n = C.c_size_t(0)
    rc = _lib.lib().b2_kv4_page_bytes(*a, C.addressof(n))
    return n.value if rc == 0 else rc


@pytest.mark.parametrize("page,heads,dim,want", [(16, 4, 128, 16 * 4 * 144), (8, 1, 64, 8 * 72), (64, 3, 64, 64 * 3 * 72)])
def test_page_bytes(page, heads, dim, want):
    assert _page_bytes(page, heads, dim) == want


@pytest.mark.parametrize("kw,word", [(dict(page_size=12), "page_size"), (dict(page_size=4), "page_size"),
                                     (dict(head_dim=80), "head_dim"), (dict(kv_heads=0), "kv_heads"),
                                     (dict(pages=1), "null"), (dict(seqs=1, max_pages=1), "null"),
                                     (dict(data=8, pages=1), "aligned"), (dict(pages=1 << 33, data=16), "32 bits")])
def test_cache_description_is_checked(kw, word):
    lib, c = _lib.lib(), _cache(**kw)
    assert lib.b2_kv4_read(C.byref(c), None, None, 0, None, None, 0, None) == BAD
    assert word in _lib.last_error()
    assert lib.b2_kv4_append(None, 0, 0, 0, None, None, 0, 0, None, 0, 0, 0, 0, None, None, None, None, 0, C.byref(c),
                             None) == BAD
    assert lib.b2_attention_kv4(None, 0, 0, None, 0, 1, 2, None, None, 1, 1, 1.0, 0, 0, C.byref(c), None, 0, None) == BAD


def test_null_and_empty():
    lib, c = _lib.lib(), _cache()
    args = lambda rows, dtype=0, cos=None: (None, 0, 0, 0, None, None, 0, 0, None, 0, 0, dtype, rows, None, None, cos,  # noqa: E731
                                            None, 0, C.byref(c), None)
    assert lib.b2_kv4_append(*args(0)) == 0
    assert lib.b2_kv4_append(*args(3)) == BAD
    assert lib.b2_kv4_append(*args(3, dtype=2)) == BAD
    assert lib.b2_kv4_append(*args(0, cos=16)) == BAD
    assert lib.b2_kv4_read(C.byref(c), None, None, 0, None, None, 0, None) == 0
    assert lib.b2_kv4_read(C.byref(c), None, None, 2, None, None, 0, None) == BAD
    assert lib.b2_kv4_read(None, None, None, 2, None, None, 0, None) == BAD
    attn = lambda **kw: lib.b2_attention_kv4(*{**dict(  # noqa: E731
        q=None, rs=0, hs=0, out=None, dtype=0, rows=0, heads=4, off=None, lens=None, mq=1, ml=1, scale=1.0, w=0, s=0,
        cache=C.byref(c), ws=None, wb=0, stream=None), **kw}.values())
    assert attn() == 0
    assert attn(heads=3) == BAD and "multiple" in _lib.last_error()
    assert attn(dtype=7) == BAD


def test_moe_decode_arguments():
    lib, n = _lib.lib(), C.c_size_t(0)
    call = lambda **kw: lib.b2_moe_decode(*{**dict(  # noqa: E731
        x=None, ldx=64, xd=0, lg=None, T=2, H=64, E=4, I=16, q=1e-3, t=2e-2, gates=0, gu=None, dn=None, wd=0, out=None,
        ldo=64, ws=None, wb=0, stream=None), **kw}.values())
    assert call() == BAD and "null" in _lib.last_error()
    assert call(E=33) == BAD and call(E=1) == BAD and call(xd=2) == BAD and call(wd=2) == BAD and call(gates=2) == BAD
    assert call(ldx=63) == BAD and call(H=0) == BAD
    assert call(T=0) == 0
    assert call(T=129) == _lib.B2_ERR_UNSUPPORTED
    assert lib.b2_moe_decode_workspace_size(128, 448, C.addressof(n)) == 0 and n.value >= 2 * 128 * 448 * 4
    assert lib.b2_moe_decode_workspace_size(129, 448, C.addressof(n)) == BAD
    assert lib.b2_attention_kv4_workspace_size(96, C.addressof(n)) == BAD
    assert lib.b2_attention_kv4_workspace_size(128, C.addressof(n)) == 0 and n.value > 0


def test_host_tensors_are_refused():
    import torch

    x = torch.zeros(2, 64)
    with pytest.raises(ops.InvalidArgument):
        decode.moe_decode_gpu(x, torch.zeros(2, 4), torch.zeros(4, 32, 64), torch.zeros(4, 64, 16), x.clone())
    cache = decode.KVCache4(1, 8, 1, 64, "cpu")
    with pytest.raises(ops.InvalidArgument):
        decode.kv4_append_gpu(torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), torch.zeros(1, dtype=torch.int32),
                              torch.zeros(1, dtype=torch.int32), cache, torch.zeros(1, 1, dtype=torch.int32))


def test_python_calls_refuse_what_is_no_tensor_or_not_on_a_gpu():
    import torch

    x = torch.zeros(2, 8)
    for bad in (x, None, "x"):
        with pytest.raises(ops.InvalidArgument):
            decode.moe_decode_gpu(bad, x, x, x.view(2, 2, 4), x, ws=decode.MoeWorkspace(2, 4, "cpu"))
    with pytest.raises(ops.InvalidArgument):
        decode.moe_decode_gpu(x, x, x, x.view(2, 2, 4), x)
    with pytest.raises(TypeError):
        decode._decode_calls.moe_decode(x)

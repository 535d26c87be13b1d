"""The decode operators where memory is least convenient: rows that start
anywhere, tensors inside others, scales of every sign, arguments that are no
tensors."""
import math

import pytest

from test_decode_gpu import _gen, _moe64, _randn

pytestmark = pytest.mark.gpu


def _inside_nan(t, offset, after=5):
    """t as a contiguous view that starts `offset` elements into a buffer of NaN."""
    import torch

    buf = torch.full((offset + t.numel() + after,), float("nan"), dtype=t.dtype, device=t.device)
    view = buf[offset:offset + t.numel()].view(t.shape)
    return view.copy_(t)


@pytest.mark.parametrize("T", [1, 6, 40, 100])
@pytest.mark.parametrize("H,I,E", [(264, 37, 4), (263, 40, 4), (2501, 37, 3), (2504, 33, 5), (40, 250, 2), (31, 3, 32)])
@pytest.mark.parametrize("xt,wt", [("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("float32", "float32"),
                                   ("bfloat16", "float32")])
@pytest.mark.parametrize("offset", [0, 1, 6])
def test_moe_rows_that_start_anywhere(cuda, T, H, I, E, xt, wt, offset):
    """Nothing around a tensor or between its rows (all NaN) is let in."""
    import torch

    from aps2026_b200 import decode

    g = _gen(T * H + I + offset)
    gu = _inside_nan((_randn(g, E, 2 * I, H) / math.sqrt(H)).to(getattr(torch, wt)), offset)
    dn = _inside_nan((_randn(g, E, H, I) / math.sqrt(I)).to(getattr(torch, wt)), offset)
    wide = torch.full((T, H + 3 * offset), float("nan"), dtype=getattr(torch, xt), device="cuda")
    x = wide[:, offset:offset + H].copy_(_randn(g, T, H))
    logits = _randn(g, T, E)
    out = torch.full((T, H + offset), float("nan"), dtype=x.dtype, device="cuda")
    decode.moe_decode_gpu(x, logits, gu, dn, out[:, :H])
    want, mag = _moe64(x, logits, gu, dn, 1e-3, 2e-2, "equal")
    # sums of inputs held to 16 bits or more, as for aligned rows
    bound = 2.0 ** -14 * (mag + mag.mean()) + (2.0 ** -8 * want.abs() if xt == "bfloat16" else 0)
    assert bool(((out[:, :H].double() - want).abs() <= bound).all())
    assert bool(out[:, H:].isnan().all())


def _filled(g, lens, page, kv_heads, dim):
    import torch

    from aps2026_b200 import decode

    width = -(-max(lens) // page)
    table = torch.randperm(len(lens) * width, generator=g, device="cuda").to(torch.int32).view(len(lens), width)
    cache = decode.KVCache4(len(lens) * width, page, kv_heads, dim, "cuda")
    seq = torch.cat([torch.full((n,), s, dtype=torch.int32, device="cuda") for s, n in enumerate(lens)])
    pos = torch.cat([torch.arange(n, dtype=torch.int32, device="cuda") for n in lens])
    k, v = _randn(g, seq.numel(), kv_heads, dim), _randn(g, seq.numel(), kv_heads, dim)
    decode.kv4_append_gpu(k, v, seq, pos, cache, table)
    decode.kv4_read_gpu(cache, table, seq, pos, k, v)
    return cache, table, k, v


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30, 4.0])
@pytest.mark.parametrize("q_heads", [4, 16])
def test_attention_scales(cuda, scale, q_heads):
    import torch

    from aps2026_b200 import decode

    g, n = _gen(q_heads), 777
    cache, table, k, v = _filled(g, [n], 16, 2, 64)
    q = _randn(g, 1, q_heads, 64)
    out = torch.empty_like(q)
    decode.attention_kv4_gpu(q, cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"), out, scale=scale)
    w = torch.softmax(q.double().view(2, -1, 64) @ k.double().permute(1, 2, 0) * scale, -1)
    want = (w @ v.double().transpose(0, 1)).view(out.shape)
    mag = (w @ v.double().abs().transpose(0, 1)).view(out.shape)
    # scores reach 4 * 64 * 3^2 = 2^11 and carry 2^-20 of their terms' size
    bound = 2.0 ** -14 + max(1.0, scale) * 64 * 9 * 2.0 ** -20
    assert bool(((out.double() - want).abs() <= bound * (mag + 0.1)).all())


def test_attention_refuses(cuda):
    import torch

    from aps2026_b200 import decode, ops

    g = _gen(1)
    cache, table, _, _ = _filled(g, [20], 8, 2, 64)
    q = _randn(g, 1, 4, 64)
    lens = torch.tensor([20], dtype=torch.int32, device="cuda")
    ok = dict(q=q, cache=cache, page_table=table, lens=lens, out=torch.empty_like(q))
    for bad in (dict(scale=float("nan")), dict(scale=float("inf")), dict(max_len=2 ** 29), dict(max_queries=2 ** 40),
                dict(max_queries=0), dict(window=-1), dict(sinks=-1), dict(q=[1.0]), dict(lens=None),
                dict(out=torch.empty(1, 4, 64)), dict(ws=decode.AttentionWorkspace(64, "cpu"))):
        with pytest.raises(ops.InvalidArgument):
            decode.attention_kv4_gpu(**{**ok, **bad})
    with pytest.raises(TypeError):
        decode.attention_kv4_gpu(**{**ok, "max_queries": 1.5})
    decode.attention_kv4_gpu(**ok)
    assert bool(ok["out"].isfinite().all()) and ops.device_status() == 0


@pytest.mark.parametrize("q_heads", [4, 16])
def test_attention_queries_of_any_size(cuda, q_heads):
    """Queries times 2^k at a scale of 2^-k are the same queries, bit for bit."""
    import torch

    from aps2026_b200 import decode

    g, n = _gen(q_heads + 7), 333
    cache, table, _, _ = _filled(g, [n], 16, 2, 64)
    q, lens = _randn(g, 1, q_heads, 64), torch.tensor([n], dtype=torch.int32, device="cuda")
    want = torch.empty_like(q)
    decode.attention_kv4_gpu(q, cache, table, lens, want, scale=0.125)
    assert bool(want.isfinite().all())
    for k in (-90, 60, 115):
        out = torch.empty_like(q)
        decode.attention_kv4_gpu(q * 2.0 ** k, cache, table, lens, out, scale=0.125 * 2.0 ** -k)
        assert torch.equal(out, want), k

"""The decode step's operators (aps2026_b200.decode) against 64-bit
restatements: the 4-bit cache's append and read, the attention over it, and
the expert layer for few tokens."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

GROUP = 64


def _gen(seed):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    import torch

    return torch.randn(shape, generator=g, device="cuda")


def _i32(v):
    import torch

    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _status():
    from aps2026_b200 import ops

    return ops.device_status()


def _held(x):
    """What the cache holds for fp32 rows x [..., D], in numpy fp32, each
    operation rounded on its own."""
    import torch

    f = np.float32
    x = x.float().cpu().numpy().astype(f)
    shape = x.shape
    x = x.reshape(*shape[:-1], shape[-1] // GROUP, GROUP)
    bf = lambda a: torch.from_numpy(np.ascontiguousarray(a)).bfloat16().float().numpy()  # noqa: E731
    m = bf(x.min(-1))
    s = bf(np.maximum(x.max(-1) - m, f(0)) * f(1.0 / 15.0))
    with np.errstate(divide="ignore"):
        inv = np.where(s < f(2.0 ** -126), f(0), f(1) / s).astype(f)
    c = np.clip(np.rint((x - m[..., None]) * inv[..., None]), 0, 15).astype(f)
    return (c * s[..., None] + m[..., None]).reshape(shape)


def _rotate32(x, cos, sin):
    """x [rows, heads, D] fp32 numpy; cos, sin [rows, D/2]."""
    h = x.shape[-1] // 2
    a, b, c, s = x[..., :h], x[..., h:], cos[:, None], sin[:, None]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def _cache(pages, page, heads, dim):
    from aps2026_b200 import decode

    return decode.KVCache4(pages, page, heads, dim, "cuda")


def _table(seqs, width, pages, seed=0):
    """A page table handing `pages` >= seqs * width pages out in random order."""
    import torch

    order = torch.randperm(pages, generator=_gen(seed), device="cuda").to(torch.int32)
    return order[: seqs * width].reshape(seqs, width).contiguous()


# ---- append and read --------------------------------------------------------------


@pytest.mark.parametrize("dim,page,heads,q_heads", [(128, 16, 4, 16), (128, 8, 1, 3), (64, 64, 3, 6), (64, 8, 8, 8)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 5, 300])
def test_append_then_read_is_the_formula(cuda, dim, page, heads, q_heads, dtype, rows):
    import torch

    from aps2026_b200 import decode

    dt = getattr(torch, dtype)
    g = _gen(rows)
    q, k, v = (_randn(g, rows, h, dim).to(dt) for h in (q_heads, heads, heads))
    k[..., 3] *= 9
    seq = torch.arange(rows, device="cuda", dtype=torch.int32) % 3
    pos = (torch.arange(rows, device="cuda", dtype=torch.int32) // 3) + 11
    width = (11 + rows // 3 + page) // page + 1
    table = _table(3, width, 3 * width)
    cache = _cache(3 * width, page, heads, dim)
    angle = torch.rand(11 + rows // 3 + 1, dim // 2, generator=g, device="cuda") * 6.28
    cos, sin = torch.cos(angle), torch.sin(angle)
    q_out = torch.full_like(q, float("nan"))
    decode.kv4_append_gpu(k, v, seq, pos, cache, table, q=q, q_out=q_out, cos=cos, sin=sin)
    ko, vo = (torch.full((rows, heads, dim), float("nan"), device="cuda") for _ in range(2))
    decode.kv4_read_gpu(cache, table, seq, pos, ko, vo)
    at = pos.cpu().numpy()
    c, s = cos.cpu().numpy()[at], sin.cpu().numpy()[at]
    rot = lambda t: torch.from_numpy(_rotate32(t.float().cpu().numpy(), c, s))  # noqa: E731
    assert torch.equal(q_out.cpu(), rot(q).to(dt))
    assert torch.equal(ko.cpu(), torch.from_numpy(_held(rot(k))))
    assert torch.equal(vo.cpu(), torch.from_numpy(_held(v)))
    # the value held is within half a step of the value, plus what the bf16 step costs at code 15
    x = v.float().view(rows, heads, dim // GROUP, GROUP)
    span = (x.amax(-1) - x.amin(-1) + 2.0 ** -8 * x.abs().amax(-1)) / 15
    worst = (vo.view_as(x) - x).abs().amax(-1)
    assert bool((worst <= span * 0.54).all())
    kb, vb = (torch.empty(rows, heads, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    decode.kv4_read_gpu(cache, table, seq, pos, kb, vb)
    assert torch.equal(kb, ko.bfloat16()) and torch.equal(vb, vo.bfloat16())
    assert _status() == 0


@pytest.mark.parametrize("layout", ["fused", "head_major", "offset"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_append_takes_strides(cuda, layout, dtype):
    import torch

    from aps2026_b200 import decode

    dt = getattr(torch, dtype)
    rows, heads, qh, dim, page = 37, 2, 6, 128, 16
    g = _gen(5)
    if layout == "fused":
        f = _randn(g, rows, qh + 2 * heads, dim).to(dt)
        q, k, v = f[:, :qh], f[:, qh:qh + heads], f[:, qh + heads:]
    elif layout == "head_major":
        q, k, v = (_randn(g, h, rows, dim).to(dt).transpose(0, 1) for h in (qh, heads, heads))
    else:  # one element off every 16-byte boundary
        q, k, v = (_randn(g, rows * h * dim + 1).to(dt)[1:].view(rows, h, dim) for h in (qh, heads, heads))
    seq, pos = _i32([0] * rows), _i32(list(range(rows)))
    table = _table(1, 3, 3)
    got = []
    for a, b, c in ((q, k, v), (q.contiguous().clone(), k.contiguous().clone(), v.contiguous().clone())):
        cache = _cache(3, page, heads, dim)
        cos = torch.cos(torch.arange(rows * 64, device="cuda").float()).view(rows, 64)
        sin = torch.sin(torch.arange(rows * 64, device="cuda").float()).view(rows, 64)
        out = torch.empty(rows, qh, dim, dtype=dt, device="cuda")
        decode.kv4_append_gpu(b, c, seq, pos, cache, table, q=a, q_out=out, cos=cos, sin=sin)
        got.append((out, cache.data))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert _status() == 0


def test_append_in_place_padding_and_no_rotation(cuda):
    import torch

    from aps2026_b200 import decode

    g = _gen(1)
    q, k, v = (_randn(g, 4, h, 64) for h in (2, 1, 1))
    want = q.clone()
    want[2] = 0
    table, cache = _table(1, 2, 2), _cache(2, 8, 1, 64)
    cache.data.fill_(0x5A)
    before = cache.data.clone()
    seq = _i32([0, 0, decode.PADDING, 0])
    decode.kv4_append_gpu(k, v, seq, _i32([0, 9, 3, 15]), cache, table, q=q, q_out=q)
    assert torch.equal(q, want)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    decode.kv4_read_gpu(cache, table, seq, _i32([0, 9, 3, 15]), ko, vo)
    assert torch.equal(ko[2], torch.zeros_like(ko[2])) and torch.equal(vo[2], torch.zeros_like(vo[2]))
    keep = torch.tensor([0, 1, 3])
    assert torch.equal(ko.cpu()[keep], torch.from_numpy(_held(k))[keep])
    # 3 rows of 72 bytes are written, nothing else
    assert int((cache.data != before).sum()) <= 3 * 72
    assert _status() == 0


def test_append_special_values(cuda):
    import torch

    from aps2026_b200 import decode

    g = _gen(2)
    k = _randn(g, 8, 1, 128)
    k[0, 0, :64] = 2.5                     # a constant group
    k[1, 0, :] = 0
    k[2, 0, 70] = float("nan")
    k[3, 0, 3] = float("inf")
    k[4, 0, 3] = -float("inf")
    k[5, 0, :] = 1e-44                     # below every step
    k[6, 0, :64] *= 1e30
    k[7, 0, :64] *= 1e-30
    table, cache = _table(1, 1, 1), _cache(1, 8, 1, 128)
    seq, pos = _i32([0] * 8), _i32(list(range(8)))
    decode.kv4_append_gpu(k, k, seq, pos, cache, table)
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    decode.kv4_read_gpu(cache, table, seq, pos, ko, vo)
    assert torch.equal(torch.nan_to_num(ko, nan=7.0), torch.nan_to_num(vo, nan=7.0))
    assert bool(ko[2, 0, 64:].isnan().all()) and bool(ko[2, 0, :64].isfinite().all())
    for r in (3, 4):
        assert bool(ko[r, 0, :64].isnan().all()) and bool(ko[r, 0, 64:].isfinite().all())
    for r in (0, 1, 5, 6, 7):
        assert torch.equal(ko[r].cpu(), torch.from_numpy(_held(k[r])))
    assert _status() == 0


def test_append_and_read_report_what_is_outside(cuda):
    import torch

    from aps2026_b200 import _lib, decode

    g = _gen(3)
    table = _i32([[1, 99], [0, 2]])        # page 99 does not exist
    cache = _cache(3, 8, 1, 64)
    before = cache.data.clone()
    q, k, v = (_randn(g, 1, 1, 64) for _ in range(3))
    out = torch.full_like(q, 7.0)
    cos = sin = torch.ones(12, 32, device="cuda")
    for seq, pos, bit in ((2, 0, _lib.B2_CHECK_KV4), (0, 9, _lib.B2_CHECK_KV4), (1, 16, _lib.B2_CHECK_KV4),
                          (0, -1, _lib.B2_CHECK_KV4)):
        decode.kv4_append_gpu(k, v, _i32([seq]), _i32([pos]), cache, table, q=q, q_out=out)
        assert _status() == bit and torch.equal(out, q)
        decode.kv4_read_gpu(cache, table, _i32([seq]), _i32([pos]), out, out.clone())
        assert _status() == bit and float(out.abs().sum()) == 0
    decode.kv4_append_gpu(k, v, _i32([1]), _i32([12]), cache, table, q=q, q_out=out, cos=cos, sin=sin)
    assert _status() == _lib.B2_CHECK_ROPE and float(out.abs().sum()) == 0
    assert torch.equal(cache.data, before)


# ---- attention -----------------------------------------------------------------------


def _filled(g, lens, page, heads, dim, kscale=1.0):
    """A cache of sequences of lens[b] positions; the values it holds, and its table."""
    import torch

    from aps2026_b200 import decode

    width = max(1, (max(lens) + page - 1) // page)
    table = _table(len(lens), width, len(lens) * width)
    cache = _cache(len(lens) * width, page, heads, dim)
    keys, values = [], []
    for b, n in enumerate(lens):
        k, v = _randn(g, n, heads, dim) * kscale, _randn(g, n, heads, dim) + 0.25
        if n:
            seq, pos = _i32([b] * n), torch.arange(n, device="cuda", dtype=torch.int32)
            decode.kv4_append_gpu(k, v, seq, pos, cache, table)
            decode.kv4_read_gpu(cache, table, seq, pos, k, v)
        keys.append(k)
        values.append(v)
    return cache, table, keys, values


def _attend64(q, keys, values, queries, window, sinks, scale):
    """The definition in 64 bits, and sum_j p_j |v_j| for the error bound."""
    import torch

    out, mag, row = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64), 0
    for k, v, n in zip(keys, values, queries):
        for i in range(n):
            p = k.shape[0] - n + i
            j = torch.arange(k.shape[0], device="cuda")
            seen = j <= p
            if window:
                seen &= (p - j < window) | (j < sinks)
            if bool(seen.any()):
                kk, vv = k[seen].double(), v[seen].double()
                qq = q[row].double().view(k.shape[1], -1, k.shape[2])
                w = torch.softmax(qq @ kk.permute(1, 2, 0) * scale, -1)
                out[row] = (w @ vv.transpose(0, 1)).reshape(out[row].shape)
                mag[row] = (w @ vv.abs().transpose(0, 1)).reshape(out[row].shape)
            row += 1
    return out, mag


def _close(got, want, mag, dtype):
    """Error bound, from the arithmetic allowed to the kernel: probabilities
    held to 16 bits or more and scores (about 10 in magnitude) to 2^-20 of
    their terms' sum give 2^-14 of sum p |v|; a bf16 output adds half an ulp."""
    bound = 2.0 ** -14 * mag + (2.0 ** -8 * want.abs() if dtype == "bfloat16" else 0)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err / (mag + 1e-30)).max())


SHAPES = [  # lens, queries, q_heads, kv_heads, dim, page, window, sinks
    ([1], [1], 16, 4, 128, 16, 0, 0),
    ([37], [1], 16, 4, 128, 16, 0, 0),
    ([0, 5, 16, 17, 128, 129], [1] * 6, 16, 4, 128, 8, 0, 0),
    ([1000, 3, 4097], [1] * 3, 8, 8, 128, 64, 0, 0),
    ([1000, 3, 700], [1] * 3, 12, 4, 64, 16, 100, 0),
    ([2500, 90, 33], [1] * 3, 32, 8, 64, 32, 64, 7),
    ([300, 40, 2100], [3, 1, 5], 8, 8, 64, 32, 33, 4),
    ([300, 0, 70, 9], [4, 1, 70, 8], 16, 4, 128, 16, 0, 0),
    ([2, 1, 600], [5, 0, 17], 8, 1, 128, 8, 50, 60),
    ([9000], [2], 8, 1, 128, 128, 0, 0),
    ([333, 200], [1, 1], 48, 2, 64, 8, 0, 0),
    ([40000], [1], 4, 1, 64, 64, 0, 0),
    ([513, 514], [1, 1], 5, 1, 128, 16, 1, 0),
    ([513, 514], [2, 3], 5, 1, 128, 16, 1, 1),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_attention_vs_64_bits(cuda, shape, dtype):
    import torch

    from aps2026_b200 import decode

    lens, queries, qh, kh, dim, page, window, sinks = shape
    g = _gen(sum(lens) + dim)
    cache, table, keys, values = _filled(g, lens, page, kh, dim)
    rows = sum(queries)
    q = _randn(g, rows, qh, dim).to(getattr(torch, dtype))
    out = torch.full_like(q, float("nan"))
    offsets = _i32(np.cumsum([0] + queries).tolist())
    single = all(n == 1 for n in queries)
    ws = decode.AttentionWorkspace(dim, "cuda")
    for _ in range(2):  # the workspace is left ready for the next call
        decode.attention_kv4_gpu(q, cache, table, _i32(lens), out, q_offsets=None if single else offsets,
                                 max_queries=max(queries), max_len=max(lens), window=window, sinks=sinks, ws=ws)
        want, mag = _attend64(q, keys, values, queries, window, sinks, 1 / math.sqrt(dim))
        _close(out, want, mag, dtype)
        first, out = out, torch.full_like(q, float("nan"))
    decode.attention_kv4_gpu(q, cache, table, _i32(lens), out, q_offsets=offsets, max_queries=max(queries) + 2,
                             max_len=max(lens), window=window, sinks=sinks, ws=ws)
    assert _status() == 0
    _close(out, first.double(), mag * 2, dtype)


def test_attention_repeats_bit_for_bit(cuda):
    import torch

    from aps2026_b200 import decode

    g = _gen(11)
    lens = [5000, 70, 2222, 0, 16]
    cache, table, _, _ = _filled(g, lens, 16, 4, 128)
    q = _randn(g, 5, 16, 128)
    ws = decode.AttentionWorkspace(128, "cuda")
    outs = []
    for _ in range(20):
        outs.append(torch.empty_like(q))
        decode.attention_kv4_gpu(q, cache, table, _i32(lens), outs[-1], ws=ws)
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("magnitude", [1e-30, 1e-3, 60.0, 3e4])
def test_attention_score_range(cuda, magnitude):
    """Scores from all-equal to one key taking everything; the running
    maximum moves with every later key."""
    import torch

    from aps2026_b200 import decode

    g = _gen(12)
    n, dim = 700, 128
    cache, table, keys, values = _filled(g, [n], 16, 1, dim)
    q = keys[0].mean(0, keepdim=True).repeat(1, 4, 1) * 0 + _randn(g, 1, 4, dim) * magnitude
    out = torch.empty_like(q)
    decode.attention_kv4_gpu(q, cache, table, _i32([n]), out, scale=1 / magnitude)
    want, mag = _attend64(q, keys, values, [1], 0, 0, 1 / magnitude)
    _close(out, want, mag, "float32")


def test_attention_unseen_keys_do_not_matter(cuda):
    """Pages no row sees may be missing; NaN beyond a row's sight or in a
    page's unused slots does not reach it, NaN in sight does."""
    import torch

    from aps2026_b200 import decode

    g = _gen(13)
    n, dim, page, window, sinks = 500, 128, 16, 40, 3
    cache, table, keys, values = _filled(g, [n], page, 2, dim)
    q = _randn(g, 3, 8, dim)
    args = dict(q_offsets=_i32([0, 3]), max_queries=3, window=window, sinks=sinks)
    want, mag = _attend64(q, keys, values, [3], window, sinks, dim ** -0.5)
    # only the sinks' page and the window's pages stay in the table
    kept = table.clone()
    kept[0, 1:(n - 3 - window + 1) // page] = -1
    out = torch.empty_like(q)
    decode.attention_kv4_gpu(q, cache, kept, _i32([n]), out, **args)
    _close(out, want, mag, "float32")
    assert _status() == 0
    # poison unused slots of the last page, and keys between sinks and window
    nan = torch.full((1, 2, dim), float("nan"), device="cuda")
    for p in (3, 100, n, n + 5):
        decode.kv4_append_gpu(nan, nan, _i32([0]), _i32([p]), cache, table)
    out = torch.empty_like(q)
    decode.attention_kv4_gpu(q, cache, table, _i32([n]), out, **args)
    _close(out, want, mag, "float32")
    # the newest key is NaN: the last query row alone sees it
    decode.kv4_append_gpu(nan, values[0][n - 1:n], _i32([0]), _i32([n - 1]), cache, table)
    out = torch.empty_like(q)
    decode.attention_kv4_gpu(q, cache, table, _i32([n]), out, **args)
    _close(out[:2], want[:2], mag[:2], "float32")
    assert bool(out[2].isnan().all())
    # a NaN value, in 64 of its dimensions
    half = values[0][n - 1:n].clone()
    half[:, 1, 64:] = float("nan")
    decode.kv4_append_gpu(keys[0][n - 1:n], half, _i32([0]), _i32([n - 1]), cache, table)
    out = torch.empty_like(q)
    decode.attention_kv4_gpu(q, cache, table, _i32([n]), out, **args)
    _close(out[:2], want[:2], mag[:2], "float32")
    heads = out[2].view(2, 4, dim)
    assert bool(heads[1, :, 64:].isnan().all()) and bool(heads[1, :, :64].isfinite().all())
    assert bool(heads[0].isfinite().all())


def test_attention_strided_queries_and_streams(cuda):
    import torch

    from aps2026_b200 import decode

    g = _gen(14)
    lens = [333, 90]
    cache, table, keys, values = _filled(g, lens, 16, 4, 128)
    fused = _randn(g, 2, 24, 128)
    q = fused[:, :16]
    odd = torch.empty(2 * 16 * 128 + 1, device="cuda")[1:].view(2, 16, 128)
    odd.copy_(q)
    want, mag = _attend64(q, keys, values, [1, 1], 0, 0, 128 ** -0.5)
    outs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in (q, odd, q.transpose(0, 1).contiguous().transpose(0, 1)):
            out = torch.empty(2, 16, 128, device="cuda")
            decode.attention_kv4_gpu(x, cache, table, _i32(lens), out)
            outs.append(out)
    torch.cuda.current_stream().wait_stream(side)
    for out in outs:
        _close(out, want, mag, "float32")
        assert torch.equal(out, outs[0])


def test_attention_reports_what_is_outside(cuda):
    import torch

    from aps2026_b200 import _lib, decode

    g = _gen(15)
    cache, table, keys, values = _filled(g, [30, 30], 16, 1, 64)
    q = _randn(g, 2, 4, 64)
    want, mag = _attend64(q, keys, values, [1, 1], 0, 0, 0.125)
    # a length past the table: that sequence's rows are zero, the other's are right
    out = torch.full_like(q, float("nan"))
    decode.attention_kv4_gpu(q, cache, table, _i32([33, 30]), out, max_len=64)
    assert _status() == _lib.B2_CHECK_KV4
    assert float(out[0].abs().sum()) == 0
    _close(out[1], want[1], mag[1], "float32")
    # a length past max_len
    decode.attention_kv4_gpu(q, cache, table, _i32([30, 30]), out, max_len=29)
    assert _status() == _lib.B2_CHECK_KV4 and float(out.abs().sum()) == 0
    # a page outside the cache: its keys are not seen
    bad = table.clone()
    bad[0, 0] = 77
    decode.attention_kv4_gpu(q, cache, bad, _i32([30, 30]), out)
    assert _status() == _lib.B2_CHECK_KV4
    half, half_mag = _attend64(q[:1], [keys[0][16:]], [values[0][16:]], [1], 0, 0, 0.125)
    _close(out[:1], half, half_mag, "float32")
    _close(out[1], want[1], mag[1], "float32")
    # query offsets that do not fit: not written
    out.fill_(5.0)
    decode.attention_kv4_gpu(q, cache, table, _i32([30, 30]), out, q_offsets=_i32([0, 1, 9]), max_queries=8)
    assert _status() == _lib.B2_CHECK_KV4 and bool((out[1] == 5.0).all())
    _close(out[0], want[0], mag[0], "float32")


# ---- experts ---------------------------------------------------------------------------


def _moe64(x, logits, gate_up, down, quantum, tie, gates):
    import torch

    f = np.float32
    T, E = logits.shape
    inter = down.shape[2]
    out = torch.zeros(T, x.shape[1], dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    grid = logits.cpu().numpy()
    grid = np.where(grid < 0, f(-1), f(1)) * (np.floor(np.abs(grid) / f(quantum) + f(0.5)) * f(quantum))
    for t in range(T):
        pair = []
        for _ in range(2):
            lead = None
            for e in range(E):
                if e not in pair and (lead is None or grid[t, e] > f(grid[t, lead] + f(tie))):
                    lead = e
            pair.append(lead)
        raw = logits[t, pair].double()
        w = torch.softmax(raw, 0) if gates == "softmax" else torch.full_like(raw, 0.5)
        for e, g in zip(pair, w):
            gu = gate_up[e].double() @ x[t].double()
            a = gu[:inter] * torch.sigmoid(gu[:inter]) * gu[inter:]
            out[t] += g * (down[e].double() @ a)
            mag[t] += g * (down[e].double().abs() @ a.abs())
    return out, mag


MOE = [  # T, H, I, E
    (1, 4096, 448, 16), (2, 256, 96, 4), (9, 4096, 448, 16), (17, 512, 448, 2), (61, 1024, 64, 32),
    (128, 1001, 333, 7), (3, 1, 1, 2), (5, 33, 7, 5), (128, 264, 40, 2), (40, 2048, 8, 3), (128, 72, 200, 16),
]


@pytest.mark.parametrize("T,H,I,E", MOE)
@pytest.mark.parametrize("xt,wt", [("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("float32", "float32"),
                                   ("bfloat16", "float32")])
@pytest.mark.parametrize("gates", ["equal", "softmax"])
def test_moe_decode_vs_64_bits(cuda, T, H, I, E, xt, wt, gates):
    import torch

    from aps2026_b200 import decode

    g = _gen(T * H + I)
    x = _randn(g, T, H).to(getattr(torch, xt))
    logits = _randn(g, T, E)
    gu = (_randn(g, E, 2 * I, H) / math.sqrt(H)).to(getattr(torch, wt))
    dn = (_randn(g, E, H, I) / math.sqrt(I)).to(getattr(torch, wt))
    out = torch.full_like(x, float("nan"))
    decode.moe_decode_gpu(x, logits, gu, dn, out, gates=gates)
    want, mag = _moe64(x, logits, gu, dn, 1e-3, 2e-2, gates)
    # fp32 sums of up to 4096 products of inputs held to 16 bits or more, and
    # of activations to 16 or more: 2^-14 of the sum of magnitudes; a gate
    # and up product that nearly cancels carries its own sum's error, hence a
    # second term in the size of a typical output
    bound = 2.0 ** -14 * (mag + mag.mean()) + (2.0 ** -8 * want.abs() if xt == "bfloat16" else 0)
    err = (out.double() - want).abs()
    assert bool((err <= bound).all()), float((err / mag.mean()).max())
    again = torch.empty_like(x)
    decode.moe_decode_gpu(x, logits, gu, dn, again, gates=gates)
    assert torch.equal(again, out)


def test_moe_decode_matches_routing_and_strides(cuda):
    """Ties and the scan's margin pick as b2_moe_route picks: every token to
    one expert pair, all tokens on one expert, strided rows."""
    import torch

    from aps2026_b200 import decode, ops

    g = _gen(21)
    T, H, I, E = 128, 128, 64, 16
    gu, dn = _randn(g, E, 2 * I, H) / 11, _randn(g, E, H, I) / 8
    fused = _randn(g, T, H + 40)
    x = fused[:, 8:8 + H]
    for logits in (torch.zeros(T, E, device="cuda"), (_randn(g, T, E) * 0.03),
                   torch.tensor([[float(e == 11) + 0.5 * float(e == 3) for e in range(E)]] * T, device="cuda")):
        routing = ops.moe_route_gpu(logits)
        pairs = routing.routes.long()
        out = torch.full((T, H + 4), float("nan"), device="cuda")
        decode.moe_decode_gpu(x, logits, gu, dn, out[:, :H])
        want = torch.zeros(T, H, dtype=torch.float64, device="cuda")
        for s in range(2):
            w1, w2 = gu[pairs[:, s]].double(), dn[pairs[:, s]].double()
            y = torch.einsum("tih,th->ti", w1, x.double())
            a = y[:, :I] * torch.sigmoid(y[:, :I]) * y[:, I:]
            want += 0.5 * torch.einsum("thi,ti->th", w2, a)
        assert float((out[:, :H].double() - want).abs().max()) <= 2.0 ** -14 * float(want.abs().max()) * 4
        assert bool(out[:, H:].isnan().all())


def test_moe_decode_nan_stays_in_its_token(cuda):
    import torch

    from aps2026_b200 import decode

    g = _gen(22)
    T, H, I, E = 20, 256, 64, 4
    x, logits = _randn(g, T, H), _randn(g, T, E)
    gu, dn = _randn(g, E, 2 * I, H) / 16, _randn(g, E, H, I) / 8
    clean, dirty = torch.empty_like(x), torch.empty_like(x)
    decode.moe_decode_gpu(x, logits, gu, dn, clean)
    x[7, 3] = float("nan")
    x[9, 3] = float("inf")
    decode.moe_decode_gpu(x, logits, gu, dn, dirty)
    others = [t for t in range(T) if t not in (7, 9)]
    assert torch.equal(clean[others], dirty[others])
    assert bool(dirty[7].isnan().all()) and not bool(dirty[9].isfinite().any())


# ---- refusals ----------------------------------------------------------------------------


def test_refusals(cuda):
    import torch

    from aps2026_b200 import decode, ops

    g = _gen(30)
    cache, table = _cache(2, 8, 2, 64), _i32([[0, 1]])
    k = _randn(g, 3, 2, 64)
    seq, pos = _i32([0] * 3), _i32([0, 1, 2])
    ok = dict(k=k, v=k, row_seq=seq, row_pos=pos, cache=cache, page_table=table)
    for bad in (dict(k=k[:, :1]), dict(v=k.double()), dict(v=k.bfloat16()), dict(row_seq=seq.long()),
                dict(row_pos=pos[:2]), dict(page_table=table[0]), dict(page_table=table.cpu()), dict(k=k.cpu()),
                dict(q=k), dict(q=k, q_out=k.bfloat16()), dict(cos=torch.ones(4, 32, device="cuda")),
                dict(cos=torch.ones(4, 16, device="cuda"), sin=torch.ones(4, 16, device="cuda")),
                dict(k=k.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ops.InvalidArgument):
            decode.kv4_append_gpu(**{**ok, **bad})
    for bad in ((0, 2, 64), (12, 2, 64), (4, 2, 64), (8, 0, 64), (8, 2, 96)):
        with pytest.raises(ops.InvalidArgument):
            decode.KVCache4(1, *bad, "cuda")
    with pytest.raises(ops.InvalidArgument):
        decode.kv4_read_gpu(cache, table, seq, pos, k, k[:2])
    q = _randn(g, 1, 4, 64)
    ok = dict(q=q, cache=cache, page_table=table, lens=_i32([3]), out=torch.empty_like(q))
    for bad in (dict(q=_randn(g, 1, 3, 64)), dict(q=q[0]), dict(out=q.bfloat16()), dict(lens=_i32([3, 3])),
                dict(window=-1), dict(max_queries=0), dict(q=q.repeat(2, 1, 1), out=torch.empty(2, 4, 64, device="cuda")),
                dict(q_offsets=_i32([0])), dict(q=q.double(), out=q.double()),
                dict(ws=decode.AttentionWorkspace(64, "cpu"))):
        with pytest.raises(ops.InvalidArgument):
            decode.attention_kv4_gpu(**{**ok, **bad})
    x, lg = _randn(g, 2, 64), _randn(g, 2, 4)
    gu, dn = _randn(g, 4, 32, 64), _randn(g, 4, 64, 16)
    ok = dict(x=x, logits=lg, w_gate_up=gu, w_down=dn, out=torch.empty_like(x))
    many = _randn(g, 129, 64)
    for bad in (dict(x=x.double(), out=x.double()), dict(logits=lg[:, :3]), dict(w_gate_up=gu[:, :31]),
                dict(w_down=dn.bfloat16()), dict(out=x[:, :3]), dict(gates="top1"), dict(logits=lg.bfloat16()),
                dict(x=many, out=torch.empty_like(many), logits=_randn(g, 129, 4)),
                dict(x=x.t().contiguous().t()), dict(ws=decode.MoeWorkspace(1, 16, "cuda"))):
        with pytest.raises(ops.InvalidArgument):
            decode.moe_decode_gpu(**{**ok, **bad})
    assert _status() == 0


def test_empty_calls_do_nothing(cuda):
    import torch

    from aps2026_b200 import decode

    cache, table = _cache(2, 8, 2, 64), _i32([[0, 1]])
    none, nothing = _i32([]), torch.empty(0, 2, 64, device="cuda")
    decode.kv4_append_gpu(nothing, nothing, none, none, cache, table)
    decode.kv4_read_gpu(cache, table, none, none, nothing, nothing.clone())
    decode.attention_kv4_gpu(torch.empty(0, 4, 64, device="cuda"), cache, table, _i32([0]),
                             torch.empty(0, 4, 64, device="cuda"), q_offsets=_i32([0, 0]))
    decode.moe_decode_gpu(torch.empty(0, 64, device="cuda"), torch.empty(0, 4, device="cuda"),
                          torch.zeros(4, 32, 64, device="cuda"), torch.zeros(4, 64, 16, device="cuda"),
                          torch.empty(0, 64, device="cuda"))
    assert _status() == 0

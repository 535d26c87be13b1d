"""The decode operators at the ends of what they take: batches in which no row
sees a key, and the largest and smallest numbers."""
import math

import pytest

from test_decode_edges_gpu import _filled
from test_decode_gpu import _gen, _i32, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs,kv_heads,q_heads", [(3, 2, 8), (128, 4, 16), (300, 1, 8), (300, 4, 4)])
@pytest.mark.parametrize("why", ["empty", "past max_len", "no queries"])
@pytest.mark.parametrize("offsets", [False, True])
def test_attention_without_a_key_in_sight(cuda, seqs, kv_heads, q_heads, why, offsets):
    """Zero rows (left as they are where no sequence has them), the status
    that says why, and a workspace that is ready for the next call."""
    import torch

    from aps2026_b200 import _lib, decode, ops

    if why == "no queries" and not offsets:
        pytest.skip("without offsets every sequence has a row")
    g = _gen(seqs)
    real = [1 + s % 5 for s in range(seqs)]
    cache, table, _, _ = _filled(g, real, 8, kv_heads, 64)
    q = _randn(g, seqs, q_heads, 64)
    ws = decode.AttentionWorkspace(64, "cuda")
    each = _i32(list(range(seqs + 1))) if offsets else None
    lens, kw, status = _i32([0] * seqs), dict(max_len=8), 0
    if why == "past max_len":
        lens, kw, status = _i32(real), dict(max_len=0), _lib.B2_CHECK_KV4
    out = torch.full_like(q, 5.0)
    first = _i32([0] * (seqs + 1)) if why == "no queries" else each
    for _ in range(2):
        decode.attention_kv4_gpu(q, cache, table, _i32(real) if why == "no queries" else lens, out, q_offsets=first,
                                 ws=ws, **kw)
        assert ops.device_status() == status
    assert bool((out == (5.0 if why == "no queries" else 0.0)).all())
    want = torch.empty_like(q)
    decode.attention_kv4_gpu(q, cache, table, _i32(real), want, q_offsets=each)
    decode.attention_kv4_gpu(q, cache, table, _i32(real), out, q_offsets=each, ws=ws)
    assert torch.equal(out, want) and bool((want != 0).any(-1).all()) and ops.device_status() == 0


def test_attention_captured_at_zero_lengths(cuda):
    import torch

    from aps2026_b200 import decode, ops

    seqs, g = 130, _gen(9)
    real = [1 + s % 40 for s in range(seqs)]
    cache, table, _, _ = _filled(g, real, 8, 4, 128)
    q, lens = _randn(g, seqs, 16, 128), _i32([0] * seqs)
    ws, out = decode.AttentionWorkspace(128, "cuda"), torch.full_like(q, 5.0)
    run = lambda: decode.attention_kv4_gpu(q, cache, table, lens, out, ws=ws)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    graph.replay()
    assert bool((out == 0).all())
    lens.copy_(_i32(real))
    graph.replay()
    want = torch.empty_like(q)
    decode.attention_kv4_gpu(q, cache, table, lens, want)
    assert torch.equal(out, want) and bool((want != 0).any(-1).all())
    lens.zero_()
    graph.replay()
    assert bool((out == 0).all()) and ops.device_status() == 0


@pytest.mark.parametrize("window", [2 ** 31 - 2, 2 ** 31 - 9, 2 ** 31, 2 ** 40, 20, 21])
@pytest.mark.parametrize("q_heads", [1, 6])
def test_attention_window_past_every_length(cuda, window, q_heads):
    """The same as no window, with more query rows than positions too."""
    import torch

    from aps2026_b200 import decode, ops

    g = _gen(q_heads)
    lens, queries = [3, 20], [8, 4]
    cache, table, _, _ = _filled(g, lens, 8, 1, 64)
    q = _randn(g, 12, q_heads, 64)
    outs = []
    for w in (0, window):
        outs.append(torch.full_like(q, 5.0))
        decode.attention_kv4_gpu(q, cache, table, _i32(lens), outs[-1], q_offsets=_i32([0, 8, 12]), max_queries=8,
                                 max_len=20, window=w, sinks=1)
    assert torch.equal(*outs) and ops.device_status() == 0
    assert bool((outs[0][:5] == 0).all()) and bool((outs[0][5:] != 0).any(-1).all())


def _append_at(cache, table, pos, k, v):
    from aps2026_b200 import decode

    decode.kv4_append_gpu(k, v, _i32([0]), _i32([pos]), cache, table)
    decode.kv4_read_gpu(cache, table, _i32([0]), _i32([pos]), k, v)


def _one_row64(q, k, v, scale):
    import torch

    kv_heads = k.shape[1]
    w = torch.softmax(q.double().view(kv_heads, -1, q.shape[-1]) @ k.double().permute(1, 2, 0) * scale, -1)
    return (w @ v.double().transpose(0, 1)).view(q.shape)


# what the arithmetic below may cost a row: scores of some 2^3 held to 2^-20 of
# their terms' sum move every weight by 2^-17 of itself
ROW = 2.0 ** -17


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_heads", [2, 8])       # four rows of a KV head, and more
@pytest.mark.parametrize("outlier", [2.0 ** 12, 2.0 ** 36, 2.0 ** 100])
@pytest.mark.parametrize("where", ["behind the mask", "out of the window", "far below in score"])
def test_attention_large_values_that_carry_no_weight(cuda, dim, q_heads, outlier, where):
    """A value with a step many times the others', which a row does not see or
    gives no weight, costs the row nothing."""
    import torch

    from aps2026_b200 import decode, ops

    g, n, kv_heads = _gen(dim + q_heads), 75, 1
    cache, table, k, v = _filled(g, [n], 16, kv_heads, dim)
    q = _randn(g, 2, q_heads, dim)
    window, at = (0, n - 1) if where != "out of the window" else (40, n - 41)
    far_k = k[at:at + 1].clone()
    if where == "far below in score":
        # against every query row's sum
        at, far_k = n - 2, torch.full_like(far_k, 0.0)
        q = q.abs()
        far_k -= 200.0
    far_v = _randn(g, 1, kv_heads, dim) * outlier
    _append_at(cache, table, at, far_k, far_v)
    out = torch.empty_like(q)
    decode.attention_kv4_gpu(q, cache, table, _i32([n]), out, q_offsets=_i32([0, 2]), max_queries=2, window=window)
    if where == "behind the mask":        # of the first row
        rows, seen = [0], [slice(0, n - 1)]
    elif where == "out of the window":    # of the last row
        rows, seen = [1], [slice(n - 40, n)]
    else:
        keep = [j for j in range(n) if j != at]
        rows, seen = [0, 1], [[j for j in keep if j < n - 1], keep]
    for row, s in zip(rows, seen):
        want = _one_row64(q[row], k[s], v[s], dim ** -0.5)
        assert float((out[row].double() - want).norm() / want.norm()) < ROW
    assert ops.device_status() == 0


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_heads", [2, 8])
@pytest.mark.parametrize("value", [1e10, -1e16, 3e25, -2.0 ** 100])
@pytest.mark.parametrize("first_group_alone", [False, True])
def test_attention_constant_values(cuda, dim, q_heads, value, first_group_alone):
    """Groups of one value have steps of zero; their weighted sum is that value."""
    import torch

    from aps2026_b200 import decode, ops

    g, n = _gen(dim), 333
    cache, table, k, v = _filled(g, [n], 16, 1, dim)
    value = float(torch.tensor(value).bfloat16())  # held as it is
    v[..., :64 if first_group_alone else dim] = value
    seq, pos = _i32([0] * n), torch.arange(n, device="cuda", dtype=torch.int32)
    decode.kv4_append_gpu(k, v, seq, pos, cache, table)
    decode.kv4_read_gpu(cache, table, seq, pos, k, v)
    q, out = _randn(g, 1, q_heads, dim), torch.empty(1, q_heads, dim, device="cuda")
    decode.attention_kv4_gpu(q, cache, table, _i32([n]), out)
    want = _one_row64(q, k, v, dim ** -0.5)
    for part in range(0, dim, 64):
        a, b = out[..., part:part + 64].double(), want[..., part:part + 64]
        assert float((a - b).norm() / b.norm()) < (ROW if abs(value) < 2.0 ** 90 or part == 0 else 2.0 ** -12)
    assert ops.device_status() == 0


@pytest.mark.parametrize("q_heads", [2, 8])
@pytest.mark.parametrize("k", [-100, 126])
def test_attention_queries_of_one_sign_and_any_size(cuda, q_heads, k):
    """Queries times 2^k at a scale of 2^-k are the same queries, bit for bit,
    also where their sum passes fp32's end, or the scale its start in base 2."""
    import torch

    from aps2026_b200 import decode

    g, n = _gen(q_heads + 8), 333
    cache, table, _, _ = _filled(g, [n], 16, 2, 128)
    q, want = torch.rand((1, q_heads, 128), generator=g, device="cuda") + 0.9, torch.empty(1, q_heads, 128, device="cuda")
    out = torch.empty_like(want)
    decode.attention_kv4_gpu(q, cache, table, _i32([n]), want, scale=0.0625)
    decode.attention_kv4_gpu(q * 2.0 ** k, cache, table, _i32([n]), out, scale=0.0625 * 2.0 ** -k)
    assert bool(want.isfinite().all()) and torch.equal(out, want)


def test_workspaces_smaller_than_they_say_are_refused(cuda):
    import torch

    from aps2026_b200 import decode, ops

    g = _gen(3)
    cache, table, _, _ = _filled(g, [5], 8, 1, 64)
    q, x = _randn(g, 1, 4, 64), _randn(g, 2, 64)
    gate_up, down, logits = _randn(g, 4, 32, 64), _randn(g, 4, 64, 16), _randn(g, 2, 4)
    for cut in (slice(16), slice(0, None, 2)):
        attention, moe = decode.AttentionWorkspace(64, "cuda"), decode.MoeWorkspace(2, 16, "cuda")
        attention.buf, moe.buf = attention.buf[cut], moe.buf[cut]
        with pytest.raises(ops.InvalidArgument, match="workspace: expected"):
            decode.attention_kv4_gpu(q, cache, table, _i32([5]), torch.empty_like(q), ws=attention)
        with pytest.raises(ops.InvalidArgument, match="workspace: expected"):
            decode.moe_decode_gpu(x, logits, gate_up, down, torch.empty_like(x), ws=moe)
    cache.pages += 1
    with pytest.raises(ops.InvalidArgument, match="cache: expected"):
        decode.attention_kv4_gpu(q, cache, table, _i32([5]), torch.empty_like(q))
    assert ops.device_status() == 0


def _experts_plain(x, logits, gate_up, down):
    """The expert layer in 64 bits, but infinite where its activations or its
    result are so in the operator's types."""
    import torch

    from aps2026_b200 import ops

    pairs = ops.moe_route_gpu(logits).routes.long().sort(1).values
    inter, rows, mag = down.shape[2], [], []
    for t, pair in enumerate(pairs.tolist()):
        y, m = 0.0, 0.0
        for e in pair:
            gate, up = (gate_up[e].double() @ x[t].double()).split(inter)
            a = (gate / (1 + torch.exp(-gate)) * up).float().double()
            y, m = y + 0.5 * (down[e].double() @ a), m + 0.5 * (down[e].double().abs() @ a.abs())
        rows.append(y)
        mag.append(m)
    out = torch.stack(rows)
    held = out.to(x.dtype).double()
    return torch.where(held.isfinite(), out, held), torch.stack(mag)


@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("H,I", [(64, 24), (65, 27), (3000, 40)])
@pytest.mark.parametrize("xt,wt", [("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("float32", "float32"), ("bfloat16", "float32")])
@pytest.mark.parametrize("what", ["x infinite", "x at the end", "gate weight infinite", "down weight infinite", "activation overflows"])
def test_experts_keep_infinities_and_the_largest_numbers(cuda, T, H, I, xt, wt, what):
    """Infinite where a plain sum is, of its sign, and finite where that is."""
    import torch

    from aps2026_b200 import decode

    g, E = _gen(T + H), 4
    xt, wt = getattr(torch, xt), getattr(torch, wt)
    x, logits = _randn(g, T, H), _randn(g, T, E)
    gate_up, down = _randn(g, E, 2 * I, H) / math.sqrt(H), _randn(g, E, H, I) / math.sqrt(I)
    sign = torch.where(torch.arange(H, device="cuda") % 3 == 0, -1.0, 1.0)[:, None]
    if what == "x infinite":
        x[1, H // 2] = float("inf")
        gate_up, down = gate_up.abs(), down.abs() * sign
    elif what == "x at the end":
        x[1] = x[1].sign() * 3.4e38
        gate_up = gate_up * 2.0 ** -100
    elif what == "gate weight infinite":
        gate_up[2, I // 2, H // 2] = float("inf")
        down = down.abs() * sign
    elif what == "down weight infinite":
        down[2, H // 2, I // 2] = float("inf")
    else:
        x[1] = x[1].abs() * 1e20
        gate_up, down = gate_up.abs(), down.abs() * sign
    x = x.to(xt) if what != "x at the end" else torch.where(x.to(xt).isinf(), 3.3e38 * x.sign(), x).to(xt)
    gate_up, down = gate_up.to(wt), down.to(wt)
    out = torch.full_like(x, 5.0)
    decode.moe_decode_gpu(x, logits, gate_up, down, out)
    want, mag = _experts_plain(x, logits, gate_up, down)
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.isinf(), want.isinf()) and torch.equal(out[out.isinf()].double(), want[want.isinf()])
    if what in ("x infinite", "activation overflows"):
        assert bool(out[1].isinf().all())
    # sums of inputs held to 16 bits or more, a row at a time
    fine = want.isfinite()
    scale = torch.where(fine, mag, 0.0).mean(1, keepdim=True)
    bound = 2.0 ** -14 * (mag + scale) + (2.0 ** -8 * want.abs() if xt == torch.bfloat16 else 0)
    assert bool(((out.double() - want).abs() <= bound)[fine].all())


@pytest.mark.parametrize("E", [2, 3, 15, 16, 17, 31, 32])
@pytest.mark.parametrize("spread", [0.0, 0.004, 0.03, 1.0])
def test_experts_are_those_of_the_routing(cuda, E, spread):
    """Two implementations of one rule: around the margin and on the grid's
    boundaries, with infinities and NaN among the scores."""
    import torch

    from aps2026_b200 import decode, ops

    g, T = _gen(E), 128
    # expert e writes coordinate e
    x, gate_up = torch.ones(T, 32, device="cuda"), torch.ones(E, 2, 32, device="cuda")
    down = torch.eye(32, device="cuda")[:E, :, None].contiguous()
    for odd in (None, float("nan"), float("inf"), -float("inf")):
        logits = _randn(g, T, E) * spread
        logits[::2] = (logits[::2] / 5e-4).round() * 5e-4      # grid points and the middles between them
        logits[1::4] = (logits[1::4] / 2e-2).round() * 2e-2    # margins
        if odd is not None:
            logits[torch.rand(T, E, generator=g, device="cuda") < 0.2] = odd
        out = torch.empty(T, 32, device="cuda")
        decode.moe_decode_gpu(x, logits, gate_up, down, out)
        want = torch.zeros(T, 32, device="cuda").scatter_(1, ops.moe_route_gpu(logits).routes.long(), 1.0)
        assert torch.equal((out != 0).float(), want)


@pytest.mark.parametrize("q_heads", [4, 16])
@pytest.mark.parametrize("dim,key,first,second", [(64, 0, -70, 0), (64, 0, 100, 0), (64, 100, 0, 0), (64, -70, 0, 0), (128, 0, 0, 12),
                                                  (128, 0, 12, 0), (128, 0, -70, -58), (128, 0, 100, 88), (128, 100, 100, 100)])
def test_attention_in_the_stated_range(cuda, q_heads, dim, key, first, second):
    """Keys 2^key, values' halves 2^first and 2^second times the usual size:
    each half as close as at the usual size."""
    import torch

    from aps2026_b200 import decode, ops

    g, n, kv_heads = _gen(dim), 1500, 2
    cache, table, k, v = _filled(g, [n], 16, kv_heads, dim)
    k *= 2.0 ** key
    v[..., :64] *= 2.0 ** first
    v[..., 64:] *= 2.0 ** second
    seq, pos = _i32([0] * n), torch.arange(n, device="cuda", dtype=torch.int32)
    decode.kv4_append_gpu(k, v, seq, pos, cache, table)
    decode.kv4_read_gpu(cache, table, seq, pos, k, v)
    q, out = _randn(g, 1, q_heads, dim) * 2.0 ** -key, torch.empty(1, q_heads, dim, device="cuda")
    decode.attention_kv4_gpu(q, cache, table, _i32([n]), out)
    want = _one_row64(q, k, v, dim ** -0.5)
    for part in range(0, dim, 64):
        a, b = out[..., part:part + 64].double(), want[..., part:part + 64]
        assert float((a - b).norm() / b.norm()) < ROW
    assert ops.device_status() == 0


def test_outputs_off_a_16_byte_boundary_are_refused(cuda):
    import torch

    from aps2026_b200 import decode, ops

    g = _gen(4)
    cache, table, k, v = _filled(g, [3], 8, 1, 64)
    off = torch.empty(1 + 3 * 64, device="cuda")[1:].view(3, 1, 64)
    seq, pos, q = _i32([0] * 3), _i32([0, 1, 2]), _randn(g, 3, 1, 64)
    for call in (lambda: decode.kv4_append_gpu(k, v, seq, pos, cache, table, q=q, q_out=off),
                 lambda: decode.kv4_read_gpu(cache, table, seq, pos, off, v),
                 lambda: decode.kv4_read_gpu(cache, table, seq, pos, k, off),
                 lambda: decode.attention_kv4_gpu(q, cache, table, _i32([3]), off, q_offsets=_i32([0, 3]), max_queries=3)):
        with pytest.raises(ops.InvalidArgument, match="16-byte"):
            call()
    assert ops.device_status() == 0

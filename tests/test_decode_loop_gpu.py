"""The decode operators together (examples/decode_loop.py): prompts fed whole
against token by token, the step as a CUDA graph against eager, and more
sequences than a CTA keeps sizes of."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _i32(v):
    import torch

    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 2)])
def test_prompts_whole_and_token_by_token(cuda, window, sinks):
    import torch

    from aps2026_b200 import ops
    from examples.decode_loop import Decoder

    prompts = [[7, 3, 900, 41, 8, 8], list(range(100, 140)), [5]]
    kw = dict(seqs=3, max_len=64, window=window, sinks=sinks, seed=4)
    whole, lens = Decoder(**kw).prefill(prompts)
    model, row = Decoder(**kw), 0
    for s, prompt in enumerate(prompts):
        now = _i32([0, 0, 0])
        for p, token in enumerate(prompt):
            now[s] = p + 1
            # one sequence's row at a time: the others have none
            offsets = _i32([0] * (s + 1) + [1] * (3 - s))
            got = model.forward(_i32([token]), _i32([s]), _i32([p]), now, offsets, 1)
            # the projections' sums may differ in their last bits between one
            # row and many; should such a bit turn one 4-bit code (a step of a
            # fifteenth of a range), a key's weight moves by some percent of
            # itself and a row by well under this
            err = (got[0] - whole[row]).norm() / whole[row].norm()
            assert float(err) < 1e-2, (s, p, float(err))
            row += 1
    assert lens.tolist() == [6, 40, 1] and ops.device_status() == 0


def test_step_in_a_graph_is_the_eager_step(cuda):
    import torch

    from aps2026_b200 import ops
    from examples.decode_loop import Decoder, Stepper

    prompts = [[1, 2, 3], list(range(50)), [9] * 17, [4]]
    eager, graphed = Decoder(seed=5), Decoder(seed=5)
    _, lens = eager.prefill(prompts)
    graphed.prefill(prompts)
    token = _i32([10, 20, 30, 40])
    step = Stepper(graphed, token, lens)
    seq = _i32([0, 1, 2, 3])
    for _ in range(20):
        pos = lens.clone()
        lens += 1
        hidden = eager.forward(token, seq, pos, lens)
        token = (hidden @ eager.head.t()).argmax(-1).to(torch.int32)
        assert torch.equal(step(), token)
        assert torch.equal(step.hidden, hidden)
    assert step.lens.tolist() == lens.tolist() and ops.device_status() == 0


@pytest.mark.parametrize("seqs,q_heads,kv_heads,queries,longest", [(300, 4, 2, 1, 70), (700, 8, 1, 1, 40), (40, 8, 8, 3, 900),
                                                                   (300, 6, 2, 2, 333), (5, 8, 8, 40, 700)])
def test_attention_over_many_sequences(cuda, seqs, q_heads, kv_heads, queries, longest):
    import torch

    from aps2026_b200 import decode, ops

    g = torch.Generator(device="cuda").manual_seed(seqs)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    dim, page = 64, 8
    lens = [(s * 37) % (longest + 1) for s in range(seqs)]
    width = -(-longest // page)
    table = torch.randperm(seqs * width, generator=g, device="cuda").to(torch.int32).view(seqs, width)
    cache = decode.KVCache4(seqs * width, page, kv_heads, dim, "cuda")
    seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), torch.tensor(lens, device="cuda")).to(torch.int32)
    pos = torch.cat([torch.arange(n, device="cuda", dtype=torch.int32) for n in lens])
    k, v = rand(seq.numel(), kv_heads, dim), rand(seq.numel(), kv_heads, dim) + 0.25
    decode.kv4_append_gpu(k, v, seq, pos, cache, table)
    decode.kv4_read_gpu(cache, table, seq, pos, k, v)
    q, out = rand(seqs * queries, q_heads, dim), torch.full((seqs * queries, q_heads, dim), float("nan"), device="cuda")
    ws = decode.AttentionWorkspace(dim, "cuda")
    for _ in range(2):
        decode.attention_kv4_gpu(q, cache, table, _i32(lens), out,
                                 q_offsets=_i32([s * queries for s in range(seqs + 1)]), max_queries=queries, ws=ws)
    start = 0
    for s, n in enumerate(lens):
        kk, vv = k[start:start + n].double(), v[start:start + n].double()
        start += n
        for i in range(queries):
            row, seen = s * queries + i, n - queries + i + 1
            if seen <= 0:
                assert float(out[row].abs().sum()) == 0
                continue
            w = torch.softmax(q[row].double().view(kv_heads, -1, dim) @ kk[:seen].permute(1, 2, 0) / math.sqrt(dim), -1)
            want = (w @ vv[:seen].transpose(0, 1)).view(q_heads, dim)
            mag = (w @ vv[:seen].abs().transpose(0, 1)).view(q_heads, dim)
            # probabilities held to 16 bits or more, scores to 2^-20 of their
            # terms' sum: 2^-14 of sum p |v|, and as much of a typical value
            # for a value next to zero, whose code and minimum cancel
            assert bool(((out[row].double() - want).abs() <= 2.0 ** -14 * (mag + 0.1)).all()), (s, i)
    assert ops.device_status() == 0


@pytest.mark.parametrize("q_heads,kv_heads,dim", [(4, 1, 128), (8, 1, 64)])
def test_long_context_relative_to_its_output(cuda, q_heads, kv_heads, dim):
    """Flat weights over many keys: outputs are a hundredth of a value, and
    every sum that is larger and cancels shows."""
    import torch

    from aps2026_b200 import decode

    g = torch.Generator(device="cuda").manual_seed(dim)
    n, page = 30001, 64
    width = -(-n // page)
    table = torch.randperm(width, generator=g, device="cuda").to(torch.int32).view(1, width)
    cache = decode.KVCache4(width, page, kv_heads, dim, "cuda")
    k, v = (torch.randn((n, kv_heads, dim), generator=g, device="cuda") for _ in range(2))
    seq, pos = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    decode.kv4_append_gpu(k, v, seq, pos, cache, table)
    decode.kv4_read_gpu(cache, table, seq, pos, k, v)
    q = torch.randn((1, q_heads, dim), generator=g, device="cuda")
    out = torch.empty_like(q)
    decode.attention_kv4_gpu(q, cache, table, _i32([n]), out)
    w = torch.softmax(q.double().view(kv_heads, -1, dim) @ k.double().permute(1, 2, 0) / math.sqrt(dim), -1)
    want = (w @ v.double().transpose(0, 1)).view(1, q_heads, dim)
    # each weight is off by some 2^-21 of itself (exp2, its argument) and p s
    # by 2^-22, apart from each other, as the values are: the sum's error is
    # that fraction of the sum. Three times it.
    assert float((out.double() - want).norm() / want.norm()) < 3 * (2.0 ** -21)

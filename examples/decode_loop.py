"""Prefill a few prompts into a 4-bit paged cache and decode on, token by token.

A small randomly initialised decoder (LayerNorm, rotated grouped-query
attention, top-2 mixture of experts) built from the library's operators, with
torch matrix products for the projections around them. It shows the decode
operators together, as a serving loop uses them:

    kv4_append_gpu     rotates q and k, keeps k and v in 4 bits
    attention_kv4_gpu  the rows' attention over their sequence's cache
    moe_decode_gpu     routing, experts and their weighted sum

The same `Decoder.forward` takes whole prompts (many rows per sequence) and
single tokens; the single-token step is captured in a CUDA graph.

    python examples/decode_loop.py
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from aps2026_b200 import decode, ops  # noqa: E402

MOE_ROWS = 128  # moe_decode_gpu takes this many rows at a time


class Decoder:
    """Weights, cache and workspaces of `layers` decoder layers for up to
    `seqs` sequences of `max_len` tokens."""

    def __init__(self, layers=2, hidden=512, q_heads=8, kv_heads=2, head_dim=64, experts=8, inter=96, vocab=1000,
                 seqs=4, max_len=512, page_size=16, window=0, sinks=0, seed=0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        rand = lambda *shape, std=1.0: torch.randn(shape, generator=g, device=device) * std  # noqa: E731
        self.hidden, self.q_heads, self.kv_heads, self.head_dim = hidden, q_heads, kv_heads, head_dim
        self.window, self.sinks, self.max_len = window, sinks, max_len
        self.emb, self.head = rand(vocab, hidden), rand(vocab, hidden, std=hidden ** -0.5)
        one, zero = torch.ones(hidden, device=device), torch.zeros(hidden, device=device)
        self.norm, self.layers = (one, zero), []
        pages = -(-max_len // page_size)
        # each sequence owns its pages here; a server hands them out as sequences grow
        self.table = torch.randperm(seqs * pages, generator=g, device=device).to(torch.int32).view(seqs, pages)
        for _ in range(layers):
            self.layers.append(dict(
                ln1=(one, zero), ln2=(one, zero),
                qkv=rand((q_heads + 2 * kv_heads) * head_dim, hidden, std=hidden ** -0.5),
                out=rand(hidden, q_heads * head_dim, std=(q_heads * head_dim) ** -0.5),
                router=rand(experts, hidden, std=hidden ** -0.5),
                gate_up=rand(experts, 2 * inter, hidden, std=hidden ** -0.5).bfloat16(),
                down=rand(experts, hidden, inter, std=inter ** -0.5).bfloat16(),
                cache=decode.KVCache4(seqs * pages, page_size, kv_heads, head_dim, device)))
        cos, sin = ops.rope_table_host(max_len, head_dim, ops.ROPE_THETA)
        self.cos, self.sin = cos.to(device), sin.to(device)
        self.attention_ws = decode.AttentionWorkspace(head_dim, device)
        self.moe_ws = decode.MoeWorkspace(MOE_ROWS, inter, device)

    def forward(self, ids, row_seq, row_pos, lens, q_offsets=None, max_queries=1):
        """Hidden states [rows, hidden] of new rows: token ids[r] is position
        row_pos[r] of sequence row_seq[r], and lens counts the new rows in."""
        rows = ids.numel()
        x = torch.empty(rows, self.hidden, device=ids.device)
        ops.gather_rows_gpu(self.emb, ids, x)
        y = torch.empty_like(x)
        heads = (self.q_heads, self.kv_heads, self.kv_heads)
        for layer in self.layers:
            ops.layer_norm_gpu(x, *layer["ln1"], ops.NORM_EPS, y)
            q, k, v = (y @ layer["qkv"].t()).view(rows, sum(heads), self.head_dim).split(heads, 1)
            q_rot = torch.empty(rows, self.q_heads, self.head_dim, device=x.device)
            decode.kv4_append_gpu(k, v, row_seq, row_pos, layer["cache"], self.table, q=q, q_out=q_rot, cos=self.cos,
                                  sin=self.sin)
            attended = torch.empty_like(q_rot)
            decode.attention_kv4_gpu(q_rot, layer["cache"], self.table, lens, attended, q_offsets=q_offsets,
                                     max_queries=max_queries, max_len=self.max_len, window=self.window,
                                     sinks=self.sinks, ws=self.attention_ws)
            projected = attended.view(rows, -1) @ layer["out"].t()
            ops.add_layer_norm_gpu(x, projected, *layer["ln2"], ops.NORM_EPS, y)
            logits, mixed = y @ layer["router"].t(), torch.empty_like(y)
            for r in range(0, rows, MOE_ROWS):
                part = slice(r, min(rows, r + MOE_ROWS))
                decode.moe_decode_gpu(y[part], logits[part], layer["gate_up"], layer["down"], mixed[part],
                                      ws=self.moe_ws)
            ops.add_inplace_gpu(x, mixed)
        ops.layer_norm_gpu(x, *self.norm, ops.NORM_EPS, y)
        return y

    def prefill(self, prompts):
        """Feeds whole prompts at once; returns every row's hidden state and lens."""
        dev, counts = self.emb.device, [len(p) for p in prompts]
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        seq = i32([s for s, n in enumerate(counts) for _ in range(n)])
        pos = i32([p for n in counts for p in range(n)])
        offsets = i32([sum(counts[:s]) for s in range(len(counts) + 1)])
        lens = i32(counts)
        return self.forward(i32(sum(map(list, prompts), [])), seq, pos, lens, offsets, max(counts)), lens


class Stepper:
    """The single-token step of a batch as a CUDA graph: token -> next token."""

    def __init__(self, model: Decoder, tokens, lens):
        self.token, self.lens = tokens.clone(), lens.clone()
        self.seq = torch.arange(tokens.numel(), dtype=torch.int32, device=tokens.device)
        self.hidden = None

        def step():
            pos = self.lens.clone()       # the new token's position
            self.lens += 1
            self.hidden = model.forward(self.token, self.seq, pos, self.lens)
            self.token.copy_((self.hidden @ model.head.t()).argmax(-1))

        side = torch.cuda.Stream()        # warm up outside the capture, then undo its step
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        self.token.copy_(tokens)
        self.lens.copy_(lens)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            step()

    def __call__(self):
        self.graph.replay()
        return self.token


def main():
    prompts = [[7, 3, 900, 41], list(range(100, 170)), [5], [11, 12, 13] * 9]
    model = Decoder()
    hidden, lens = model.prefill(prompts)
    last = torch.tensor([sum(map(len, prompts[:s + 1])) - 1 for s in range(len(prompts))], device="cuda")
    first = (hidden[last] @ model.head.t()).argmax(-1).to(torch.int32)
    step, steps = Stepper(model, first, lens), 64
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    out = [first.tolist()]
    start.record()
    for _ in range(steps):
        step()
    stop.record()
    torch.cuda.synchronize()
    out.append(step.token.tolist())
    assert ops.device_status() == 0
    print(f"{len(prompts)} sequences, {steps} steps, {start.elapsed_time(stop) / steps * 1e3:.1f} us per step; "
          f"lengths {lens.tolist()} -> {step.lens.tolist()}, first tokens {out[0]}, last {out[1]}")


if __name__ == "__main__":
    main()

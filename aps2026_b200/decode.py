"""The decode step on torch CUDA tensors: a 4-bit paged KV cache, the
attention over it, and the expert layer for a few tokens.

What carries a prefilled model on, token by token. There is no reference
counterpart (ezzy0654/aps2026 recomputes every prompt); the definitions are
those of ``include/aps2026_b200.h``. Every call runs on the current torch CUDA
stream through the C ABI; refusals raise ``ops.InvalidArgument``, CUDA
failures ``ops.CudaError``. Positions, pages, lengths and offsets live on the
device: what is out of range there is skipped and reported by
``ops.device_status()`` (``B2_CHECK_KV4``, ``B2_CHECK_ROPE``).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .ops import ROUTER_SCORE_QUANTUM, ROUTER_TIE_EPS, InvalidArgument, _check

_lib.lib()  # says so when nothing is built
try:
    from . import _decode_calls  # checks the tensors and makes the C ABI call (pyext/decode_calls.cpp)
except ImportError as e:
    raise ImportError("aps2026_b200/_decode_calls.so: not built, or for another torch; run `python -m aps2026_b200.build`") from e

PADDING = -1  # row_seq of a row that is not there

_GATES = {"equal": _lib.B2_GATES_EQUAL, "softmax": _lib.B2_GATES_SOFTMAX}


class _CacheStruct(C.Structure):
    """b2_kv4_cache, for calls of the C ABI through _lib.lib()"""
    _fields_ = [("data", C.c_void_p), ("pages", C.c_size_t), ("page_size", C.c_size_t), ("kv_heads", C.c_size_t),
                ("head_dim", C.c_size_t), ("page_table", C.c_void_p), ("seqs", C.c_size_t),
                ("max_pages", C.c_size_t)]


class KVCache4:
    """Keys and values of many sequences in 4 bits, in `pages` pages of
    `page_size` positions. A page table [seqs, max_pages] (int32, device)
    says which page holds which positions of a sequence; the user's program
    hands pages out."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, device):
        n = C.c_size_t(0)
        _check(_lib.lib().b2_kv4_page_bytes(page_size, kv_heads, head_dim, C.addressof(n)), "KVCache4")
        self.pages, self.page_size, self.kv_heads, self.head_dim = pages, page_size, kv_heads, head_dim
        self.data = torch.zeros(pages, n.value, dtype=torch.uint8, device=device)


def kv4_append_gpu(k, v, row_seq, row_pos, cache: KVCache4, page_table, q=None, q_out=None, cos=None,
                   sin=None) -> None:
    """Appends rows to the cache (b2_kv4_append): keys rotated at row_pos and
    rounded to 4 bits, values rounded, stored at (row_seq, row_pos); with q,
    q_out = the rotated queries. k, v: [rows, kv_heads, head_dim], q and q_out
    [rows, q_heads, head_dim], fp32 or bf16, q_out contiguous and 16-byte
    aligned; cos, sin: the fp32 tables
    [positions, head_dim / 2] of rope_table_host on the device, or None for no
    rotation. row_seq = PADDING marks a row that is not there."""
    rc = _decode_calls.kv4_append(k, v, row_seq, row_pos, cache.data, cache.pages, cache.page_size, cache.kv_heads,
                                  cache.head_dim, page_table, q, q_out, cos, sin)
    if rc:
        _check(rc, "kv4_append_gpu")


def kv4_read_gpu(cache: KVCache4, page_table, row_seq, row_pos, k_out, v_out) -> None:
    """k_out, v_out [rows, kv_heads, head_dim], contiguous and 16-byte aligned,
    = the values the cache holds at (row_seq, row_pos) (b2_kv4_read), e.g. the K
    and V of a cached prefix for attention_tree_gpu."""
    rc = _decode_calls.kv4_read(cache.data, cache.pages, cache.page_size, cache.kv_heads, cache.head_dim, page_table,
                                row_seq, row_pos, k_out, v_out)
    if rc:
        _check(rc, "kv4_read_gpu")


class AttentionWorkspace:
    """Scratch of attention_kv4_gpu, kept between calls; calls that overlap on
    the GPU (other streams) must not share one."""

    def __init__(self, head_dim: int, device):
        n = C.c_size_t(0)
        _check(_lib.lib().b2_attention_kv4_workspace_size(head_dim, C.addressof(n)), "workspace size")
        self.bytes = n.value
        self.buf = torch.zeros(self.bytes, dtype=torch.uint8, device=device)


def attention_kv4_gpu(q, cache: KVCache4, page_table, lens, out, q_offsets=None, max_queries: int = 1,
                      max_len: int | None = None, scale: float | None = None, window: int = 0, sinks: int = 0,
                      ws: AttentionWorkspace | None = None) -> None:
    """out = attention of each sequence's newest query rows over its cached
    keys and values (b2_attention_kv4). q, out: [rows, q_heads, head_dim],
    fp32 or bf16, out contiguous and 16-byte aligned; lens [seqs] counts the
    cached positions, the query rows' own among them; q_offsets [seqs + 1] splits the rows between the sequences
    (None: one row each). Key j is visible at position p when j <= p and
    (p - j < window or j < sinks); window 0: no window. max_queries and
    max_len (default: the page table's reach) bound a sequence's query rows
    and length."""
    if ws is None:
        ws = AttentionWorkspace(cache.head_dim, cache.data.device)
    rc = _decode_calls.attention_kv4(q, cache.data, cache.pages, cache.page_size, cache.kv_heads, cache.head_dim,
                                     page_table, lens, out, q_offsets, max_queries, max_len, scale, window, sinks,
                                     ws.buf, ws.bytes)
    if rc:
        _check(rc, "attention_kv4_gpu")


class MoeWorkspace:
    """Scratch of moe_decode_gpu for up to `tokens` tokens; calls that overlap
    on the GPU must not share one."""

    def __init__(self, tokens: int, inter: int, device):
        n = C.c_size_t(0)
        _check(_lib.lib().b2_moe_decode_workspace_size(tokens, inter, C.addressof(n)), "workspace size")
        self.bytes = n.value
        self.buf = torch.empty(self.bytes, dtype=torch.uint8, device=device)


def moe_decode_gpu(x, logits, w_gate_up, w_down, out, quantum: float = ROUTER_SCORE_QUANTUM,
                   tie_eps: float = ROUTER_TIE_EPS, gates: str = "equal", ws: MoeWorkspace | None = None) -> None:
    """out = the whole expert layer of up to 128 tokens (b2_moe_decode): the
    top-2 routing of moe_route_gpu, silu(gate) * up, down, and the sum over a
    token's two experts weighed by `gates`: "equal" (0.5 each, as
    moe_combine_gpu) or "softmax" over the two picked logits. x, out: [T, H]
    fp32 or bf16 (row strides allowed); logits [T, E] fp32; w_gate_up
    [E, 2I, H] and w_down [E, H, I] fp32 or bf16."""
    code = _GATES.get(gates)
    if code is None:
        raise InvalidArgument(f"moe_decode: gates must be one of {sorted(_GATES)}")
    if ws is None:
        if not all(isinstance(t, torch.Tensor) for t in (x, w_down)) or x.dim() != 2 or w_down.dim() != 3:
            raise InvalidArgument("moe_decode: expected x [T, H] and w_down [E, H, I]")
        ws = MoeWorkspace(x.shape[0], w_down.shape[2], x.device)
    rc = _decode_calls.moe_decode(x, logits, w_gate_up, w_down, out, quantum, tie_eps, code, ws.buf, ws.bytes)
    if rc:
        _check(rc, "moe_decode_gpu")

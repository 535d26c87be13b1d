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
import struct

import torch

from . import _lib
from .ops import ROUTER_SCORE_QUANTUM, ROUTER_TIE_EPS, InvalidArgument, _check

PADDING = -1  # row_seq of a row that is not there

_DTYPES = {torch.float32: _lib.B2_DTYPE_F32, torch.bfloat16: _lib.B2_DTYPE_BF16}
_GATES = {"equal": _lib.B2_GATES_EQUAL, "softmax": _lib.B2_GATES_SOFTMAX}
_INDEX = (torch.int32, torch.uint32)


class _CacheStruct(C.Structure):
    """b2_kv4_cache"""
    _fields_ = [("data", C.c_void_p), ("pages", C.c_size_t), ("page_size", C.c_size_t), ("kv_heads", C.c_size_t),
                ("head_dim", C.c_size_t), ("page_table", C.c_void_p), ("seqs", C.c_size_t),
                ("max_pages", C.c_size_t)]


# The same struct as bytes: a call's own immutable copy, cheaper to make.
_pack_cache = struct.Struct("@PNNNNPNN").pack
assert struct.calcsize("@PNNNNPNN") == C.sizeof(_CacheStruct)


def _dtype(t: torch.Tensor, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise InvalidArgument(f"{what}: expected float32 or bfloat16, got {t.dtype}")
    return code


# The checks below compare device indices (get_device() is -1 on the host) and
# leave the wording of what is wrong to the refusal: a decode step makes them
# some twenty times.


def _index(t: torch.Tensor, n: int, device: int, what: str) -> int:
    """Address of a contiguous device vector of n 32-bit indices."""
    if t.dtype not in _INDEX or t.numel() != n or t.get_device() != device or not t.is_contiguous():
        raise InvalidArgument(f"{what}: expected {n} contiguous 32-bit indices on CUDA device {device}")
    return t.data_ptr()


def _heads(t: torch.Tensor, rows: int, heads: int, dim: int, device: int, what: str) -> tuple[int, int, int]:
    """Address and strides of [rows, heads, dim] activations whose last
    dimension is contiguous (slices of a fused projection are)."""
    if t.shape != (rows, heads, dim) or t.get_device() != device:
        raise InvalidArgument(f"{what}: expected [{rows}, {heads}, {dim}] on CUDA device {device}")
    by_row, by_head, by_dim = t.stride()
    if by_dim != 1 and rows:
        raise InvalidArgument(f"{what}: the last dimension must be contiguous")
    return t.data_ptr(), by_row, by_head


def _whole(t: torch.Tensor, shape: tuple, dtype: torch.dtype, device: int, what: str) -> int:
    if t.dtype != dtype or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        raise InvalidArgument(f"{what}: expected a contiguous {tuple(shape)} {dtype} tensor on CUDA device {device}")
    return t.data_ptr()


def _on_gpu(device: int) -> int:
    """The current stream of CUDA device `device`, which must be the current one."""
    if device < 0:
        raise InvalidArgument("tensor is not on a CUDA device")
    if device != _current_device():
        raise InvalidArgument(f"tensors are on CUDA device {device}, the current one is {_current_device()}")
    # torch.cuda.current_stream().cuda_stream without the 3 us of building a Stream
    return torch._C._cuda_getCurrentRawStream(device)


def _current_device() -> int:
    # torch.cuda.current_device() without its lazy initialisation: a tensor is there
    return torch._C._cuda_getDevice()


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
        self._device = self.data.get_device()

    def _struct(self, page_table: torch.Tensor) -> bytes:
        shape = page_table.shape
        if (len(shape) != 2 or page_table.dtype not in _INDEX or page_table.get_device() != self._device
                or not page_table.is_contiguous()):
            raise InvalidArgument("page_table: expected contiguous 32-bit indices [seqs, max_pages] on the cache's device")
        seqs, max_pages = shape
        return _pack_cache(self.data.data_ptr(), self.pages, self.page_size, self.kv_heads, self.head_dim,
                           page_table.data_ptr(), seqs, max_pages)


def kv4_append_gpu(k, v, row_seq, row_pos, cache: KVCache4, page_table, q=None, q_out=None, cos=None,
                   sin=None) -> None:
    """Appends rows to the cache (b2_kv4_append): keys rotated at row_pos and
    rounded to 4 bits, values rounded, stored at (row_seq, row_pos); with q,
    q_out = the rotated queries. k, v: [rows, kv_heads, head_dim], q and q_out
    [rows, q_heads, head_dim], fp32 or bf16; cos, sin: the fp32 tables
    [positions, head_dim / 2] of rope_table_host on the device, or None for no
    rotation. row_seq = PADDING marks a row that is not there."""
    device = cache._device
    stream = _on_gpu(device)
    rows, heads, dim = k.shape[0], cache.kv_heads, cache.head_dim
    dtype = _dtype(k, "kv4_append k")
    if v.dtype != k.dtype:
        raise InvalidArgument("kv4_append: q, k and v must have one dtype")
    kp, kr, kh = _heads(k, rows, heads, dim, device, "kv4_append k")
    vp, vr, vh = _heads(v, rows, heads, dim, device, "kv4_append v")
    qp = qo = None
    qr = qh = q_heads = 0
    if q is not None:
        if q.dtype != k.dtype:
            raise InvalidArgument("kv4_append: q, k and v must have one dtype")
        if q_out is None:
            raise InvalidArgument("kv4_append: q without q_out")
        q_heads = q.shape[1]
        qp, qr, qh = _heads(q, rows, q_heads, dim, device, "kv4_append q")
        qo = _whole(q_out, (rows, q_heads, dim), q.dtype, device, "kv4_append q_out")
    cp = sp = None
    positions = 0
    if (cos is None) != (sin is None):
        raise InvalidArgument("kv4_append: one rotation table without the other")
    if cos is not None:
        positions = cos.shape[0]
        cp = _whole(cos, (positions, dim // 2), torch.float32, device, "kv4_append cos")
        sp = _whole(sin, (positions, dim // 2), torch.float32, device, "kv4_append sin")
    rc = _lib.lib().b2_kv4_append(
        qp, qr, qh, q_heads, qo, kp, kr, kh, vp, vr, vh, dtype, rows, _index(row_seq, rows, device, "row_seq"),
        _index(row_pos, rows, device, "row_pos"), cp, sp, positions, cache._struct(page_table), stream)
    if rc:
        _check(rc, "kv4_append_gpu")


def kv4_read_gpu(cache: KVCache4, page_table, row_seq, row_pos, k_out, v_out) -> None:
    """k_out, v_out [rows, kv_heads, head_dim] = the values the cache holds at
    (row_seq, row_pos) (b2_kv4_read), e.g. the K and V of a cached prefix for
    attention_tree_gpu."""
    device = cache._device
    stream = _on_gpu(device)
    rows = row_seq.numel()
    shape = (rows, cache.kv_heads, cache.head_dim)
    rc = _lib.lib().b2_kv4_read(
        cache._struct(page_table), _index(row_seq, rows, device, "row_seq"), _index(row_pos, rows, device, "row_pos"),
        rows, _whole(k_out, shape, k_out.dtype, device, "kv4_read k_out"),
        _whole(v_out, shape, k_out.dtype, device, "kv4_read v_out"), _dtype(k_out, "kv4_read k_out"), stream)
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
    fp32 or bf16; lens [seqs] counts the cached positions, the query rows'
    own among them; q_offsets [seqs + 1] splits the rows between the sequences
    (None: one row each). Key j is visible at position p when j <= p and
    (p - j < window or j < sinks); window 0: no window. max_queries and
    max_len (default: the page table's reach) bound a sequence's query rows
    and length."""
    device = cache._device
    stream = _on_gpu(device)
    shape = q.shape
    if len(shape) != 3:
        raise InvalidArgument("attention_kv4 q: expected [rows, q_heads, head_dim]")
    rows, q_heads, dim = shape
    qp, qr, qh = _heads(q, rows, q_heads, cache.head_dim, device, "attention_kv4 q")
    seqs, max_pages = page_table.shape if page_table.dim() == 2 else (0, 0)
    if max_len is None:
        max_len = max_pages * cache.page_size
    if max_queries < 0 or max_len < 0 or window < 0 or sinks < 0:
        raise InvalidArgument("attention_kv4: negative max_queries, max_len, window or sinks")
    if ws is None:
        ws = AttentionWorkspace(cache.head_dim, cache.data.device)
    elif ws.buf.get_device() != device:
        raise InvalidArgument("attention_kv4: the workspace is on another device")
    rc = _lib.lib().b2_attention_kv4(
        qp, qr, qh, _whole(out, shape, q.dtype, device, "attention_kv4 out"), _dtype(q, "attention_kv4 q"), rows, q_heads,
        None if q_offsets is None else _index(q_offsets, seqs + 1, device, "q_offsets"),
        _index(lens, seqs, device, "lens"), max_queries, max_len, dim ** -0.5 if scale is None else scale, window,
        sinks, cache._struct(page_table), ws.buf.data_ptr(), ws.bytes, stream)
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
    device = x.get_device()
    stream = _on_gpu(device)
    if x.dim() != 2 or w_down.dim() != 3:
        raise InvalidArgument("moe_decode: expected x [T, H] and w_down [E, H, I]")
    T, H = x.shape
    E, _, I = w_down.shape  # noqa: E741
    code = _GATES.get(gates)
    if code is None:
        raise InvalidArgument(f"moe_decode: gates must be one of {sorted(_GATES)}")
    if out.shape != (T, H) or out.dtype != x.dtype or out.get_device() != device:
        raise InvalidArgument(f"moe_decode out: expected [{T}, {H}] {x.dtype} on CUDA device {device}")
    (x_row, x_dim), (out_row, out_dim) = x.stride(), out.stride()
    if H > 1 and (x_dim != 1 or out_dim != 1):
        raise InvalidArgument("moe_decode: the last dimension of x and out must be contiguous")
    weights = w_down.dtype
    if ws is None:
        ws = MoeWorkspace(T, I, x.device)
    elif ws.buf.get_device() != device:
        raise InvalidArgument("moe_decode: the workspace is on another device")
    rc = _lib.lib().b2_moe_decode(
        x.data_ptr(), x_row if T > 1 else H, _dtype(x, "moe_decode x"),
        _whole(logits, (T, E), torch.float32, device, "moe_decode logits"), T, H, E, I, quantum, tie_eps, code,
        _whole(w_gate_up, (E, 2 * I, H), weights, device, "moe_decode w_gate_up"),
        _whole(w_down, (E, H, I), weights, device, "moe_decode w_down"), _dtype(w_down, "moe_decode w_down"),
        out.data_ptr(), out_row if T > 1 else H, ws.buf.data_ptr(), ws.bytes, stream)
    if rc:
        _check(rc, "moe_decode_gpu")

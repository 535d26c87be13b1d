"""The decode step's operators as a user's program calls them, each next to
its plain form in elementary torch operations.

Three operators carry a model past its prefill:

- ``append``: new rows' queries and keys are rotated, keys and values are
  rounded to 4 bits (one scale and one minimum per 64 dimensions, both bf16)
  and stored in a paged cache; the rows are then read back as the values the
  cache holds.
- ``attention``: each sequence's newest rows attend over its cached keys and
  values. Key j is visible at position p when j <= p and either p - j < window
  or j < sinks.
- ``moe``: a whole mixture-of-experts layer for a few tokens: top-2 routing of
  router logits, the gated expert products and the weighted sum.

``own`` selects the framework's kernels (true) or the plain form (false).
"""
import math
import struct

import torch

own = False

GROUP = 64                      # dimensions that share a scale and a minimum
SMALLEST_STEP = 2.0 ** -126     # steps below it count as zero
QUANTUM, TIE_EPS = 1.0e-3, 2.0e-2   # routing: score grid and tie margin
F32, BF16 = "float32", "bfloat16"


def _dtype(name):
    return torch.bfloat16 if name == BF16 else torch.float32


def _bytes(name):
    return 2 if name == BF16 else 4


# ---- the cases ----------------------------------------------------------------


def _append(name, **kw):
    """batch sequences; sequence b gets new_b rows (ragged between new_min and
    new_max) after the past rows it already has."""
    case = dict(op="append", batch=1, new_min=1, new_max=1, past=0, q_heads=16, kv_heads=4, head_dim=128,
                page=16, dtype=F32, fused_qkv=False)
    case.update(kw)
    if name:
        case["name"] = name
    return case


def _attention(name, **kw):
    """batch sequences of len_min..len_max cached tokens, the last `queries`
    of which ask; window 0 means no window; empty marks the first sequence as
    one with nothing cached."""
    case = dict(op="attention", batch=1, len_min=1, len_max=1, queries=1, q_heads=16, kv_heads=4, head_dim=128,
                page=16, window=0, sinks=0, dtype=F32, empty=False)
    case.update(kw)
    if name:
        case["name"] = name
    return case


def _moe(name, **kw):
    case = dict(op="moe", tokens=1, hidden=4096, inter=448, experts=16, dtype=F32, weights=BF16, gates="equal")
    case.update(kw)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one user's next token enters the cache: pure latency
        _append("append_one_token", past=611),
        # a step of a serving batch, every sequence one token
        _append("append_batch_step", batch=64, past=1500, page=64, dtype=BF16),
        # ragged prompts enter the cache after prefill, k and v being slices
        # of one fused projection
        _append("append_prompts", batch=13, new_min=37, new_max=2048, fused_qkv=True),
        # a short chat, one token: latency
        _attention("attention_short", len_min=37, len_max=37),
        # a serving batch inside the model's window of 2047
        _attention("attention_batch", batch=32, len_min=129, len_max=4096, window=2047, dtype=BF16),
        # one long document, one token: only the split over keys fills the GPU
        _attention("attention_one_long", len_min=131069, len_max=131069, page=64, dtype=BF16),
        # streaming sequences far past the window with 4 sink tokens, three
        # drafted tokens checked at once, one sequence still empty
        _attention("attention_window_sinks", batch=24, len_min=7001, len_max=60007, queries=3, q_heads=8,
                   kv_heads=8, head_dim=64, window=2047, sinks=4, page=32, empty=True),
        # the largest: a full batch of long ragged contexts
        _attention("attention_large", batch=64, len_min=4095, len_max=32768, page=64),
        # one token through the expert layer, experts in bf16
        _moe("moe_one_token"),
        # a small serving batch, softmax gates, all bf16
        _moe("moe_batch_9", tokens=9, dtype=BF16, gates="softmax"),
        # weights kept in fp32, a batch that reaches every expert
        _moe("moe_batch_61_fp32", tokens=61, weights=F32),
        # the most tokens, odd sizes that no vector load divides
        _moe("moe_odd_128", tokens=128, hidden=1001, inter=333, experts=7),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    op = rng.choice(["append", "attention", "moe"])
    q_heads, kv_heads = rng.choice([(16, 4), (8, 8), (32, 8), (8, 1), (12, 4)])
    head_dim = rng.choice([64, 128, 128])
    page = rng.choice([8, 16, 32, 64, 128])
    dtype = rng.choice([F32, BF16])
    if op == "append":
        rows = _log_int(rng, 1, 6000)
        batch = _log_int(rng, 1, min(rows, 64))
        most = max(1, (2 * rows) // batch)
        return _append(None, batch=batch, new_min=rng.randint(1, most), new_max=most, past=_log_int(rng, 1, 4000) - 1,
                       q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype,
                       fused_qkv=rng.random() < 0.5)
    if op == "attention":
        batch = _log_int(rng, 1, 64)
        longest = _log_int(rng, 1, min(131072, 4194304 // (batch * kv_heads)))
        shortest = rng.randint(max(1, longest // 8), longest)
        window, sinks = rng.choice([(0, 0), (2047, 0), (rng.randint(1, 3000), 0),
                                    (2047, rng.randint(1, 9)), (rng.randint(1, 3000), rng.randint(1, 100))])
        return _attention(None, batch=batch, len_min=shortest, len_max=longest,
                          queries=min(rng.choice([1, 1, 1, 2, 3, 5, 8]), shortest), q_heads=q_heads,
                          kv_heads=kv_heads, head_dim=head_dim, page=page, window=window, sinks=sinks, dtype=dtype,
                          empty=rng.random() < 0.2)
    odd = rng.random() < 0.4
    hidden = _log_int(rng, 256, 4096)
    inter = _log_int(rng, 64, 1024)
    if not odd:
        hidden, inter = max(256, hidden // 64 * 64), max(64, inter // 32 * 32)
    experts = rng.choice([4, 7, 8, 16, 32])
    while experts * hidden * inter > 16 * 4096 * 448:
        inter = max(64, inter // 2)
        hidden = max(256, hidden // 2 if inter == 64 else hidden)
    return _moe(None, tokens=_log_int(rng, 1, 128), hidden=hidden, inter=inter, experts=experts, dtype=dtype,
                weights=F32 if dtype == F32 and rng.random() < 0.5 else BF16, gates=rng.choice(["equal", "softmax"]))


def _spread(lo, hi, n):
    """n ragged sizes from lo to hi, both ends among them (out of order unless
    n shares a factor with 37)."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * ((i * 37 + 11) % n if math.gcd(37, n) == 1 else i) // (n - 1) for i in range(n)]


def _lens(case):
    lens = _spread(case["len_min"], case["len_max"], case["batch"])
    if case["empty"]:
        lens[0] = 0
    return lens


def _visible(case, length):
    """Keys that one of a sequence's query rows can see."""
    first = max(0, length - case["queries"])      # oldest query position
    if length == 0:
        return 0
    if not case["window"]:
        return length
    low = max(0, first - case["window"] + 1)
    return length - low + min(case["sinks"], low)


# ---- inputs ----------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _channel_gain(g, heads, dim):
    """Keys have a few large channels, as trained models' do."""
    gain = torch.ones(heads, dim, device="cuda")
    big = torch.randint(0, dim, (heads, 3), generator=g, device="cuda")
    return gain.scatter_(1, big, 4.0)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _page_table(case, g, needed):
    """A table of needed[b] = the logical pages that sequence b keeps, in
    physical pages handed out in random order; the others are -1."""
    width = max([1] + [p + 1 for pages in needed for p in pages[-1:]])
    count = sum(len(p) for p in needed)
    order = torch.randperm(max(count, 1), generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(needed), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, pages in enumerate(needed):
        if pages:
            table[b, torch.tensor(pages, device="cuda")] = order[at:at + len(pages)]
            at += len(pages)
    return table, max(count, 1)


def _rope_tables(positions, head_dim):
    half = head_dim // 2
    inv = 10000.0 ** (-2.0 * torch.arange(half, dtype=torch.float32, device="cuda") / head_dim)
    angle = torch.arange(positions, dtype=torch.float32, device="cuda")[:, None] * inv
    return torch.cos(angle), torch.sin(angle)


class _PlainCache:
    """The 4-bit cache in plain tensors, one byte for each code."""

    def __init__(self, pages, page, heads, dim):
        shape = (pages, page, heads, dim)
        groups = (pages, page, heads, dim // GROUP, 2)
        self.codes = [torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in range(2)]
        self.params = [torch.zeros(groups, dtype=torch.bfloat16, device="cuda") for _ in range(2)]

    def store(self, which, x, page_ids, slots):
        codes, params = _quantise(x)
        self.codes[which][page_ids, slots] = codes
        self.params[which][page_ids, slots] = params

    def load(self, which, page_ids, slots):
        return _values(self.codes[which][page_ids, slots], self.params[which][page_ids, slots])


def _quantise(x):
    """x [rows, heads, dim] -> codes (uint8) and (scale, minimum) per group."""
    rows, heads, dim = x.shape
    x = x.float().view(rows, heads, dim // GROUP, GROUP)
    low = x.amin(-1).to(torch.bfloat16)
    step = ((x.amax(-1) - low.float()).clamp(min=0.0) * (1.0 / 15.0)).to(torch.bfloat16)
    wide = step.float()
    inverse = torch.where(wide < SMALLEST_STEP, torch.zeros_like(wide), torch.ones_like(wide) / wide)
    codes = torch.round((x - low.float()[..., None]) * inverse[..., None]).clamp(0.0, 15.0)
    codes = codes.to(torch.uint8).view(rows, heads, dim)
    return codes, torch.stack([step, low], -1)


def _values(codes, params):
    wide = params.float()
    shape = codes.shape
    grouped = codes.view(*shape[:-1], shape[-1] // GROUP, GROUP).float()
    return (grouped * wide[..., 0:1] + wide[..., 1:2]).view(shape)


def _locate(table, seq, pos, page):
    return table[seq, pos // page].long(), pos % page


def _append_inputs(case, seed):
    g = _generator(seed)
    new = _spread(case["new_min"], case["new_max"], case["batch"])
    page = case["page"]
    table, pages = _page_table(case, g, [list(range((case["past"] + n + page - 1) // page)) for n in new])
    rows = sum(new)
    qh, kh, dim = case["q_heads"], case["kv_heads"], case["head_dim"]
    dtype = _dtype(case["dtype"])
    if case["fused_qkv"]:
        fused = _normal(g, (rows, qh + 2 * kh, dim), dtype)
        q, k, v = fused[:, :qh], fused[:, qh:qh + kh], fused[:, qh + kh:]
    else:
        q, k, v = (_normal(g, (rows, h, dim), dtype) for h in (qh, kh, kh))
    k.mul_(_channel_gain(g, kh, dim).to(dtype))
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
    pos = torch.cat([torch.arange(n, device="cuda") for n in new]) + case["past"]
    cos, sin = _rope_tables(case["past"] + max(new), dim)
    return dict(q=q, k=k, v=v, seq=seq, pos=pos, cos=cos, sin=sin, table=table, pages=pages)


def _fill_pieces(case, g, table):
    """The cached rows of every sequence, one piece at a time."""
    page = case["page"]
    kh, dim = case["kv_heads"], case["head_dim"]
    gain = _channel_gain(g, kh, dim)
    for b, length in enumerate(_lens(case)):
        pages = _kept_pages(case, length)
        if not pages:
            continue
        kept = torch.tensor(pages, device="cuda")
        pos = (kept[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)
        pos = pos[pos < length]
        k = _normal(g, (pos.numel(), kh, dim)) * gain
        v = _normal(g, (pos.numel(), kh, dim))
        yield torch.full_like(pos, b), pos, k, v


def _kept_pages(case, length):
    """Logical pages that hold a key some query row sees."""
    if length == 0:
        return []
    page = case["page"]
    last = (length - 1) // page
    if not case["window"]:
        return list(range(last + 1))
    low = max(0, length - case["queries"] - case["window"] + 1)
    sink = (min(case["sinks"], length) + page - 1) // page
    return list(range(min(sink, low // page))) + list(range(low // page, last + 1))


def _attention_inputs(case, seed):
    g = _generator(seed)
    lens = _lens(case)
    table, pages = _page_table(case, g, [_kept_pages(case, n) for n in lens])
    q = _normal(g, (case["batch"] * case["queries"], case["q_heads"], case["head_dim"]), _dtype(case["dtype"]))
    return g, q, lens, table, pages


def _moe_inputs(case, seed):
    g = _generator(seed)
    t, h, i, e = case["tokens"], case["hidden"], case["inter"], case["experts"]
    wdt = _dtype(case["weights"])
    return dict(x=_normal(g, (t, h), _dtype(case["dtype"])), logits=_normal(g, (t, e)),
                gate_up=(_normal(g, (e, 2 * i, h)) / math.sqrt(h)).to(wdt),
                down=(_normal(g, (e, h, i)) / math.sqrt(i)).to(wdt))


def prepare(case, seed):
    state = dict(case=case)
    op = case["op"]
    if own:
        from aps2026_b200 import decode

        state["decode"] = decode
    if op == "append":
        state.update(_append_inputs(case, seed))
        if own:
            state["seq"], state["pos"] = state["seq"].to(torch.int32), state["pos"].to(torch.int32)
            state["cache"] = decode.KVCache4(state["pages"], case["page"], case["kv_heads"], case["head_dim"], "cuda")
            rows = state["q"].shape[0]
            state["q_out"] = torch.empty(rows, case["q_heads"], case["head_dim"], dtype=state["q"].dtype,
                                         device="cuda")
            state["k_out"], state["v_out"] = (torch.empty(rows, case["kv_heads"], case["head_dim"],
                                                          dtype=state["q"].dtype, device="cuda") for _ in range(2))
        else:
            state["cache"] = _PlainCache(state["pages"], case["page"], case["kv_heads"], case["head_dim"])
    elif op == "attention":
        g, q, lens, table, pages = _attention_inputs(case, seed)
        state.update(q=q, lens=_int32(lens), table=table)
        page, kh, dim = case["page"], case["kv_heads"], case["head_dim"]
        if own:
            cache = decode.KVCache4(pages, page, kh, dim, "cuda")
            for seq, pos, k, v in _fill_pieces(case, g, table):
                decode.kv4_append_gpu(k, v, seq.to(torch.int32), pos.to(torch.int32), cache, table)
            n = case["queries"]
            state["q_offsets"] = _int32([n * b for b in range(case["batch"] + 1)])
            state["workspace"] = decode.AttentionWorkspace(dim, "cuda")
            state["out"] = torch.empty_like(q)
        else:
            cache = _PlainCache(pages, page, kh, dim)
            for seq, pos, k, v in _fill_pieces(case, g, table):
                where = _locate(table, seq, pos, page)
                cache.store(0, k, *where)
                cache.store(1, v, *where)
        state["cache"] = cache
    else:
        state.update(_moe_inputs(case, seed))
        if own:
            state["out"] = torch.empty_like(state["x"])
            state["workspace"] = decode.MoeWorkspace(case["tokens"], case["inter"], "cuda")
    return state


# ---- one pass ----------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return dict(append=_own_append, attention=_own_attention, moe=_own_moe)[op](state)
    return dict(append=_plain_append, attention=_plain_attention, moe=_plain_moe)[op](state)


def _own_append(s):
    decode = s["decode"]
    decode.kv4_append_gpu(s["k"], s["v"], s["seq"], s["pos"], s["cache"], s["table"], q=s["q"], q_out=s["q_out"],
                          cos=s["cos"], sin=s["sin"])
    decode.kv4_read_gpu(s["cache"], s["table"], s["seq"], s["pos"], s["k_out"], s["v_out"])
    return s["q_out"], s["k_out"], s["v_out"]


def _own_attention(s):
    c = s["case"]
    s["decode"].attention_kv4_gpu(s["q"], s["cache"], s["table"], s["lens"], s["out"], q_offsets=s["q_offsets"],
                                  max_queries=c["queries"], max_len=c["len_max"], window=c["window"],
                                  sinks=c["sinks"], ws=s["workspace"])
    return s["out"]


def _own_moe(s):
    s["decode"].moe_decode_gpu(s["x"], s["logits"], s["gate_up"], s["down"], s["out"], quantum=QUANTUM,
                               tie_eps=TIE_EPS, gates=s["case"]["gates"], ws=s["workspace"])
    return s["out"]


def _rotate(x, cos, sin):
    x = x.float()
    half = x.shape[-1] // 2
    first, second = x[..., :half], x[..., half:]
    return torch.cat([first * cos - second * sin, second * cos + first * sin], -1)


def _plain_append(s):
    dtype = s["q"].dtype
    cos, sin = s["cos"][s["pos"]][:, None], s["sin"][s["pos"]][:, None]
    where = _locate(s["table"], s["seq"], s["pos"], s["case"]["page"])
    cache = s["cache"]
    cache.store(0, _rotate(s["k"], cos, sin), *where)
    cache.store(1, s["v"], *where)
    return (_rotate(s["q"], cos, sin).to(dtype), cache.load(0, *where).to(dtype), cache.load(1, *where).to(dtype))


def _key_positions(case, length, count):
    """Positions of the keys that a sequence of `length` (device scalar) may
    show its query rows, `count` of them at most; the rest are >= length."""
    u = torch.arange(count, device="cuda")
    if not case["window"]:
        return u
    low = (length - case["queries"] - case["window"] + 1).clamp(min=0)
    sinks = low.clamp(max=case["sinks"])
    return torch.where(u < sinks, u, u - sinks + low)


def _plain_attention(s):
    case, q, lens, table, cache = s["case"], s["q"], s["lens"], s["table"], s["cache"]
    kh, dim, n = case["kv_heads"], case["head_dim"], case["queries"]
    group = case["q_heads"] // kh
    most = _visible(case, case["len_max"])
    capacity = table.shape[1] * case["page"]
    outs = []
    for b in range(case["batch"]):
        length = lens[b].long()
        keys = _key_positions(case, length, most)
        live = keys < length
        where = _locate(table[b:b + 1], torch.zeros_like(keys), torch.where(live, keys, 0).clamp(max=capacity - 1),
                        case["page"])
        k = cache.load(0, *where)
        v = torch.where(live[:, None, None], cache.load(1, *where), 0.0)
        rows = q[b * n:(b + 1) * n].float().view(n, kh, group, dim)
        scores = torch.einsum("nhgd,khd->hgnk", rows, k) * (1.0 / math.sqrt(dim))
        pos = length - n + torch.arange(n, device="cuda")
        seen = live & (keys <= pos[:, None])
        if case["window"]:
            seen = seen & ((pos[:, None] - keys < case["window"]) | (keys < case["sinks"]))
        scores = torch.where(seen, scores, float("-inf"))
        top = scores.amax(-1, keepdim=True)
        weights = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
        total = weights.sum(-1, keepdim=True)
        weights = weights / torch.where(total > 0, total, 1.0)
        outs.append(torch.einsum("hgnk,khd->nhgd", weights, v).reshape(n, kh * group, dim))
    return torch.cat(outs).to(q.dtype)


def _pick(logits, quantum, tie_eps):
    """The two experts of each token: scores on a grid, scanned in ascending
    order, an expert taking the lead by more than tie_eps only."""
    logits = logits.float()
    score = torch.sign(logits) * (torch.floor(logits.abs() / torch.full_like(logits, quantum) + 0.5) * quantum)
    chosen = []
    for _ in range(2):
        best = torch.full_like(score[:, 0], -torch.inf)
        lead = torch.full_like(best, -1, dtype=torch.long)
        for e in range(score.shape[1]):
            better = (lead < 0) | (score[:, e] > best + tie_eps)
            if chosen:
                better = better & (chosen[0] != e)
            best = torch.where(better, score[:, e], best)
            lead = torch.where(better, e, lead)
        chosen.append(lead)
    return torch.stack(chosen, 1)


def _gates(picked, logits, how):
    if how == "equal":
        return torch.full(picked.shape, 0.5, device=picked.device)
    raw = torch.gather(logits.float(), 1, picked)
    e = torch.exp(raw - raw.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def _plain_moe(s):
    case, x = s["case"], s["x"].float()
    picked = _pick(s["logits"], QUANTUM, TIE_EPS)
    gates = _gates(picked, s["logits"], case["gates"])
    inter, tokens, experts = case["inter"], case["tokens"], case["experts"]
    if 2 * tokens <= experts:      # fewer assignments than experts: their weights alone
        both = torch.einsum("tpih,th->tpi", s["gate_up"][picked].float(), x)
        gate, up = both[..., :inter], both[..., inter:]
        hidden = gate / (1.0 + torch.exp(-gate)) * up
        out = torch.einsum("tphi,tpi->tph", s["down"][picked].float(), hidden * gates[..., None])
        return out.sum(1).to(s["x"].dtype)
    share = torch.zeros(tokens, experts, device="cuda").scatter_(1, picked, gates)
    both = torch.matmul(x, s["gate_up"].float().transpose(1, 2))
    gate, up = both[..., :inter], both[..., inter:]
    hidden = gate / (1.0 + torch.exp(-gate)) * up * share.t()[..., None]
    return torch.matmul(hidden, s["down"].float().transpose(1, 2)).sum(0).to(s["x"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------


def work(case):
    op = case["op"]
    size = _bytes(case["dtype"])
    if op == "append":
        rows = sum(_spread(case["new_min"], case["new_max"], case["batch"]))
        dim, qh, kh = case["head_dim"], case["q_heads"], case["kv_heads"]
        packed = dim // 2 + dim // GROUP * 4
        per_row = (2 * qh + 2 * kh) * dim * size          # q in and out, k and v in
        per_row += 2 * kh * (2 * packed + dim * size)     # stored, read back, values out
        per_row += dim * 4 + 8                            # cos and sin, sequence and position
        return dict(bytes=rows * per_row, flops=rows * (qh * 3 + kh * 12) * dim)
    if op == "attention":
        dim, qh, kh = case["head_dim"], case["q_heads"], case["kv_heads"]
        keys = sum(_visible(case, n) for n in _lens(case))
        packed = dim // 2 + dim // GROUP * 4
        rows = case["batch"] * case["queries"]
        return dict(bytes=keys * kh * 2 * packed + 2 * rows * qh * dim * size,
                    flops=4 * keys * case["queries"] * qh * dim)
    t, h, i, e = case["tokens"], case["hidden"], case["inter"], case["experts"]
    active = e * (1.0 - (1.0 - 2.0 / e) ** t)             # experts that are reached, on average
    return dict(bytes=int(active * 3 * h * i * _bytes(case["weights"])) + 2 * t * h * size + 4 * t * e,
                flops=2 * 2 * t * 3 * h * i)


# ---- the definitions in 64 bits ------------------------------------------------------


def exact(case, seed):
    return dict(append=_exact_append, attention=_exact_attention, moe=_exact_moe)[case["op"]](case, seed)


def _exact_append(case, seed):
    s = _append_inputs(case, seed)
    q, k, v = (s[n].double() for n in "qkv")
    cos, sin = (s[n].double()[s["pos"]].unsqueeze(1) for n in ("cos", "sin"))

    def rotated(x):
        a, b = x.chunk(2, dim=2)
        return torch.cat((a * cos - b * sin, a * sin + b * cos), dim=2)

    def held(x):
        parts = []
        for part in x.split(GROUP, dim=2):
            low = part.min(dim=2, keepdim=True).values.to(torch.bfloat16).double()
            high = part.max(dim=2, keepdim=True).values
            step = ((high - low).clamp_min(0) / 15).to(torch.bfloat16).double()
            code = ((part - low) / step.masked_fill(step == 0, math.inf)).round().clamp(0, 15)
            parts.append(low + step * code)
        return torch.cat(parts, dim=2)

    return rotated(q), held(rotated(k)), held(v)


def _exact_attention(case, seed):
    g, q, lens, table, _ = _attention_inputs(case, seed)
    n, kh, dim = case["queries"], case["kv_heads"], case["head_dim"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for seq, pos, k, v in _fill_pieces(case, g, table):
        b = int(seq[0])
        keys, values = (_values(*_quantise(t)).double() for t in (k, v))
        for i in range(n):
            at = lens[b] - n + i
            seen = pos <= at
            if case["window"]:
                seen &= (at - pos < case["window"]) | (pos < case["sinks"])
            if not bool(seen.any()):
                continue
            kk, vv = keys[seen], values[seen]
            row = q[b * n + i].double().view(kh, -1, dim)
            p = torch.softmax(row @ kk.permute(1, 2, 0) / math.sqrt(dim), dim=-1)
            out[b * n + i] = (p @ vv.transpose(0, 1)).reshape(-1, dim)
    return out


def _f32(value):
    """value rounded to 32 bits: routing's grid and margin are defined there."""
    return struct.unpack("f", struct.pack("f", value))[0]


def _exact_moe(case, seed):
    s = _moe_inputs(case, seed)
    x = s["x"].double()
    inter = case["inter"]
    scores = s["logits"].cpu().numpy()
    out = torch.zeros_like(x)
    quantum, margin = _f32(QUANTUM), _f32(TIE_EPS)
    for t in range(case["tokens"]):
        row = [float(value) for value in scores[t]]
        grid = [math.copysign(_f32(math.floor(_f32(_f32(abs(r) / quantum) + 0.5)) * quantum), r) for r in row]
        pair = []
        for _ in range(2):
            lead = None
            for e, value in enumerate(grid):
                if e in pair:
                    continue
                if lead is None or value > _f32(grid[lead] + margin):
                    lead = e
            pair.append(lead)
        if case["gates"] == "equal":
            weight = [0.5, 0.5]
        else:
            first = 1.0 / (1.0 + math.exp(row[pair[1]] - row[pair[0]]))
            weight = [first, 1.0 - first]
        for e, w in zip(pair, weight):
            both = s["gate_up"][e].double() @ x[t]
            gate, up = both[:inter], both[inter:]
            out[t] += w * (s["down"][e].double() @ (gate * torch.sigmoid(gate) * up))
    return out

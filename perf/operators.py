"""Operators of a paged key/value cache, as cases that can be timed and compared.

  append   ``KVCache.append`` and ``KVCache.read``: rotates the new queries and keys by their positions, stores keys and values in the
           sequences' pages, and hands back what the cache now holds for them.
  attend   ``KVCache.attend``: attention of the new rows over their sequences' pages, causal, grouped heads.

``run`` computes them in elementary torch operations, or with the framework's calls where ``own`` is true.

The cache: a pool of pages, [page][kv head][tiles of 16 tokens].  A tile holds the keys and the values of 16 tokens of a
head, each as a plane of quants and a plane of fp16 scales, one per token and 32 dimensions (GGUF blocks Q4_0 and Q8_0;
fp16 caches have no scales).  ``_maps`` says where a value lies in its tile.
"""
from __future__ import annotations

import math

import torch

own = False

FMT = {"f16": 0, "q4_0": 1, "q8_0": 5}
UNIT = {"f16": 16, "q4_0": 4, "q8_0": 8}         # bytes of eight values
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
TYPE_ID = {"f32": 0, "bf16": 1}
WORKSPACE_BYTES = 16 << 20
MOST_CACHED = 16 * 8192 * 8 * 128                # values of keys a case may cache, over all sequences and heads
MOST_SCORES = 64 * 512 * 16896                   # query row x head x key triples
MOST_APPENDED = 8192 * 64 * 128                  # values of queries a case may append


def _append(name, fmt, heads, kv_heads, head_dim, page, batch, rows_min, rows_max, past, kind, rope_dim, rope, yarn):
    """``past``: tokens already cached.  ``rope``: which dimensions are pairs, "pairs" (2i, 2i+1) or "halves".  ``yarn``:
    how many times longer than trained the context is made, 1 for not at all."""
    return {"name": name, "kind": "append", "fmt": fmt, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "batch": batch, "rows_min": rows_min, "rows_max": rows_max, "past": past, "type": kind,
            "rope_dim": rope_dim, "rope": rope, "yarn": yarn}


def _attend(name, fmt, heads, kv_heads, head_dim, page, batch, rows_min, rows_max, len_min, len_max, q, out, window=0):
    """``len_*``: tokens cached before the rows of the call; the sequences' lengths and rows are spread between the two."""
    return {"name": name, "kind": "attend", "fmt": fmt, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page, "batch": batch, "rows_min": rows_min, "rows_max": rows_max, "len_min": len_min,
            "len_max": len_max, "q": q, "out": out, "window": window}


def listed():
    return [
        # the new token of each of sixteen 7B-shape sequences, one layer
        _append("append_q4_step_16", "q4_0", 32, 32, 128, 64, 16, 1, 1, 512, "f32", 128, "pairs", 1),
        # one 70B-shape sequence, deep into a context four times longer than trained
        _append("append_q8_step_1", "q8_0", 64, 8, 128, 16, 1, 1, 1, 30000, "f32", 128, "pairs", 4),
        # a long document's prompt, fp32 projections
        _append("append_q4_prompt_1999", "q4_0", 32, 32, 128, 64, 1, 1999, 1999, 0, "f32", 128, "pairs", 1),
        # ragged prompts of a server behind their histories, bf16 projections, half of the head rotated
        _append("append_f16_ragged_16", "f16", 64, 8, 128, 32, 16, 33, 901, 1000, "bf16", 64, "halves", 1),
        # a small model's step: launches and latency
        _attend("attend_small_step", "f16", 8, 2, 64, 16, 1, 1, 1, 20, 20, "f32", "f32"),
        # a chat answer of the 7B shape: every head has its own keys
        _attend("attend_q4_7b_step", "q4_0", 32, 32, 128, 64, 1, 1, 1, 639, 639, "f32", "f32"),
        # sixteen 70B-shape sequences of a server, lengths from short to long
        _attend("attend_q4_70b_step_16", "q4_0", 64, 8, 128, 64, 16, 1, 1, 700, 8191, "f32", "f32"),
        # one very long document, grouped heads
        _attend("attend_q4_long_step", "q4_0", 64, 8, 128, 128, 1, 1, 1, 131071, 131071, "bf16", "bf16"),
        # eight bits, a handful of drafted tokens verified for each of eight sequences
        _attend("attend_q8_draft_8", "q8_0", 32, 8, 128, 32, 8, 3, 5, 100, 4000, "f32", "f32"),
        # fp16 cache of a batch, 7B shape, fp32 all the way
        _attend("attend_f16_7b_step_16", "f16", 32, 32, 128, 64, 16, 1, 1, 500, 2000, "f32", "f32"),
        # a long document's prompt over its own 4-bit keys
        _attend("attend_q4_prompt_1999", "q4_0", 32, 32, 128, 64, 1, 1999, 1999, 0, 0, "f32", "bf16"),
        # the next piece of a long prompt, grouped heads
        _attend("attend_q4_piece_512", "q4_0", 64, 8, 128, 64, 1, 512, 512, 16384, 16384, "bf16", "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    fmt = rng.choice(["f16", "q8_0", "q4_0", "q4_0"])
    head_dim = rng.choice([64, 96, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 4, 7, 8])
    page = rng.choice([16, 32, 64, 128])
    if rng.random() < 0.33:
        step = rng.random() < 0.5
        batch = _log(rng, 1, 64) if step else _log(rng, 1, 16)
        most = max(2, min(2048, MOST_APPENDED // (batch * heads * head_dim)))
        rows = 1 if step else _log(rng, 2, most)
        rope_dim = rng.choice([head_dim, head_dim, head_dim // 2])
        case = _append("", fmt, heads, kv_heads, head_dim, page, batch, rng.randint(1, rows), rows,
                       rng.choice([0, _log(rng, 1, 4096), _log(rng, 1, 100000)]), rng.choice(["f32", "bf16"]), rope_dim,
                       rng.choice(["pairs", "halves"]), rng.choice([1, 1, 4, 8]))
        tokens = case["batch"] * (case["past"] + rows)
        if tokens * kv_heads * head_dim > MOST_CACHED:
            case["past"] = max(0, MOST_CACHED // (batch * kv_heads * head_dim) - rows)
    else:
        form = rng.choice(["step", "step", "draft", "prompt"])
        batch = _log(rng, 1, 64) if form != "prompt" else _log(rng, 1, 4)
        rows = 1 if form == "step" else rng.randint(2, 9) if form == "draft" else _log(rng, 10, 2048)
        deepest = max(1, min(131071, MOST_CACHED // (batch * kv_heads * head_dim), MOST_SCORES // (batch * heads * rows)) - rows)
        longest = _log(rng, 1, max(2, deepest))
        q, out = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
        case = _attend("", fmt, heads, kv_heads, head_dim, page, batch, rng.randint(1, rows), rows,
                       rng.choice([longest, rng.randint(0, longest)]), longest, q, out,
                       rng.choice([0, 0, 0, _log(rng, 16, 4096)]))
    del case["name"]
    return case


# ---- where a value lies -----------------------------------------------------------------------------------------------

def _spread(lo, hi, n):
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _rows_lens(case):
    """Rows of this call of each sequence, and the length its cache has with them."""
    rows = _spread(case["rows_min"], case["rows_max"], case["batch"])
    if case["kind"] == "append":
        return rows, [case["past"] + r for r in rows]
    return rows, [p + r for p, r in zip(_spread(case["len_min"], case["len_max"], case["batch"]), rows)]


def _tile_bytes(fmt, head_dim):
    return 2 * (64 * (head_dim // 32) * UNIT[fmt] + (0 if fmt == "f16" else head_dim))


def _maps(fmt, head_dim, device):
    """Byte of each value in its tile and, for 4 bits, how far it is shifted ([16 tokens, head_dim], keys and values), byte of
    each scale ([16, blocks])."""
    blocks, unit = head_dim // 32, UNIT[fmt]
    lane_bytes = blocks * unit
    vec = 16 if lane_bytes % 16 == 0 else 8 if lane_bytes % 8 == 0 else 4
    token = torch.arange(16, device=device).view(16, 1)
    dim = torch.arange(head_dim, device=device).view(1, head_dim)

    def place(half, g, t, sub, second):
        if fmt == "q4_0":
            at, shift = (sub >> 1) + 2 * second, 4 * (sub & 1)
        else:
            at, shift = (2 * sub + second) * (2 if fmt == "f16" else 1), torch.zeros_like(sub + second)
        x = (dim >> 5) * unit + at
        return half * 32 * lane_bytes + x // vec * (32 * vec) + (4 * g + t) * vec + x % vec, shift + 0 * x

    k, k_shift = place(token >> 3, token & 7, dim >> 3 & 3, dim >> 1 & 3, dim & 1)
    v, v_shift = place(token >> 3, dim >> 2 & 7, token >> 1 & 3, dim & 3, token & 1)
    block = torch.arange(blocks, device=device).view(1, blocks)
    scale = ((((token >> 1 & 3) * 2 + (token >> 3)) * blocks + block) * 2 + (token & 1)) * 2
    plane, scales = 64 * lane_bytes, 0 if fmt == "f16" else head_dim
    return {"k": k, "k_shift": k_shift, "k_scale": plane + scale, "v": plane + scales + v, "v_shift": v_shift,
            "v_scale": 2 * plane + scales + scale}


# ---- inputs -------------------------------------------------------------------------------------------------------------

def _inv_freq(case, device):
    """Angle per position of each pair of dimensions, base 10000.  Stretched contexts: the fast pairs as trained, the slow
    ones interpolated, a ramp between (YaRN), for a model trained on 8192 positions."""
    n, stretch = case["rope_dim"] // 2, case["yarn"]
    i = torch.arange(n, dtype=torch.float64, device=device)
    freq = torch.exp(-i / n * math.log(10000.0))
    if stretch == 1:
        return freq, 1.0
    turn = lambda beta: 2 * n * math.log(8192 / (beta * 2 * math.pi)) / (2 * math.log(10000.0))  # noqa: E731
    low, high = max(0.0, math.floor(turn(32.0))), min(2.0 * n - 1, math.ceil(turn(1.0)))
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return freq * (1 - ramp) + freq / stretch * ramp, 0.1 * math.log(stretch) + 1


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rows, lens = _rows_lens(case)
    batch, kv_heads, hd, page = case["batch"], case["kv_heads"], case["head_dim"], case["page"]
    width = max(1, max(-(-n // page) for n in lens))
    pages = batch * width + 3
    table = torch.randperm(pages, device="cuda", generator=gen)[:batch * width].view(batch, width)
    total = sum(rows)
    begin = torch.tensor([0] + rows, device="cuda").cumsum(0)
    state = {"case": case, "table": table.int(), "pages": pages, "total": total, "max_len": max(lens), "max_rows": max(rows),
             "len": torch.tensor(lens, device="cuda", dtype=torch.int32), "begin": begin.int(),
             "pool": torch.zeros(pages * kv_heads * (page // 16) * _tile_bytes(case["fmt"], hd), device="cuda", dtype=torch.uint8)}
    if case["kind"] == "append":
        kind = TYPE[case["type"]]
        # one projection makes queries, keys and values, as a fused weight does
        qkv = torch.randn(total, (case["heads"] + 2 * kv_heads) * hd, device="cuda", generator=gen)
        qkv[:, ::37] *= 4  # some channels are larger than the others
        state["qkv"] = qkv.to(kind)
        state["freq"], state["gain"] = _inv_freq(case, "cuda")
        state["q_out"] = torch.empty(total, case["heads"] * hd, device="cuda", dtype=kind)
        state["k_out"] = torch.empty(total, kv_heads, hd, device="cuda", dtype=torch.bfloat16)
        state["v_out"] = torch.empty_like(state["k_out"])
        return state
    # the cache as earlier appends left it, one sequence after the other
    for s, n in enumerate(lens):
        for at in range(0, n, 65536):
            m = min(65536, n - at)
            pos = torch.arange(at, at + m, device="cuda")
            k, v = torch.randn(2, m, kv_heads, hd, device="cuda", generator=gen)
            k[:, :, ::37] *= 2
            _store(state, torch.full_like(pos, s), pos, k, v)
    q = torch.randn(total, case["heads"] * hd, device="cuda", generator=gen) * 2
    state["q"] = q.to(TYPE[case["q"]])
    state["out"] = torch.empty(total, case["heads"] * hd, device="cuda", dtype=TYPE[case["out"]])
    state["scale"] = 1 / math.sqrt(hd)
    state["workspace"] = torch.zeros(WORKSPACE_BYTES, device="cuda", dtype=torch.uint8)
    return state


# ---- the plain form -------------------------------------------------------------------------------------------------------

def _tile_base(state, seq, pos):
    """Byte where the tile of a token starts, for each kv head: [tokens, kv heads]."""
    case = state["case"]
    page, kv_heads = case["page"], case["kv_heads"]
    at = state["table"].long()[seq, pos // page]
    head = torch.arange(kv_heads, device=pos.device)
    tile = (at.unsqueeze(-1) * kv_heads + head) * (page // 16) + (pos % page // 16).unsqueeze(-1)
    return tile * _tile_bytes(case["fmt"], case["head_dim"])


def _quantize(x, fmt):
    """fp32 [..., blocks, 32] to quants (whole numbers, as they are stored) and fp16 scales, by GGUF's rules."""
    size = x.abs()
    top = size.amax(-1, keepdim=True)
    if fmt == "q4_0":
        lane = torch.arange(32, device=x.device)
        first = torch.where(size == top, lane, 32).amin(-1, keepdim=True)  # the lowest index of equals
        d = x.gather(-1, first) / -8
    else:
        d = top / 127
    d = d.clamp(-65504, 65504)
    inverse = torch.where(d == 0, torch.zeros_like(d), 1 / d)
    if fmt == "q4_0":
        quants = (x * inverse + 8.5).floor().clamp(0, 15)
    else:
        y = x * inverse
        quants = ((y.abs() + 0.5).floor() * y.sign()).clamp(-127, 127) + 128
    return quants.to(torch.uint8), d.squeeze(-1).half()


def _store(state, seq, pos, k, v):
    """Puts fp32 keys and values [tokens, kv heads, head_dim] where they belong."""
    case, pool = state["case"], state["pool"]
    fmt, hd = case["fmt"], case["head_dim"]
    maps = _maps(fmt, hd, pool.device)
    base = _tile_base(state, seq, pos).unsqueeze(-1)
    row = pos % 16
    dims = torch.arange(hd, device=pool.device)
    for x, name, step in ((k, "k", 2), (v, "v", 1)):
        if fmt == "f16":
            pool.view(torch.float16)[(base + maps[name][row].unsqueeze(1)) // 2] = x.half()
            continue
        quants, scales = _quantize(x.reshape(*x.shape[:-1], hd // 32, 32), fmt)
        quants = quants.reshape(x.shape)
        pool.view(torch.float16)[(base + maps[name + "_scale"][row].unsqueeze(1)) // 2] = scales
        if fmt == "q4_0":  # two values of a token share a byte
            low = dims[(dims // step) % 2 == 0]
            quants = quants[..., low] | quants[..., low + step] << 4
            pool[base + maps[name][row][:, low].unsqueeze(1)] = quants
        else:
            pool[base + maps[name][row].unsqueeze(1)] = quants


def _load(tiles, maps, name, fmt):
    """fp32 values of tiles [..., bytes]: [..., 16, head_dim]."""
    half = tiles.view(torch.float16)
    if fmt == "f16":
        return half[..., maps[name] // 2].float()
    quants = tiles[..., maps[name]]
    quants = (quants >> maps[name + "_shift"].to(torch.uint8) & 15).float() - 8 if fmt == "q4_0" else quants.float() - 128
    return quants * half[..., maps[name + "_scale"] // 2].float().repeat_interleave(32, -1)


def _row_places(state):
    """Sequence of each row of the call, and its place among that sequence's rows."""
    begin = state["begin"].long()
    row = torch.arange(state["total"], device=begin.device)
    seq = torch.searchsorted(begin, row, right=True) - 1
    return seq, row - begin[seq]


def _rotate(x, pos, case, freq, gain):
    """fp32 of [rows, heads, head_dim], rotated in 64 bits: far positions have large angles."""
    n = case["rope_dim"] // 2
    angle = pos.double().unsqueeze(-1) * freq
    c, s = (torch.cos(angle) * gain).unsqueeze(1), (torch.sin(angle) * gain).unsqueeze(1)
    y, x = x.float(), x.double()
    first, second = (slice(0, n), slice(n, 2 * n)) if case["rope"] == "halves" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = (a * c - b * s).float(), (a * s + b * c).float()
    return y


def _run_append(state):
    case = state["case"]
    heads, kv_heads, hd = case["heads"], case["kv_heads"], case["head_dim"]
    seq, place = _row_places(state)
    begin = state["begin"].long()
    pos = state["len"].long()[seq] - (begin[seq + 1] - begin[seq]) + place
    q, k, v = state["qkv"].view(state["total"], heads + 2 * kv_heads, hd).split((heads, kv_heads, kv_heads), 1)
    q = _rotate(q.clone(), pos, case, state["freq"], state["gain"])
    _store(state, seq, pos, _rotate(k.clone(), pos, case, state["freq"], state["gain"]), v.float())
    tile_bytes = _tile_bytes(case["fmt"], hd)
    tiles = state["pool"].view(-1, tile_bytes)[_tile_base(state, seq, pos) // tile_bytes]
    maps = _maps(case["fmt"], hd, "cuda")
    at = (pos % 16).view(-1, 1, 1, 1).expand(-1, kv_heads, 1, hd)
    k, v = (_load(tiles, maps, name, case["fmt"]).gather(2, at).squeeze(2).bfloat16() for name in ("k", "v"))
    return {"q": q.reshape(state["total"], heads * hd).to(TYPE[case["type"]]), "k": k, "v": v}


def _run_attend(state):
    case = state["case"]
    heads, kv_heads, hd = case["heads"], case["kv_heads"], case["head_dim"]
    batch, rows, group = case["batch"], state["max_rows"], heads // kv_heads
    tiles = -(-state["max_len"] // 16)
    seq = torch.arange(batch, device="cuda").view(-1, 1)
    tile_bytes = _tile_bytes(case["fmt"], hd)
    base = _tile_base(state, seq, torch.arange(tiles, device="cuda").view(1, -1) * 16) // tile_bytes
    cached = state["pool"].view(-1, tile_bytes)[base.transpose(1, 2)]  # [batch, kv heads, tiles, bytes]
    maps = _maps(case["fmt"], hd, "cuda")
    k, v = (_load(cached, maps, name, case["fmt"]).reshape(batch, kv_heads, tiles * 16, hd) for name in ("k", "v"))
    seq, place = _row_places(state)
    q = torch.zeros(batch, rows, heads, hd, device="cuda")
    q[seq, place] = state["q"].float().view(-1, heads, hd)
    q = q.view(batch, rows, kv_heads, group, hd).transpose(1, 2).reshape(batch, kv_heads, rows * group, hd)
    begin, length = state["begin"].long(), state["len"].long().view(-1, 1, 1)
    first = length - (begin[1:] - begin[:-1]).view(-1, 1, 1)
    row_pos = first + torch.arange(rows, device="cuda").view(1, -1, 1)
    key = torch.arange(tiles * 16, device="cuda").view(1, 1, -1)
    seen = (key <= row_pos) & (key < length)
    if case["window"]:
        seen &= key > row_pos - case["window"]
    seen = seen.repeat_interleave(group, 1).unsqueeze(1)
    scores = torch.matmul(q, k.transpose(2, 3)) * state["scale"]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)  # a row that sees nothing
    p = torch.exp(scores - top)
    del scores
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1)
    out = out.view(batch, kv_heads, rows, group, hd).transpose(1, 2).reshape(batch, rows, heads * hd)
    return out[seq, place].to(TYPE[case["out"]])


# ---- one pass -------------------------------------------------------------------------------------------------------------

def _handles(state):
    """What the framework's calls take of the cache and of the batch, made once."""
    from litenn_b200 import capi
    case = state["case"]
    cache = capi.KVCache(FMT[case["fmt"]], case["kv_heads"], case["head_dim"], case["page"], state["pages"],
                         state["pool"].data_ptr())
    step = case["rows_min"] == case["rows_max"] == 1
    batch = capi.KVBatch(case["batch"], state["table"].shape[1], state["table"].data_ptr(), state["len"].data_ptr(),
                         0 if step else state["begin"].data_ptr(), state["total"])
    rope = capi.Rope(case["rope_dim"], 1 if case["rope"] == "halves" else 0, state["freq"].data_ptr(), state["gain"]) \
        if case["kind"] == "append" else None
    state["handles"] = cache, batch, rope
    return state["handles"]


def run(state):
    case = state["case"]
    if not own:
        return _run_append(state) if case["kind"] == "append" else _run_attend(state)
    cache, batch, rope = state.get("handles") or _handles(state)
    stream = torch.cuda.current_stream().cuda_stream
    hd, heads, kv_heads = case["head_dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        qkv, kind, stride = state["qkv"], TYPE_ID[case["type"]], (heads + 2 * kv_heads) * hd
        at, item = qkv.data_ptr(), qkv.element_size()
        cache.append(batch, rope, heads, kind, at, stride, at + heads * hd * item, stride, at + (heads + kv_heads) * hd * item,
                     stride, state["q_out"].data_ptr(), kind, heads * hd, stream)
        cache.read(batch, state["k_out"].data_ptr(), kv_heads * hd, state["v_out"].data_ptr(), kv_heads * hd, 1, stream)
        return {"q": state["q_out"], "k": state["k_out"], "v": state["v_out"]}
    cache.attend(batch, heads, state["q"].data_ptr(), TYPE_ID[case["q"]], heads * hd, state["out"].data_ptr(),
                 TYPE_ID[case["out"]], heads * hd, state["scale"], case["window"], state["workspace"].data_ptr(), stream)
    return state["out"]


# ---- what a pass cannot do without, and what it should give ------------------------------------------------------------------

def _token_bytes(case):
    """Keys and values of one token, all kv heads."""
    return case["kv_heads"] * _tile_bytes(case["fmt"], case["head_dim"]) // 16


def work(case):
    rows, lens = _rows_lens(case)
    hd, heads, kv_heads, total = case["head_dim"], case["heads"], case["kv_heads"], sum(rows)
    if case["kind"] == "append":
        item = 4 if case["type"] == "f32" else 2
        return {"bytes": total * (item * hd * (2 * heads + 2 * kv_heads) + _token_bytes(case) + 2 * 2 * kv_heads * hd),
                "flops": total * (3 * case["rope_dim"] * (heads + kv_heads) + 4 * kv_heads * hd)}
    window = case["window"]
    keys = pairs = 0
    for n, r in zip(lens, rows):
        first = n - r
        keys += n if not window else n - max(0, first - window + 1)
        pairs += sum(min(first + i + 1, window) if window else first + i + 1 for i in range(r))
    item = (4 if case["q"] == "f32" else 2) + (4 if case["out"] == "f32" else 2)
    return {"bytes": keys * _token_bytes(case) + total * heads * hd * item, "flops": 4 * hd * heads * pairs}


def _unpack(plane, fmt, blocks, keys):
    """Stored whole numbers (or fp16 values) of a plane, [tiles, bytes], as [tiles, 16, head_dim] in 64 bits: undoes the
    lanes' order step by step."""
    unit = UNIT[fmt]
    lane = blocks * unit
    vec = 16 if lane % 16 == 0 else 8 if lane % 8 == 0 else 4
    x = plane.reshape(-1, 2, lane // vec, 32, vec).permute(0, 1, 3, 2, 4).reshape(-1, 2, 8, 4, blocks, unit)
    if fmt == "q4_0":
        x = torch.stack([x & 15, x >> 4], -1)                  # [.., 4 bytes, 2]: four subs of the first, four of the second
        x = x.reshape(*x.shape[:-2], 2, 4).transpose(-1, -2)   # [.., sub, second]
    elif fmt == "q8_0":
        x = x.reshape(*x.shape[:-1], 4, 2)
    else:
        x = x.contiguous().view(torch.float16).reshape(*x.shape[:-1], 4, 2)
    # [tile, half, g, t, block, sub, second]
    if keys:   # token = half, g; dimension = block, t, sub, second
        return x.permute(0, 1, 2, 4, 3, 5, 6).reshape(-1, 16, blocks * 32).double()
    # token = half, t, second; dimension = block, g, sub
    return x.permute(0, 1, 3, 6, 4, 2, 5).reshape(-1, 16, blocks * 32).double()


def _unscale(plane, blocks):
    """[tiles, bytes] of scales as [tiles, 16, blocks] in 64 bits."""
    s = plane.contiguous().view(torch.float16).reshape(-1, 4, 2, blocks, 2)
    return s.permute(0, 2, 1, 4, 3).reshape(-1, 16, blocks).double()


def _exact_attend(case, seed):
    state = prepare(case, seed)
    rows, lens = _rows_lens(case)
    hd, heads, kv_heads, page, fmt = (case[n] for n in ("head_dim", "heads", "kv_heads", "page", "fmt"))
    group, blocks, window = heads // kv_heads, hd // 32, case["window"]
    tile_bytes = _tile_bytes(fmt, hd)
    plane, scales = 64 * blocks * UNIT[fmt], 0 if fmt == "f16" else hd
    pages = state["pool"].view(state["pages"], kv_heads, page // 16, tile_bytes)
    out = torch.empty(state["total"], heads, hd, dtype=torch.float64, device="cuda")
    q = state["q"].double().view(-1, heads, hd)
    at = 0
    for s, (n, r) in enumerate(zip(lens, rows)):
        mine = pages[state["table"][s, :-(-n // page)].long()]
        for h in range(kv_heads):
            raw = mine[:, h].reshape(-1, tile_bytes)
            kv = []
            for first, keys in ((0, True), (plane + scales, False)):
                x = _unpack(raw[:, first:first + plane], fmt, blocks, keys)
                if fmt != "f16":
                    d = _unscale(raw[:, first + plane:first + plane + scales], blocks).unsqueeze(-1)
                    x = ((x - (8 if fmt == "q4_0" else 128)).reshape(-1, 16, blocks, 32) * d)
                kv.append(x.reshape(-1, hd)[:n])
            for r0 in range(0, r, 256):
                r1 = min(r, r0 + 256)
                heads_of = slice(h * group, (h + 1) * group)
                score = torch.einsum("rgd,nd->rgn", q[at + r0:at + r1, heads_of], kv[0]) / math.sqrt(hd)
                pos = torch.arange(n - r + r0, n - r + r1, device="cuda").view(-1, 1, 1)
                key = torch.arange(n, device="cuda")
                hidden = key > pos
                if window:
                    hidden = hidden | (key <= pos - window)
                p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
                out[at + r0:at + r1, heads_of] = torch.einsum("rgn,nd->rgd", p, kv[1])
        at += r
    return out.view(-1, heads * hd)


def _exact_append(case, seed):
    state = prepare(case, seed)
    rows, lens = _rows_lens(case)
    hd, heads, kv_heads, fmt, n = case["head_dim"], case["heads"], case["kv_heads"], case["fmt"], case["rope_dim"] // 2
    pos = torch.cat([torch.arange(length - r, length, device="cuda") for r, length in zip(rows, lens)]).double()
    turn = torch.polar(torch.full((len(pos), n), float(state["gain"]), dtype=torch.float64, device="cuda"),
                       pos.view(-1, 1) * state["freq"]).unsqueeze(1)
    x = state["qkv"].double().view(-1, heads + 2 * kv_heads, hd)
    rot, v = x[:, :heads + kv_heads].clone(), x[:, heads + kv_heads:]
    if case["rope"] == "halves":
        z = torch.complex(rot[..., :n], rot[..., n:2 * n]) * turn
        rot[..., :n], rot[..., n:2 * n] = z.real, z.imag
    else:
        z = torch.complex(rot[..., 0:2 * n:2], rot[..., 1:2 * n:2]) * turn
        rot[..., 0:2 * n:2], rot[..., 1:2 * n:2] = z.real, z.imag
    out = {"q": rot[:, :heads].reshape(-1, heads * hd)}
    for name, y in (("k", rot[:, heads:]), ("v", v)):
        if fmt == "f16":
            out[name] = y.half().double()
            continue
        blk = y.reshape(-1, kv_heads, hd // 32, 32)
        largest = blk.abs().amax(-1, keepdim=True)
        if fmt == "q4_0":
            is_top = blk.abs() == largest
            top = (blk * (is_top & (is_top.cumsum(-1) == 1))).sum(-1, keepdim=True)  # the first of equals, with its sign
            code = (blk / torch.where(top == 0, 1, top / -8) + 8.5).floor().clamp(0, 15) - 8
            scale = (top / -8).half().double()
        else:
            top = largest
            code = blk / torch.where(top == 0, 1, top / 127)
            code = torch.where(code < 0, (code - 0.5).ceil(), (code + 0.5).floor()).clamp(-127, 127)
            scale = (top / 127).half().double()
        out[name] = (code * scale).reshape(-1, kv_heads, hd)
    return out


def exact(case, seed):
    return _exact_append(case, seed) if case["kind"] == "append" else _exact_attend(case, seed)

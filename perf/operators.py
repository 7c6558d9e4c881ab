"""The model step's operators on a compressed paged cache, timed at real sizes.

A case is a dict of plain values; ``kind`` names the operator:

  tables   serving.build_step_tables: block table, slot mapping, positions and
           attention lengths of a step from the requests' lengths
  rotate   serving.rotate_and_store: rotary positions with one to three axes,
           queries rotated, keys rotated into the cache, values beside them
  attend   serving.attend_paged: new tokens of every request over its cached
           keys and values; ``window`` > 0 hides keys that many or more tokens
           back, except the first ``sinks``

Lengths of a case are the same for every seed.  ``n_seq`` requests, the last
``chunks`` of which bring ``min_new`` to ``max_new`` tokens, the others ``few``.
Where ``own`` is false an operator runs in its plain form, in float32.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

PAGE = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

# Attention shapes of the repository's workloads: query heads, KV heads, head dim.
_QWEN25 = {"heads": 40, "kv": 8, "head_dim": 128}
_QWEN35 = {"heads": 16, "kv": 2, "head_dim": 256}
_TINY = {"heads": 8, "kv": 2, "head_dim": 128}
_DECODE = {"few": 1, "chunks": 0, "min_new": 1, "max_new": 1}
_FULL = {"window": 0, "sinks": 0}


def listed():
    return [
        # One user, one token: launches and latency count.
        {"name": "attend-decode-1x4096", "kind": "attend", **_TINY, "dtype": "bf16", "n_seq": 1, **_DECODE, "min_len": 4096,
         "max_len": 4096, **_FULL},
        # The headline batch before its compression: one layer of a decode step.
        {"name": "attend-decode-16x16384", "kind": "attend", **_QWEN25, "dtype": "bf16", "n_seq": 16, **_DECODE,
         "min_len": 16384, "max_len": 16384, **_FULL},
        # A serving batch of unequal lengths, fp16.
        {"name": "attend-decode-48x2k-32k-fp16", "kind": "attend", **_QWEN25, "dtype": "fp16", "n_seq": 48, **_DECODE,
         "min_len": 2048, "max_len": 32768, **_FULL},
        # A chunk of a long prompt: matrix products count.
        {"name": "attend-chunk-2048-of-16384", "kind": "attend", **_QWEN25, "dtype": "bf16", "n_seq": 1, "few": 1, "chunks": 1,
         "min_new": 2048, "max_new": 2048, "min_len": 16384, "max_len": 16384, **_FULL},
        # Hybrid model, head_dim 256: six requests with two draft tokens each beside two prompts' chunks.
        {"name": "attend-mixed-8x700-8k-hd256", "kind": "attend", **_QWEN35, "dtype": "bf16", "n_seq": 8, "few": 3, "chunks": 2,
         "min_new": 200, "max_new": 600, "min_len": 700, "max_len": 8192, **_FULL},
        # Sliding window beside a few first tokens, one token each.
        {"name": "window-decode-32x4k-16k", "kind": "attend", **_QWEN25, "dtype": "bf16", "n_seq": 32, **_DECODE, "min_len": 4096,
         "max_len": 16384, "window": 1024, "sinks": 4},
        # A whole prompt under a window with a protected prefix, head_dim 96, an odd length.
        {"name": "window-prompt-4001-hd96-fp16", "kind": "attend", "heads": 32, "kv": 8, "head_dim": 96, "dtype": "fp16",
         "n_seq": 1, "few": 1, "chunks": 1, "min_new": 4001, "max_new": 4001, "min_len": 4001, "max_len": 4001, "window": 512,
         "sinks": 64},
        # A decode step's tokens.
        {"name": "rotate-decode-16", "kind": "rotate", **_QWEN25, "rotary": 128, "theta": 1e6, "dtype": "bf16", "style": "half",
         "axes": 1, "order": "blocked", "tokens": 16, "max_position": 32768},
        # A prompt with images: time, height and width.
        {"name": "rotate-image-8192", "kind": "rotate", **_QWEN25, "rotary": 128, "theta": 1e6, "dtype": "bf16", "style": "half",
         "axes": 3, "order": "blocked", "tokens": 8192, "max_position": 32768},
        # Partial rotation, axes in turn, adjacent pairs, far positions, an odd number of tokens.
        {"name": "rotate-hybrid-3001-fp16", "kind": "rotate", **_QWEN35, "rotary": 64, "theta": 1e7, "dtype": "fp16",
         "style": "interleaved", "axes": 3, "order": "cycled", "tokens": 3001, "max_position": 262144},
        # Tables of a decode step.
        {"name": "tables-decode-64", "kind": "tables", "n_seq": 64, **_DECODE, "min_len": 300, "max_len": 32768,
         "page_tokens": 128, "max_model_len": 32768},
        # Many requests beside chunks of prompts, scheduler pages of 2048 tokens.
        {"name": "tables-mixed-512", "kind": "tables", "n_seq": 512, "few": 1, "chunks": 24, "min_new": 128, "max_new": 1024,
         "min_len": 1024, "max_len": 65536, "page_tokens": 2048, "max_model_len": 65536},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# Head shapes a drawn case takes: (head_dim, rotated dims).
_SHAPES = ((64, 64), (80, 80), (96, 96), (128, 128), (128, 64), (192, 192), (256, 64), (256, 256))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "attend", "rotate", "rotate", "tables"))
    if kind == "tables":
        n_seq = _log_int(rng, 1, 512)
        hi = _log_int(rng, 400, 65536)
        new = _log_int(rng, 1, min(hi, 1024))
        return {"kind": kind, "n_seq": n_seq, "few": rng.randint(1, 3), "chunks": rng.randint(0, min(n_seq, 24)), "min_new": min(new, 8),
                "max_new": new, "min_len": _log_int(rng, 300, hi), "max_len": hi, "page_tokens": 128 * rng.choice((1, 1, 2, 16)),
                "max_model_len": 65536}
    head_dim, rotary = rng.choice(_SHAPES)
    kv = rng.choice((1, 2, 4, 8))
    heads = kv * rng.randint(1, 8)
    shape = {"heads": heads, "kv": kv, "head_dim": head_dim, "dtype": rng.choice(("bf16", "bf16", "fp16"))}
    if kind == "rotate":
        return {"kind": kind, **shape, "rotary": rotary, "theta": rng.choice((1e4, 1e6, 1e7)),
                "style": rng.choice(("half", "half", "interleaved")), "axes": rng.choice((1, 2, 3, 3)),
                "order": rng.choice(("blocked", "cycled")), "tokens": _log_int(rng, 1, 8192), "max_position": rng.choice((32768, 262144))}
    window = rng.choice((0, 0, _log_int(rng, 1, 4096)))
    case = {"kind": kind, **shape, "window": window, "sinks": rng.choice((0, 4, rng.randint(1, 128))) if window else 0}
    if rng.random() < 0.5:  # single tokens, or a few drafted ones
        n_seq, few = _log_int(rng, 1, 64), rng.choice((1, 1, 1, 2, 3, 4))
        hi = _log_int(rng, 20, max(24, min(32768, int(2.6e8 / (n_seq * kv * head_dim)))))
        return {**case, "n_seq": n_seq, "few": few, "chunks": 0, "min_new": 1, "max_new": 1, "min_len": max(few, _log_int(rng, max(1, hi // 8), hi)),
                "max_len": max(few, hi)}
    n_seq = _log_int(rng, 1, 8)
    most = 1.6e11 / (n_seq * heads * head_dim)  # new tokens x length of a request, padded: no more than the listed chunk's
    new = _log_int(rng, 8, min(2048, int(math.sqrt(most / 2))))
    hi = new + _log_int(rng, 1, max(2, min(14000, int(most / new) - new)))
    return {**case, "n_seq": n_seq, "few": rng.randint(1, 3), "chunks": rng.randint(1, n_seq), "min_new": _log_int(rng, 4, new), "max_new": new,
            "min_len": new, "max_len": hi}


def _lengths(case):
    """(new tokens, length after the step) of every request, on the host."""
    n, chunks = case["n_seq"], case["chunks"]
    g = torch.Generator().manual_seed(7 * n + 13 * case["max_len"] + case["max_new"])
    total = torch.randint(case["min_len"], case["max_len"] + 1, (n,), generator=g)
    new = torch.full((n,), case["few"])
    if chunks:
        new[n - chunks:] = torch.randint(case["min_new"], case["max_new"] + 1, (chunks,), generator=g)
    return new, torch.maximum(total, new)


def _block_tables(lengths, g, device):
    """Random disjoint pages: int32 [n, most pages] (-1 behind a request's last) and the pool's size."""
    need = (lengths + PAGE - 1) // PAGE
    pool = int(need.sum()) + 3
    order = torch.randperm(pool, generator=g, device=device).to(torch.int32)
    column = torch.arange(int(need.max()))
    table = torch.full((len(lengths), len(column)), -1, dtype=torch.int32, device=device)
    inside = (column[None] < need[:, None]).to(device)
    table[inside] = order[: int(need.sum())]
    return table, pool


def _start_loc(new):
    return torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).to(torch.int32)


def _prepare_attend(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    new, lengths = _lengths(case)
    dtype, kv, dim = DTYPES[case["dtype"]], case["kv"], case["head_dim"]
    table, pool = _block_tables(lengths, g, device)
    channel = 1 + 0.25 * torch.randn((2, 1, 1, kv, dim), generator=g, device=device)
    cache = torch.randn((2, pool, PAGE, kv, dim), generator=g, device=device)
    cache = (cache.mul_(channel)).to(dtype)
    tokens = int(new.sum())
    q = (2 * torch.randn((tokens, case["heads"], dim), generator=g, device=device)).to(dtype)
    return {
        "kind": "attend", "q": q, "k_cache": cache[0], "v_cache": cache[1], "out": torch.empty_like(q),
        "query_start_loc": _start_loc(new).to(device), "seq_lens": lengths.to(torch.int32).to(device), "block_table": table,
        "max_query_len": int(new.max()), "max_seq_len": int(lengths.max()), "scale": 1 / math.sqrt(dim), "window": case["window"],
        "sinks": case["sinks"],
    }


def _prepare_rotate(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    heads, kv, dim, n = case["heads"], case["kv"], case["head_dim"], case["tokens"]
    dtype, freq = DTYPES[case["dtype"]], case["rotary"] // 2
    # Queries, keys and values are parts of one projection's rows.
    qkv = torch.randn((n, heads + 2 * kv, dim), generator=g, device=device).to(dtype)
    omega = 1.0 / (case["theta"] ** (torch.arange(freq, dtype=torch.float64, device=device) / freq))
    start = torch.randint(0, case["max_position"] - n, (), generator=g, device=device)
    time = start + torch.arange(n, device=device)
    # Images of 24 x 20 patches: time stands still inside one, height and width run.
    patch = torch.arange(n, device=device) % 480
    image = time - patch
    axes = torch.stack([image, image + patch // 20, image + patch % 20])[: case["axes"]] if case["axes"] > 1 else time[None]
    axes = torch.where((torch.arange(n, device=device) // 480 % 2 == 1)[None], axes, time[None])
    pool = n // PAGE + 2
    slots = torch.randperm(pool * PAGE, generator=g, device=device)[:n]
    caches = [torch.randn((pool, PAGE, kv, dim), generator=g, device=device).to(dtype) for _ in range(2)]
    share = [freq // case["axes"]] * case["axes"]
    share[0] += freq - sum(share)
    return {
        "kind": "rotate", "q": qkv[:, :heads], "k": qkv[:, heads : heads + kv], "v": qkv[:, heads + kv :], "omega": omega.float(),
        "positions": axes.contiguous(), "slot_mapping": slots, "k_cache": caches[0], "v_cache": caches[1], "sections": share,
        "axis_order": case["order"], "rope_style": case["style"], "q_out": torch.empty((n, heads, dim), dtype=dtype, device=device),
    }


def _prepare_tables(case, seed):
    device = torch.device("cuda")
    g = torch.Generator().manual_seed(seed)
    new, lengths = _lengths(case)
    n, page = case["n_seq"], case["page_tokens"]
    # Half of the requests were compressed once: their physical length is less than what they have computed.
    removed = torch.randint(0, 30000, (n,), generator=g) * torch.randint(0, 2, (n,), generator=g)
    pages = (lengths + page - 1) // page
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), pages.cumsum(0)])
    ids = torch.randperm(int(offsets[-1]) + 7, generator=g)[: int(offsets[-1])]
    tokens, most = int(new.sum()), case["max_model_len"] // PAGE
    return {
        "kind": "tables", "computed_tokens": (lengths - new + removed).to(torch.int32).to(device), "new_tokens": new.to(torch.int32).to(device),
        "request_offsets": removed.to(device), "block_ids": ids.to(device), "block_offsets": offsets.to(device), "page_tokens": page,
        "max_query_len": int(new.max()),
        "buffers": {
            "query_start_loc": torch.empty(n + 1, dtype=torch.int32, device=device),
            "seq_lens": torch.empty(n, dtype=torch.int32, device=device),
            "positions": torch.empty(tokens, dtype=torch.int64, device=device),
            "slot_mapping": torch.empty(tokens, dtype=torch.int64, device=device),
            "block_table": torch.empty((n, most), dtype=torch.int32, device=device),
        },
    }


def prepare(case, seed):
    return {"attend": _prepare_attend, "rotate": _prepare_rotate, "tables": _prepare_tables}[case["kind"]](case, seed)


def _serving():
    root = str(Path(__file__).resolve().parents[1] / "vllm-ascend-kvcompress-hust_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from kvcompress_mi355x.methods.triattention import serving

    return serving


def _attend_own(s):
    return _serving().attend_paged(
        s["q"], s["k_cache"], s["v_cache"], s["query_start_loc"], s["seq_lens"], s["block_table"], max_query_len=s["max_query_len"],
        max_seq_len=s["max_seq_len"], scale=s["scale"], window=s["window"], sinks=s["sinks"], out=s["out"])


def _attend_plain(s):
    q, table, start = s["q"], s["block_table"].long(), s["query_start_loc"].long()
    tokens, heads, dim = q.shape
    device, n, kv = q.device, table.shape[0], s["k_cache"].shape[2]
    lengths, new = s["seq_lens"].long(), start[1:] - start[:-1]
    most_new, most = s["max_query_len"], s["max_seq_len"]
    # Every request's new tokens and cached rows, padded to the longest.
    i, j = torch.arange(most_new, device=device), torch.arange(most, device=device)
    token = (start[:-1, None] + i).clamp_max(tokens - 1)
    slot = table[:, j // PAGE] * PAGE + j % PAGE
    slot = torch.where(j < lengths[:, None], slot, slot[:, :1])
    k, v = (s[c].reshape(-1, kv, dim)[slot].float().transpose(1, 2) for c in ("k_cache", "v_cache"))
    queries = q.float()[token].view(n, most_new, kv, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, dim)
    scores = torch.matmul(queries, k.transpose(-1, -2).contiguous()).mul_(s["scale"]).view(n, kv, most_new, heads // kv, most)
    place = (lengths - new)[:, None] + i
    hidden = j > place[..., None]
    if s["window"]:
        hidden |= (place[..., None] - j >= s["window"]) & (j >= s["sinks"])
    scores.masked_fill_(hidden[:, None, :, None], -torch.inf)
    weights = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = weights.sum(-1, keepdim=True)
    out = (torch.matmul(weights.view(n, kv, -1, most), v).view(n, kv, most_new, heads // kv, dim) / total).permute(0, 2, 1, 3, 4)
    flat = torch.arange(tokens, device=device)
    request = torch.searchsorted(start[1:], flat, right=True)
    return out.reshape(n, most_new, heads, dim)[request, flat - start[request]].to(q.dtype)


def _rotate_own(s):
    serving = _serving()
    serving.rotate_and_store(
        s["q"], s["k"], s["v"], s["positions"], s["omega"], s["slot_mapping"], s["k_cache"], s["v_cache"], sections=s["sections"],
        axis_order=s["axis_order"], rope_style=s["rope_style"], q_out=s["q_out"])
    return s["q_out"], s["k_cache"], s["v_cache"]


def _axis_of(freq, sections, order, device):
    """The axis whose position turns each frequency: runs of `sections`, or axes in turn while their sections last."""
    f, sizes = torch.arange(freq, device=device), torch.tensor(sections, device=device)
    if order == "blocked":
        return torch.searchsorted(sizes.cumsum(0), f, right=True)
    axis = f % len(sections)
    return torch.where(f // len(sections) < sizes[axis], axis, 0)


def _turn(x, cos, sin, style):
    """Pairs of the first 2F dims turned by the angles; the others stay. float32."""
    x, freq = x.float(), cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    turned, rest = x[..., : 2 * freq], x[..., 2 * freq :]
    if style == "half":
        a, b = turned[..., :freq], turned[..., freq:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _rotate_plain(s):
    dtype, omega = s["q"].dtype, s["omega"]
    axis = _axis_of(omega.numel(), s["sections"], s["axis_order"], omega.device)
    angle = s["positions"][axis].t().double() * omega.double()
    cos, sin = angle.cos().float(), angle.sin().float()
    kv, dim = s["k"].shape[1:]
    s["q_out"].copy_(_turn(s["q"], cos, sin, s["rope_style"]))
    s["k_cache"].view(-1, kv, dim)[s["slot_mapping"]] = _turn(s["k"], cos, sin, s["rope_style"]).to(dtype)
    s["v_cache"].view(-1, kv, dim)[s["slot_mapping"]] = s["v"]
    return s["q_out"], s["k_cache"], s["v_cache"]


def _tables_own(s):
    b = s["buffers"]
    _serving().build_step_tables(
        s["computed_tokens"], s["new_tokens"], s["request_offsets"], s["block_ids"], s["block_offsets"], s["page_tokens"],
        max_query_len=s["max_query_len"], **b)
    return b


def _tables_plain(s):
    b, k = s["buffers"], s["page_tokens"] // PAGE
    new, removed = s["new_tokens"].long(), s["request_offsets"]
    n, device = new.numel(), new.device
    start = torch.zeros(n + 1, dtype=torch.int64, device=device)
    start[1:] = new.cumsum(0)
    lengths = s["computed_tokens"].long() + new - removed
    flat = torch.arange(b["positions"].numel(), device=device)
    request = torch.searchsorted(start[1:], flat, right=True)
    positions = s["computed_tokens"].long()[request] + flat - start[request]
    j = torch.arange(b["block_table"].shape[1], device=device)
    at = (s["block_offsets"][:-1, None] + j // k).clamp_max(s["block_ids"].numel() - 1)
    table = torch.where(j * PAGE < lengths[:, None], s["block_ids"][at] * k + j % k, -1)
    place = positions - removed[request]
    b["query_start_loc"].copy_(start)
    b["seq_lens"].copy_(lengths)
    b["positions"].copy_(positions)
    b["slot_mapping"].copy_(table[request, place // PAGE] * PAGE + place % PAGE)
    b["block_table"].copy_(table)
    return b


def run(state):
    if own:
        return {"attend": _attend_own, "rotate": _rotate_own, "tables": _tables_own}[state["kind"]](state)
    return {"attend": _attend_plain, "rotate": _rotate_plain, "tables": _tables_plain}[state["kind"]](state)


def work(case):
    if case["kind"] == "rotate":
        values = case["tokens"] * (case["heads"] + 2 * case["kv"]) * case["head_dim"]
        turned = case["tokens"] * (case["heads"] + case["kv"]) * case["rotary"]
        return {"bytes": 2 * values * 2 + case["tokens"] * 8 * (case["axes"] + 1) + 2 * case["rotary"], "flops": 3 * turned}
    new, lengths = _lengths(case)
    if case["kind"] == "tables":
        n, tokens = case["n_seq"], int(new.sum())
        pages = int(((lengths + case["page_tokens"] - 1) // case["page_tokens"]).sum())
        return {"bytes": n * (4 + 4 + 8 + 8) + 8 * pages + 8 * n + 16 * tokens + 4 * n * (case["max_model_len"] // PAGE), "flops": 0}
    seen = pairs = 0
    for fresh, length in zip(new.tolist(), lengths.tolist()):
        p = torch.arange(length - fresh, length)
        if case["window"]:
            low = (p - case["window"] + 1).clamp_min(0)
            first = low.clamp_max(case["sinks"])
            pairs += int((p + 1 - low + first).sum())
            seen += length - int(low[0]) + int(first[0])
        else:
            pairs += int((p + 1).sum())
            seen += length
    row = case["head_dim"] * 2
    return {"bytes": 2 * int(new.sum()) * case["heads"] * row + 2 * seen * case["kv"] * row,
            "flops": 4 * case["head_dim"] * case["heads"] * pairs}


def exact(case, seed):
    if case["kind"] == "tables":
        return None
    s = prepare(case, seed)
    if case["kind"] == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        start, lengths = s["query_start_loc"].tolist(), s["seq_lens"].tolist()
        group = case["heads"] // case["kv"]
        for r, length in enumerate(lengths):
            pages = s["block_table"][r, : -(-length // PAGE)].long()
            rows = slice(start[r], start[r + 1])
            place = torch.arange(length - (start[r + 1] - start[r]), length, device="cuda")[:, None]
            key = torch.arange(length, device="cuda")[None]
            seen = (key <= place) & ((place - key < (case["window"] or length + 1)) | (key < case["sinks"]))
            for h in range(case["kv"]):
                k = s["k_cache"][pages, :, h].reshape(-1, case["head_dim"])[:length].double()
                v = s["v_cache"][pages, :, h].reshape(-1, case["head_dim"])[:length].double()
                for head in range(h * group, (h + 1) * group):
                    logits = (s["q"][rows, head].double() @ k.T) * s["scale"]
                    out[rows, head] = torch.softmax(torch.where(seen, logits, -torch.inf), -1) @ v
        return out
    angle = torch.empty((case["tokens"], case["rotary"] // 2), dtype=torch.float64, device="cuda")
    ends = [sum(s["sections"][: a + 1]) for a in range(case["axes"])]
    for f in range(angle.shape[1]):
        if case["order"] == "blocked":
            axis = next(a for a in range(case["axes"]) if f < ends[a])
        else:
            axis = f % case["axes"] if f // case["axes"] < s["sections"][f % case["axes"]] else 0
        angle[:, f] = s["positions"][axis].double() * s["omega"][f].double()
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    outs = [torch.empty_like(s["q"], dtype=torch.float64), torch.empty_like(s["k"], dtype=torch.float64)]
    for x, y in zip((s["q"], s["k"]), outs):
        y.copy_(x)
        near = slice(0, case["rotary"] // 2) if case["style"] == "half" else slice(0, case["rotary"], 2)
        far = slice(case["rotary"] // 2, case["rotary"]) if case["style"] == "half" else slice(1, case["rotary"], 2)
        z = torch.complex(x[..., near].double(), x[..., far].double()) * turn
        y[..., near], y[..., far] = z.real, z.imag
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    page, row = s["slot_mapping"] // PAGE, s["slot_mapping"] % PAGE
    k_cache[page, row], v_cache[page, row] = outs[1], s["v"].double()
    return outs[0], k_cache, v_cache

"""The model step's operators on a paged cache against float64 on the host (needs a GPU)."""

from __future__ import annotations

import pytest
import torch

from oracle import serving_ref as ref

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _serving():
    from kvcompress_mi355x.methods.triattention import serving

    return serving


# ------------------------------------------------------------------ tables --

TABLE_CASES = [
    # (computed, new, removed or None, pages a request, page_tokens, padding tokens, max_blocks)
    ([0], [1], None, [1], 128, 0, 1),
    ([0, 127, 128, 129, 4095], [1, 1, 1, 1, 1], None, [1, 1, 2, 2, 32], 128, 3, 40),
    ([5000, 0, 300, 7, 9999], [3, 700, 0, 129, 1], [4000, 0, 20, 0, 9000], [8, 6, 3, 2, 8], 128, 11, 17),
    ([100, 5000], [2000, 1], [0, 3000], [1, 1], 2048, 0, 33),  # page expansion; the second row's last page is reached
    ([300, 10], [5, 5], None, [1, 0], 128, 2, 4),  # too few pages: slots of -1
    ([10, 10, 10], [-4, 5, 2], [0, 30, 0], [1, 1, 1], 128, 0, 2),  # negative counts, physical places below zero
    (list(range(0, 900)), [1 + (i % 3) for i in range(900)], [i // 2 for i in range(900)], [8] * 900, 256, 5, 9),
    ([0], [9000], None, [80], 128, 100, 71),  # more than one share of a request; the table is full
]


@pytest.mark.parametrize("case", TABLE_CASES, ids=range(len(TABLE_CASES)))
@pytest.mark.parametrize("hint", [True, False])
def test_step_tables_match_definition(hip_device, case, hint) -> None:
    computed, new, removed, pages, page_tokens, padding, max_blocks = case
    n = len(computed)
    g = torch.Generator().manual_seed(n + page_tokens)
    ids = torch.randperm(sum(pages) + 5, generator=g)
    offsets = torch.tensor([0, *torch.tensor(pages).cumsum(0).tolist()])
    rows = [ids[offsets[r] : offsets[r + 1]].tolist() for r in range(n)]
    total = sum(max(x, 0) for x in new) + padding
    d = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device=hip_device)  # noqa: E731
    start, lens = torch.full((n + 1,), -7, dtype=torch.int32, device=hip_device), torch.full((n + 3,), -7, dtype=torch.int32, device=hip_device)
    positions, slots = (torch.full((total,), -7, device=hip_device) for _ in range(2))
    wide = torch.full((n + 2, max_blocks + 3), -7, dtype=torch.int32, device=hip_device)
    _serving().build_step_tables(
        d(computed), d(new), None if removed is None else d(removed, torch.int64), ids.to(hip_device), offsets.to(hip_device), page_tokens,
        query_start_loc=start, seq_lens=lens, positions=positions, slot_mapping=slots, block_table=wide[:, :max_blocks],
        max_query_len=max(new) if hint else None)
    want = ref.step_tables(computed, new, removed or [0] * n, rows, page_tokens, total, max_blocks)
    assert start.tolist() == want[0] and lens.tolist() == want[1] + [-7] * 3
    assert positions.tolist() == want[2] and slots.tolist() == want[3]
    assert wide[:n, :max_blocks].tolist() == want[4]
    assert (wide[n:] == -7).all() and (wide[:, max_blocks:] == -7).all()


def test_step_tables_drop_what_the_buffers_cannot_hold(hip_device) -> None:
    d = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device=hip_device)  # noqa: E731
    start, lens = torch.empty(4, dtype=torch.int32, device=hip_device), torch.empty(3, dtype=torch.int32, device=hip_device)
    positions, slots = torch.full((10,), -7, device=hip_device), torch.full((10,), -7, device=hip_device)
    table = torch.empty((3, 2), dtype=torch.int32, device=hip_device)
    _serving().build_step_tables(
        d([100, 50, 20]), d([8, 8, 8]), None, d([4, 1 << 40, -3, 2], torch.int64), d([0, 1, 2, 4], torch.int64), 128,
        query_start_loc=start, seq_lens=lens, positions=positions, slot_mapping=slots, block_table=table)
    assert start.tolist() == [0, 8, 10, 10] and lens.tolist() == [108, 52, 20]
    assert positions.tolist() == [*range(100, 108), 50, 51]
    assert slots.tolist() == [*range(612, 620), -1, -1]  # a page id past 32 bits is none
    assert table.tolist() == [[4, -1], [-1, -1], [-1, -1]]


def test_step_tables_without_requests(hip_device) -> None:
    e = lambda t, *s: torch.full(s, 5, dtype=t, device=hip_device)  # noqa: E731
    start, positions, slots = e(torch.int32, 1), e(torch.int64, 6), e(torch.int64, 6)
    _serving().build_step_tables(
        e(torch.int32, 0), e(torch.int32, 0), None, e(torch.int64, 0), torch.zeros(1, dtype=torch.int64, device=hip_device), 128,
        query_start_loc=start, seq_lens=e(torch.int32, 0), positions=positions, slot_mapping=slots, block_table=e(torch.int32, 0, 4))
    assert start.tolist() == [0] and positions.tolist() == [0] * 6 and slots.tolist() == [-1] * 6


def test_step_tables_beside_each_other_in_one_buffer(hip_device) -> None:
    """Lengths in the gap behind a table's rows are no overlap; lengths written over
    their own input are."""
    d = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device=hip_device)  # noqa: E731
    wide = torch.full((3, 12), -7, dtype=torch.int32, device=hip_device)
    args = (d([200, 5, 300]), d([1, 2, 1]), None, d([4, 9, 1, 2, 7, 8], torch.int64), d([0, 2, 3, 6], torch.int64), 128)
    buffers = {"query_start_loc": wide[0, 4:8], "positions": torch.empty(4, dtype=torch.int64, device=hip_device),
               "slot_mapping": torch.empty(4, dtype=torch.int64, device=hip_device), "block_table": wide[:, :4]}
    _serving().build_step_tables(*args, seq_lens=wide[0, 8:11], **buffers)
    assert wide.tolist() == [[4, 9, -1, -1, 0, 1, 3, 4, 201, 7, 301, -7], [1, -1, -1, -1] + [-7] * 8, [2, 7, 8, -1] + [-7] * 8]
    for lens in (args[0], wide[0, 7:10], wide[1, :3]):
        with pytest.raises(ValueError, match="overlap"):
            _serving().build_step_tables(*args, seq_lens=lens, **buffers)


# ------------------------------------------------------------------ rotary --

ROTARY_CASES = [
    # (tokens, heads, kv, head_dim, sections, order, style, dtype, strided)
    (1, 8, 2, 128, (64,), "blocked", "half", BF16, True),
    (16, 40, 8, 128, (64,), "blocked", "half", BF16, True),
    (130, 16, 2, 256, (16, 8, 8), "cycled", "half", FP16, True),
    (130, 16, 2, 256, (12, 10, 10), "blocked", "interleaved", BF16, False),
    (67, 5, 1, 64, (8, 16, 8), "blocked", "half", FP16, False),
    (33, 6, 3, 80, (14, 13, 13), "cycled", "interleaved", BF16, True),
    (33, 6, 3, 80, (20, 0, 20), "blocked", "half", BF16, True),
    (9, 4, 4, 72, (9, 9), "cycled", "half", FP16, False),  # 18 frequencies: no whole 16-byte words
    (9, 3, 1, 10, (1, 1, 1, 1), "cycled", "interleaved", BF16, False),
    (9, 3, 1, 34, (0, 5), "cycled", "half", BF16, False),
    (5, 2, 2, 512, (256,), "blocked", "half", BF16, True),
    (2000, 4, 2, 64, (32,), "blocked", "half", BF16, True),
    (300, 0, 2, 64, (32,), "blocked", "half", BF16, True),  # keys only
]


@pytest.mark.parametrize("far", [0, 1 << 20, (1 << 31) + 12345])
@pytest.mark.parametrize("case", ROTARY_CASES, ids=range(len(ROTARY_CASES)))
def test_rotate_and_store_matches_definition(hip_device, case, far) -> None:
    n, heads, kv, dim, sections, order, style, dtype, strided = case
    freq = sum(sections)
    g = torch.Generator().manual_seed(n + dim)
    qkv = torch.randn((n, heads + 2 * kv, dim + (24 if strided else 0)), generator=g).to(dtype)
    omega = 1.0 / (1e4 ** (torch.arange(freq, dtype=torch.float64) / freq)).float()
    positions = far + torch.randint(-3 if far == 0 else 0, 5000, (len(sections), n), generator=g)
    pages = n // 128 + 2
    cache = torch.randn((pages, 2, 128, kv, dim), generator=g).to(dtype)  # K and V pages of one buffer
    slots = torch.randperm(pages * 128, generator=g)[:n]
    slots[n // 2] = -1 if n % 2 else pages * 128
    dev_qkv, dev_cache = qkv.to(hip_device), cache.to(hip_device)
    q, k, v = dev_qkv[:, :heads, :dim], dev_qkv[:, heads : heads + kv, :dim], dev_qkv[:, heads + kv :, :dim]
    got = _serving().rotate_and_store(
        q, k, v, positions.to(hip_device) if len(sections) > 1 else positions[0].to(hip_device), omega.to(hip_device), slots.to(hip_device),
        dev_cache[:, 0], dev_cache[:, 1], sections=sections if len(sections) > 1 else None, axis_order=order, rope_style=style)
    half_step, least = torch.finfo(dtype).eps / 2, 2.0**-25
    # float32: the angle's last bit, cosine and sine, two products and a sum.
    slack = 2.0**-21

    def check(out, want, x):
        pair = x.double().abs().amax(-1, keepdim=True) * 2
        assert ((out.double().cpu() - want).abs() <= half_step * want.abs() + slack * pair + least).all()

    host_q, host_k = qkv[:, :heads, :dim], qkv[:, heads : heads + kv, :dim]
    if heads:
        check(got, ref.rotate(host_q, positions, omega, sections, order, style), host_q)
    turned = ref.rotate(host_k, positions, omega, sections, order, style)
    after = dev_cache.cpu()
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < pages * 128:
            check(after[slot // 128, 0, slot % 128], turned[t], host_k[t])
            assert torch.equal(after[slot // 128, 1, slot % 128], qkv[t, heads + kv :, :dim])
            after[slot // 128, :, slot % 128] = cache[slot // 128, :, slot % 128]
    assert torch.equal(after, cache)  # other rows are left alone


def test_rotate_in_place_and_pass_through(hip_device) -> None:
    g = torch.Generator(device=hip_device).manual_seed(3)
    q = torch.randn((200, 6, 96), generator=g, device=hip_device).to(BF16)
    kv = torch.randn((2, 200, 2, 96), generator=g, device=hip_device).to(BF16)
    omega = torch.rand(16, generator=g, device=hip_device)
    positions = torch.arange(200, device=hip_device)
    caches = [torch.zeros((2, 128, 2, 96), dtype=BF16, device=hip_device) for _ in range(4)]
    slots = torch.arange(255, 55, -1, device=hip_device)
    apart = _serving().rotate_and_store(q, kv[0], kv[1], positions, omega, slots, *caches[:2])
    same = q.clone()
    assert _serving().rotate_and_store(same, kv[0], kv[1], positions, omega, slots, *caches[2:], q_out=same) is same
    assert torch.equal(same, apart) and torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])
    assert torch.equal(apart[..., 32:], q[..., 32:])
    assert torch.equal(apart[0], q[0])  # position 0


def test_rotate_more_tokens_than_one_dispatch_takes(hip_device) -> None:
    """2^24 tokens of 256 threads: the values of two calls of about half of them."""
    n, dim = (1 << 24) + 5, 8
    g = torch.Generator(device=hip_device).manual_seed(8)
    q, k, v = (torch.randn((n, 1, dim), generator=g, device=hip_device, dtype=BF16) for _ in range(3))
    omega = torch.tensor([1.0, 0.5, 0.25, 0.125], device=hip_device)
    positions = torch.randint(0, 1000, (2, n), generator=g, device=hip_device)
    slots = torch.arange(n - 1, -1, -1, device=hip_device)
    pages = -(-n // 128)
    caches = [torch.zeros((pages, 128, 1, dim), dtype=BF16, device=hip_device) for _ in range(4)]
    rotate = lambda part, *to: _serving().rotate_and_store(  # noqa: E731
        q[part], k[part], v[part], positions[:, part], omega, slots[part], *to, sections=(3, 1))
    whole = rotate(slice(0, n), *caches[:2])
    half = (1 << 23) - 101
    for part in (slice(0, half), slice(half, 2 * half), slice(2 * half, n)):
        assert torch.equal(rotate(part, *caches[2:]), whole[part])
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])
    assert torch.equal(caches[1].view(-1, 1, dim)[:n].flip(0), v)


# --------------------------------------------------------------- attention --


def _paged(lens, kv, dim, dtype, g, *, max_blocks=None, extra=3, hidden=float("nan")):
    """Host K and V caches whose rows outside every request hold ``hidden``."""
    need = [-(-n // 128) for n in lens]
    pool = sum(need) + extra
    order = torch.randperm(pool, generator=g)
    width = max_blocks or max([1, *need]) + 2
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    caches = [torch.full((pool, 128, kv, dim), hidden, dtype=dtype) for _ in range(2)]
    at = 0
    for r, n in enumerate(lens):
        pages = order[at : at + need[r]]
        at += need[r]
        keep = min(need[r], width)
        table[r, :keep] = pages[:keep].int()
        slots = (pages[:, None] * 128 + torch.arange(128)).reshape(-1)[:n]
        for cache in caches:
            cache.view(-1, kv, dim)[slots] = torch.randn((n, kv, dim), generator=g).to(dtype)
    return caches[0], caches[1], table


def _check(got, q, caches, start, lens, table, dtype, *, scale, window, sinks, rows_most):
    """Derived tolerance: the output's rounding (half a step of its value); of
    weights rounded to the cache's type (requests of more than 32 rows) half a
    step of the mean |v|, else what two words leave (2^-16 bf16, 2^-22 fp16);
    float32 scores twice (weights and their sum); weights below fp16's normal
    range, whose step is 2^-25 of a largest weight of at least 1."""
    want, spread, rel = ref.attend(q, *caches, start, lens, table, scale=scale, window=window, sinks=sinks)
    half_step = torch.finfo(dtype).eps / 2
    weight = half_step if rows_most > 32 else half_step**2
    keys = max(max(lens), 1)
    tiny = keys * 2.0**-25 * 4 if dtype == FP16 else 0.0
    bound = half_step * want.abs() + spread * (weight + 2 * rel) * (1 + half_step) + tiny * spread.amax() + 2.0**-25
    inside = start[-1]
    assert torch.equal(torch.isnan(got[:inside].cpu()), torch.isnan(want[:inside]))
    err = (got.double().cpu() - want).abs()[:inside]
    worst = (err / bound[:inside]).nan_to_num(0.0)
    assert worst.numel() == 0 or float(worst.max()) <= 1.0, f"error {float(worst.max()):.2f} x its bound"


ATTEND_CASES = [
    # (heads, kv, head_dim, dtype, lengths, new tokens, window, sinks)
    (8, 2, 128, BF16, [1], [1], 0, 0),
    (8, 2, 128, BF16, [4096], [1], 0, 0),
    (40, 8, 128, BF16, [127, 128, 129, 1000, 1], [1, 1, 1, 1, 1], 0, 0),
    (40, 8, 128, FP16, [300, 2000, 31, 33, 513], [1, 3, 1, 2, 1], 0, 0),
    (16, 2, 256, BF16, [700, 200, 64], [3, 4, 1], 0, 0),
    (16, 2, 256, FP16, [700, 400], [1, 1], 0, 0),
    (6, 2, 64, BF16, [257, 900], [1, 5], 0, 0),
    (4, 4, 80, BF16, [130, 300], [1, 2], 0, 0),
    (12, 4, 96, FP16, [130, 300, 17], [2, 1, 1], 0, 0),
    (8, 1, 192, BF16, [600, 129], [1, 2], 0, 0),
    (3, 3, 8, BF16, [200, 5], [1, 1], 0, 0),
    (17, 1, 40, FP16, [333], [1], 0, 0),  # one token's heads fill more than 16 rows
    (33, 1, 64, BF16, [333, 40], [1, 2], 0, 0),  # more than 32 rows a token
    (2, 1, 72, BF16, [100, 200], [7, 1], 0, 0),
    # chunks
    (40, 8, 128, BF16, [300], [300], 0, 0),
    (8, 2, 128, FP16, [1100, 260], [400, 131], 0, 0),
    (8, 8, 64, BF16, [129, 200], [129, 64], 0, 0),
    (16, 2, 256, BF16, [500, 90], [77, 90], 0, 0),
    (6, 2, 192, FP16, [300], [45], 0, 0),
    (12, 4, 96, BF16, [700], [130], 0, 0),
    (5, 1, 80, FP16, [400, 3], [100, 3], 0, 0),
    (40, 8, 128, BF16, [900, 17, 500, 1], [1, 17, 200, 1], 0, 0),  # single tokens beside chunks
    (8, 2, 128, BF16, [20, 0, 3, 50], [40, 1, 8, 0], 0, 0),  # rows without keys, a request without tokens
    # windows and sinks
    (8, 2, 128, BF16, [1000, 300, 64], [1, 1, 1], 1, 0),
    (8, 2, 128, BF16, [1000, 300, 64], [1, 2, 3], 100, 4),
    (40, 8, 128, FP16, [2000, 129], [1, 1], 128, 130),
    (16, 2, 256, BF16, [1500, 1400], [3, 1], 300, 257),
    (8, 2, 128, BF16, [1500], [1], 5000, 3),  # wider than the request
    (8, 2, 128, BF16, [1100], [400], 1, 0),
    (8, 2, 128, BF16, [1100, 300], [400, 300], 64, 1),
    (12, 4, 96, FP16, [900], [333], 200, 150),
    (16, 2, 256, BF16, [600], [200], 33, 65),
    (4, 4, 64, BF16, [2000], [50], 700, 2000),  # sinks cover everything
    (5, 1, 128, BF16, [70, 900], [70, 1], 10, 0),
    (8, 2, 128, BF16, [30], [50], 8, 2),
]


@pytest.mark.parametrize("case", ATTEND_CASES, ids=[f"{c[0]}q{c[1]}kv{c[2]}-{i}" for i, c in enumerate(ATTEND_CASES)])
def test_attend_matches_float64(hip_device, case) -> None:
    heads, kv, dim, dtype, lens, new, window, sinks = case
    g = torch.Generator().manual_seed(sum(lens) + dim)
    caches = _paged(lens, kv, dim, dtype, g)
    start = [0]
    for x in new:
        start.append(start[-1] + x)
    pad = 3
    q = (2 * torch.randn((start[-1] + pad, heads, dim), generator=g)).to(dtype)
    out = torch.full_like(q, 7.0, device=hip_device)
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    got = _serving().attend_paged(
        q.to(hip_device), caches[0].to(hip_device), caches[1].to(hip_device), d(start), d(lens), caches[2].to(hip_device),
        max_query_len=max(new), max_seq_len=max(lens), window=window, sinks=sinks, out=out)
    assert got is out and (out[start[-1] :] == 7).all()
    _check(got, q, caches[:2], start, lens, caches[2], dtype, scale=dim**-0.5, window=window, sinks=sinks,
           rows_most=max(new) * heads // kv)


@pytest.mark.parametrize("seed", range(12))
def test_attend_random_shapes(hip_device, seed) -> None:
    g = torch.Generator().manual_seed(seed)
    pick = lambda *x: x[int(torch.randint(len(x), (), generator=g))]  # noqa: E731
    kv, dim, dtype = pick(1, 2, 3, 8), pick(16, 64, 80, 96, 128, 192, 256), pick(BF16, FP16)
    heads = kv * pick(1, 2, 3, 5, 7, 8)
    n = pick(1, 2, 5)
    new = [pick(1, 1, 2, 9, 40, 150) for _ in range(n)]
    lens = [x + int(torch.randint(0, pick(2, 200, 900), (), generator=g)) for x in new]
    window = pick(0, 0, 1, 17, 128, 300)
    sinks = pick(0, 1, 4, 100, 140)
    caches = _paged(lens, kv, dim, dtype, g)
    start = [0, *torch.tensor(new).cumsum(0).tolist()]
    q = torch.randn((start[-1], heads, dim), generator=g).to(dtype)
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    got = _serving().attend_paged(q.to(hip_device), caches[0].to(hip_device), caches[1].to(hip_device), d(start), d(lens),
                                  caches[2].to(hip_device), scale=0.3, window=window, sinks=sinks)
    _check(got, q, caches[:2], start, lens, caches[2], dtype, scale=0.3, window=window, sinks=sinks, rows_most=max(new) * heads // kv)


@pytest.mark.parametrize("window, sinks", [(0, 0), (100, 5)])
@pytest.mark.parametrize("heads, kv, dim, dtype", [
    (16, 8, 64, BF16), (24, 8, 96, FP16), (40, 8, 128, BF16), (8, 8, 192, BF16), (16, 8, 192, FP16), (16, 8, 256, BF16), (64, 8, 256, BF16),
])
def test_attend_short_requests_apart_from_chunks(hip_device, heads, kv, dim, dtype, window, sinks) -> None:
    """A table so wide that short requests and chunks get a launch each, and a
    narrow one that gives them one: both are the definition's values."""
    g = torch.Generator().manual_seed(dim + heads)
    lens, new = [700, 1, 300, 2100, 5, 0], [2, 1, 150, 1, 5, 0]
    start = [0, *torch.tensor(new).cumsum(0).tolist()]
    q = torch.randn((start[-1], heads, dim), generator=g).to(dtype)
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    for width in (600, 20):
        caches = _paged(lens, kv, dim, dtype, torch.Generator().manual_seed(dim), max_blocks=width)
        got = _serving().attend_paged(q.to(hip_device), caches[0].to(hip_device), caches[1].to(hip_device), d(start), d(lens),
                                      caches[2].to(hip_device), max_query_len=max(new), window=window, sinks=sinks)
        _check(got, q, caches[:2], start, lens, caches[2], dtype, scale=dim**-0.5, window=window, sinks=sinks,
               rows_most=max(new) * heads // kv)


@pytest.mark.parametrize("dim, dtype", [(128, BF16), (128, FP16), (256, BF16), (96, BF16), (192, BF16), (64, FP16), (256, FP16)])
@pytest.mark.parametrize("new, window, sinks", [(3, 0, 0), (4, 7, 2), (60, 0, 0), (60, 9, 1)])
def test_hidden_values_reach_no_row_that_does_not_see_them(hip_device, dim, dtype, new, window, sinks) -> None:
    """Infinities and NaN in keys and values that some rows see and others do
    not: the ones that do get them, the others what they get without."""
    g = torch.Generator().manual_seed(dim + new)
    lens, heads, kv = [200, 90], 4, 2
    k, v, table = _paged(lens, kv, dim, dtype, g)
    for r, n in enumerate(lens):
        for back, what in ((new // 2, float("inf")), (new // 3, float("nan")), (new + 5, float("-inf"))):
            key = n - 1 - back
            page = int(table[r, key // 128])
            v[page, key % 128, 0, 1 + back % 5] = what
        key = n - 1 - new // 4
        k[int(table[r, key // 128]), key % 128, 1, 3] = float("nan")
    start = [0, new, 2 * new]
    q = torch.randn((2 * new, heads, dim), generator=g).to(dtype)
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    got = _serving().attend_paged(q.to(hip_device), k.to(hip_device), v.to(hip_device), d(start), d(lens), table.to(hip_device),
                                  max_query_len=new, window=window, sinks=sinks).cpu()
    want, _, _ = ref.attend(q, k, v, start, lens, table, scale=dim**-0.5, window=window, sinks=sinks)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(got)].double(), want[torch.isinf(want)])
    fine = torch.isfinite(want)
    assert fine.any() and not fine.all()
    assert ((got.double() - want).abs()[fine] <= 4 * torch.finfo(dtype).eps * (want.abs()[fine] + 1)).all()


@pytest.mark.parametrize("dim, dtype", [(64, BF16), (96, FP16), (128, BF16), (192, FP16), (256, BF16)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (6, 2)])
def test_hidden_values_beside_drafts_of_many_heads(hip_device, dim, dtype, window, sinks) -> None:
    """The same for three tokens of eight heads a KV head, by tokens that see a
    key and those that do not."""
    g = torch.Generator().manual_seed(dim)
    lens, heads, kv, new = [300, 131, 64], 16, 2, 3
    k, v, table = _paged(lens, kv, dim, dtype, g)
    for r, n in enumerate(lens):
        for key, what in ((n - 1, float("inf")), (n - 2, float("nan")), (n - 9, float("-inf"))):
            v[int(table[r, key // 128]), key % 128, r % 2, 1 + key % 7] = what
    start = [0, new, 2 * new, 3 * new]
    q = torch.randn((3 * new, heads, dim), generator=g).to(dtype)
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    got = _serving().attend_paged(q.to(hip_device), k.to(hip_device), v.to(hip_device), d(start), d(lens), table.to(hip_device),
                                  max_query_len=new, window=window, sinks=sinks).cpu()
    want, _, _ = ref.attend(q, k, v, start, lens, table, scale=dim**-0.5, window=window, sinks=sinks)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(got)].double(), want[torch.isinf(want)])
    fine = torch.isfinite(want)
    assert fine.any() and not fine.all()
    assert ((got.double() - want).abs()[fine] <= 4 * torch.finfo(dtype).eps * (want.abs()[fine] + 1)).all()


@pytest.mark.parametrize("dim, dtype", [(64, FP16), (128, BF16), (192, FP16), (256, BF16)])
@pytest.mark.parametrize("new, window, sinks", [(1, 0, 0), (3, 1500, 4), (130, 0, 0), (130, 1500, 4), (300, 0, 0)])
def test_hidden_values_in_pieces_that_are_joined(hip_device, dim, dtype, new, window, sinks) -> None:
    """Infinities and NaN in some of the pieces that a request's keys are split into,
    a piece of which holds no key for some rows: as many pieces as the launch is
    for, by a hint of 20000 keys."""
    g = torch.Generator().manual_seed(dim + new)
    lens, heads, kv = [3000, 1700], 4, 2
    k, v, table = _paged(lens, kv, dim, dtype, g, max_blocks=160)
    for r, n in enumerate(lens):
        first = n - new
        for key, what in ((10, float("nan")), (first - 700, float("inf")), (first + new // 2, float("-inf")), (n - 1, float("nan")), (2, float("inf"))):
            v[int(table[r, key // 128]), key % 128, r, 1 + key % 7] = what
        v[int(table[r, (first - 300) // 128]), (first - 300) % 128, 1 - r, :] = float("inf")
        key = first + new // 3
        k[int(table[r, key // 128]), key % 128, 1 - r, 3] = float("nan")
    start = [0, new, 2 * new]
    q = (0.5 * torch.randn((2 * new, heads, dim), generator=g)).to(dtype)
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    got = _serving().attend_paged(q.to(hip_device), k.to(hip_device), v.to(hip_device), d(start), d(lens), table.to(hip_device),
                                  max_query_len=new, max_seq_len=20000, window=window, sinks=sinks).cpu()
    want, _, _ = ref.attend(q, k, v, start, lens, table, scale=dim**-0.5, window=window, sinks=sinks)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(got)].double(), want[torch.isinf(want)])
    fine = torch.isfinite(want)
    assert fine.any() and not fine.all()
    assert ((got.double() - want).abs()[fine] <= 4 * torch.finfo(dtype).eps * (want.abs()[fine] + 1)).all()


@pytest.mark.parametrize("dim, dtype", [(64, BF16), (128, BF16), (192, FP16), (256, BF16)])
@pytest.mark.parametrize("lens, new", [([5000, 700, 3000], [1, 1, 1]), ([5000, 700, 3000], [4, 1, 3]), ([5000], [100]), ([4000, 2500], [90, 300]),
                                       ([9000] * 16, [1, 200, 2, 1] * 4)])
def test_workspace_of_split_calls(hip_device, dim, dtype, lens, new) -> None:
    """Nothing behind the workspace is written and nothing it held before is read:
    pieces of single tokens, drafts, chunks, and of both kinds after one another."""
    serving = _serving()
    g = torch.Generator(device=hip_device).manual_seed(dim)
    heads, kv = 16, 4
    pool = torch.randn((2, 300, 128, kv, dim), generator=g, device=hip_device).to(dtype)
    table = torch.stack([torch.randperm(300, generator=g, device=hip_device)[:80] for _ in lens]).int()
    q = torch.randn((sum(new), heads, dim), generator=g, device=hip_device).to(dtype)
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    start = d([0, *torch.tensor(new).cumsum(0).tolist()])
    args = (q, pool[0], pool[1], start, d(lens), table)
    sizes = {"max_query_len": max(new), "max_seq_len": max(lens)}
    size = serving.attend_workspace_bytes(heads, kv, dim, len(lens), sum(new), *sizes.values())
    outs = []
    for fill in (0x00, 0xFF, 0x7F):
        kept = torch.full((size + 4096,), fill, dtype=torch.uint8, device=hip_device)
        outs.append(serving.attend_paged(*args, **sizes, workspace=kept[:size]))
        assert (kept[size:] == fill).all()
    outs.append(serving.attend_paged(*args, **sizes, workspace=kept[:size]))
    assert all(torch.equal(out, outs[0]) for out in outs) and torch.isfinite(outs[0]).all()


@pytest.mark.parametrize("dim, heads, kv, new", [
    (64, 2, 2, 1), (128, 4, 1, 1), (64, 16, 2, 3), (256, 8, 1, 2), (64, 4, 2, 40), (128, 16, 2, 6), (256, 4, 2, 20),
])
def test_small_weights_of_many_keys_add_up(hip_device, dim, heads, kv, new) -> None:
    """fp16: a key of a large weight in each of the first page's four slices, and
    131068 of 2^-25 of it, whose values are 0 and 1: the many add up to 2^-10.  A
    hint of one key leaves all pages to one workgroup.

    Bounds.  Output: half a step, 2^-11 of it.  Scores are one product of 16-bit
    numbers each, exact; their float32 product with scale * log2(e), 25, is off by
    25 * 2^-24 twice, a weight by ln 2 times that and an exponential's last bits:
    2^-18.  Sums of positive numbers: at most 131072 / 32 products one after
    another, each 2^-24 of the sum, 2^-12; the sum of the weights likewise.
    Weights: one word, half a step, 2^-11, and 2^-34 of the largest each (fp16's
    half step at its end, 2^-25, where the largest is held as 2^9)."""
    length = 131072
    k = torch.zeros((length // 128, 128, kv, dim), dtype=FP16, device=hip_device)
    v = torch.ones_like(k)
    k[0, 5::32, :, 3], v[0, 5::32] = 17.390625, 0.0
    q = torch.zeros((new, heads, dim), dtype=FP16, device=hip_device)
    q[..., 3] = 1.0
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    table = torch.arange(length // 128, dtype=torch.int32, device=hip_device)[None]
    got = _serving().attend_paged(q, k, v, d([0, new]), d([length]), table, scale=1.0, max_query_len=new,
                                  max_seq_len=1).double().cpu()
    small = torch.arange(length - new - 3, length - 3, dtype=torch.float64)[:, None, None] * torch.exp(torch.tensor(-17.390625, dtype=torch.float64))
    want = small / (4 + small)
    bound = want * (2 * 2.0**-11 + 2 * 2.0**-12 + 2.0**-18) + length * 2.0**-34
    assert ((got - want).abs() <= bound).all(), (float(got.min()), float(got.max()), float(want.min()))


@pytest.mark.parametrize("dim, heads, kv, new", [(64, 2, 2, 1), (64, 16, 2, 3), (64, 4, 2, 40), (128, 16, 2, 6), (192, 4, 2, 20), (256, 4, 2, 20)])
def test_small_weights_count_in_the_sum(hip_device, dim, heads, kv, new) -> None:
    """fp16: values of 1 give 1, whatever the weights: 131068 of 2^-23 to 2^-25 of
    the largest, which the many-rows kernel holds below fp16's normal range, are
    2^-9 of the sum.

    Bounds.  Output: half a step, 2^-11.  Both sums are of the same rounded weights
    (two words leave 2^-40 of the largest each, 2^-23 in all): what differs is
    float32's rounding of 4096 products one after another, 2^-12 each."""
    length = 131072
    k = torch.zeros((length // 128, 128, kv, dim), dtype=FP16, device=hip_device)
    g = torch.Generator(device=hip_device).manual_seed(dim)
    k[..., 3] = -16 - 1.3 * torch.rand(k.shape[:3], generator=g, device=hip_device).half()
    k[0, 5::32, :, 3] = 0.0
    v = torch.ones_like(k)
    q = torch.zeros((new, heads, dim), dtype=FP16, device=hip_device)
    q[..., 3] = 1.0
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    table = torch.arange(length // 128, dtype=torch.int32, device=hip_device)[None]
    got = _serving().attend_paged(q, k, v, d([0, new]), d([length]), table, scale=1.0, max_query_len=new, max_seq_len=1).double()
    assert float((got - 1).abs().max()) <= 2.0**-11 + 2 * 2.0**-12


@pytest.mark.parametrize("dim, new", [(64, 1), (128, 40), (192, 40), (256, 40)])
def test_weights_of_huge_scores_stay_in_range(hip_device, dim, new) -> None:
    """fp16: scores of 2^27 + 16 and, in later tiles, one float32 step more, 16.  A
    row whose last keys have those gives their mean, as 2^-16 of 128 values of 1
    beside 217 or more of 3 is less than half a step of 3."""
    k = torch.zeros((4, 128, 1, dim), dtype=FP16)
    v = torch.ones_like(k)
    k[..., 0], k[..., 1] = 8192.0, 16.0
    k[1:, ..., 1] = 32.0
    v[1:] = 3.0
    q = torch.zeros((new, 1, dim), dtype=FP16)
    q[..., 0], q[..., 1] = 16384.0, 1.0
    table = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32, device=hip_device)
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    scale = 0.6931471824645996  # times float32's log2(e): exactly 1
    got = _serving().attend_paged(q.to(hip_device), k.to(hip_device), v.to(hip_device), d([0, new]), d([384]), table, scale=scale)
    assert (got == 3).all()


@pytest.mark.parametrize("dim, heads, new", [(64, 16, 1), (128, 8, 4), (256, 16, 1)])
def test_two_words_of_a_small_weight(hip_device, dim, heads, new) -> None:
    """fp16, few rows: weights of 2^-10 of the largest keep 2^-22 of their own.
    Two of them meet values of opposite sign, so their difference shows.

    Bounds.  Output: 2^-11 of it.  Scores are exact; times scale * log2(e) they
    are at most 11, off by 11 * 2^-24 in the factor, the product and the
    difference to the maximum: ln 2 * 33 * 2^-24 < 2^-19 of a weight, which
    covers the exponential's last bit too; words: 2^-22."""
    g = torch.Generator().manual_seed(dim)
    k = torch.zeros((1, 128, 1, dim), dtype=FP16)
    v = torch.zeros_like(k)
    k[0, 0, 0, 0], k[0, 1, 0, 1] = 6.5, 1.0
    v[0, 1], v[0, 2] = 32768.0, -32768.0
    q = torch.zeros((new, heads, dim), dtype=FP16)
    q[..., 0] = (1 + torch.rand((new, heads), generator=g) / 8).half()
    q[..., 1] = (2.0**-11 * (1 + torch.rand((new, heads), generator=g))).half()
    length = new + 3
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    got = _serving().attend_paged(q.to(hip_device), k.to(hip_device), v.to(hip_device), d([0, new]), d([length]), d([[0]]), scale=1.0,
                                  max_query_len=new).double().cpu()
    seen = torch.arange(length - new + 1, length + 1, dtype=torch.float64)[:, None]
    first, second = (q[..., 0].double() * 6.5).exp(), q[..., 1].double().exp()
    total = first + second + seen - 2
    want = (32768 * (second - 1) / total)[..., None]
    spread = (32768 * (second + 1) / total)[..., None]
    assert ((got - want).abs() <= 2.0**-11 * want + spread * (2.0**-19 + 2.0**-22)).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim, heads, kv, new", [(64, 8, 2, 40), (96, 4, 2, 40), (128, 40, 8, 30), (192, 4, 1, 50), (256, 8, 2, 70)])
def test_weights_of_chunks_add_up_to_one(hip_device, dim, heads, kv, new, dtype) -> None:
    """Values of c and one step above it, in another share in each dim: outputs are
    the mean, rounded, whatever step the weights lie off.  All keys but the first
    have a weight of (1 + 0.98 half steps) / 2, which rounds down, or (for every
    other head) of (1 + 3.02 half steps) / 2, which rounds up.

    Bounds.  Output: half a step of it.  Weights: half a step, of the distance of
    two values, which is one step of c; the first key's in proportion.  Sums of
    positive numbers in float32: 600 / 16 products and as many additions, each
    2^-24 of the sum: 2^-18."""
    length, step = 600, torch.finfo(dtype).eps
    k, v, table = _paged([length], kv, dim, dtype, torch.Generator().manual_seed(dim), hidden=0.0)
    slots = (table[0, : -(-length // 128), None].long() * 128 + torch.arange(128)).reshape(-1)[:length]
    share = (torch.arange(length)[:, None] * dim % (length + 1)) < (torch.arange(dim) * length / dim)[None]
    v.view(-1, kv, dim)[slots] = torch.where(share, 1 + step, 1.0).to(dtype)[:, None]
    # q.k of 0 for the first key, -x for the others, by the first two dims.
    k.zero_()
    k.view(-1, kv, dim)[slots[1:], :, 0] = -1.0
    k.view(-1, kv, dim)[slots[1:], :, 1] = -1.0
    off = torch.where(torch.arange(heads) % 2 == 0, 0.98, 3.02).double()
    x = -torch.log((1 + off * step / 2) / 2)
    q = torch.zeros((new, heads, dim), dtype=dtype)
    q[..., 0] = x.to(dtype)
    q[..., 1] = (x - x.to(dtype).double()).to(dtype)
    d = lambda y: torch.tensor(y, dtype=torch.int32, device=hip_device)  # noqa: E731
    got = _serving().attend_paged(q.to(hip_device), k.to(hip_device), v.to(hip_device), d([0, new]), d([length]), table.to(hip_device),
                                  scale=1.0)
    want, spread, _ = ref.attend(q, k, v, [0, new], [length], table, scale=1.0)
    assert ((got.double().cpu() - want).abs() <= want * (step / 2 + 2.0**-18) + step * step / 2).all()


@pytest.mark.parametrize("new", [1, 40])
def test_pages_outside_the_pool_are_not_seen(hip_device, new) -> None:
    g = torch.Generator().manual_seed(new)
    lens, heads, kv, dim = [700, 256, 90], 8, 2, 128
    k, v, table = _paged(lens, kv, dim, BF16, g)
    table[0, 1], table[0, 3], table[1, 0], table[1, 1], table[2, 0] = -1, k.shape[0], -5, 1 << 30, k.shape[0]
    table = table[:, :5].contiguous()  # the first request's last keys are past the table
    start = [0, new, 2 * new, 3 * new]
    q = torch.randn((3 * new, heads, dim), generator=g).to(BF16)
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    got = _serving().attend_paged(q.to(hip_device), k.to(hip_device), v.to(hip_device), d(start), d(lens), table.to(hip_device))
    _check(got, q, (k, v), start, lens, table, BF16, scale=dim**-0.5, window=0, sinks=0, rows_most=new * 4)
    assert (got[start[1] :] == 0).all()


@pytest.mark.parametrize("new", [1, 6, 70])
@pytest.mark.parametrize("dim, dtype", [(64, FP16), (96, BF16), (192, BF16), (192, FP16), (256, BF16)])
def test_pages_outside_the_pool_at_other_head_sizes(hip_device, dim, dtype, new) -> None:
    """Holes between a request's pages, at its first and last ones, odd and even
    numbers of key tiles, with a window over some."""
    g = torch.Generator().manual_seed(dim + new)
    lens, heads, kv = [1500, 1000, 500, 129], 8, 2
    k, v, table = _paged(lens, kv, dim, dtype, g)
    table[0, 2:5], table[0, 7], table[1, 0], table[2, 3] = -1, k.shape[0], -1, 1 << 30
    start = [0, new, 2 * new, 3 * new, 4 * new]
    q = torch.randn((4 * new, heads, dim), generator=g).to(dtype)
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    for window, sinks in ((0, 0), (300, 130)):
        got = _serving().attend_paged(q.to(hip_device), k.to(hip_device), v.to(hip_device), d(start), d(lens), table.to(hip_device),
                                      max_query_len=new, window=window, sinks=sinks)
        _check(got, q, (k, v), start, lens, table, dtype, scale=dim**-0.5, window=window, sinks=sinks, rows_most=new * 4)


@pytest.mark.parametrize("new", [1, 3, 50])
def test_attend_strided_views_and_padded_pages(hip_device, new) -> None:
    """q from a fused projection, out a part of a wider buffer, K and V views of
    one padded page buffer: the values of contiguous tensors, bit for bit."""
    g = torch.Generator().manual_seed(new)
    lens, heads, kv, dim = [500, 129], 10, 2, 128
    k, v, table = (x.to(hip_device) for x in _paged(lens, kv, dim, BF16, g))
    start = torch.tensor([0, new, 2 * new], dtype=torch.int32, device=hip_device)
    seq = torch.tensor(lens, dtype=torch.int32, device=hip_device)
    fused = torch.randn((2 * new, heads + 2 * kv, dim), generator=g).to(BF16).to(hip_device)
    q = fused[:, kv : kv + heads]
    plain = _serving().attend_paged(q.contiguous(), k, v, start, seq, table, window=90, sinks=3)
    page = 128 * kv * dim
    buffer = torch.full((k.shape[0], 2 * page + 64), float("nan"), dtype=BF16, device=hip_device)
    buffer[:, :page], buffer[:, page : 2 * page] = k.reshape(-1, page), v.reshape(-1, page)
    views = [torch.as_strided(buffer, k.shape, (2 * page + 64, kv * dim, dim, 1), at) for at in (0, page)]
    wide = torch.full((heads, 2 * new, dim + 8), 5.0, dtype=BF16, device=hip_device)
    out = wide.transpose(0, 1)[..., :dim]
    tables = torch.full((2, table.shape[1] + 3), 9, dtype=torch.int32, device=hip_device)
    tables[:, : table.shape[1]] = table
    got = _serving().attend_paged(q, *views, start, seq, tables[:, : table.shape[1]], window=90, sinks=3, out=out)
    assert torch.equal(got, plain) and (wide[..., dim:] == 5).all()


@pytest.mark.parametrize("new", [1, 40])
def test_outputs_beside_inputs_in_one_buffer(hip_device, new) -> None:
    """Outputs between a projection's parts, heads taking turns, or tokens taking
    turns are no overlap; the inputs themselves, shifted or widened, are."""
    g = torch.Generator().manual_seed(new)
    lens, heads, kv, dim, tokens = [500, 129], 8, 2, 64, 2 * new
    k, v, table = (x.to(hip_device) for x in _paged(lens, kv, dim, BF16, g, hidden=0.0))
    start = torch.tensor([0, new, 2 * new], dtype=torch.int32, device=hip_device)
    seq = torch.tensor(lens, dtype=torch.int32, device=hip_device)
    host = torch.randn((tokens, heads, dim), generator=g).to(BF16).to(hip_device)
    attend = lambda q, out=None: _serving().attend_paged(q, k, v, start, seq, table, out=out)  # noqa: E731
    plain = attend(host)
    fused = torch.zeros((tokens, 3 * heads, dim), dtype=BF16, device=hip_device)
    flat = torch.zeros((2 * heads, tokens, dim), dtype=BF16, device=hip_device)
    turns = torch.zeros((tokens, 2, heads, dim), dtype=BF16, device=hip_device)
    places = [(fused[:, heads : 2 * heads], fused[:, :heads]), (fused[:, :heads], fused[:, 2 * heads :]), (fused[:, 0 : 2 * heads : 2], fused[:, 1 : 2 * heads : 2]),
              (flat[:heads].transpose(0, 1), flat[heads:].transpose(0, 1)), (flat[1::2].transpose(0, 1), flat[0::2].transpose(0, 1)),
              (turns[:, 1], turns[:, 0])]
    for q, out in places:
        q.copy_(host)
        out.fill_(7.0)
        assert attend(q, out) is out and torch.equal(out, plain) and torch.equal(q, host)
    q = fused[:, :heads].copy_(host)
    for out in (q, fused[:, 1 : heads + 1], turns[:, 0, :1].expand(-1, heads, -1), turns[:1, 0].expand(tokens, -1, -1)):
        with pytest.raises(ValueError, match="overlap"):
            attend(q, out)
    omega = torch.ones(dim // 2, device=hip_device)
    positions, slots = torch.arange(tokens, device=hip_device), torch.arange(tokens, device=hip_device)
    pages = [torch.zeros((2, 128, kv, dim), dtype=BF16, device=hip_device) for _ in range(2)]
    kk, vv = (torch.randn((tokens, kv, dim), generator=g).to(BF16).to(hip_device) for _ in range(2))
    rotate = lambda q, k, v, out=None: _serving().rotate_and_store(q, k, v, positions, omega, slots, *pages, q_out=out)  # noqa: E731
    plain = rotate(host, kk, vv)
    for q, out in places:
        q.copy_(host)
        assert torch.equal(rotate(q, kk, vv, out), plain) and torch.equal(q, host)
        assert rotate(q, kk, vv, q) is q and torch.equal(q, plain)
    q = fused[:, :heads].copy_(host)
    for out in (fused[:, 1 : heads + 1], fused[:, heads : 2 * heads], turns[:, 0, :1].expand(-1, heads, -1)):
        with pytest.raises(ValueError, match="overlap|another view"):
            rotate(q, fused[:, heads : heads + kv], fused[:, 2 * heads - kv : 2 * heads], out)


def test_attend_far_pages(hip_device) -> None:
    """Rows behind 2^32 elements of the pool, and slots behind 2^31 rows' bytes."""
    g = torch.Generator().manual_seed(5)
    kv, dim, heads, stride = 2, 128, 8, 1 << 20
    pages = 6000  # 6000 x 2^20 elements: 12.6 GB a cache
    pools = [torch.empty(pages * stride, dtype=BF16, device=hip_device) for _ in range(2)]
    caches = [torch.as_strided(p, (pages, 128, kv, dim), (stride, kv * dim, dim, 1)) for p in pools]
    table = torch.tensor([[5999, 4097, 2], [2048, 4096, 5000]], dtype=torch.int32)
    small = [torch.randn((6, 128, kv, dim), generator=g).to(BF16) for _ in range(2)]
    for cache, host in zip(caches, small):
        cache[table.view(-1).long().to(hip_device)] = host.to(hip_device)
    lens = [300, 384]
    near = torch.arange(6, dtype=torch.int32).view(2, 3)
    for new in (1, 30):
        start = [0, new, 2 * new]
        q = torch.randn((2 * new, heads, dim), generator=g).to(BF16)
        d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
        got = _serving().attend_paged(q.to(hip_device), *caches, d(start), d(lens), table.to(hip_device))
        _check(got, q, small, start, lens, near, BF16, scale=dim**-0.5, window=0, sinks=0, rows_most=new * 4)
    token = torch.randn((2, kv, dim), generator=g).to(BF16).to(hip_device)
    _serving().rotate_and_store(
        token[:, :0], token, token, torch.zeros(2, dtype=torch.int64, device=hip_device), torch.ones(64, device=hip_device),
        torch.tensor([5999 * 128 + 127, 4096 * 128], device=hip_device), *caches)
    assert torch.equal(caches[0][5999, 127], token[0]) and torch.equal(caches[1][4096, 0], token[1])


@pytest.mark.parametrize("new", [1, 2, 33])
def test_attend_splits_and_joins_long_requests(hip_device, new) -> None:
    """One long request beside short ones: its keys are spread over workgroups and joined."""
    g = torch.Generator().manual_seed(new)
    lens, heads, kv, dim = [20000, 40, 3000], 8, 2, 128
    k, v, table = _paged(lens, kv, dim, BF16, g)
    start = [0, new, new + 1, 2 * new + 1]
    q = torch.randn((start[-1], heads, dim), generator=g).to(BF16)
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    args = (q.to(hip_device), k.to(hip_device), v.to(hip_device), d(start), d(lens), table.to(hip_device))
    got = _serving().attend_paged(*args, max_query_len=new, max_seq_len=20000)
    _check(got, q, (k, v), start, lens, table, BF16, scale=dim**-0.5, window=0, sinks=0, rows_most=new * 4)
    again = _serving().attend_paged(*args, max_query_len=new, max_seq_len=20000)
    assert torch.equal(got, again)
    # Sizes that shape the launch only: the same values to rounding.
    hint = _serving().attend_paged(*args, max_query_len=new, max_seq_len=1)
    _check(hint, q, (k, v), start, lens, table, BF16, scale=dim**-0.5, window=0, sinks=0, rows_most=new * 4)


def test_attend_more_requests_than_one_launch_takes(hip_device) -> None:
    g = torch.Generator(device=hip_device).manual_seed(1)
    n, kv, dim = 5000, 1, 64
    pool = torch.randn((2, 300, 128, kv, dim), generator=g, device=hip_device).to(BF16)
    table = torch.randint(0, 300, (n, 2), generator=g, device=hip_device).int()
    lens = torch.randint(1, 200, (n,), generator=g, device=hip_device).int()
    q = torch.randn((n, 2, dim), generator=g, device=hip_device).to(BF16)
    start = torch.arange(n + 1, dtype=torch.int32, device=hip_device)
    got = _serving().attend_paged(q, pool[0], pool[1], start, lens, table, max_query_len=1)
    for r in (0, 1023, 1024, 2047, 2048, 4095, 4096, 4999):
        one = _serving().attend_paged(q[r : r + 1], pool[0], pool[1], start[:2], lens[r : r + 1], table[r : r + 1])
        torch.testing.assert_close(got[r : r + 1], one, rtol=2.0**-7, atol=2.0**-12)


@pytest.mark.parametrize("n, longest, heads", [(70, 90, 8), (300, 40, 4), (5000, 12, 8)])
def test_attend_chunks_of_many_requests(hip_device, n, longest, heads) -> None:
    """Row tiles of more requests than a wave has lanes, between ones without any:
    each request's rows are what it gets alone."""
    g = torch.Generator(device=hip_device).manual_seed(n)
    kv, dim = 2, 64
    pool = torch.randn((2, 200, 128, kv, dim), generator=g, device=hip_device).to(BF16)
    table = torch.randint(0, 200, (n, 3), generator=g, device=hip_device).int()
    new = torch.randint(0, longest, (n,), generator=g, device=hip_device).int()
    new[n // 3 : n // 2] = 0
    new[[0, n // 2, n - 1]] = longest
    lens = new + torch.randint(0, 250, (n,), generator=g, device=hip_device).int()
    start = torch.cat([new.new_zeros(1), new.cumsum(0, dtype=torch.int32)])
    host = start.tolist()
    q = torch.randn((host[-1], heads, dim), generator=g, device=hip_device).to(BF16)
    got = _serving().attend_paged(q, pool[0], pool[1], start, lens, table, max_query_len=longest)
    assert torch.isfinite(got).all()
    two = torch.empty(2, dtype=torch.int32, device=hip_device)
    for r in sorted({0, 1, n // 3 - 1, n // 2, n // 2 + 1, 63 % n, 64, 65, n - 2, n - 1}):
        size = host[r + 1] - host[r]
        two[0], two[1] = 0, size
        one = _serving().attend_paged(q[host[r] : host[r + 1]], pool[0], pool[1], two, lens[r : r + 1], table[r : r + 1])
        torch.testing.assert_close(got[host[r] : host[r + 1]], one, rtol=2.0**-6, atol=2.0**-9)


@pytest.mark.parametrize("tokens, total, kv, heads, window", [(900, 3000, 8, 40, 0), (700, 2500, 8, 40, 700), (1300, 1300, 2, 16, 0)])
def test_attend_splits_what_whole_rounds_leave(hip_device, tokens, total, kv, heads, window) -> None:
    """More (row tile, head) items than the device takes at once, or fewer: the ones left over are split."""
    g = torch.Generator().manual_seed(tokens)
    dim = 128
    k, v, table = _paged([total], kv, dim, BF16, g)
    q = torch.randn((tokens, heads, dim), generator=g).to(BF16)
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    got = _serving().attend_paged(q.to(hip_device), k.to(hip_device), v.to(hip_device), d([0, tokens]), d([total]), table.to(hip_device),
                                  window=window, max_seq_len=total)
    # Rows of the first, middle and last tiles, as requests of one token each.
    picked = sorted({0, 1, 25, 26, 300, 301, tokens // 2, tokens - 27, tokens - 1})
    lens = [total - tokens + i + 1 for i in picked]
    _check(got[picked], q[picked], (k, v), list(range(len(picked) + 1)), lens, table.expand(len(picked), -1), BF16, scale=dim**-0.5,
           window=window, sinks=0, rows_most=tokens)


@pytest.mark.parametrize("heads, kv, dim, tokens, total", [(40, 8, 64, 10000, 10100), (24, 3, 64, 17000, 20000), (64, 8, 256, 3170, 6000)])
def test_attend_splits_behind_many_rounds(hip_device, heads, kv, dim, tokens, total) -> None:
    """Six rounds of (row tile, head) items and a few more, which are split as well."""
    g = torch.Generator().manual_seed(tokens)
    k, v, table = _paged([total], kv, dim, BF16, g)
    q = torch.randn((tokens, heads, dim), generator=g).to(BF16)
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    got = _serving().attend_paged(q.to(hip_device), k.to(hip_device), v.to(hip_device), d([0, tokens]), d([total]), table.to(hip_device),
                                  max_seq_len=total)
    assert torch.isfinite(got).all()
    picked = sorted({0, 1, 15, 16, 31, 32, 50, 51, 52, 300, tokens // 2, tokens - 27, tokens - 1})
    lens = [total - tokens + i + 1 for i in picked]
    _check(got[picked], q[picked], (k, v), list(range(len(picked) + 1)), lens, table.expand(len(picked), -1), BF16, scale=dim**-0.5,
           window=0, sinks=0, rows_most=tokens)


@pytest.mark.parametrize("tokens, total, kv, heads, dim, dtype", [
    (300, 5000, 2, 8, 64, BF16), (300, 5000, 2, 8, 96, FP16), (300, 5000, 2, 8, 192, BF16), (300, 5000, 2, 8, 256, BF16),
    (700, 2500, 8, 40, 256, FP16), (900, 2500, 8, 40, 192, BF16),
])
def test_attend_splits_at_other_head_sizes(hip_device, tokens, total, kv, heads, dim, dtype) -> None:
    g = torch.Generator().manual_seed(dim)
    k, v, table = _paged([total], kv, dim, dtype, g)
    q = torch.randn((tokens, heads, dim), generator=g).to(dtype)
    d = lambda x: torch.tensor(x, dtype=torch.int32, device=hip_device)  # noqa: E731
    got = _serving().attend_paged(q.to(hip_device), k.to(hip_device), v.to(hip_device), d([0, tokens]), d([total]), table.to(hip_device))
    picked = sorted({0, 1, 25, 26, 31, 32, 63, 64, tokens // 2, tokens - 27, tokens - 1})
    lens = [total - tokens + i + 1 for i in picked]
    _check(got[picked], q[picked], (k, v), list(range(len(picked) + 1)), lens, table.expand(len(picked), -1), dtype, scale=dim**-0.5,
           window=0, sinks=0, rows_most=tokens)


@pytest.mark.parametrize("new", [1, 40])
def test_attend_under_capture_and_on_another_stream(hip_device, new) -> None:
    g = torch.Generator(device=hip_device).manual_seed(new)
    kv, dim, heads, n = 2, 128, 8, 3
    pool = torch.randn((2, 60, 128, kv, dim), generator=g, device=hip_device).to(BF16)
    table = torch.randperm(60, generator=g, device=hip_device).int().view(n, 20)
    start = new * torch.arange(n + 1, dtype=torch.int32, device=hip_device)
    lens = torch.tensor([300, 2560, 1000], dtype=torch.int32, device=hip_device)
    q = torch.randn((n * new, heads, dim), generator=g, device=hip_device).to(BF16)
    run = lambda out=None: _serving().attend_paged(q, pool[0], pool[1], start, lens, table, max_query_len=new, out=out)  # noqa: E731
    eager = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(eager, other)
    graphs, outs = [], []
    for _ in range(2):
        graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(q)
        with torch.cuda.graph(graph):
            run(out)
        graphs.append(graph)
        outs.append(out)
    for step in range(4):
        q.normal_(generator=g)
        lens.sub_(7)
        eager = run().clone()
        for graph, out in zip(graphs, outs):
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, eager) for out in outs), step


def test_attend_workspace(hip_device) -> None:
    serving = _serving()
    g = torch.Generator(device=hip_device).manual_seed(2)
    pool = torch.randn((2, 40, 128, 2, 64), generator=g, device=hip_device).to(FP16)
    q = torch.randn((1, 4, 64), generator=g, device=hip_device).to(FP16)
    table = torch.arange(40, dtype=torch.int32, device=hip_device)[None]
    start = torch.tensor([0, 1], dtype=torch.int32, device=hip_device)
    lens = torch.tensor([5000], dtype=torch.int32, device=hip_device)
    size = serving.attend_workspace_bytes(4, 2, 64, 1, 1, 1, 40 * 128)
    guard = torch.full((size + 64,), 0xA5, dtype=torch.uint8, device=hip_device)
    kept = serving.attend_paged(q, pool[0], pool[1], start, lens, table, workspace=guard[:size])
    assert (guard[size:] == 0xA5).all()
    assert torch.equal(kept, serving.attend_paged(q, pool[0], pool[1], start, lens, table))
    with pytest.raises(ValueError, match="workspace"):
        serving.attend_paged(q, pool[0], pool[1], start, lens, table, workspace=guard[: size - 16])


def test_attend_nothing_to_do(hip_device) -> None:
    serving = _serving()
    cache = torch.zeros((1, 128, 2, 64), dtype=BF16, device=hip_device)
    empty = torch.zeros((0, 4, 64), dtype=BF16, device=hip_device)
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=hip_device)  # noqa: E731
    assert serving.attend_paged(empty, cache, cache, i(3), i(2), i(2, 1)).shape == (0, 4, 64)
    assert serving.attend_paged(empty, cache, cache, i(1), i(0), i(0, 1)).shape == (0, 4, 64)
    out = torch.full((2, 4, 64), 3.0, dtype=BF16, device=hip_device)
    serving.attend_paged(torch.zeros_like(out), cache, cache, i(4), i(3), i(3, 1), out=out)  # requests without tokens
    assert (out == 3).all()
    start = torch.tensor([0, 2], dtype=torch.int32, device=hip_device)
    serving.attend_paged(torch.zeros_like(out), cache[:0], cache[:0], start, i(1) + 50, i(1, 0), out=out)  # no pages at all
    assert (out == 0).all()


# -------------------------------------------------------------- a whole step --


def test_step_after_a_compression(hip_device) -> None:
    """Compress two of three requests, then run a step on the cache that is left:
    tables from the lengths, rotation at semantic positions into physical slots,
    attention over the kept rows and the new ones."""
    from kvcompress_mi355x import workloads

    serving = _serving()
    spec = workloads.config_spec(
        1, seq_lens=(700, 1100), budget=256, recent=32, permute_pages=True, num_attention_heads=8, num_kv_heads=2)
    cache = workloads.build_synthetic_cache(spec, hip_device, seed=4)
    k, v = cache.k_caches[0], cache.v_caches[0]
    third = torch.randn((2, 2, 128, 2, 128), device=hip_device).to(k.dtype)
    k, v = torch.cat([k, third[0]]), torch.cat([v, third[1]])
    cache.k_caches[0], cache.v_caches[0] = k, v
    pipeline, batch = workloads.build_pipeline(cache)
    _, tables, _ = pipeline.step(batch)
    pages = k.shape[0]
    # The kept pages and one more for each compressed request (a freed one), the
    # third request's own two.
    rows = [[*tables[0].tolist(), int(cache.source_tables[0][0])], [*tables[1].tolist(), int(cache.source_tables[1][0])], [pages - 2, pages - 1]]
    computed, new, removed = [700, 1100, 250], [1, 3, 2], [700 - 256, 1100 - 256, 0]
    total, width, heads, dim = 8, 4, 8, 128
    d = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device=hip_device)  # noqa: E731
    buffers = {
        "query_start_loc": torch.empty(4, dtype=torch.int32, device=hip_device), "seq_lens": torch.empty(3, dtype=torch.int32, device=hip_device),
        "positions": torch.empty(total, dtype=torch.int64, device=hip_device), "slot_mapping": torch.empty(total, dtype=torch.int64, device=hip_device),
        "block_table": torch.empty((3, width), dtype=torch.int32, device=hip_device)}
    flat = [i for row in rows for i in row]
    lengths = d([0, 3, 6, 8], torch.int64)
    g = torch.Generator().manual_seed(9)
    host = torch.randn((total, heads + 4, dim), generator=g).to(k.dtype)
    qkv = host.to(hip_device)
    omega = 1.0 / (1e6 ** (torch.arange(64) / 64))
    out, q_out = torch.full((total, heads, dim), 9.0, dtype=k.dtype, device=hip_device), torch.empty((total, heads, dim), dtype=k.dtype, device=hip_device)
    device_args = (d(computed), d(new), d(removed, torch.int64), d(flat, torch.int64), lengths)
    device_omega = omega.to(hip_device)

    def step():
        serving.build_step_tables(*device_args, 128, max_query_len=3, **buffers)
        serving.rotate_and_store(qkv[:, :heads], qkv[:, heads : heads + 2], qkv[:, heads + 2 :], buffers["positions"], device_omega,
                                 buffers["slot_mapping"], k, v, q_out=q_out)
        serving.attend_paged(q_out, k, v, buffers["query_start_loc"], buffers["seq_lens"], buffers["block_table"], max_query_len=3,
                             window=200, sinks=4, out=out)

    before = (k.cpu(), v.cpu())
    step()
    want = ref.step_tables(computed, new, removed, rows, 128, total, width)
    for name, value in zip(("query_start_loc", "seq_lens", "positions", "slot_mapping", "block_table"), want):
        assert buffers[name].tolist() == value, name
    kept_k, kept_v = k.cpu(), v.cpu()
    turned = ref.rotate(host[:, heads : heads + 2], torch.tensor([want[2]]), omega, (64,), "blocked", "half")
    for t, slot in enumerate(want[3]):
        if slot >= 0:
            assert ((kept_k[slot // 128, slot % 128].double() - turned[t]).abs() <= 2.0**-8 * turned[t].abs() + 2.0**-17).all()
            assert torch.equal(kept_v[slot // 128, slot % 128], host[t, heads + 2 :])
            before[0][slot // 128, slot % 128], before[1][slot // 128, slot % 128] = kept_k[slot // 128, slot % 128], kept_v[slot // 128, slot % 128]
    assert torch.equal(before[0], kept_k) and torch.equal(before[1], kept_v)
    _check(out, q_out.cpu(), (kept_k, kept_v), want[0], want[1], torch.tensor(want[4]), k.dtype, scale=dim**-0.5, window=200, sinks=4, rows_most=12)
    assert (out[6:] == 9).all()
    # The same step as a graph, replayed with other lengths.
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        device_args[0].add_(1)
        out.fill_(9.0)
        step()
        eager = [x.clone() for x in (out, k, v, buffers["slot_mapping"])]
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, (out, k, v, buffers["slot_mapping"])))

"""What the model step's operators refuse, before anything reaches a device, and
their float64 definitions on small cases worked out by hand."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import serving_ref as ref

BF16 = torch.bfloat16


@pytest.fixture
def launches(monkeypatch):
    """Host tensors pass for device tensors; launches are recorded, not made."""
    from kvcompress_mi355x import _native
    from kvcompress_mi355x.methods.triattention import _device as dev

    made = []
    monkeypatch.setattr(dev, "require_hip", lambda tensor, name: None)
    monkeypatch.setattr(dev, "stream_handle", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(_native, "call", lambda entry, *args: made.append((entry, args)))
    return made


def _serving():
    from kvcompress_mi355x.methods.triattention import serving

    return serving


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _i64(*shape):
    return torch.zeros(shape, dtype=torch.int64)


def _table_args(n=3, tokens=5, blocks=4):
    args = [_i32(n), _i32(n), _i64(n), _i64(7), _i64(n + 1), 128]
    buffers = {"query_start_loc": _i32(n + 1), "seq_lens": _i32(n), "positions": _i64(tokens), "slot_mapping": _i64(tokens),
               "block_table": _i32(n, blocks)}
    return args, buffers


def test_host_tensors_are_refused() -> None:
    args, buffers = _table_args()
    with pytest.raises(ValueError, match="HIP device"):
        _serving().build_step_tables(*args, **buffers)
    cache = torch.zeros(2, 128, 1, 16, dtype=BF16)
    q = torch.zeros(1, 1, 16, dtype=BF16)
    with pytest.raises(ValueError, match="HIP device"):
        _serving().attend_paged(q, cache, cache, _i32(2), _i32(1), _i32(1, 1))
    with pytest.raises(ValueError, match="HIP device"):
        _serving().rotate_and_store(q, q, q, _i64(1), torch.zeros(8), _i64(1), cache, cache)


@pytest.mark.parametrize("at, value, message", [
    (0, _i64(3), "computed_tokens must have dtype"),
    (1, _i32(4), "new_tokens must have 3 entries"),
    (1, _i32(6)[::2], "new_tokens must be a contiguous vector"),
    (2, _i32(3), "request_offsets must have dtype"),
    (2, _i64(2), "request_offsets must have 3 entries"),
    (3, _i32(7), "block_ids must have dtype"),
    (4, _i64(3), "block_offsets must have 4 entries"),
    ("query_start_loc", _i32(3), "query_start_loc must have 4 entries"),
    ("seq_lens", _i32(2), "seq_lens must have an entry"),
    ("positions", _i32(5), "positions must have dtype"),
    ("slot_mapping", _i64(4), "slot_mapping must have 5 entries"),
    ("block_table", _i64(3, 4), "block_table must have dtype"),
    ("block_table", _i32(2, 4), "block_table must be"),
    ("block_table", _i32(4, 3).t(), "block_table must be"),
    ("max_query_len", -1, "max_query_len"),
])
def test_step_tables_refusals(launches, at, value, message) -> None:
    args, buffers = _table_args()
    if isinstance(at, int):
        args[at] = value
    else:
        buffers[at] = value
    with pytest.raises(ValueError, match=message):
        _serving().build_step_tables(*args, **buffers)
    assert launches == []
    args, buffers = _table_args()
    _serving().build_step_tables(*args, **buffers)
    assert [entry for entry, _ in launches] == ["kvc_step_tables"]


def _rotary_args(tokens=5, heads=4, kv=2, dim=32, pages=2):
    cache = torch.zeros(pages, 128, kv, dim, dtype=BF16)
    return {"q": torch.zeros(tokens, heads, dim, dtype=BF16), "k": torch.zeros(tokens, kv, dim, dtype=BF16),
            "v": torch.zeros(tokens, kv, dim, dtype=BF16), "positions": _i64(3, tokens), "omega": torch.zeros(16), "slot_mapping": _i64(tokens),
            "k_cache": cache, "v_cache": cache.clone(), "sections": (8, 4, 4)}


@pytest.mark.parametrize("change, message", [
    ({"q": torch.zeros(5, 4, 32)}, "q must have the cache's dtype"),
    ({"q": torch.zeros(4, 4, 32, dtype=BF16)}, "q must have shape"),
    ({"q": torch.zeros(5, 4, 64, dtype=BF16)[..., ::2]}, "q must have contiguous heads"),
    ({"k": torch.zeros(5, 3, 32, dtype=BF16)}, "k must have the cache's 2 heads"),
    ({"v": torch.zeros(5, 2, 16, dtype=BF16)}, "v must have shape"),
    ({"positions": _i64(3, 4)}, "positions must be"),
    ({"positions": _i32(3, 5)}, "positions must have dtype"),
    ({"positions": _i64(5, 3).t()}, "positions must be"),
    ({"positions": _i64(5)}, "sections must name"),
    ({"positions": _i64(5, 5), "sections": (4, 4, 4, 2, 2)}, "one to four"),
    ({"sections": None}, "sections must name"),
    ({"sections": (8, 4, 5)}, "add up to 16"),
    ({"sections": (20, -2, -2)}, "non-negative"),
    ({"omega": torch.zeros(17), "sections": (8, 4, 5)}, "omega must hold"),
    ({"omega": torch.zeros(16, dtype=torch.float64)}, "omega must have dtype"),
    ({"slot_mapping": _i32(5)}, "slot_mapping must have dtype"),
    ({"axis_order": "mixed"}, "axis_order"),
    ({"rope_style": "full"}, "rope style"),
    ({"v_cache": torch.zeros(3, 128, 2, 32, dtype=BF16)}, "K and V caches"),
    ({"k_cache": torch.zeros(2, 64, 2, 32, dtype=BF16)}, "k_cache must have shape"),
    ({"q_out": torch.zeros(5, 3, 32, dtype=BF16)}, "q_out must have q's heads"),
])
def test_rotary_refusals(launches, change, message) -> None:
    with pytest.raises(ValueError, match=message):
        _serving().rotate_and_store(**{**_rotary_args(), **change})
    assert launches == []


def test_rotary_takes_q_itself_but_no_other_view_of_it(launches) -> None:
    args = _rotary_args()
    assert _serving().rotate_and_store(**args, q_out=args["q"]) is args["q"]
    args["q"] = torch.zeros(5 * 4 * 32 + 64, dtype=BF16)[: 5 * 128].view(5, 4, 32)
    with pytest.raises(ValueError, match="another view"):
        _serving().rotate_and_store(**args, q_out=torch.as_strided(args["q"], (5, 4, 32), (64, 32, 1)))
    assert len(launches) == 1


def _attend_args(tokens=5, heads=4, kv=2, dim=32, pages=2, n=2):
    cache = torch.zeros(pages, 128, kv, dim, dtype=BF16)
    return {"q": torch.zeros(tokens, heads, dim, dtype=BF16), "k_cache": cache, "v_cache": cache.clone(), "query_start_loc": _i32(n + 1),
            "seq_lens": _i32(n), "block_table": _i32(n, 4)}


@pytest.mark.parametrize("change, message", [
    ({"q": torch.zeros(5, 4, 32)}, "q must have the cache's dtype"),
    ({"q": torch.zeros(5, 3, 32, dtype=BF16)}, "multiple of the cache's KV heads"),
    ({"q": torch.zeros(5, 0, 32, dtype=BF16)}, "multiple of the cache's KV heads"),
    ({"q": torch.zeros(5, 128, dtype=BF16)}, "q must have shape"),
    ({"query_start_loc": _i64(3)}, "query_start_loc must have dtype"),
    ({"query_start_loc": _i32(0)}, "one entry more"),
    ({"query_start_loc": _i32(4)}, "row for every request"),
    ({"seq_lens": _i32(1)}, "row for every request"),
    ({"block_table": _i64(2, 4)}, "block_table must have dtype"),
    ({"block_table": _i32(4, 2).t()}, "contiguous rows"),
    ({"scale": 0.0}, "scale"),
    ({"scale": -1.0}, "scale"),
    ({"scale": math.inf}, "scale"),
    ({"scale": math.nan}, "scale"),
    ({"window": -1}, "non-negative"),
    ({"sinks": -1}, "non-negative"),
    ({"max_query_len": -1}, "non-negative"),
    ({"max_seq_len": -2}, "non-negative"),
    ({"out": torch.zeros(5, 2, 32, dtype=BF16)}, "out must have q's shape"),
    ({"out": torch.zeros(5, 4, 32)}, "out must have the cache's dtype"),
    ({"workspace": torch.zeros(8, dtype=torch.uint8)}, "workspace must be contiguous"),
    ({"k_cache": torch.zeros(2, 128, 2, 32), "v_cache": torch.zeros(2, 128, 2, 32)}, "cache dtype"),
])
def test_attend_refusals(launches, change, message) -> None:
    with pytest.raises(ValueError, match=message):
        _serving().attend_paged(**{**_attend_args(), **change})
    assert launches == []


@pytest.mark.parametrize("dim", [4, 20, 264])
def test_attend_refuses_head_sizes(launches, dim) -> None:
    with pytest.raises(ValueError, match="multiple of 8 up to 256"):
        _serving().attend_paged(**_attend_args(dim=dim))
    assert launches == []


def _attend_c(lib, **change):
    fake = 4096  # 16-byte aligned placeholders; every refusal comes before a dereference
    a = dict(dtype=0, q=fake, qt=256, qh=128, k=fake, v=fake, pages=4, page=128 * 2 * 128, kv=2, qpk=1, dim=128, n=1, tokens=1, start=fake,
             lens=fake, table=fake, stride=4, blocks=4, longest=1, reach=512, scale=1.0, window=0, sinks=0, out=fake, ot=256, oh=128, ws=fake,
             size=1 << 40)
    a.update(change)
    return lib.kvc_attend_paged(None, *a.values())


@pytest.mark.parametrize("change, message", [
    ({"dtype": 2}, "dtype"),
    ({"dim": 12}, "head_dim 12"),
    ({"kv": 0}, "bad sizes"),
    ({"n": -1}, "bad sizes"),
    ({"tokens": 1 << 24}, "bad sizes"),
    ({"page": 128 * 2 * 128 - 8}, "page_stride"),
    ({"page": 128 * 2 * 128 + 4}, "page_stride"),
    ({"page": 1 << 31}, "page_stride"),
    ({"blocks": 5}, "block_table_stride"),
    ({"blocks": 1 << 23, "stride": 1 << 23}, "max_blocks"),
    ({"scale": -1.0}, "scale"),
    ({"scale": float("nan")}, "scale"),
    ({"window": -1}, "window"),
    ({"q": None}, "null pointer"),
    ({"table": None}, "null pointer"),
    ({"out": 4100}, "aligned"),
    ({"qt": 130}, "strides"),
    ({"size": 64}, "workspace too small"),
    ({"ws": None}, "workspace too small"),
    ({"kv": 512, "page": 128 * 512 * 128, "blocks": (1 << 22) + 1, "stride": 1 << 23}, "2\\^30"),
])
def test_attend_entry_refusals(change, message) -> None:
    from kvcompress_mi355x import _native

    lib = _native.load()
    assert _attend_c(lib, **change) == _native.EINVAL
    import re

    assert re.search(message, lib.kvc_last_error().decode()), lib.kvc_last_error()


@pytest.mark.parametrize("tokens, qpk", [(1 << 23, 256), ((1 << 24) - 1, 1024), (1 << 21, 1024), ((1 << 24) - 2, 128)])
def test_rows_past_32_bits_are_refused(launches, tokens, qpk) -> None:
    """Rows are numbered in 32 bits, the last tile's places behind them too."""
    from kvcompress_mi355x import _native

    lib = _native.load()
    assert tokens * qpk >= (1 << 31) - 256
    assert lib.kvc_attend_workspace_bytes(1, qpk, 8, 1, tokens, tokens, 512) == 0
    assert _attend_c(lib, kv=1, qpk=qpk, dim=8, page=128 * 8, tokens=tokens, longest=tokens, qt=8 * qpk, qh=8, ot=8 * qpk, oh=8) == _native.EINVAL
    assert "num_tokens * qpk" in lib.kvc_last_error().decode()
    with pytest.raises(ValueError, match="below 2\\^31"):
        _serving().attend_workspace_bytes(qpk, 1, 8, 1, tokens, tokens, 512)
    assert lib.kvc_attend_workspace_bytes(1, 64, 8, 1, (1 << 24) - 1, (1 << 24) - 1, 512) > 0


def test_launches_past_32_bits_of_work_items_are_refused() -> None:
    from kvcompress_mi355x import _native

    lib, fake, most = _native.load(), 4096, (1 << 24) - 1
    # 2^19 row tiles x 1024 KV heads x 512 threads.
    assert _attend_c(lib, kv=1024, qpk=8, dim=8, page=128 * 1024 * 8, tokens=most, longest=most, qt=8 * 8192, qh=8, ot=8 * 8192, oh=8) == _native.EINVAL
    assert "too many rows" in lib.kvc_last_error().decode()
    assert lib.kvc_step_tables(None, most, fake, fake, None, fake, fake, 128, 1, 5, 4, 8, fake, fake, fake, fake, fake) == _native.EINVAL
    assert "bad sizes" in lib.kvc_last_error().decode()


# Two tokens of two heads of 128 elements, 2 bytes each: rows of 256 bytes, at 0, 256, 512 and 768.
@pytest.mark.parametrize("change, message", [
    ({}, "out overlaps q"),
    ({"out": 4096 + 752}, "out overlaps q"),
    ({"out": 4096 - 1008}, "out overlaps q"),
    ({"qt": 512, "ot": 512, "out": 4096 + 256}, "out overlaps q"),  # the second head's rows are the first one's
    ({"qt": 384, "ot": 384, "out": 4096 + 512 + 128}, "out overlaps q"),  # a token's rows end in the next one's
    ({"ot": 512, "out": 4096 + 512}, "out overlaps q"),  # other strides in one range
    ({"out": 8192, "oh": 0}, "rows of out"),
    ({"out": 8192, "ot": 0}, "rows of out"),
    ({"out": 8192, "oh": 120}, "rows of out"),
    ({"out": 8192, "ot": 128, "oh": 128}, "rows of out"),  # the second token's first row is the first one's second
    ({"out": 8192, "ot": 200, "oh": 128}, "rows of out"),
])
def test_attend_refuses_outputs_that_overlap(change, message) -> None:
    from kvcompress_mi355x import _native

    lib = _native.load()
    assert _attend_c(lib, **{"tokens": 2, "longest": 2, **change}) == _native.EINVAL
    assert message in lib.kvc_last_error().decode()


@pytest.mark.parametrize("change, message", [
    ({"out": 4096 + 16}, "without being q"),
    ({"ot": 512}, "without being q"),
    ({"out": (1 << 20) + 3 * 256}, "overlaps k or v"),
    ({"out": (2 << 20) - 256}, "overlaps k or v"),
    ({"out": 8 << 20, "oh": 0}, "rows of q_out"),
    ({"out": 8 << 20, "ot": 64}, "rows of q_out"),
])
def test_rotary_refuses_outputs_that_overlap(change, message) -> None:
    import ctypes

    from kvcompress_mi355x import _native

    lib, fake = _native.load(), 4096
    a = {"out": fake, "ot": 256, "oh": 128, **change}
    rc = lib.kvc_rotate_and_store(
        None, 0, 0, 3, 2, 2, 128, 128, fake, 256, 128, 1 << 20, 256, 128, 2 << 20, 256, 128, fake, 0, 1, (ctypes.c_int * 1)(64), 0, fake, fake,
        a["out"], a["ot"], a["oh"], fake, fake, 4, 128 * 2 * 128)
    assert rc == _native.EINVAL and message in lib.kvc_last_error().decode()


def test_entries_without_work_return_before_any_launch() -> None:
    from kvcompress_mi355x import _native

    lib = _native.load()
    assert _attend_c(lib, n=0, start=None) == 0
    assert _attend_c(lib, tokens=0, q=None) == 0
    assert lib.kvc_attend_workspace_bytes(8, 5, 128, 16, 16, 1, 16384) > 0
    assert lib.kvc_attend_workspace_bytes(8, 5, 130, 16, 16, 1, 16384) == 0
    assert lib.kvc_attend_workspace_bytes(0, 5, 128, 16, 16, 1, 16384) == 0


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("heads, kv", [(8, 1), (16, 8), (32, 1), (64, 8), (40, 1)])
def test_workspace_of_the_largest_step_serves_smaller_ones(dim, heads, kv) -> None:
    """No size needs less than a smaller one: a step of single tokens, of drafts, of
    chunks, short requests and long ones, apart and in one launch."""
    bytes_of = _serving().attend_workspace_bytes
    sizes = [(n, n * new, new, longest) for n in (0, 1, 7, 64, 2000) for new in (0, 1, 2, 4, 5, 40, 700)
             for longest in (0, 1, 128, 896, 1024, 5000, 65536)]
    need = {s: bytes_of(heads, kv, dim, *s) for s in sizes}
    for large, most in need.items():
        assert all(least <= most for small, least in need.items() if all(a <= b for a, b in zip(small, large))), large


@pytest.mark.parametrize("change, message", [
    ({"dtype": 2}, "dtype"), ({"style": 2}, "rope style"), ({"rotary": 130}, "rotary_dim"), ({"rotary": 63}, "rotary_dim"),
    ({"axes": 5}, "axes"), ({"axes": 0}, "axes"), ({"sections": (60, 5, 0, 0)}, "add up"), ({"sections": (70, -6, 0, 0)}, "section"),
    ({"page": 100}, "page_stride"), ({"kv": 0}, "bad sizes"), ({"q": None}, "null pointer"), ({"omega": None}, "null pointer"),
])
def test_rotary_entry_refusals(change, message) -> None:
    import ctypes

    from kvcompress_mi355x import _native

    lib, fake = _native.load(), 4096
    a = dict(dtype=0, style=0, tokens=1, heads=2, kv=2, dim=128, rotary=128, q=fake, k=fake, v=fake, axes=2, sections=(60, 4, 0, 0), omega=fake,
             page=128 * 2 * 128)
    a.update(change)
    rc = lib.kvc_rotate_and_store(
        None, a["dtype"], a["style"], a["tokens"], a["heads"], a["kv"], a["dim"], a["rotary"], a["q"], 256, 128, a["k"], 256, 128, a["v"], 256,
        128, fake, 1, a["axes"], (ctypes.c_int * 4)(*a["sections"]), 0, a["omega"], fake, fake, 256, 128, fake, fake, 4, a["page"])
    assert rc == _native.EINVAL and message in lib.kvc_last_error().decode()


@pytest.mark.parametrize("change, message", [
    ({"n": -1}, "bad sizes"), ({"page": 100}, "page_tokens"), ({"page": 0}, "page_tokens"), ({"blocks": 9}, "max_blocks"),
    ({"start": None}, "null pointer"), ({"lens": None}, "null pointer"), ({"positions": None}, "null pointer"),
])
def test_step_tables_entry_refusals(change, message) -> None:
    from kvcompress_mi355x import _native

    lib, fake = _native.load(), 4096
    a = dict(n=2, page=128, blocks=4, start=fake, lens=fake, positions=fake)
    a.update(change)
    rc = lib.kvc_step_tables(None, a["n"], fake, fake, None, fake, fake, a["page"], 1, 5, a["blocks"], 8, a["start"], a["lens"], a["positions"],
                             fake, fake)
    assert rc == _native.EINVAL and message in lib.kvc_last_error().decode()


def test_rotary_refuses_one_pool_for_keys_and_values() -> None:
    import ctypes

    from kvcompress_mi355x import _native

    lib, fake = _native.load(), 4096
    rc = lib.kvc_rotate_and_store(
        None, 0, 0, 3, 2, 2, 128, 128, fake, 256, 128, 1 << 20, 256, 128, 2 << 20, 256, 128, fake, 0, 1, (ctypes.c_int * 1)(64), 0, fake, fake,
        fake, 256, 128, 1 << 24, 1 << 24, 4, 128 * 2 * 128)
    assert rc == _native.EINVAL and "one pool" in lib.kvc_last_error().decode()


# Tables of 3 requests and 5 tokens, 4096 bytes apart; 4 blocks of a row of 8.
@pytest.mark.parametrize("change, message", [
    ({"lens": 1}, "inputs and outputs"),  # lengths written over the computed tokens
    ({"start": 2}, "inputs and outputs"),
    ({"start": 2 - 3 / 1024}, "inputs and outputs"),  # its last entry is the first new token count
    ({"slots": 3}, "inputs and outputs"),
    ({"positions": 5 + 24 / 4096}, "inputs and outputs"),
    ({"table": 1 - 64 / 4096}, "inputs and outputs"),  # its third row
    ({"positions": 9}, "outputs overlap"),
    ({"lens": 6 + 12 / 4096}, "outputs overlap"),
    ({"table": 7 - 32 / 4096}, "outputs overlap"),  # its second row
    ({"lens": 10 + 76 / 4096}, "outputs overlap"),
    ({"lens": 10 + 8 / 4096}, "outputs overlap"),
    ({"lens": 10 + 24 / 4096}, "outputs overlap"),  # two entries in the gap behind the first row (bytes 16 to 32), one in the second
])
def test_step_tables_refuse_tensors_that_overlap(change, message) -> None:
    from kvcompress_mi355x import _native

    lib = _native.load()
    at = dict(computed=1, new=2, offsets=3, ids=4, id_offsets=5, start=6, lens=7, positions=8, slots=9, table=10)
    a = {name: int(4096 * place) for name, place in {**at, **change}.items()}
    rc = lib.kvc_step_tables(None, 3, a["computed"], a["new"], a["offsets"], a["ids"], a["id_offsets"], 128, 1, 5, 4, 8, a["start"], a["lens"],
                             a["positions"], a["slots"], a["table"])
    assert rc == _native.EINVAL and message in lib.kvc_last_error().decode()


# ------------------------------------------------------- definitions by hand --


def test_definition_of_tables() -> None:
    start, lens, positions, slots, table = ref.step_tables([254, 4], [4, 1], [0, 4], [[7, 2, 9], [5]], 128, 6, 3)
    assert start == [0, 4, 5] and lens == [258, 1]
    assert positions == [254, 255, 256, 257, 4, 0]
    assert slots == [2 * 128 + 126, 2 * 128 + 127, 9 * 128, 9 * 128 + 1, 5 * 128, -1]
    assert table == [[7, 2, 9], [5, -1, -1]]
    assert ref.step_tables([200], [1], [0], [[3]], 256, 1, 4)[4] == [[6, 7, -1, -1]]


def test_definition_of_axes_and_rotation() -> None:
    assert ref.axis_of_frequency(6, (3, 1, 2), "blocked") == [0, 0, 0, 1, 2, 2]
    assert ref.axis_of_frequency(8, (4, 2, 2), "cycled") == [0, 1, 2, 0, 1, 2, 0, 0]
    x = torch.tensor([[[1.0, 0.0, 5.0]]])
    turned = ref.rotate(x, torch.tensor([[1]]), torch.tensor([math.pi / 2]), (1,), "half", "half")
    assert torch.allclose(turned, torch.tensor([[[0.0, 1.0, 5.0]]], dtype=torch.float64), atol=1e-7)


def test_definition_of_attention() -> None:
    k = torch.zeros(1, 128, 1, 8)
    v = torch.zeros(1, 128, 1, 8)
    v[0, :, 0, 0] = torch.arange(128.0)
    q = torch.zeros(3, 1, 8)
    table = torch.zeros(1, 1, dtype=torch.int32)
    see = lambda n, **kw: ref.attend(q, k, v, [0, 3], [n], table, scale=1.0, **kw)[0][:, 0, 0].tolist()  # noqa: E731
    assert see(10) == pytest.approx([3.5, 4.0, 4.5])  # means of 0..7, 0..8, 0..9
    assert see(10, window=2) == pytest.approx([6.5, 7.5, 8.5])
    assert see(10, window=2, sinks=1) == pytest.approx([13 / 3, 15 / 3, 17 / 3])
    assert see(2) == pytest.approx([0.0, 0.0, 0.5])  # the first token is before the cache: it sees nothing

"""The 4-bit K/V cache without a GPU: the number format's oracle, and every refusal of the C entry points and of the Python
object (all of them are decided on the host before anything is launched)."""
import math

import pytest
import torch

from fish_speech_amd import _lib, kv4
from fish_speech_amd._lib import FishmiError
from oracle import kv4 as O

A = 1 << 20   # an aligned address that is never dereferenced: every call below is refused first


def test_representable_values_are_kept_and_ties_go_to_even_codes():
    for e in (-100, -7, 0, 3, 100):
        vals = torch.cat([O.GRID, -O.GRID, O.GRID, -O.GRID]) * 2.0 ** e
        assert torch.equal(O.stored(vals), vals)
    # borders between neighbours, next to a 6 that fixes the power
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0] + [6.0] * 25, dtype=torch.float64)
    assert O.stored(border)[:7].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]


def test_block_power_is_the_smallest_that_holds_the_largest_value():
    for top, e in ((7.0, 0), (7.03125, 1), (3.5, -1), (3.515625, 0), (6.0, 0), (2.0 ** -90, -92), (2.0 ** -120, -100), (0.0, -100)):
        y = torch.zeros(32, dtype=torch.float64)
        y[5] = top
        assert int(O.quantise(y)[1]) == e + 127, (top, e)


def test_error_is_at_most_half_a_step():
    g = torch.Generator().manual_seed(0)
    y = torch.randn(400, 64, generator=g, dtype=torch.float64)
    code, scale = O.quantise(y)
    unit = torch.ldexp(torch.ones(400, 2, dtype=torch.float64), scale.long() - 127).repeat_interleave(32, 1)
    a = y.abs() / unit
    half = torch.where(a <= 2, 0.25, torch.where(a <= 4, 0.5, 1.0))
    assert bool(((O.stored(y) - y).abs() <= half * unit).all())


def test_nonfinite_blocks_read_as_nan_and_leave_their_neighbours():
    y = torch.ones(1, 96)
    y[0, 40] = math.inf
    y[0, 70] = math.nan
    s = O.stored(y)
    assert s[0, :32].eq(1).all() and s[0, 32:].isnan().all()


# ------------------------------------------------------------------------------------------------ refusals: C ABI


def _pack(layout, fields, kw):
    """The fields in the order of include/fishmi.h -> the packed struct."""
    assert set(kw) <= set(fields)
    return layout.pack(*[v or 0 for v in dict(fields, **kw).values()])


def test_packed_structs_match_the_header():
    """Field types and order of the three structs in include/fishmi.h, and their sizes as the C compiler lays them out."""
    import os
    import re

    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "fishmi.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    kinds = {"int32_t": "i", "int64_t": "q", "float": "f", "double": "d"}
    for name, layout in (("fmi_kv4_cache", kv4._CACHE), ("fmi_kv4_rows", kv4._ROWS), ("fmi_kv4_query", kv4._QUERY)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, src, flags=re.S).group(1)
        fmt = "@"
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            base = re.sub(r"^const\s+", "", decl).split()[0].rstrip("*")
            for var in re.sub(r"^(const\s+)?\w+", "", decl).split(","):
                fmt += "P" if "*" in var else kinds[base]
        assert fmt == layout.format, name


def _cache(**kw):
    d = dict(pool_dev=A, block_table_dev=A, n_pages=4, n_kv_head=2, head_dim=64, n_seqs=3, max_pages=5)
    return _pack(kv4._CACHE, d, kw)


def _rows(**kw):
    d = dict(q_dev=A, k_dev=A, v_dev=A, q_stride=256, k_stride=128, v_stride=128, q_out_dev=A, q_out_stride=256, n_head=4,
             q_norm_dev=None, k_norm_dev=None, norm_eps=1e-6, rope_dev=A, rope_len=10, rope_dim=64, rope_half=0,
             row_seq_dev=A, row_pos_dev=A, rows=7)
    return _pack(kv4._ROWS, d, kw)


def _query(**kw):
    d = dict(q_dev=A, q_stride=256, n_head=4, q_start_dev=A, kv_len_dev=A, n_seqs=3, total_q=5, max_q=2, max_kv=100,
             scale=0.1, splits=1)
    return _pack(kv4._QUERY, d, kw)


BAD_CACHES = [dict(pool_dev=None), dict(pool_dev=A + 8), dict(block_table_dev=None), dict(block_table_dev=A + 2), dict(head_dim=48),
              dict(head_dim=256), dict(n_pages=0), dict(n_kv_head=0), dict(n_kv_head=-1), dict(n_seqs=0), dict(max_pages=0),
              dict(max_pages=(1 << 24) + 1)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_every_entry_point_refuses_a_bad_cache(bad):
    lib = _lib.load()
    c = _cache(**bad)
    assert lib.fmi_op_kv4_append(c, _rows(), None) == -1
    assert lib.fmi_op_kv4_read(c, A, A, 3, A, A, None) == -1
    assert lib.fmi_op_kv4_attention(c, _query(), A, 256, None, 0, None) == -1
    assert lib.fmi_op_kv4_step(c, _rows(q_out_dev=None), 0.1, 100, 1, A, 256, None, 0, None) == -1
    assert b"kv4" in lib.fmi_last_error()


@pytest.mark.parametrize("bad", [
    dict(k_dev=None), dict(v_dev=None), dict(k_dev=A + 2), dict(v_stride=120), dict(v_stride=132), dict(k_stride=64),
    dict(q_out_dev=None), dict(q_out_dev=A + 4), dict(q_stride=128), dict(q_out_stride=250), dict(n_head=0), dict(n_head=-4),
    dict(row_seq_dev=None), dict(row_pos_dev=None), dict(rows=-1), dict(rope_dim=0), dict(rope_dim=8), dict(rope_dim=24),
    dict(rope_dim=80), dict(rope_len=0), dict(rope_dev=A + 4), dict(q_norm_dev=A + 2), dict(k_norm_dev=A + 8),
    dict(q_dev=None, q_norm_dev=A), dict(rope_half=1), dict(q_out_stride=264)], ids=str)    # (q_out is q itself here)
def test_append_refusals(bad):
    assert _lib.load().fmi_op_kv4_append(_cache(), _rows(**bad), None) == -1


@pytest.mark.parametrize("bad", [
    dict(q_dev=None), dict(q_dev=A + 8), dict(q_stride=252), dict(q_stride=192), dict(n_head=0), dict(n_head=3), dict(q_start_dev=None),
    dict(kv_len_dev=None), dict(n_seqs=-1), dict(n_seqs=4), dict(n_seqs=65536), dict(total_q=-1), dict(max_q=-1), dict(max_kv=-1),
    dict(scale=math.inf), dict(scale=-math.inf), dict(scale=math.nan), dict(splits=-1), dict(splits=257), dict(max_q=1 << 30), dict(max_q=1 << 26, splits=3)], ids=str)
def test_attention_refusals(bad):
    lib = _lib.load()
    c, q = _cache(), _query(**bad)
    assert lib.fmi_op_kv4_attention(c, q, A, 256, A, 1 << 30, None) == -1


def test_attention_refuses_a_missing_or_small_workspace_and_bad_outputs():
    lib = _lib.load()
    c, q = _cache(), _query(splits=3)
    need = lib.fmi_kv4_attention_ws_bytes(c, q)
    assert need >= 3 * 5 * 4 * 64 * 4
    assert lib.fmi_op_kv4_attention(c, q, A, 256, A, need - 1, None) == -1
    assert lib.fmi_op_kv4_attention(c, q, A, 256, None, need, None) == -1
    assert lib.fmi_op_kv4_attention(c, q, A, 256, A + 4, need, None) == -1
    assert lib.fmi_op_kv4_attention(c, q, None, 256, A, need, None) == -1
    assert lib.fmi_op_kv4_attention(c, q, A, 192, A, need, None) == -1
    assert lib.fmi_kv4_attention_ws_bytes(c, _query(splits=1)) == 0


@pytest.mark.parametrize("bad", [
    dict(k_dev=None), dict(v_dev=A + 2), dict(k_stride=64), dict(q_dev=None), dict(q_dev=A + 8), dict(q_stride=128), dict(q_out_dev=A),
    dict(n_head=0), dict(n_head=3), dict(row_seq_dev=None), dict(row_pos_dev=None), dict(rows=-1), dict(rows=65536), dict(rope_dim=8),
    dict(rope_len=0), dict(rope_dev=A + 4), dict(q_norm_dev=A + 2), dict(k_norm_dev=A + 8)], ids=str)
def test_step_refuses_bad_rows(bad):
    rows = _rows(**{**dict(q_out_dev=None), **bad})
    assert _lib.load().fmi_op_kv4_step(_cache(), rows, 0.1, 100, 1, A, 256, None, 0, None) == -1


def test_step_refuses_bad_outputs_scales_and_workspaces():
    lib = _lib.load()
    c, rows = _cache(), _rows(q_out_dev=None)
    ok = dict(scale=0.1, max_kv=100, splits=1, out=A, stride=256, ws=None, ws_bytes=0)
    need = lib.fmi_kv4_attention_ws_bytes(c, _query(n_seqs=7, total_q=7, max_q=1, splits=3))
    assert need > 0
    for bad in (dict(out=None), dict(out=A + 4), dict(stride=192), dict(stride=252), dict(scale=math.nan), dict(scale=math.inf),
                dict(max_kv=-1), dict(splits=-1), dict(splits=257), dict(splits=3, ws=A, ws_bytes=need - 1),
                dict(splits=3, ws=None, ws_bytes=need), dict(splits=3, ws=A + 4, ws_bytes=need)):
        a = {**ok, **bad}
        assert lib.fmi_op_kv4_step(c, rows, a["scale"], a["max_kv"], a["splits"], a["out"], a["stride"], a["ws"], a["ws_bytes"],
                                   None) == -1, bad
    assert lib.fmi_op_kv4_step(None, rows, 0.1, 100, 1, A, 256, None, 0, None) == -1
    assert lib.fmi_op_kv4_step(c, None, 0.1, 100, 1, A, 256, None, 0, None) == -1
    assert lib.fmi_op_kv4_step(c, _rows(q_out_dev=None, rows=0), 0.1, 100, 1, A, 256, None, 0, None) == 0


def test_null_arguments_and_empty_calls():
    lib = _lib.load()
    assert lib.fmi_op_kv4_append(None, _rows(), None) == -1
    assert lib.fmi_op_kv4_append(_cache(), None, None) == -1
    assert lib.fmi_op_kv4_read(None, A, A, 3, A, A, None) == -1
    assert lib.fmi_op_kv4_read(_cache(), None, A, 3, A, A, None) == -1
    assert lib.fmi_op_kv4_read(_cache(), A, A, -3, A, A, None) == -1
    assert lib.fmi_op_kv4_read(_cache(), A, A, 3, A + 2, A, None) == -1
    assert lib.fmi_op_kv4_attention(None, _query(), A, 256, None, 0, None) == -1
    # nothing to do: fine, and nothing is launched
    assert lib.fmi_op_kv4_append(_cache(), _rows(rows=0), None) == 0
    assert lib.fmi_op_kv4_read(_cache(), None, None, 0, None, None, None) == 0
    assert lib.fmi_op_kv4_attention(_cache(), _query(total_q=0), A, 256, None, 0, None) == 0
    none = _cache(n_seqs=0, block_table_dev=None)
    for c in (_cache(), none):
        assert lib.fmi_op_kv4_attention(c, _query(n_seqs=0, q_start_dev=None, kv_len_dev=None), A, 256, None, 0, None) == 0
    assert lib.fmi_op_kv4_append(none, _rows(rows=0), None) == 0
    assert lib.fmi_op_kv4_read(none, None, None, 0, None, None, None) == 0


def test_page_bytes():
    assert kv4.page_bytes(8, 128) == 8 * 2 * 64 * (64 + 4)
    assert kv4.page_bytes(2, 32) == 2 * 2 * 64 * (16 + 1)
    for heads, dim in ((0, 128), (8, 96), (-1, 64)):
        with pytest.raises(FishmiError):
            kv4.page_bytes(heads, dim)


# ------------------------------------------------------------------------------------------------ refusals: Python


def test_cache_needs_a_gpu():
    with pytest.raises(FishmiError, match="GPU"):
        kv4.KV4Cache(4, 2, 64, device="cpu")


@pytest.fixture
def cache():
    """A cache object whose tensors live on the CPU: good enough for checks that end before any launch."""
    c = kv4.KV4Cache.__new__(kv4.KV4Cache)
    c._setup(torch.zeros(4, 2, 2, 64 * 34, dtype=torch.uint8), 64)
    return c


def _call(cache, what, **kw):
    i32, bf = torch.int32, torch.bfloat16
    a = dict(k=torch.zeros(3, 2, 64, dtype=bf), v=torch.zeros(3, 2, 64, dtype=bf), row_seq=torch.zeros(3, dtype=i32),
             row_pos=torch.zeros(3, dtype=i32), block_table=torch.zeros(2, 3, dtype=i32))
    if what == "attend":
        a = dict(q=torch.zeros(3, 4, 64, dtype=bf), q_start=torch.zeros(3, dtype=i32), kv_len=torch.zeros(2, dtype=i32),
                 block_table=torch.zeros(2, 3, dtype=i32), max_q=3, max_kv=10)
    if what == "step":
        a.update(q=torch.zeros(3, 4, 64, dtype=bf), max_kv=10)
    if what == "read":
        a = {k: a[k] for k in ("row_seq", "row_pos", "block_table")}
    a.update(kw)
    return getattr(cache, what)(**a)


BF = torch.bfloat16


@pytest.mark.parametrize("what, kw", [
    ("append", dict(k=torch.zeros(3, 2, 64))), ("append", dict(k=torch.zeros(3, 3, 64, dtype=BF))),
    ("append", dict(v=torch.zeros(2, 2, 64, dtype=BF))), ("append", dict(v=torch.zeros(3, 2, 32, dtype=BF))),
    ("append", dict(k=torch.zeros(3, 64, 2, dtype=BF).transpose(1, 2))), ("append", dict(row_seq=torch.zeros(3))),
    ("append", dict(row_pos=torch.zeros(4, dtype=torch.int32))), ("append", dict(row_pos=torch.zeros(6, dtype=torch.int32)[::2])),
    ("append", dict(block_table=torch.zeros(3, dtype=torch.int32))),
    ("append", dict(block_table=torch.zeros(3, 2, dtype=torch.int32).t())),
    ("append", dict(rope=torch.zeros(9, 32, 2))), ("append", dict(rope=torch.zeros(9, 64, dtype=BF))),
    ("append", dict(rope=torch.zeros(9, 32, 2, dtype=BF), rope_layout="other")),
    ("append", dict(k_norm=torch.zeros(32, dtype=BF))), ("append", dict(q_norm=torch.zeros(64, dtype=BF))),
    ("append", dict(q_out=torch.zeros(3, 4, 64, dtype=BF))),
    ("append", dict(q=torch.zeros(3, 4, 64, dtype=BF), q_out=torch.zeros(3, 5, 64, dtype=BF))),
    ("attend", dict(q=torch.zeros(3, 4, 64))), ("attend", dict(q_start=torch.zeros(2, dtype=torch.int32))),
    ("attend", dict(kv_len=torch.zeros(3, dtype=torch.int32))), ("attend", dict(kv_len=torch.zeros(2, dtype=torch.int64))),
    ("attend", dict(out=torch.zeros(2, 4, 64, dtype=BF))),
    ("step", dict(q=torch.zeros(3, 4, 64))), ("step", dict(q=torch.zeros(2, 4, 64, dtype=BF))), ("step", dict(k=torch.zeros(3, 3, 64, dtype=BF))),
    ("step", dict(row_seq=torch.zeros(2, dtype=torch.int32))), ("step", dict(row_pos=torch.zeros(3))), ("step", dict(rope_layout="x")),
    ("step", dict(rope=torch.zeros(9, 64, dtype=BF))), ("step", dict(k_norm=torch.zeros(32, dtype=BF))),
    ("step", dict(out=torch.zeros(3, 5, 64, dtype=BF))), ("step", dict(block_table=torch.zeros(3, dtype=torch.int32))),
    ("read", dict(row_seq=torch.zeros(2, dtype=torch.int32))), ("read", dict(row_pos=torch.zeros(3, 1, dtype=torch.int32))),
])
def test_python_argument_errors(cache, what, kw):
    with pytest.raises(ValueError):
        _call(cache, what, **kw)


# ------------------------------------------------------------------------------------------------ the model's setup


class _Handle:
    """The library's part of MiDualAR.setup_caches: caches of at most 1024 positions."""

    def __init__(self):
        self.bits, self.calls = 16, []

    def fmi_dualar_set_kv_bits(self, h, bits):
        self.bits = bits
        return 0

    def fmi_dualar_setup_caches(self, h, max_batch, max_seq_len):
        self.calls.append((self.bits, max_batch, max_seq_len))
        return -1 if max_seq_len > 1024 else 0


def test_a_refused_setup_does_not_choose_the_caches_type():
    from fish_speech_amd.dual_ar import MiDualAR

    m = MiDualAR.__new__(MiDualAR)
    m.lib, m._h = _Handle(), None
    m._cache_setup_done, m.max_batch_size, m.max_seq_len, m.kv_bits = False, -1, -1, 16
    with pytest.raises(FishmiError):
        m.setup_caches(1, 2048, kv_bits=4)
    assert m.kv_bits == 16 and not m._cache_setup_done
    m.setup_caches(1, 512)
    assert m.kv_bits == 16 and m.lib.calls == [(4, 1, 2048), (16, 1, 512)]
    m.setup_caches(1, 256, kv_bits=16)
    with pytest.raises(FishmiError, match="already set up"):
        m.setup_caches(1, 256, kv_bits=4)


@pytest.mark.parametrize("what, kw", [
    ("attend", dict(max_q=1 << 31)), ("attend", dict(max_kv=1 << 40)), ("attend", dict(max_q=2.0)), ("attend", dict(max_kv=None)),
    ("attend", dict(max_q=torch.tensor(3.0))), ("attend", dict(splits=1 << 31)), ("attend", dict(splits="2")), ("attend", dict(scale="x")),
    ("attend", dict(scale=1e50)), ("step", dict(max_kv=1 << 31)), ("step", dict(splits=2.5)), ("step", dict(scale=torch.ones(2))),
    ("step", dict(scale=-1e39)), ("step", dict(eps="x")), ("append", dict(eps=None))], ids=str)
def test_numbers_that_are_none_or_out_of_range(cache, what, kw, monkeypatch):
    """A ValueError of the argument's name, not one of the packing's; outputs are not what is refused here."""
    monkeypatch.setattr(cache, "_new", lambda rows, heads: torch.zeros(rows, heads, 64, dtype=BF), raising=False)
    with pytest.raises(ValueError, match=next(iter(kw))):
        _call(cache, what, **kw)


def test_numbers_held_in_tensors_are_taken_by_value(cache, monkeypatch):
    """A one-element tensor counts as the number it holds at the call; no size is remembered by a tensor's identity."""
    monkeypatch.setattr(cache, "_new", lambda rows, heads: torch.zeros(rows, heads, 64, dtype=BF), raising=False)
    sizes = []
    real = kv4._attention_ws_bytes
    monkeypatch.setattr(kv4, "_attention_ws_bytes", lambda *a: sizes.append(a) or real(*a) and 0)
    calls = []
    monkeypatch.setattr(cache, "_call", lambda fn, *a: calls.append(a), raising=False)
    n = torch.tensor(3)
    _call(cache, "attend", max_q=n, max_kv=torch.tensor(2000), splits=torch.tensor(2), scale=torch.tensor(0.5))
    n += 1
    _call(cache, "attend", max_q=n, max_kv=2000, splits=2)
    assert [a[5:] for a in sizes] == [(3, 2000, 2), (4, 2000, 2)] and all(type(x) is int for a in sizes for x in a)
    assert kv4._QUERY.unpack(calls[0][1])[7:] == (3, 2000, 0.5, 2)

"""The 4-bit K/V cache in the forms that only larger calls take: sequences split over key ranges (few and many query columns), and
the append and the read that hold eight heads per wave.  Each test asserts that its sizes reach the form."""
import math
import os
import re

import pytest
import torch

from oracle import kv4 as O
from tests.test_kv4_gpu import (append_then_attend, check_attention, cuda, make_cache, make_table, page_bytes_expected, randn,
                                rope_table, rows_of, same, setup_attention, setup_step)
from tests.test_kv4_ranges_gpu import reference, weight_bits, worst

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF = torch.bfloat16
I32 = torch.int32

_CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fish_speech_amd", "csrc")


def _source(name):
    with open(os.path.join(_CSRC, name)) as f:
        return f.read()


def key_ranges(keys, splits):
    """The ranges that the last row of `keys` keys is divided into (the constants are the kernels')."""
    single = int(re.search(r"KV4_SINGLE_PAGES = (\d+)", _source("kv4_kernels.h")).group(1))
    least = int(re.search(r"KV4_MIN_PAGES = (\d+)", _source("kv4.hip")).group(1))
    pages = (keys + 63) // 64
    return 1 if pages < single else max(1, min(splits, pages // least))


def many(what, values):
    """Whether a call of so many values takes the eight-heads kernel."""
    limit = int(re.search(r"launch_kv4_%s.*?many = .*? > \(int64_t\)1 << (\d+)" % what, _source("kv4.hip"), flags=re.S).group(1))
    return values > 1 << limit


SHAPES = [(128, 8, 2), (64, 14, 2), (32, 17, 1)]


# ------------------------------------------------------------------------------------------------ key ranges


def check_rows(got, q, kv, new, D):
    bits = weight_bits(max(new), q.shape[1] // kv[0][0].shape[1])
    r = 0
    for n, (k, v) in zip(new, kv):
        if n and k.shape[0]:
            ref, tol = reference(q[r:r + n], k, v, 1 / math.sqrt(D), bits)
            assert worst(got[r:r + n], ref, tol) <= 1
        else:
            assert got[r:r + n].eq(0).all()
        r += n


@pytest.mark.parametrize("D, H, KVH", SHAPES)
@pytest.mark.parametrize("splits", [0, 3, 20, 256])
def test_single_tokens_in_several_ranges(D, H, KVH, splits):
    keys = [704, 705, 768, 769, 1023, 1024, 1025, 1500, 2050, 0, 3]
    assert key_ranges(2050, splits or 2) > 1 and key_ranges(705, 2) > 1 and key_ranges(704, 256) == 1
    new = [1] * len(keys)
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, new, keys, seed=3, fill=0xFF)
    got = cache.attend(qd, start, kv_len, t, max_q=1, max_kv=max(keys), splits=splits)
    check_rows(got, q, kv, new, D)


@pytest.mark.parametrize("D, H, KVH", SHAPES)
@pytest.mark.parametrize("new, keys", [([70, 66, 68, 90], [1500, 705, 704, 90]), ([130, 1], [900, 2000]), ([40, 3], [1100, 769])], ids=str)
@pytest.mark.parametrize("splits", [0, 3, 20])
def test_chunks_in_several_ranges(D, H, KVH, new, keys, splits):
    assert key_ranges(max(keys), splits or 2) > 1
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, new, keys, seed=11, fill=0xFF)
    got = cache.attend(qd, start, kv_len, t, max_q=max(new), max_kv=max(keys), splits=splits)
    check_rows(got, q, kv, new, D)


@pytest.mark.parametrize("D, H, KVH", [(128, 8, 2), (64, 4, 2), (32, 4, 2)])
@pytest.mark.parametrize("n", [1, 16, 150])
@pytest.mark.parametrize("splits", [1, 3, 20])
def test_nan_values_inside_one_of_several_ranges(D, H, KVH, n, splits):
    """A NaN in the second of three ranges, seen by every row, and one at a key that only the later rows see."""
    keys, late = 1500, 1500 - (n + 1) // 2
    assert splits == 1 or key_ranges(keys, splits) >= 3
    G, q = H // KVH, randn(n, H, D, seed=3)
    for which in (0, 1):
        k, v = randn(keys, KVH, D, seed=1), randn(keys, KVH, D, seed=2)
        bad = (k, v)[which]
        bad[750, 1, D - 1] = math.nan
        bad[late, 0, 3] = math.inf
        table, n_pages = make_table([keys])
        cache = make_cache(n_pages, KVH, D, fill=0xFF)
        t, s, p, kd, vd, qd = cuda(table, *rows_of([keys]), k, v, q)
        cache.append(kd, vd, s, p, t)
        start, kv_len = torch.tensor([0, n], dtype=I32, device=DEV), torch.tensor([keys], dtype=I32, device=DEV)
        got = cache.attend(qd, start, kv_len, t, max_q=n, max_kv=keys, splits=splits).cpu()
        nan = torch.zeros(n, H, D, dtype=torch.bool)
        first = late - (keys - n)                                   # the first row that sees the late key
        if which == 0:
            nan[:, G:2 * G] = True
            nan[first:, :G] = True
        else:
            nan[:, G:2 * G, D - 32:] = True
            nan[first:, :G, :32] = True
        assert torch.equal(got.isnan(), nan)
        clean = torch.nan_to_num(O.stored(k), nan=0.0), torch.nan_to_num(O.stored(v), nan=0.0)
        ref, tol = reference(q, *clean, 1 / math.sqrt(D), weight_bits(n, G))
        assert bool(((got.double() - ref).abs() <= tol)[~nan].all())


@pytest.mark.parametrize("D, H, KVH", [(128, 8, 2), (64, 4, 2), (32, 4, 2)])
@pytest.mark.parametrize("n", [1, 2, 70])
@pytest.mark.parametrize("splits", [1, 3])
def test_missing_pages_and_a_range_without_any(D, H, KVH, n, splits):
    """24 pages in three ranges of 8: the second range has none of its pages; another sequence has a few holes, a third nothing."""
    keys, new = [1536, 1300, 800], [n, n, n]
    assert splits == 1 or (key_ranges(1536, splits), key_ranges(1300, splits), key_ranges(800, splits)) == (3, 3, 3)
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, new, keys, seed=21)
    t = t.clone()
    t[0, 8:16] = -1
    t[1, 0], t[1, 7], t[1, 20] = -1, cache.n_pages, 2 ** 31 - 1
    t[2] = -2 ** 31
    seen = [torch.ones(m, dtype=torch.bool) for m in keys]
    seen[0][512:1024] = False
    seen[1][:64] = seen[1][448:512] = seen[1][1280:] = False
    seen[2][:] = False
    got = cache.attend(qd, start, kv_len, t, max_q=n, max_kv=1536, splits=splits)
    check_attention(got, q, kv, new, D, seen=seen)
    assert got[2 * n:].eq(0).all()


@pytest.mark.parametrize("H, n, max_q", [(4, 5, 2), (8, 90, 40)])
def test_rows_beyond_max_q_in_several_ranges(H, n, max_q):
    D, KVH, keys = 64, 2, [1300]
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, [n], keys, seed=13)
    for splits in (1, 3):
        assert splits == 1 or key_ranges(1300 - n + 1, splits) == 3
        out = torch.full((n + 2, H + 1, D), 3.0, dtype=BF, device=DEV)
        wide = torch.cat([qd, qd[:2]])
        cache.attend(wide, start, kv_len, t, max_q=max_q, max_kv=1300, out=out[:, :H], splits=splits)
        have = keys[0] - n + max_q
        check_attention(out[:max_q, :H], q[:max_q], [(kv[0][0][:have], kv[0][1][:have])], [max_q], D)
        assert out[max_q:].eq(3).all() and out[:, H].eq(3).all()


@pytest.mark.parametrize("n", [1, 16, 80])
def test_rows_in_several_ranges_do_not_depend_on_their_batch(n):
    """With fixed splits and max_q, alone or with others, also where the others are longer or do not exist."""
    D, H, KVH = 128, 8, 2
    keys, new = [1400, 90, 2100, 800], [n, n, n, n]
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, new, keys, seed=4)
    whole = cache.attend(qd, start, kv_len, t, max_q=n, max_kv=2100, splits=3)
    for i in range(4):
        one = cache.attend(qd[i * n:(i + 1) * n], torch.tensor([0, n], dtype=I32, device=DEV), kv_len[i:i + 1], t[i:i + 1].contiguous(),
                           max_q=n, max_kv=keys[i], splits=3)
        assert torch.equal(one, whole[i * n:(i + 1) * n])


@pytest.mark.parametrize("n", [1, 40])
def test_an_output_over_its_queries(n):
    """`out` may be q itself: every work-group reads its own rows before they are written."""
    D, H, KVH = 64, 8, 2
    keys, new = [1400, 200], [n, n]
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, new, keys, seed=5)
    for splits in (1, 3):
        want = cache.attend(qd, start, kv_len, t, max_q=n, max_kv=1400, splits=splits)
        over = qd.clone()
        assert cache.attend(over, start, kv_len, t, max_q=n, max_kv=1400, splits=splits, out=over) is over
        assert torch.equal(over, want)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("splits", [1, 3])
def test_a_steps_output_over_its_queries(half, splits):
    D, H, KVH, at = 64, 40, 1, [1300, 30]                          # 40 heads per kv head: three tiles
    cache, t, qkv, rope, wq, wk, _, _ = setup_step(D, H, KVH, at, D, True, seed=5)
    d, s, p, r, dq, dk = cuda(qkv, torch.arange(2, dtype=I32), torch.tensor(at, dtype=I32), rope, wq, wk)
    q, k, v = d.split([H, KVH, KVH], dim=1)
    kw = dict(max_kv=1301, rope=r, rope_layout="half" if half else "interleaved", q_norm=dq, k_norm=dk, splits=splits)
    want = cache.step(q, k, v, s, p, t, **kw)
    assert cache.step(q, k, v, s, p, t, out=q, **kw) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("n", [1, 40])
def test_split_calls_on_two_streams_and_in_two_graphs(n):
    """Workspaces: two captured graphs of split calls replayed in turn and eager calls between them; two streams at once."""
    D, H, KVH = 128, 8, 2
    keys = [1500, 900]
    assert key_ranges(1500, 4) == 4 and key_ranges(900, 20) == 3
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, [n, n], keys, seed=6)

    def call(x, splits):
        return cache.attend(x, start, kv_len, t, max_q=n, max_kv=1500, splits=splits)

    want = call(qd, 4)
    check_rows(want, q, kv, [n, n], D)
    q2 = randn(2 * n, H, D, seed=99).to(DEV)
    want2 = call(q2, 20)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, (x, splits) in enumerate(((qd, 4), (q2, 20))):
            with torch.cuda.stream(streams[i]):
                outs[i].append(call(x, splits))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs[0]) and all(torch.equal(o, want2) for o in outs[1])

    qin = torch.zeros_like(qd)
    graphs = []
    for splits in (4, 20):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(qin, splits)
        graphs.append((g, out, splits))
    for rep in range(6):
        g, out, splits = graphs[rep % 2]
        kv_len.copy_(torch.tensor([1500 - 100 * rep, 900 - 30 * rep], dtype=I32))
        qin.copy_(randn(2 * n, H, D, seed=300 + rep))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(qin, splits)), rep
        cut = [(a[:int(m)], b[:int(m)]) for (a, b), m in zip(kv, kv_len)]
        check_rows(out, qin.cpu(), cut, [n, n], D)


@pytest.mark.parametrize("splits", [3, 20])
def test_a_split_steps_padding_rows_and_missing_pages(splits):
    D, H, KVH = 64, 8, 2
    at = [1300, 960, 1500, 5, 800]
    assert key_ranges(801, splits) > 1
    cache, t, qkv, rope, _, _, _, _ = setup_step(D, H, KVH, at, 64, False, seed=31)
    t = t.clone()
    t[1, 15] = -1                                                  # sequence 1: the new token's page
    t[2, 10:16] = cache.n_pages                                    # sequence 2: pages in the middle
    rows = [(3, 5), (-1, 5), (0, 1300), (5, 3), (2, 1500), (4, -1), (1, 960), (4, 800)]
    seq, pos = (torch.tensor([x[i] for x in rows], dtype=I32) for i in range(2))
    M = len(rows)
    d, s, p, r = cuda(randn(M, H + 2 * KVH, D, seed=33), seq, pos, rope)
    q, k, v = d.split([H, KVH, KVH], dim=1)
    real = [i for i, x in enumerate(rows) if 0 <= x[0] < 5 and x[1] >= 0]
    idx = torch.tensor(real, device=DEV)
    want, after = append_then_attend(cache, q[idx].contiguous(), k[idx].contiguous(), v[idx].contiguous(),
                                     torch.arange(len(real), dtype=I32, device=DEV), p[idx], t[s[idx].long()].contiguous(), 1501,
                                     splits, r, "interleaved", None, None)
    out = torch.full((M, H, D), 7.0, dtype=BF, device=DEV)
    cache.step(q, k, v, s, p, t, max_kv=1501, rope=r, eps=1e-5, splits=splits, out=out)
    assert torch.equal(out[idx], want) and torch.equal(cache.pool, after)
    assert out[[i for i in range(M) if i not in real]].eq(7.0).all()


# ------------------------------------------------------------------------------------------------ eight heads per wave


@pytest.mark.parametrize("D, H, KVH, rot, half, norm", [
    (128, 14, 2, 128, False, True), (128, 12, 4, 64, True, True), (128, 20, 5, 0, False, False), (128, 9, 9, 128, True, False),
    (64, 14, 2, 32, True, True), (64, 20, 5, 64, False, True), (64, 17, 17, 64, True, True), (32, 12, 4, 32, False, True),
    (32, 20, 5, 16, True, True), (32, 9, 3, 32, True, False), (64, 0, 24, 32, True, True)])
def test_large_appends_store_the_same_bytes_as_small_ones(D, H, KVH, rot, half, norm):
    """Bit for bit against calls of the one-head form over pieces of the rows, and against the definition on some of them."""
    M = (1 << 23) // ((H + 2 * KVH) * D) + 61
    piece = M // 3 + 1
    assert many("append", M * (H + 2 * KVH) * D) and not many("append", piece * (H + 2 * KVH) * D)
    lens = [M // 2 - 7, M - M // 2, 7]
    seq, pos = rows_of(lens)
    order = torch.randperm(M, generator=torch.Generator().manual_seed(D))
    seq, pos = seq[order].contiguous(), pos[order].contiguous()
    table, n_pages = make_table(lens, seed=H)
    table[1, 3] = -1                                               # a page that is not there
    seq[5::97] = -1                                                # padding in between
    qkv = randn(M, H + 2 * KVH, D, seed=1)
    qkv[:, H::2] *= 23.0
    qn, kn = (randn(D, seed=2) + 1, randn(D, seed=3) + 1) if norm else (None, None)
    rope = rope_table(max(lens), rot) if rot else None
    d, t, s, p, r, wq, wk = cuda(qkv, table, seq, pos, rope, qn if H else None, kn)
    layout = "half" if half else "interleaved"

    def run(cache, a, b, inplace=False):
        x = d[a:b].clone() if inplace else d[a:b]
        q, k, v = x.split([H, KVH, KVH], dim=1)
        kw = dict(q=q, q_norm=wq, q_out=q if inplace else torch.full((b - a, H, D), 9.0, dtype=BF, device=DEV)) if H else {}
        return cache.append(k, v, s[a:b], p[a:b], t, rope=r, rope_layout=layout, k_norm=wk, eps=1e-5, **kw)

    big, small = make_cache(n_pages, KVH, D, fill=0xA5), make_cache(n_pages, KVH, D, fill=0xA5)
    got = run(big, 0, M)
    parts = [run(small, a, min(M, a + piece)) for a in range(0, M, piece)]
    assert torch.equal(big.pool, small.pool)
    if H:
        assert torch.equal(got, torch.cat(parts))
        if not half:
            over = run(big, 0, M, inplace=True)
            there = (seq >= 0).to(DEV)
            assert torch.equal(over[there], got[there]) and torch.equal(big.pool, small.pool)
            assert torch.equal(over[~there], d[:, :H][~there])
    some = torch.arange(0, M, max(1, M // 50))
    cs = rope[pos[some].long()] if rot else None
    if H:
        want = O.rotate(O.head_norm(qkv[some, :H], qn, 1e-5), cs, half)
        pad = seq[some] < 0
        assert same(got[some.to(DEV)][~pad.to(DEV)], want[~pad]) and got[some.to(DEV)][pad.to(DEV)].eq(9).all()
    want_k, want_v = O.rotate(O.head_norm(qkv[some, H:H + KVH], kn, 1e-5), cs, half), qkv[some, H + KVH:]
    pool = big.pool.cpu()
    for j, i in enumerate(some.tolist()):
        page = int(table[seq[i], pos[i] // 64]) if seq[i] >= 0 else -1
        for h in range(KVH if page >= 0 else 0):
            for which, val in enumerate((want_k, want_v)):
                b, mask = page_bytes_expected(val[j:j + 1, h], pos[i:i + 1].long() % 64)
                assert torch.equal(pool[page, h, which] & mask, b & mask), (i, h, which)


@pytest.mark.parametrize("D, KVH", [(128, 8), (128, 5), (128, 1), (64, 5), (64, 2), (32, 3), (32, 8)])
def test_large_reads_return_what_small_ones_do(D, KVH):
    M = (1 << 21) // (KVH * D) + 37
    piece = M // 2 + 1
    assert many("read", M * KVH * D) and not many("read", piece * KVH * D)
    n = 400
    table, n_pages = make_table([n, 70], seed=D)
    k, v = randn(n + 70, KVH, D, seed=4), randn(n + 70, KVH, D, seed=5)
    v[:, -1] *= 1000.0
    k[17, 0, 1] = math.nan
    cache = make_cache(n_pages, KVH, D)
    t, s, p, kd, vd = cuda(table, *rows_of([n, 70]), k, v)
    cache.append(kd, vd, s, p, t)
    g = torch.Generator().manual_seed(1)
    pick = torch.randint(0, n + 70, (M,), generator=g)
    seq, pos = (x[pick].contiguous() for x in rows_of([n, 70]))
    gone = torch.arange(M) % 89 == 3
    seq[gone] = 2
    ds, dp = cuda(seq, pos)
    gk, gv = cache.read(ds, dp, t)
    parts = [cache.read(ds[a:a + piece], dp[a:a + piece], t) for a in range(0, M, piece)]
    bits = lambda x: x.view(torch.int16)
    assert torch.equal(bits(gk), bits(torch.cat([a for a, _ in parts]))) and torch.equal(bits(gv), bits(torch.cat([b for _, b in parts])))
    for got, val in ((gk, k), (gv, v)):
        want = O.stored(val)[pick].masked_fill(gone[:, None, None], 0.0)
        assert same(got, want)

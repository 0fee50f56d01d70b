"""The 4-bit paged K/V cache on the GPU against its 64-bit oracle (oracle/kv4.py): stored codes bit for bit, attention within
one bf16 rounding (half a step, 2^-8 of the value) plus the oracle's bound of the fp32 arithmetic."""
import math

import pytest
import torch

from oracle import kv4 as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF = torch.bfloat16
I32 = torch.int32


def make_cache(n_pages, kvh, D, fill=0):
    from fish_speech_amd.kv4 import KV4Cache

    c = KV4Cache(n_pages, kvh, D, device=DEV)
    c.pool.fill_(fill)
    return c


def make_table(lens, seed=0, extra=2, width=None):
    """Pages in no order; entries past a sequence's own pages are -1."""
    need = [(n + 63) // 64 for n in lens]
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(sum(need) + extra, generator=g)
    t = torch.full((len(lens), width or max(1, max(need))), -1, dtype=I32)
    o = 0
    for i, n in enumerate(need):
        t[i, :n] = perm[o:o + n].to(I32)
        o += n
    return t, sum(need) + extra


def rows_of(lens, start=None):
    seq = torch.cat([torch.full((n,), i, dtype=I32) for i, n in enumerate(lens)])
    pos = torch.cat([torch.arange(n, dtype=I32) + (start[i] if start else 0) for i, n in enumerate(lens)])
    return seq, pos


def randn(*shape, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(BF)


def rope_table(n, rot):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return torch.stack([ang.cos(), ang.sin()], -1).to(BF)


def same(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def cuda(*ts):
    return tuple(t.to(DEV) if t is not None else None for t in ts)


def page_bytes_expected(values, tok):
    """values (tokens, D) of one page block at token offsets tok -> (bytes, which of them are written)."""
    D = values.shape[1]
    code, scale = O.quantise(values)
    c, s = torch.zeros(64, D, dtype=torch.uint8), torch.zeros(64, D // 32, dtype=torch.uint8)
    cw, sw = torch.zeros(64, D, dtype=torch.uint8), torch.zeros(64, D // 32, dtype=torch.uint8)
    c[tok], s[tok], cw[tok], sw[tok] = code, scale, 15, 255
    return O.pack_block(c, s), O.pack_block(cw, sw)


# ------------------------------------------------------------------------------------------------ append and read


@pytest.mark.parametrize("D, H, KVH, rot, half, norm, lens", [
    (128, 32, 8, 128, False, True, [1]), (128, 32, 8, 128, False, True, [70, 1, 129]), (128, 5, 5, 64, True, True, [33, 64]),
    (128, 16, 2, 0, False, False, [17]), (64, 14, 2, 32, True, False, [65, 3]), (64, 3, 3, 64, True, True, [9, 0, 63]),
    (64, 8, 4, 16, False, True, [5]), (32, 4, 2, 32, False, True, [200, 31]), (32, 6, 2, 16, True, False, [64]),
    (32, 2, 1, 32, True, True, [1, 1, 1])])
def test_append_stores_the_definitions_bits(D, H, KVH, rot, half, norm, lens):
    start = [7 * i + 60 for i in range(len(lens))]
    ends = [s + n for s, n in zip(start, lens)]
    table, n_pages = make_table(ends, seed=D + H)
    seq, pos = rows_of(lens, start)
    M = len(seq)
    qkv = randn(M, H + 2 * KVH, D, seed=1)
    qkv[:, H::2] *= 37.0
    qn, kn = (randn(D, seed=2) + 1, randn(D, seed=3) + 1) if norm else (None, None)
    rope = rope_table(max(ends), rot) if rot else None
    cache = make_cache(n_pages, KVH, D, fill=0xA5)
    dq = qkv.to(DEV)
    q, k, v = dq.split([H, KVH, KVH], dim=1)                       # slices of a fused projection, as the model has them
    t, s, p, r, wq, wk = cuda(table, seq, pos, rope, qn, kn)
    got = cache.append(k, v, s, p, t, q=q, rope=r, rope_layout="half" if half else "interleaved", q_norm=wq, k_norm=wk, eps=1e-5)
    cs = rope[pos.long()] if rot else None
    want_q = O.rotate(O.head_norm(qkv[:, :H], qn, 1e-5), cs, half)
    want_k = O.rotate(O.head_norm(qkv[:, H:H + KVH], kn, 1e-5), cs, half)
    want_v = qkv[:, H + KVH:]
    assert same(got, want_q)
    gk, gv = cache.read(s, p, t)
    assert same(gk, O.stored(want_k)) and same(gv, O.stored(want_v))
    # byte for byte, and nothing else of the pool was touched
    want = torch.full(cache.pool.shape, 0xA5, dtype=torch.uint8)
    for i in range(len(lens)):
        for page in range(table.shape[1]):
            rows = (seq == i) & (pos // 64 == page)
            if rows.any():
                for h in range(KVH):
                    for j, val in enumerate((want_k, want_v)):
                        b, mask = page_bytes_expected(val[rows, h], pos[rows].long() % 64)
                        w = want[table[i, page], h, j]
                        want[table[i, page], h, j] = (w & ~mask) | (b & mask)
    assert torch.equal(cache.pool.cpu(), want)


def test_number_format_at_its_edges():
    """Ties, the block power's border, the smallest and largest powers, zeros of both signs, blocks with inf or NaN."""
    rows = []
    for e in (-133, -128, -103, -100, -99, -30, -1, 0, 1, 40, 124, 125):
        for top in (1.0, 1.5, 1.75, 1.7578125, 1.9921875):          # 1.f of the largest value, around f = 1.75
            base = torch.linspace(0, 1, 64, dtype=torch.float64) * top
            rows.append(torch.ldexp(base, torch.tensor(e)))
            rows.append(-torch.ldexp(base.flip(0), torch.tensor(e)))
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.5, 7.0] * 6 + [0.0, -0.0, 7.0, -7.0], dtype=torch.float64)
    rows += [ties, -ties * 2.0 ** -60, torch.zeros(64, dtype=torch.float64), -torch.zeros(64, dtype=torch.float64)]
    for bad in (math.inf, -math.inf, math.nan):
        r = torch.ones(64, dtype=torch.float64)
        r[40] = bad
        rows.append(r)
    big = torch.full((64,), 3.3895313892515355e38, dtype=torch.float64)     # the largest bf16
    rows += [big, -big]
    y = torch.stack(rows).to(BF)[:, None, :]
    M = y.shape[0]
    table, n_pages = make_table([M])
    cache = make_cache(n_pages, 1, 64)
    seq, pos = rows_of([M])
    t, s, p = cuda(table, seq, pos)
    cache.append(y.to(DEV), y.flip(0).contiguous().to(DEV), s, p, t)
    k, v = cache.read(s, p, t)
    assert same(k, O.stored(y)) and same(v, O.stored(y.flip(0)))
    code, scale = O.quantise(y[:64, 0])
    want = O.pack_block(code, scale)
    assert torch.equal(cache.pool[table[0, 0], 0, 0].cpu(), want)


def test_head_norm_of_tiny_and_huge_rows():
    D, KVH, M = 64, 2, 64
    k = randn(M, KVH, D, seed=1)
    for i in range(M):
        k[i] = (k[i].float() * 10.0 ** ((i - 32) * 1.1)).to(BF)
    table, n_pages = make_table([M])
    cache = make_cache(n_pages, KVH, D)
    seq, pos = rows_of([M])
    w = randn(D, seed=4) + 1
    t, s, p, kd, wd = cuda(table, seq, pos, k, w)
    cache.append(kd, kd, s, p, t, k_norm=wd, eps=1e-6)
    assert same(cache.read(s, p, t)[0], O.stored(O.head_norm(k, w, 1e-6)))


def test_padding_rows_and_missing_pages_write_nothing():
    D, KVH, H = 64, 2, 4
    table = torch.tensor([[3, 1], [-1, 9], [0, 2 ** 31 - 1], [-2 ** 31, 4]], dtype=I32)   # pool of 5 pages: 9 and the extremes are none
    cache = make_cache(5, KVH, D, fill=0x5A)
    rope = rope_table(100, 32)
    cases = [(0, 5, True, True), (-1, 5, False, False), (4, 5, False, False), (2 ** 31 - 1, 0, False, False), (-2 ** 31, 0, False, False),
             (0, -1, False, False), (0, -2 ** 31, False, False), (0, 99, True, True), (0, 100, False, False), (0, 128, False, False),
             (0, 2 ** 31 - 1, False, False), (1, 5, True, False), (1, 70, True, False), (2, 3, True, True), (2, 66, True, False),
             (3, 0, True, False), (3, 64, True, True)]                      # (sequence, position, q written, k and v written)
    M = len(cases)
    seq, pos = (torch.tensor([c[i] for c in cases], dtype=I32) for i in range(2))
    q, k, v = (randn(M, n, D, seed=n) for n in (H, KVH, KVH))
    t, s, p, r, qd, kd, vd = cuda(table, seq, pos, rope, q, k, v)
    qo = torch.full((M, H, D), 77.0, dtype=BF, device=DEV)
    assert cache.append(kd, vd, s, p, t, q=qd, q_out=qo, rope=r) is qo
    qo = qo.cpu()
    want = torch.full(cache.pool.shape, 0x5A, dtype=torch.uint8)
    for i, (sq, ps, wq, wkv) in enumerate(cases):
        if wq:
            cs = rope[ps:ps + 1]
            assert same(qo[i], O.rotate(q[i:i + 1], cs, False)[0]), cases[i]
        else:
            assert qo[i].eq(77.0).all(), cases[i]
        if wkv:
            for h in range(KVH):
                for j, val in enumerate((O.rotate(k[i:i + 1], rope[ps:ps + 1], False), v[i:i + 1])):
                    b, mask = page_bytes_expected(val[:, h], torch.tensor([ps % 64]))
                    page = int(table[sq, ps // 64])
                    want[page, h, j] = (want[page, h, j] & ~mask) | (b & mask)
    assert torch.equal(cache.pool.cpu(), want)
    gk, gv = cache.read(s, p, t)
    for i, (sq, ps, _, wkv) in enumerate(cases):
        inside = 0 <= sq < 4 and 0 <= ps < 128 and 0 <= int(table[sq, ps // 64]) < 5
        if not inside:
            assert gk[i].eq(0).all() and gv[i].eq(0).all(), cases[i]
        if wkv:
            assert same(gv[i], O.stored(v[i]))


def test_strided_inputs_and_outputs_and_writing_q_over_itself():
    D, KVH, H, M = 128, 4, 8, 21
    wide = randn(2 * M, H + 2 * KVH + 3, D, seed=9).to(DEV)
    q, k, v = wide[1::2, 1:1 + H], wide[::2, H:H + KVH], wide[1::2, -KVH:]
    table, n_pages = make_table([M])
    seq, pos = rows_of([M])
    rope = rope_table(M, D)
    t, s, p, r = cuda(table, seq, pos, rope)
    cache = make_cache(n_pages, KVH, D)
    out = torch.full((M, H + 2, D), 5.0, dtype=BF, device=DEV)
    cache.append(k, v, s, p, t, q=q, q_out=out[:, 1:1 + H], rope=r)
    want_q = O.rotate(q.cpu(), rope, False)
    assert same(out[:, 1:1 + H], want_q) and out[:, 0].eq(5).all() and out[:, -1].eq(5).all()
    gk, gv = cache.read(s, p, t)
    assert same(gk, O.stored(O.rotate(k.cpu(), rope, False))) and same(gv, O.stored(v.cpu()))
    kc, vc = k.contiguous(), v.contiguous()
    got = cache.append(kc, vc, s, p, t, q=q, q_out=q, rope=r)
    assert same(got, want_q)
    with pytest.raises(ValueError, match="half-split"):
        cache.append(kc, vc, s, p, t, q=q, q_out=q, rope=r, rope_layout="half")


# ------------------------------------------------------------------------------------------------ attention


def check_attention(got, q, kv, new, D, scale=None, seen=None):
    """kv: per sequence the stored (k, v) float64 of its keys.  Calls of more than 64 query columns (rows x heads per kv
    head) per sequence keep their softmax weights in fp16: 2^-11 of a weight, at most 2^-11 max|v| of an output."""
    G = q.shape[1] // kv[0][0].shape[1]
    weight = 2.0 ** -11 if max(new) * G > 64 else 2.0 ** -16
    scale = 1 / math.sqrt(D) if scale is None else scale
    r = 0
    for i, n in enumerate(new):
        k, v = kv[i]
        ref, bound = O.attend(q[r:r + n], k, v, k.shape[0] - n, scale, None if seen is None else seen[i], weight)
        err = (got[r:r + n].double().cpu() - ref).abs()
        tol = 2.0 ** -8 * ref.abs() + bound
        assert bool((err <= tol).all()), (i, float((err - tol).max()), float(err.max()))
        r += n


def setup_attention(D, H, KVH, new, keys, seed=0, fill=0, width=None, kscale=1.0):
    table, n_pages = make_table(keys, seed=seed, width=width)
    cache = make_cache(n_pages, KVH, D, fill=fill)
    k, v = randn(sum(keys), KVH, D, seed=seed + 1, scale=kscale), randn(sum(keys), KVH, D, seed=seed + 2)
    q = randn(sum(new), H, D, seed=seed + 3, scale=1.3)
    seq, pos = rows_of(keys)
    t, s, p, kd, vd, qd = cuda(table, seq, pos, k, v, q)
    cache.append(kd, vd, s, p, t)
    ks, vs = O.stored(k).split(keys), O.stored(v).split(keys)
    start = torch.tensor([0] + new).cumsum(0).to(I32).to(DEV)
    return cache, t, q, qd, start, torch.tensor(keys, dtype=I32, device=DEV), list(zip(ks, vs))


SHAPES = [(128, 32, 8), (128, 8, 8), (64, 14, 2), (64, 6, 2), (32, 4, 2), (32, 17, 1), (128, 10, 2)]


@pytest.mark.parametrize("D, H, KVH", SHAPES)
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_single_tokens_over_every_short_length(D, H, KVH, splits):
    keys = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 200, 300, 0, 513]
    new = [1] * len(keys)
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, new, keys, seed=3, fill=0xFF)
    got = cache.attend(qd, start, kv_len, t, max_q=1, max_kv=max(keys), splits=splits)
    check_attention(got, q, kv, new, D)
    assert got[17].eq(0).all()                                      # no keys


@pytest.mark.parametrize("D, H, KVH", SHAPES)
@pytest.mark.parametrize("new, keys", [([5, 1, 16, 3], [5, 40, 100, 64]), ([33, 0, 17], [33, 50, 65]), ([2, 7, 4], [0, 3, 1030]),
                                       ([130], [130]), ([65, 64, 63], [65, 128, 200])], ids=str)
@pytest.mark.parametrize("splits", [0, 2])
def test_prompts_and_chunks(D, H, KVH, new, keys, splits):
    """Chunks longer than their keys too: the first rows then lie before position 0 and see nothing."""
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, new, keys, seed=11, fill=0xFF)
    got = cache.attend(qd, start, kv_len, t, max_q=max(new), max_kv=max(keys), splits=splits)
    check_attention(got, q, kv, new, D)
    if new[0] == 2:
        assert got[:2].eq(0).all() and got[2:6].eq(0).all()


@pytest.mark.parametrize("scale", [0.0, 0.02, 1.0, -0.3])
def test_softmax_scale(scale):
    cache, t, q, qd, start, kv_len, kv = setup_attention(64, 4, 2, [3, 1], [70, 130], seed=5)
    got = cache.attend(qd, start, kv_len, t, max_q=3, max_kv=130, scale=scale)
    check_attention(got, q, kv, [3, 1], 64, scale=scale)


@pytest.mark.parametrize("splits", [0, 1, 16, 256])
def test_large_scores_and_a_long_context(splits):
    keys, new = [9001, 2500], [1, 2]
    cache, t, q, qd, start, kv_len, kv = setup_attention(128, 4, 1, new, keys, seed=7, kscale=8.0)
    got = cache.attend(qd, start, kv_len, t, max_q=2, max_kv=9001, splits=splits)
    check_attention(got, q, kv, new, 128)


def test_nan_values_reach_only_the_rows_that_see_them():
    """A NaN in V or K at some key: rows before it are untouched, rows from it on are NaN (V: in its 32-dim block only)."""
    D, H, KVH, n = 64, 4, 2, 150
    table, n_pages = make_table([n])
    seq, pos = rows_of([n])
    for which, splits in ((0, 1), (1, 1), (1, 3)):
        k, v, q = randn(n, KVH, D, seed=1), randn(n, KVH, D, seed=2), randn(n, H, D, seed=3)
        bad = (k, v)[which]
        bad[77, 1, 40] = math.nan
        bad[130, 1, 3] = math.inf
        cache = make_cache(n_pages, KVH, D)
        t, s, p, kd, vd, qd = cuda(table, seq, pos, k, v, q)
        cache.append(kd, vd, s, p, t)
        start, kv_len = torch.tensor([0, n], dtype=I32, device=DEV), torch.tensor([n], dtype=I32, device=DEV)
        got = cache.attend(qd, start, kv_len, t, max_q=n, max_kv=n, splits=splits).cpu()
        clean = torch.nan_to_num(O.stored(k), nan=0.0), torch.nan_to_num(O.stored(v), nan=0.0)
        nan = torch.zeros(n, H, D, dtype=torch.bool)
        if which == 0:
            nan[77:, 2:] = True
        else:
            nan[77:, 2:, 32:] = True
            nan[130:, 2:, :32] = True
        assert torch.equal(got.isnan(), nan)
        ref, bound = O.attend(q, *clean, 0, 1 / math.sqrt(D), weight=2.0 ** -11)
        ok = ~nan
        assert bool(((got.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + bound)[ok].all())


def test_missing_pages_are_masked():
    D, H, KVH = 64, 4, 2
    keys, new = [300, 130, 64], [2, 1, 1]
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, new, keys, seed=21)
    t = t.clone()
    t[0, 1], t[0, 4], t[1, 0], t[2, 0] = -1, cache.n_pages, 2 ** 31 - 1, -2 ** 31
    seen = [torch.ones(n, dtype=torch.bool) for n in keys]
    seen[0][64:128] = seen[0][256:] = False
    seen[1][:64] = False
    seen[2][:] = False
    for splits in (1, 4):
        got = cache.attend(qd, start, kv_len, t, max_q=2, max_kv=300, splits=splits)
        check_attention(got, q, kv, new, D, seen=seen)
        assert got[3].eq(0).all()


def test_lengths_outside_the_buffers_are_clamped():
    """Lengths and row bounds come from device memory: whatever they say, the kernel stays inside its buffers."""
    D, H, KVH = 64, 4, 2
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, [1, 1], [128, 100], seed=2)
    ok = cache.attend(qd, start, kv_len, t, max_q=1, max_kv=128)
    out = torch.full_like(ok, 9.0)
    cache.attend(qd, torch.tensor([0, 1, 2 ** 31 - 1], dtype=I32, device=DEV), kv_len, t, max_q=1, max_kv=128, out=out)
    assert torch.equal(out, ok)
    out.fill_(9.0)
    cache.attend(qd, torch.tensor([-5, 1, 1], dtype=I32, device=DEV), torch.tensor([128, -7], dtype=I32, device=DEV), t, max_q=1,
                 max_kv=128, out=out)
    assert torch.equal(out[0], ok[0]) and out[1].eq(9).all()
    out.fill_(9.0)
    big = cache.attend(qd, start, torch.tensor([2 ** 31 - 1, -2 ** 31], dtype=I32, device=DEV), t, max_q=1, max_kv=128, out=out)
    assert torch.equal(big[0], ok[0]) and big[1].eq(0).all()       # every key of the table; no key


def test_rows_behind_the_last_sequence_and_beyond_max_q_stay():
    D, H, KVH = 128, 4, 2
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, [3, 2], [70, 40], seed=2)
    wide = torch.cat([qd, qd])
    for splits in (1, 2):
        out = torch.full((10, H + 1, D), 3.0, dtype=BF, device=DEV)
        cache.attend(wide, start, kv_len, t, max_q=3, max_kv=70, out=out[:, :H], splits=splits)
        assert out[5:].eq(3).all() and out[:, H].eq(3).all()
        check_attention(out[:5, :H], q, kv, [3, 2], D)
        out.fill_(3.0)
        cache.attend(wide, start, kv_len, t, max_q=2, max_kv=70, out=out[:, :H], splits=splits)
        assert out[2].eq(3).all() and out[5:].eq(3).all()
        check_attention(out[3:5, :H], q[3:5], kv[1:], [2], D)


@pytest.mark.parametrize("H, n, max_q", [(4, 5, 2), (8, 90, 40)])
def test_rows_up_to_max_q_keep_their_positions(H, n, max_q):
    """A sequence with more rows than max_q: the first max_q are at the positions they have in the whole call."""
    D, KVH, keys = 64, 2, [150]
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, [n], keys, seed=13)
    for splits in (1, 3):
        out = torch.full((n, H, D), 3.0, dtype=BF, device=DEV)
        cache.attend(qd, start, kv_len, t, max_q=max_q, max_kv=150, out=out, splits=splits)
        seen = keys[0] - n + max_q
        check_attention(out[:max_q], q[:max_q], [(kv[0][0][:seen], kv[0][1][:seen])], [max_q], D)
        assert out[max_q:].eq(3).all()


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("n, splits", [(3, 1), (3, 2), (70, 1), (70, 2)])
def test_nonfinite_queries_give_nan_where_they_see_a_key(bad, n, splits):
    """Also if every key's score would be minus infinity; the other rows and heads do not notice."""
    D, H, KVH, keys = 64, 4, 2, 800
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, [n, 2], [keys, 1], seed=17)
    pos = torch.arange(keys, dtype=I32)
    k = torch.ones(keys, KVH, D, dtype=BF)                         # no zero, one sign: inf times k is the same infinity for every key
    v = randn(keys, KVH, D, seed=19)
    cache.append(k.to(DEV), v.to(DEV), torch.zeros(keys, dtype=I32, device=DEV), pos.to(DEV), t)
    qd[0, 1, 7], qd[2, 3, 63], qd[n, 0, 0], qd[n + 1, 2, 32] = bad, bad, bad, bad     # (row n: the 2-row sequence's row without a key)
    got = cache.attend(qd, start, kv_len, t, max_q=n, max_kv=keys, splits=splits)
    nan = torch.zeros(n + 2, H, dtype=torch.bool)
    nan[0, 1] = nan[2, 3] = nan[n + 1, 2] = True
    assert torch.equal(got.isnan().any(-1).cpu(), nan) and torch.equal(got.isnan().all(-1).cpu(), nan)
    assert got[n].eq(0).all()
    ref, bound = O.attend(q[:n], O.stored(k), O.stored(v), keys - n, 1 / math.sqrt(D), weight=2.0 ** -16 if n == 3 else 2.0 ** -11)
    err = (got[:n].double().cpu() - ref).abs()
    assert bool((err <= 2.0 ** -8 * ref.abs() + bound)[~nan[:n]].all())


def test_rows_do_not_depend_on_their_batch_with_fixed_splits():
    D, H, KVH = 128, 32, 8
    keys, new = [700, 64, 333, 1500], [1, 1, 1, 1]
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, new, keys, seed=4)
    whole = cache.attend(qd, start, kv_len, t, max_q=1, max_kv=1500, splits=8)
    for i in range(4):
        one = cache.attend(qd[i:i + 1], torch.tensor([0, 1], dtype=I32, device=DEV), kv_len[i:i + 1], t[i:i + 1].contiguous(),
                           max_q=1, max_kv=keys[i], splits=8)
        assert torch.equal(one[0], whole[i])


def test_offsets_beyond_32_bits():
    """A pool of more than 4 GiB whose used pages lie at its end."""
    D, H, KVH = 128, 16, 8
    n_pages = (1 << 32) // (KVH * 2 * 64 * 68) + 50
    cache = make_cache(n_pages, KVH, D)
    assert cache.pool.numel() > 1 << 32
    keys, new = [130, 90], [2, 1]
    table = torch.tensor([[n_pages - 1, n_pages - 7, n_pages - 2], [n_pages - 30, n_pages - 3, -1]], dtype=I32)
    seq, pos = rows_of(keys)
    k, v, q = randn(220, KVH, D, seed=1), randn(220, KVH, D, seed=2), randn(3, H, D, seed=3)
    t, s, p, kd, vd, qd = cuda(table, seq, pos, k, v, q)
    cache.append(kd, vd, s, p, t)
    gk, gv = cache.read(s, p, t)
    assert same(gk, O.stored(k)) and same(gv, O.stored(v))
    got = cache.attend(qd, torch.tensor([0, 2, 3], dtype=I32, device=DEV), torch.tensor(keys, dtype=I32, device=DEV), t, max_q=2,
                       max_kv=130)
    check_attention(got, q, list(zip(O.stored(k).split(keys), O.stored(v).split(keys))), new, D)
    assert cache.pool[: n_pages - 31].count_nonzero() == 0


def test_more_rows_than_a_grid_dimension_and_values_beyond_32_bits():
    """1.1 million rows, nearly all of them padding: q and its output pass 2^31 elements, the groups of rows pass 65 535."""
    D, H, KVH, M = 128, 16, 1, 1_100_000
    table = torch.tensor([[2, 0, 1]], dtype=I32, device=DEV)
    cache = make_cache(3, KVH, D, fill=0x11)
    rows = [0, 5, 700_001, 1_048_577, M - 1]
    pos = torch.full((M,), -1, dtype=I32, device=DEV)
    pos[rows] = torch.tensor([3, 190, 64, 70, 127], dtype=I32, device=DEV)
    seq = torch.zeros(M, dtype=I32, device=DEV)
    q = torch.zeros(M, H, D, dtype=BF, device=DEV)
    k, v = (torch.zeros(M, KVH, D, dtype=BF, device=DEV) for _ in range(2))
    q[rows], k[rows], v[rows] = (x.to(DEV) for x in (randn(5, H, D, seed=1), randn(5, KVH, D, seed=2), randn(5, KVH, D, seed=3)))
    rope = rope_table(192, D)
    out = torch.full_like(q, 7.0)
    cache.append(k, v, seq, pos, table, q=q, q_out=out, rope=rope.to(DEV))
    cs = rope[pos[rows].long().cpu()]
    assert same(out[rows], O.rotate(q[rows].cpu(), cs, False))
    out[rows] = 7.0
    assert out.eq(7.0).all()
    gk, gv = cache.read(seq, pos, table)
    assert same(gk[rows], O.stored(O.rotate(k[rows].cpu(), cs, False))) and same(gv[rows], O.stored(v[rows].cpu()))
    gk[rows] = 0
    gv[rows] = 0
    assert not gk.any() and not gv.any()
    # attention rows at the end of the same buffer
    start, n = torch.tensor([M - 2, M], dtype=I32, device=DEV), torch.tensor([128], dtype=I32, device=DEV)
    cache.attend(q, start, n, table, max_q=2, max_kv=128, out=out)
    ks, vs = (x.double().cpu() for x in cache.read(torch.zeros(128, dtype=I32, device=DEV),
                                                   torch.arange(128, dtype=I32, device=DEV), table))
    check_attention(out[-2:], q[-2:].cpu(), [(ks, vs)], [2], D)
    assert out[:M - 2].eq(7.0).all()


def test_a_conversation_prompt_steps_and_a_second_chunk():
    """The three operators as a generation loop uses them: a ragged prompt, single tokens, another chunk on top."""
    D, H, KVH = 64, 8, 4
    n_seq, cap = 3, 260
    table, n_pages = make_table([cap] * n_seq, seed=8)
    cache = make_cache(n_pages, KVH, D, fill=0xFF)
    rope, qn, kn = rope_table(cap, D), randn(D, seed=40) + 1, randn(D, seed=41) + 1
    t, r, wq, wk = cuda(table, rope, qn, kn)
    lens = [0] * n_seq
    hist = [[[], []] for _ in range(n_seq)]
    for step, new in enumerate([[70, 1, 33], [1, 1, 1], [1, 1, 1], [1, 1, 1], [65, 2, 128]]):
        seq, pos = rows_of(new, lens)
        qkv = randn(sum(new), H + 2 * KVH, D, seed=50 + step)
        s, p, d = cuda(seq, pos, qkv)
        q, k, v = d.split([H, KVH, KVH], dim=1)
        q = cache.append(k, v, s, p, t, q=q, rope=r, q_norm=wq, k_norm=wk)
        cs = rope[pos.long()]
        want_q = O.rotate(O.head_norm(qkv[:, :H], qn, 1e-6), cs, False)
        assert same(q, want_q)
        sk = O.stored(O.rotate(O.head_norm(qkv[:, H:H + KVH], kn, 1e-6), cs, False))
        sv = O.stored(qkv[:, H + KVH:])
        for i, (a, b) in enumerate(zip(sk.split(new), sv.split(new))):
            hist[i][0].append(a)
            hist[i][1].append(b)
        lens = [x + n for x, n in zip(lens, new)]
        start = torch.tensor([0] + new).cumsum(0).to(I32).to(DEV)
        got = cache.attend(q, start, torch.tensor(lens, dtype=I32, device=DEV), t, max_q=max(new), max_kv=cap)
        check_attention(got, want_q, [(torch.cat(a), torch.cat(b)) for a, b in hist], new, D)
    seq, pos = rows_of(lens)
    gk, gv = cache.read(*cuda(seq, pos), t)
    assert same(gk, torch.cat([torch.cat(a) for a, _ in hist])) and same(gv, torch.cat([torch.cat(b) for _, b in hist]))


# ------------------------------------------------------------------------------------------------ a step in one launch


STEP_POS = [0, 1, 31, 32, 63, 64, 65, 100, 127, 128, 300, 703, 704, 1500]


def setup_step(D, H, KVH, pos, rot, norm, seed=0):
    """A cache that holds the tokens before `pos` of each sequence; what it holds at and behind them reads as NaN."""
    table, n_pages = make_table([p + 1 for p in pos], seed=seed)
    cache = make_cache(n_pages, KVH, D, fill=0xFF)
    k, v = randn(sum(pos), KVH, D, seed=seed + 1), randn(sum(pos), KVH, D, seed=seed + 2)
    t, s, p, kd, vd = cuda(table, *rows_of(pos), k, v)
    cache.append(kd, vd, s, p, t)
    qkv = randn(len(pos), H + 2 * KVH, D, seed=seed + 3)
    rope = rope_table(max(pos) + 1, rot) if rot else None
    wq, wk = (randn(D, seed=seed + 4) + 1, randn(D, seed=seed + 5) + 1) if norm else (None, None)
    return cache, t, qkv, rope, wq, wk, k, v


def append_then_attend(cache, q, k, v, seq, pos, t, max_kv, splits, rope, layout, wq, wk, scale=None):
    """-> the output and the pool afterwards, by the two calls on a copy of the cache; rows in the table's order"""
    from fish_speech_amd.kv4 import KV4Cache

    c = KV4Cache(cache.n_pages, cache.n_kv_head, cache.head_dim, pool=cache.pool.clone())
    q = c.append(k, v, seq, pos, t, q=q, rope=rope, rope_layout=layout, q_norm=wq, k_norm=wk, eps=1e-5)
    start = torch.arange(len(seq) + 1, dtype=I32, device=DEV)
    return c.attend(q, start, pos + 1, t, max_q=1, max_kv=max_kv, splits=splits, scale=scale), c.pool


@pytest.mark.parametrize("D, H, KVH, rot, half, norm", [
    (128, 32, 8, 128, False, True), (128, 5, 5, 64, True, True), (128, 16, 2, 0, False, False), (64, 14, 2, 32, True, False),
    (64, 6, 2, 64, True, True), (64, 8, 4, 16, False, True), (32, 4, 2, 32, False, True), (32, 6, 2, 16, True, False),
    (32, 17, 1, 32, True, True), (64, 40, 1, 64, False, True), (128, 10, 2, 128, True, True)])
@pytest.mark.parametrize("splits", [0, 1, 3, 20])
def test_a_step_equals_append_and_attention(D, H, KVH, rot, half, norm, splits):
    cache, t, qkv, rope, wq, wk, k0, v0 = setup_step(D, H, KVH, STEP_POS, rot, norm, seed=D + H)
    seq, pos = torch.arange(len(STEP_POS), dtype=I32), torch.tensor(STEP_POS, dtype=I32)
    d, s, p, r, dq, dk = cuda(qkv, seq, pos, rope, wq, wk)
    q, k, v = d.split([H, KVH, KVH], dim=1)
    layout = "half" if half else "interleaved"
    want, pool = append_then_attend(cache, q, k, v, s, p, t, 1501, splits, r, layout, dq, dk)
    got = cache.step(q, k, v, s, p, t, max_kv=1501, rope=r, rope_layout=layout, q_norm=dq, k_norm=dk, eps=1e-5, splits=splits)
    assert torch.equal(got, want) and torch.equal(cache.pool, pool)
    if splits == 0:
        cs = rope[pos.long()] if rot else None
        wantq = O.rotate(O.head_norm(qkv[:, :H], wq, 1e-5), cs, half)
        newk = O.stored(O.rotate(O.head_norm(qkv[:, H:H + KVH], wk, 1e-5), cs, half))
        newv = O.stored(qkv[:, H + KVH:])
        kv = [(torch.cat([a, newk[i:i + 1]]), torch.cat([b, newv[i:i + 1]]))
              for i, (a, b) in enumerate(zip(O.stored(k0).split(STEP_POS), O.stored(v0).split(STEP_POS)))]
        check_attention(got, wantq, kv, [1] * len(STEP_POS), D)


def test_a_steps_padding_rows_missing_pages_strides_and_row_order():
    """Rows in another order than the table's sequences, rows that are padding, pages that are not there, strided rows."""
    D, H, KVH = 64, 8, 2
    at = [130, 64, 700, 5, 90]
    cache, t, qkv, rope, _, _, _, _ = setup_step(D, H, KVH, at, 64, False, seed=31)
    t = t.clone()
    t[1, 1] = -1                                                   # sequence 1: the new token's page
    t[2, 3] = cache.n_pages                                        # sequence 2: a page in the middle
    rows = [(3, 5), (-1, 5), (0, 130), (5, 3), (2, 700), (4, -1), (1, 64), (4, 2 ** 31 - 1), (2 ** 31 - 1, 0), (4, 701)]
    seq, pos = (torch.tensor([x[i] for x in rows], dtype=I32) for i in range(2))     # (the table of rotations ends at 700)
    M = len(rows)
    wide = randn(2 * M, H + 2 * KVH + 1, D, seed=33).to(DEV)
    q, k, v = wide[1::2, 1:1 + H], wide[::2, H:H + KVH], wide[1::2, -KVH:]
    s, p, r = cuda(seq, pos, rope)
    real = [i for i, x in enumerate(rows) if x in ((3, 5), (0, 130), (2, 700), (1, 64))]
    for splits in (1, 2):
        pool = cache.pool.clone()
        idx = torch.tensor(real, device=DEV)
        want, after = append_then_attend(cache, q[idx], k[idx], v[idx], torch.arange(4, dtype=I32, device=DEV), p[idx],
                                         t[s[idx].long()].contiguous(), 701, splits, r, "interleaved", None, None)
        out = torch.full((M, H + 1, D), 7.0, dtype=BF, device=DEV)
        assert cache.step(q, k, v, s, p, t, max_kv=701, rope=r, eps=1e-5, splits=splits, out=out[:, :H]).data_ptr() == out.data_ptr()
        assert torch.equal(out[idx][:, :H], want) and torch.equal(cache.pool, after)
        rest = [i for i in range(M) if i not in real]
        assert out[rest].eq(7.0).all() and out[:, H].eq(7.0).all()
        cache.pool.copy_(pool)


def test_a_step_with_nonfinite_inputs_and_a_negative_scale():
    D, H, KVH = 64, 4, 2
    at = [40, 70, 100, 0]
    cache, t, qkv, rope, wq, wk, _, _ = setup_step(D, H, KVH, at, 0, False, seed=41)
    qkv[0, 1, 3] = -math.inf                                       # a query
    qkv[1, H + 1, 9] = math.nan                                    # a key
    qkv[2, H + KVH, 40] = math.inf                                 # a value
    d, s, p = cuda(qkv, torch.arange(4, dtype=I32), torch.tensor(at, dtype=I32))
    q, k, v = d.split([H, KVH, KVH], dim=1)
    want, pool = append_then_attend(cache, q, k, v, s, p, t, 101, 1, None, "interleaved", None, None, scale=-0.2)
    got = cache.step(q, k, v, s, p, t, max_kv=101, scale=-0.2, splits=1)
    assert same(got, want) and torch.equal(cache.pool, pool)
    nan = torch.zeros(4, H, D, dtype=torch.bool)
    nan[0, 1] = nan[1, 2:] = True
    nan[2, :2, 32:] = True
    assert torch.equal(got.isnan().cpu(), nan)


def test_steps_in_a_captured_graph():
    """A graph of a step whose inputs and positions change from replay to replay, with eager calls on the cache between them."""
    D, H, KVH = 128, 8, 2
    cache, t, qkv, rope, wq, wk, k0, v0 = setup_step(D, H, KVH, [800, 126], 128, True, seed=51)
    wide = torch.full((2, t.shape[1] + 1), -1, dtype=I32)
    wide[:, :t.shape[1]] = t.cpu()
    wide[1, 2] = wide[0, -1] = -1
    n_free = cache.n_pages                                         # two pages more: the second sequence grows into another
    bigger = make_cache(n_free + 1, KVH, D, fill=0xFF)
    bigger.pool[:n_free] = cache.pool
    cache = bigger
    wide[1, 2] = n_free
    t, r, dq, dk = cuda(wide, rope, wq, wk)
    s, pos = cuda(torch.arange(2, dtype=I32), torch.tensor([800, 126], dtype=I32))
    d = torch.zeros(2, H + 2 * KVH, D, dtype=BF, device=DEV)
    q, k, v = d.split([H, KVH, KVH], dim=1)
    r = torch.cat([r, r[:10]])
    for _ in range(2):                                             # (position 800 is written again by the first replay)
        cache.step(q, k, v, s, pos, t, max_kv=2000, rope=r, q_norm=dq, k_norm=dk, eps=1e-5)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = cache.step(q, k, v, s, pos, t, max_kv=2000, rope=r, q_norm=dq, k_norm=dk, eps=1e-5)
    for rep in range(5):
        d.copy_(randn(2, H + 2 * KVH, D, seed=60 + rep))
        pos.copy_(torch.tensor([800 + rep, 126 + rep], dtype=I32))
        want, pool = append_then_attend(cache, q, k, v, s, pos, t, 2000, 0, r, "interleaved", dq, dk)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(cache.pool, pool)
        cache.read(s, pos, t)


def test_another_stream_and_captured_graphs_with_new_lengths():
    """Two graphs over one cache, replayed in turn with eager calls between them; lengths, rows and inputs live on the
    device and change from replay to replay."""
    D, H, KVH = 128, 8, 2
    keys = [700, 90]
    cache, t, q, qd, start, kv_len, kv = setup_attention(D, H, KVH, [1, 1], keys, seed=6)
    side = torch.cuda.Stream()
    eager = cache.attend(qd, start, kv_len, t, max_q=1, max_kv=700, splits=4)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = cache.attend(qd, start, kv_len, t, max_q=1, max_kv=700, splits=4)
    side.synchronize()
    assert torch.equal(other, eager)
    seq, pos = cuda(torch.tensor([0, 1], dtype=I32), torch.tensor([699, 89], dtype=I32))
    kin, vin, qin = (torch.zeros(2, n, D, dtype=BF, device=DEV) for n in (KVH, KVH, H))
    graphs = []
    for splits in (4, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cache.append(kin, vin, seq, pos, t)
            out = cache.attend(qin, start, kv_len, t, max_q=1, max_kv=700, splits=splits)
            rk, rv = cache.read(seq, pos, t)
        graphs.append((g, out, rk, rv, splits))
    for rep in range(6):
        g, out, rk, rv, splits = graphs[rep % 2]
        kv_len.copy_(torch.tensor([700 - 60 * rep, 90 - rep], dtype=I32))
        pos.copy_(kv_len - 1)
        kin.copy_(randn(2, KVH, D, seed=100 + rep))
        vin.copy_(randn(2, KVH, D, seed=200 + rep))
        qin.copy_(randn(2, H, D, seed=300 + rep))
        g.replay()
        torch.cuda.synchronize()
        want = cache.attend(qin, start, kv_len, t, max_q=1, max_kv=700, splits=splits)
        assert torch.equal(out, want)
        assert same(rk, O.stored(kin.cpu())) and same(rv, O.stored(vin.cpu()))
        allk, allv = cache.read(*cuda(*rows_of([int(n) for n in kv_len])), t)
        ks, vs = (x.double().cpu().split([int(n) for n in kv_len]) for x in (allk, allv))
        check_attention(out, qin.cpu(), list(zip(ks, vs)), [1, 1], D)


def test_empty_calls():
    cache = make_cache(2, 2, 64)
    e = torch.empty(0, dtype=I32, device=DEV)
    t = torch.zeros(1, 2, dtype=I32, device=DEV)
    z = torch.empty(0, 2, 64, dtype=BF, device=DEV)
    assert cache.append(z, z, e, e, t) is None
    k, v = cache.read(e, e, t)
    assert k.shape == v.shape == (0, 2, 64)
    s = torch.zeros(2, dtype=I32, device=DEV)
    out = cache.attend(torch.empty(0, 4, 64, dtype=BF, device=DEV), s, s[:1], t, max_q=0, max_kv=0)
    assert out.shape == (0, 4, 64)
    assert cache.step(torch.empty(0, 4, 64, dtype=BF, device=DEV), z, z, e, e, t, max_kv=0).shape == (0, 4, 64)
    # no sequences at all: every row is one behind the last
    none, q = torch.empty(0, 2, dtype=I32, device=DEV), torch.ones(3, 4, 64, dtype=BF, device=DEV)
    assert cache.append(z, z, e, e, none) is None
    out = torch.full((3, 4, 64), 5.0, dtype=BF, device=DEV)
    assert cache.attend(q, s[:1], e, none, max_q=3, max_kv=5000, out=out) is out and out.eq(5).all()

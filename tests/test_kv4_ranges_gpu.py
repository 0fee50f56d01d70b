"""The 4-bit K/V cache with keys and values far from the ordinary ones: weights far below a row's largest, V blocks of very
different powers, large numbers.  The tolerance is relative to what a row adds up, sum of weight times |v|, so a sum that lost
its small terms does not pass: half a bf16 step of the output (2^-8 of it), and of the sum of absolute terms the rounding of
the weights (2^-11 where fp16 holds them, else 2^-16), the fp32 exponential's 2^-16, 2^-24 per added key, and what an fp32
score's rounding moves (its D + 4 roundings of the absolute products, twice: weight and sum of the weights)."""
import math

import pytest
import torch

from oracle import kv4 as O
from tests.test_kv4_gpu import cuda, make_cache, make_table, randn, rows_of

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF = torch.bfloat16
I32 = torch.int32


def reference(q, k, v, scale, weight):
    """One sequence whose rows are its last positions; k, v (keys, KVH, D) stored values in float64.  -> output, tolerance"""
    n, H, D = q.shape
    keys, G = k.shape[0], H // k.shape[1]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    hidden = torch.arange(keys)[None, :] > torch.arange(keys - n, keys)[:, None]
    s = torch.einsum("nhd,khd->hnk", q.double(), k) * scale
    moved = torch.einsum("nhd,khd->hnk", q.double().abs(), k.abs()).amax(-1, keepdim=True) * abs(scale) * (D + 4) * 2.0 ** -24
    s = s.masked_fill(hidden, -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    out, terms = torch.matmul(p, v.transpose(0, 1)), torch.matmul(p, v.abs().transpose(0, 1))
    tol = 2.0 ** -8 * out.abs() + (weight + 2.0 ** -16 + keys * 2.0 ** -24 + 2 * moved) * terms
    return out.transpose(0, 1), tol.transpose(0, 1)


def stored_cache(k, v, seed=0):
    """One sequence in a cache of its own -> cache, table, stored k and v"""
    n, KVH, D = k.shape
    table, n_pages = make_table([n], seed=seed)
    cache = make_cache(n_pages, KVH, D, fill=0xFF)
    t, s, p, kd, vd = cuda(table, *rows_of([n]), k, v)
    cache.append(kd, vd, s, p, t)
    return cache, t, O.stored(k), O.stored(v)


def attend(cache, t, q, keys, splits=1, max_q=None, **kw):
    n = q.shape[0]
    start, kv_len = torch.tensor([0, n], dtype=I32, device=DEV), torch.tensor([keys], dtype=I32, device=DEV)
    return cache.attend(q.to(DEV), start, kv_len, t, max_q=max_q or n, max_kv=keys, splits=splits, **kw)


def weight_bits(rows, G):
    return 2.0 ** -11 if rows * G > 64 else 2.0 ** -16


def worst(got, ref, tol):
    return float(((got.double().cpu() - ref).abs() / tol.clamp(min=1e-300)).max())


def sink_case(D, H, KVH, rows, keys, gap, seed, sink_v):
    """Key 0 takes nearly all of the weight, the others' scores lie about `gap` below (natural logarithm)."""
    q = 1 + randn(rows, H, D, seed=seed).float() * 0.02
    k = (4 - gap * math.sqrt(D) / D) + randn(keys, KVH, D, seed=seed + 1).float() * 0.3
    k[0] = 4.0
    v = 1 + randn(keys, KVH, D, seed=seed + 2).float() * 0.2
    v[0] = sink_v
    return q.to(BF), k.to(BF), v.to(BF)


@pytest.mark.parametrize("D, H, KVH", [(128, 8, 2), (64, 4, 2), (32, 4, 4)])
@pytest.mark.parametrize("rows", [1, 16, 70])
@pytest.mark.parametrize("gap", [10.0, 13.0, 15.5])
@pytest.mark.parametrize("splits", [1, 3])
def test_keys_beside_an_attention_sink(D, H, KVH, rows, gap, splits):
    """The sink's V is 0 in every second dim: what comes out there are thousands of small weights."""
    keys = 4200
    sink = torch.zeros(D)
    sink[1::2] = 1.0
    q, k, v = sink_case(D, H, KVH, rows, keys, gap, 7, sink)
    cache, t, ks, vs = stored_cache(k, v)
    got = attend(cache, t, q, keys, splits)
    ref, tol = reference(q, ks, vs, 1 / math.sqrt(D), weight_bits(rows, H // KVH))
    s = torch.einsum("nhd,khd->hnk", q.double(), ks.repeat_interleave(H // KVH, 1)) / math.sqrt(D)
    below = (s[..., :1] - s[..., 1:keys - rows]).median()
    assert gap - 1 <= below <= gap + 1                              # (of the stored keys)
    assert worst(got, ref, tol) <= 1


# ------------------------------------------------------------------------------------------------ V of very different powers


def spread_case(D, H, KVH, keys, power, seed):
    """V normal times 2^power, a tensor that spreads over (keys, KVH, D)."""
    q, k = randn(keys, H, D, seed=seed), randn(keys, KVH, D, seed=seed + 1)
    v = (torch.randn(keys, KVH, D, generator=torch.Generator().manual_seed(seed + 2)).double() * 2.0 ** power.double()).to(BF)
    return q, k, v


@pytest.mark.parametrize("D, H, KVH", [(128, 8, 2), (64, 4, 2), (32, 3, 3)])
@pytest.mark.parametrize("small", [-20, -30, -60, -90])
@pytest.mark.parametrize("big_at", [1, 31, 40, 63, 64, 100, 195])
def test_a_large_value_leaves_the_rows_before_it_alone(D, H, KVH, small, big_at):
    keys = 200
    power = torch.full((keys, 1, 1), small)
    power[big_at] = 0
    q, k, v = spread_case(D, H, KVH, keys, power, 3)
    cache, t, ks, vs = stored_cache(k, v)
    got = attend(cache, t, q, keys)
    ref, tol = reference(q, ks, vs, 1 / math.sqrt(D), 2.0 ** -11)
    assert worst(got, ref, tol) <= 1
    # the few-row kernel, on the rows around the large value
    lo, n = max(0, big_at - 3), 6
    few = attend(cache, t, q[lo:lo + n], min(lo + n, keys))
    ref, tol = reference(q[lo:lo + n], ks[:lo + n], vs[:lo + n], 1 / math.sqrt(D), 2.0 ** -16)
    assert worst(few, ref, tol) <= 1


def powers(kind, keys, KVH, D):
    g = torch.Generator().manual_seed(11)
    if kind == "dims":                # one 32-dim block after the other, 2^40 apart
        return (torch.arange(D) // 32 * 40 - 60).expand(keys, KVH, D)
    if kind == "falling":             # page after page, 2^35 down
        return (40 - torch.arange(keys) // 64 * 35)[:, None, None]
    if kind == "rising":
        return (-90 + torch.arange(keys) // 64 * 35)[:, None, None]
    if kind == "window":              # about the powers that the prompt kernel holds in fp16, and a step beyond
        return torch.randint(-5, 7, (keys, KVH, D // 32), generator=g).repeat_interleave(32, -1)
    return torch.randint(-95, 100, (keys, KVH, D // 32), generator=g).repeat_interleave(32, -1)    # "random"


@pytest.mark.parametrize("D, H, KVH", [(128, 8, 2), (64, 4, 2), (32, 6, 2)])
@pytest.mark.parametrize("kind", ["dims", "falling", "rising", "window", "random"])
@pytest.mark.parametrize("rows, splits", [(300, 1), (60, 1), (3, 1), (60, 2), (3, 3)])
def test_powers_spread_over_blocks_tokens_and_pages(D, H, KVH, kind, rows, splits):
    keys = 300 if splits == 1 else 1000
    q, k, v = spread_case(D, H, KVH, keys, powers(kind if splits == 1 or kind not in ("falling", "rising") else "random", keys, KVH, D), 5)
    q = q[-rows:]
    cache, t, ks, vs = stored_cache(k, v)
    got = attend(cache, t, q, keys, splits)
    ref, tol = reference(q, ks, vs, 1 / math.sqrt(D), weight_bits(rows, H // KVH))
    assert worst(got, ref, tol) <= 1


@pytest.mark.parametrize("D, H, KVH", [(128, 8, 2), (64, 4, 2), (32, 6, 2)])
@pytest.mark.parametrize("rows", [60, 16, 1])
@pytest.mark.parametrize("gap", [20.0, 26.0])
def test_keys_far_below_a_sink_without_a_value(D, H, KVH, rows, gap):
    """Weights about 2^-29 and 2^-37, all that there is where the sink's V is 0."""
    keys = 1500
    q, k, v = sink_case(D, H, KVH, rows, keys, gap, 21, torch.zeros(D))
    cache, t, ks, vs = stored_cache(k, v)
    for splits in (1, 2):
        got = attend(cache, t, q, keys, splits)
        ref, tol = reference(q, ks, vs, 1 / math.sqrt(D), weight_bits(rows, H // KVH))
        assert worst(got, ref, tol) <= 1


@pytest.mark.parametrize("D, H, KVH", [(128, 8, 2), (64, 6, 2), (32, 3, 1)])
@pytest.mark.parametrize("odd", [None, 0, 1, 37, 64, 130, 191, 199])
def test_a_prompts_rows_do_not_depend_on_later_tokens_or_on_how_it_is_cut(D, H, KVH, odd):
    """Bit for bit, with one token (`odd`) whose V is 2^30 times the others', and with none; the last tokens replaced by
    other ones; the prompt in two calls, cut at every kind of place (each call has more than 64 query columns)."""
    keys = 260
    power = torch.zeros(keys, 1, 1)
    if odd is not None:
        power[odd] = 30
    q, k, v = spread_case(D, H, KVH, keys, power, 9)
    cache, t, _, _ = stored_cache(k, v)
    whole = attend(cache, t, q, keys)
    for cut in (66, 128, 131, 190):
        first, second = attend(cache, t, q[:cut], cut), attend(cache, t, q[cut:], keys)
        assert torch.equal(first, whole[:cut]) and torch.equal(second, whole[cut:]), cut
        v2 = v.clone()
        v2[cut:] = (v2[cut:].float() * 2.0 ** torch.randint(-60, 60, (keys - cut, 1, 1), generator=torch.Generator().manual_seed(cut))).to(BF)
        other, t2, _, _ = stored_cache(k, v2)
        assert torch.equal(attend(other, t2, q, keys)[:cut], whole[:cut]), cut


def test_nan_blocks_and_missing_pages_at_the_start_of_a_prompt():
    """A first key whose V is NaN in one block, or in all; a first page that is not there."""
    D, H, KVH, keys = 64, 4, 2, 200
    q, k, v = spread_case(D, H, KVH, keys, torch.zeros(keys, 1, 1), 13)
    for dims in (slice(0, 1), slice(0, 64, 32)):
        bad = v.clone()
        bad[0, 1, dims] = math.nan
        cache, t, ks, vs = stored_cache(k, bad)
        got = attend(cache, t, q, keys).cpu()
        nan = torch.zeros(keys, H, D, dtype=torch.bool)
        nan[:, 2:, :32] = True
        if dims.step:
            nan[:, 2:, 32:] = True
        assert torch.equal(got.isnan(), nan)
        ref, tol = reference(q, ks, vs.nan_to_num(0.0), 1 / math.sqrt(D), 2.0 ** -11)
        assert bool(((got.double() - ref).abs() <= tol)[~nan].all())
    cache, t, ks, vs = stored_cache(k, v)
    t[0, 0] = -1
    got = attend(cache, t, q, keys)
    assert got[:64].eq(0).all()
    ref, tol = reference(q[64:], ks[64:], vs[64:], 1 / math.sqrt(D), 2.0 ** -11)
    assert worst(got[64:], ref, tol) <= 1


@pytest.mark.parametrize("D, H, KVH", [(128, 8, 2), (64, 4, 2), (32, 3, 3)])
@pytest.mark.parametrize("rows", [1, 16, 70])
@pytest.mark.parametrize("power", [-99, 112, 116])
def test_sums_of_large_and_small_values_stay_in_range(D, H, KVH, rows, power):
    """Scores that rise to 2^7.5 of the first ones' weight (less than a running maximum may lag behind): no sum is larger
    than with the true maximum, 1500 times 2^116 at most, and small values keep their bits."""
    keys = 1500
    q, k = torch.ones(rows, H, D, dtype=BF), torch.zeros(keys, KVH, D, dtype=BF)
    k[256:] = 0.75
    v = ((1 + randn(keys, KVH, D, seed=3).double() * 0.1) * 2.0 ** power).to(BF)
    scale = 7.5 * math.log(2) / (0.75 * D)
    cache, t, ks, vs = stored_cache(k, v)
    ref, tol = reference(q, ks, vs, scale, weight_bits(rows, H // KVH))
    for splits in (1, 3):
        assert worst(attend(cache, t, q, keys, splits, scale=scale), ref, tol) <= 1, splits


@pytest.mark.parametrize("base, step", [(0.0, 2), (2.0 ** 20, 2), (2.0 ** 24, 2), (2.0 ** 25, 4), (2.0 ** 26, 8), (2.0 ** 27, 16), (-2.0 ** 25, 4), (-2.0 ** 27, 16)])
@pytest.mark.parametrize("rows", [1, 16, 70])
@pytest.mark.parametrize("splits", [1, 3])
def test_scores_so_large_that_fp32_rounds_their_exponents(base, step, rows, splits):
    """Scores base + a few steps, exact in fp32, that grow along the keys: the weights depend on the differences alone."""
    D, H, KVH, keys = 64, 4, 2, 1500
    scale = math.log(2)
    q, k = torch.zeros(rows, H, D), torch.zeros(keys, KVH, D)
    q[..., 0], q[..., 32] = base, 1.0
    k[..., 0] = 1.0
    g = torch.Generator().manual_seed(2)
    grid = torch.tensor([0.0, 2, 4, 6, 8, 12, 16, 24])              # (one power for the block: its largest value is in every row)
    grid = grid[(grid % step) == 0]
    pick = (torch.rand(keys, KVH, generator=g) * (1 + torch.arange(keys)[:, None] / keys * (len(grid) - 1))).long()
    k[..., 32], k[..., 33] = grid[pick], 24.0
    v = 1 + randn(keys, KVH, D, seed=3).float() * 0.3
    cache, t, ks, vs = stored_cache(k.to(BF), v.to(BF))
    assert torch.equal(ks, k.double())
    ref, _ = reference(q.to(BF), ks, vs, scale, 0.0)
    bits = weight_bits(rows, H // KVH)
    # the scores are exact, their product with the scale in units of log2 is off by a common factor: half a step of 24 at most
    tol = 2.0 ** -8 * ref.abs() + (bits + 2.0 ** -16 + keys * 2.0 ** -24) * vs.abs().max()
    assert worst(attend(cache, t, q.to(BF), keys, splits, scale=scale), ref, tol) <= 1

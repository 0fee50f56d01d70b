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

"""The 4-bit paged K/V cache of the slow transformer, as it is measured: appending rotated keys and values to it,
attention that reads it, and reading stored tokens back.

The cache holds, per token and kv head, D values of K and D of V in blocks of 32 consecutive dims: each value is a
signed 4-bit float (0, 0.5, 1, 1.5, 2, 3, 4, 6, round to nearest, ties to the even code) times 2^e of its block, where e
is the smallest exponent with max|block| <= 7 * 2^e, at least -100 (values between 6 * 2^e and 7 * 2^e read as
6 * 2^e).  Tokens live in pages of 64; a block table per sequence names the pages.

Where ``own`` is false the operators are computed in plain torch operations; where it is true by
``fish_speech_amd.kv4.KV4Cache``.
"""
import math

import torch

own = False

PAGE = 64
DEV = "cuda:0"


# ------------------------------------------------------------------------------------------------ cases


def listed():
    """Attention: what a generation loop calls per layer.  ``new`` = query tokens per sequence (ragged: down to half of
    it), ``past`` = cached tokens in front of them, ``idle`` = batch rows whose slot is empty (no keys: zeros)."""
    a = dict(op="attend", n_head=32, n_kv=8, head_dim=128, idle=0, ragged=True)
    p = dict(op="append", n_head=32, n_kv=8, head_dim=128, rot=128, half=False, norm=True)
    return [
        # one utterance in the middle of its 10 s: the latency of a single frame's attention
        dict(a, name="step_1x300", seqs=1, new=1, past=300, ragged=False),
        # the headline batch of 8 with voice-clone prompts, one slot empty
        dict(a, name="step_8x2k", seqs=8, new=1, past=2047, idle=1),
        # a full server: 32 utterances with long conversations
        dict(a, name="step_32x8k", seqs=32, new=1, past=8191),
        # one very long context: the work has to be split over the keys
        dict(a, name="step_1x128k", seqs=1, new=1, past=131000, ragged=False),
        # a few tokens per sequence (verifying drafted frames), narrow heads, seven query heads per kv head
        dict(a, name="draft_5x900", seqs=5, new=3, past=900, n_head=14, n_kv=2, head_dim=64),
        # the headline prefill: eight prompts of about 200 tokens
        dict(a, name="prompt_8x200", seqs=8, new=200, past=0),
        # the next chunk of a long conversation on top of its cached prefix
        dict(a, name="prompt_2x2k_on_4k", seqs=2, new=2048, past=4099),
        # the frame's append: one row per slot, q | k | v of the fused projection, head norm and rotation on the way
        dict(p, name="append_8", seqs=8, new=1, past=777),
        # the append of a large prefill
        dict(p, name="append_8x2k", seqs=8, new=2048, past=0),
        # half-split rotation of half of a 64-wide head, no head norm, odd lengths on top of a prefix
        dict(p, name="append_3x333_half", seqs=3, new=333, past=51, n_head=14, n_kv=2, head_dim=64, rot=32, half=True,
             norm=False),
        # one short prefix read back
        dict(op="read", name="read_1x130", seqs=1, new=130, past=0, n_kv=8, head_dim=128),
        # the caches of a whole batch read back
        dict(op="read", name="read_8x4k", seqs=8, new=4096, past=1, n_kv=8, head_dim=128),
    ]


HEADS = [(32, 8, 128), (16, 8, 128), (8, 8, 128), (12, 4, 128), (16, 2, 128), (14, 2, 64), (16, 16, 64), (20, 5, 64),
         (4, 2, 32), (6, 2, 32)]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    H, KVH, D = rng.choice(HEADS)
    op = rng.choice(["attend", "attend", "attend", "attend", "append", "append", "read"])
    if op == "attend":
        kind = rng.choice(["step", "step", "draft", "prompt", "prompt"])
        if kind == "prompt":
            seqs, new = rng.randint(1, 6), _log_int(rng, 8, 2048)
            past = rng.choice([0, _log_int(rng, 1, 4096)])
            while seqs * new * (past + new) * H * D > 2 * 2048 * 6147 * 32 * 128:
                seqs, new = max(1, seqs - 1), max(8, new * 3 // 4)
            idle = 0
        else:
            seqs, new = _log_int(rng, 1, 48), 1 if kind == "step" else rng.randint(2, 7)
            past = _log_int(rng, 1, 131000)
            while seqs * past * KVH * D > 32 * 8191 * 8 * 128:
                seqs, past = max(1, seqs * 3 // 4), past * 3 // 4
            idle = rng.randint(0, seqs // 2) if rng.random() < 0.3 else 0
        return dict(op=op, n_head=H, n_kv=KVH, head_dim=D, seqs=seqs, new=new, past=past, idle=idle,
                    ragged=rng.random() < 0.8)
    seqs, new = _log_int(rng, 1, 32), rng.choice([1, _log_int(rng, 1, 2048)])
    while seqs * new > 16384:
        seqs = max(1, seqs // 2)
    past = rng.choice([0, _log_int(rng, 1, 8000)])
    if op == "read":
        return dict(op=op, n_kv=KVH, head_dim=D, seqs=seqs, new=new, past=past)
    return dict(op=op, n_head=H, n_kv=KVH, head_dim=D, seqs=seqs, new=new, past=past, rot=rng.choice([D, D, D // 2]),
                half=rng.random() < 0.5, norm=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------ inputs


def _lengths(case):
    """(new, past) of every sequence: a spread of lengths that depends on the case alone, so ``work`` can count it."""
    out = []
    n = case["seqs"]
    for i in range(n):
        new, past = case["new"], case["past"]
        if case.get("ragged"):
            f = (i * 7919 + 13) % 97 / 96.0
            if new > 7:
                new = max(1, int(new * (0.5 + 0.5 * f)))
            past = int(past * (0.5 + 0.5 * ((i * 104729 + 5) % 89 / 88.0)))
        if i >= n - case.get("idle", 0):
            past = -new          # an empty slot: its query rows see no key
        out.append((new, past))
    return out


def _rope_table(n, rot):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return torch.stack([ang.cos(), ang.sin()], dim=-1).to(torch.bfloat16).to(DEV)


def _inputs(case, seed):
    """Everything both forms start from: raw bf16 values, lengths, the block table (pages in no order)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    D, KVH, L = case["head_dim"], case["n_kv"], _lengths(case)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    pages = [(max(0, a + b) + PAGE - 1) // PAGE for a, b in L]
    width, total = max(1, max(pages)), sum(pages) + 3
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(L), width), -1, dtype=torch.int32, device=DEV)
    o = 0
    for i, n in enumerate(pages):
        table[i, :n] = perm[o:o + n]
        o += n
    x = dict(lens=L, table=table, n_pages=total)
    # keys: a few channels are several times larger than the rest, as rotated keys have them
    chan = torch.exp(0.5 * randn(KVH, D))

    def rows(spans):
        s = torch.cat([torch.full((b - a,), i, dtype=torch.int32, device=DEV) for i, (a, b) in enumerate(spans)])
        p = torch.cat([torch.arange(a, b, dtype=torch.int32, device=DEV) for a, b in spans])
        return s, p

    if case["op"] == "append":
        H = case["n_head"]
        x["row_seq"], x["row_pos"] = rows([(b, a + b) for a, b in L])
        M = x["row_seq"].numel()
        qkv = randn(M, H + 2 * KVH, D)
        qkv[:, H:H + KVH] *= chan
        x["qkv"] = qkv.to(torch.bfloat16).view(M, -1)
        x["rope"] = _rope_table(max(a + b for a, b in L), case["rot"])
        if case["norm"]:
            x["q_norm"], x["k_norm"] = ((1 + 0.2 * randn(D)).to(torch.bfloat16) for _ in range(2))
        return x
    x["row_seq"], x["row_pos"] = rows([(0, max(0, a + b)) for a, b in L])
    M = x["row_seq"].numel()
    x["k"] = (randn(M, KVH, D) * chan).to(torch.bfloat16)
    x["v"] = randn(M, KVH, D).to(torch.bfloat16)
    if case["op"] == "read":
        x["read_seq"], x["read_pos"] = rows([(b, a + b) for a, b in L])
    else:
        T = sum(a for a, _ in L)
        q = randn(T, KVH, case["n_head"] // KVH, D) / chan[:, None] * 1.5
        x["q"] = q.to(torch.bfloat16).view(T, case["n_head"], D)
        x["q_start"] = torch.tensor([0] + [a for a, _ in L], device=DEV).cumsum(0).to(torch.int32)
        x["kv_len"] = torch.tensor([max(0, a + b) for a, b in L], dtype=torch.int32, device=DEV)
    return x


# ------------------------------------------------------------------------------------------------ plain forms


def _quantise(y):
    """(..., D) bf16 -> codes (..., D) in 0..15 and block exponents + 127 (..., D / 32), both uint8."""
    b = y.float().unflatten(-1, (-1, 32))
    mant, ex = torch.frexp(b.abs().amax(-1))
    e = torch.where(mant <= 0.875, ex - 3, ex - 2).clamp(min=-100)
    e = torch.where(mant == 0, torch.full_like(e, -100), e)
    s = torch.ldexp(b, -e[..., None])
    a = s.abs()
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    code = code + 8 * (s < 0)
    return code.to(torch.uint8).flatten(-2), (e + 127).to(torch.uint8)


def _dequantise(code, e):
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
    val = grid[code.int()].unflatten(-1, (-1, 32))
    return torch.ldexp(val, e.int()[..., None] - 127).flatten(-2)


def _slots(table, seq, pos):
    return table[seq.long(), pos.long() // PAGE].long() * PAGE + pos.long() % PAGE


def _store(planes, y, slot):
    code, e = _quantise(y)
    planes[0][slot] = code[..., 0::2] | (code[..., 1::2] << 4)
    planes[1][slot] = e


def _load(planes, slot):
    packed = planes[0][slot]
    code = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2)
    return _dequantise(code, planes[1][slot])


def _rotate(y, cs, half):
    """y (M, heads, D) fp32, cs (M, rot / 2, 2): pairs (2 i, 2 i + 1), or (i, i + rot / 2) where ``half``."""
    rot = 2 * cs.shape[1]
    c, s = cs[:, None, :, 0].float(), cs[:, None, :, 1].float()
    a, rest = y[..., :rot], y[..., rot:]
    if half:
        x0, x1 = a[..., : rot // 2], a[..., rot // 2:]
        r = torch.cat([x0 * c - x1 * s, x1 * c + x0 * s], dim=-1)
    else:
        x0, x1 = a[..., 0::2], a[..., 1::2]
        r = torch.stack([x0 * c - x1 * s, x1 * c + x0 * s], dim=-1).flatten(-2)
    return torch.cat([r, rest], dim=-1).to(torch.bfloat16)


def _head_norm(x, w, eps=1e-6):
    ss = (x.double() ** 2).mean(-1, keepdim=True)
    rstd = (1.0 / (ss + eps).sqrt()).float()
    return (x.float() * rstd * w.float()).to(torch.bfloat16)


def _plain_append(st):
    D, H, KVH = st["D"], st["H"], st["KVH"]
    q, k, v = st["qkv"].unflatten(-1, (-1, D)).split([H, KVH, KVH], dim=1)
    if "q_norm" in st:
        q, k = _head_norm(q, st["q_norm"]), _head_norm(k, st["k_norm"])
    cs = st["rope"][st["row_pos"].long()]
    q, k = _rotate(q.float(), cs, st["half"]), _rotate(k.float(), cs, st["half"])
    slot = _slots(st["table"], st["row_seq"], st["row_pos"])
    _store(st["kp"], k, slot)
    _store(st["vp"], v, slot)
    return q, _load(st["kp"], slot).to(torch.bfloat16), _load(st["vp"], slot).to(torch.bfloat16)


def _plain_read(st):
    slot = _slots(st["table"], st["read_seq"], st["read_pos"])
    return _load(st["kp"], slot).to(torch.bfloat16), _load(st["vp"], slot).to(torch.bfloat16)


def _plain_attend(st):
    q, KVH, D = st["q"], st["KVH"], st["D"]
    G = q.shape[1] // KVH
    out = torch.zeros_like(q)
    r = 0
    for i, (new, past) in enumerate(st["lens"]):
        n, r0, r = new + past, r, r + new
        if n <= 0:
            continue
        pos = torch.arange(n, device=q.device)
        slot = _slots(st["table"], torch.full_like(pos, i), pos)
        k, v = (_load(pl, slot).transpose(0, 1) for pl in (st["kp"], st["vp"]))       # (KVH, n, D)
        qi = q[r0:r].float().unflatten(1, (KVH, G)).permute(1, 0, 2, 3).reshape(KVH, new * G, D)
        s = torch.matmul(qi, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(D))
        qpos = past + torch.arange(new, device=q.device).repeat_interleave(G)
        s = torch.where(pos[None, None, :] <= qpos[None, :, None], s, float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(p, v.contiguous()) / p.sum(-1, keepdim=True)
        out[r0:r] = o.view(KVH, new, G, D).permute(1, 0, 2, 3).reshape(new, KVH * G, D).to(torch.bfloat16)
    return out


# ------------------------------------------------------------------------------------------------ measured calls


def prepare(case, seed):
    x = _inputs(case, seed)
    D, KVH = case["head_dim"], case["n_kv"]
    st = dict(x, op=case["op"], D=D, KVH=KVH, H=case.get("n_head"), half=case.get("half"))
    if case["op"] == "attend":
        st["max_q"] = max(a for a, _ in x["lens"])
        st["max_kv"] = max(0, max(a + b for a, b in x["lens"]))
    if own:
        from fish_speech_amd.kv4 import KV4Cache

        st["cache"] = KV4Cache(x["n_pages"], KVH, D, device=DEV)
        if "k" in st:
            st["cache"].append(st.pop("k"), st.pop("v"), x["row_seq"], x["row_pos"], x["table"])
        return st
    n = x["n_pages"] * PAGE
    st["kp"], st["vp"] = ((torch.zeros(n, KVH, D // 2, dtype=torch.uint8, device=DEV),
                           torch.zeros(n, KVH, D // 32, dtype=torch.uint8, device=DEV)) for _ in range(2))
    if "k" in st:
        slot = _slots(x["table"], x["row_seq"], x["row_pos"])
        k, v = st.pop("k"), st.pop("v")
        for o in range(0, slot.numel(), 32768):
            _store(st["kp"], k[o:o + 32768], slot[o:o + 32768])
            _store(st["vp"], v[o:o + 32768], slot[o:o + 32768])
    return st


def run(st):
    if not own:
        return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend}[st["op"]](st)
    cache, table = st["cache"], st["table"]
    if st["op"] == "attend":
        return cache.attend(st["q"], st["q_start"], st["kv_len"], table, max_q=st["max_q"], max_kv=st["max_kv"])
    if st["op"] == "read":
        return cache.read(st["read_seq"], st["read_pos"], table)
    q, k, v = st["qkv"].unflatten(-1, (-1, st["D"])).split([st["H"], st["KVH"], st["KVH"]], dim=1)
    q = cache.append(k, v, st["row_seq"], st["row_pos"], table, q=q, rope=st["rope"],
                     rope_layout="half" if st["half"] else "interleaved", q_norm=st.get("q_norm"),
                     k_norm=st.get("k_norm"), eps=1e-6)
    return (q, *cache.read(st["row_seq"], st["row_pos"], table))


def work(case):
    D, KVH, L = case["head_dim"], case["n_kv"], _lengths(case)
    stored = 2 * KVH * (D // 2 + D // 32)                # bytes of one token in the cache
    rows = sum(a for a, _ in L)
    if case["op"] == "attend":
        H = case["n_head"]
        keys = sum(max(0, a + b) for a, b in L)
        pairs = sum(sum(range(max(0, b + 1), a + b + 1)) for a, b in L)
        return {"bytes": keys * stored + 2 * rows * H * D * 2, "flops": 4 * H * D * pairs}
    if case["op"] == "read":
        return {"bytes": rows * (stored + 4 * KVH * D), "flops": 2 * rows * KVH * D}
    H = case["n_head"]
    # q | k | v in, q out, the cache written and read back, the values out
    return {"bytes": rows * (2 * (H + 2 * KVH) * D + 2 * H * D + 2 * stored + 4 * KVH * D) +
            max(a + b for a, b in L) * case["rot"] * 2,
            "flops": rows * (6 * (H + KVH) * D + 6 * KVH * D)}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits


def _exact_stored(y):
    """What the cache gives back for bf16 values, by search over the representable values."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=y.device)
    mid = (grid[1:] + grid[:-1]) / 2
    b = y.double().reshape(*y.shape[:-1], y.shape[-1] // 32, 32)
    top = b.abs().max(dim=-1, keepdim=True).values
    e = torch.ceil(torch.log2(top.clamp(min=7 * 2.0 ** -100) / 7))
    # the logarithm may land beside an integer: settle it by comparison
    e = torch.where(top > 7 * 2.0 ** e, e + 1, e)
    e = torch.where((top <= 7 * 2.0 ** (e - 1)) & (e > -100), e - 1, e)
    a = b.abs() / 2.0 ** e
    up, down = torch.searchsorted(mid, a, right=True), torch.searchsorted(mid, a, right=False)
    idx = torch.where(up == down, up, torch.where(up % 2 == 0, up, down))      # on a border: the even code
    return (torch.sign(b) * grid[idx] * 2.0 ** e).reshape(y.shape)


def exact(case, seed):
    x = _inputs(case, seed)
    D, KVH = case["head_dim"], case["n_kv"]
    f64, f32, bf = torch.float64, torch.float32, torch.bfloat16
    if case["op"] == "append":
        H, half = case["n_head"], case["rot"] // 2
        rows = x["qkv"].view(-1, H + 2 * KVH, D)
        done = []
        for part, w in ((rows[:, :H], x.get("q_norm")), (rows[:, H:H + KVH], x.get("k_norm"))):
            y = part.to(f64)
            if w is not None:      # the definition rounds the reciprocal norm and each product to 32 bits, the value to bf16
                rs = torch.rsqrt(y.square().sum(-1, keepdim=True) / D + 1e-6).to(f32).to(f64)
                y = ((y * rs).to(f32).to(f64) * w.to(f64)).to(f32).to(bf).to(f64)
            cos, sin = x["rope"].to(f64)[x["row_pos"].long()].unbind(-1)
            out = y.clone()
            for i in range(half):
                i0, i1 = (i, i + half) if case["half"] else (2 * i, 2 * i + 1)
                c, s = cos[:, i, None], sin[:, i, None]
                out[:, :, i0] = y[:, :, i0] * c - y[:, :, i1] * s
                out[:, :, i1] = y[:, :, i1] * c + y[:, :, i0] * s
            done.append(out)
        q, k = done
        k = k.to(f32).to(bf)       # rounded through 32 bits like the rotation's definition
        return q, _exact_stored(k), _exact_stored(rows[:, H + KVH:])
    if case["op"] == "read":
        want = torch.cat([torch.arange(a + b, device=DEV) >= b for a, b in x["lens"]])
        return _exact_stored(x["k"][want]), _exact_stored(x["v"][want])
    H = case["n_head"]
    G = H // KVH
    out = torch.zeros(x["q"].shape, dtype=f64, device=DEV)
    row = key = 0
    for new, past in x["lens"]:
        n = max(0, new + past)
        k, v = _exact_stored(x["k"][key:key + n]), _exact_stored(x["v"][key:key + n])
        q = x["q"][row:row + new].to(f64)
        hidden = torch.arange(n, device=DEV)[None, :] > past + torch.arange(new, device=DEV)[:, None]
        for h in range(H if n > 0 else 0):
            s = (q[:, h] @ k[:, h // G].T) / D ** 0.5
            s[hidden] = -math.inf
            out[row:row + new, h] = torch.softmax(s, dim=-1) @ v[:, h // G]
        row, key = row + new, key + n
    return out

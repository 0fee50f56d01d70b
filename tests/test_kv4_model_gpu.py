"""The Dual-AR model with its slow K/V cache in 4 bits (MiDualAR.setup_caches(kv_bits=4)) against the CPU oracle with the
same stored values, and the invariances the bf16 cache has: batch, graph, prefix reuse, slots."""
import pytest
import torch

from oracle import dual_ar as O
from oracle import kv4 as K4
from tests.helpers import load_dualar_case

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


class _Stored:
    """A K or V cache of the oracle that keeps what the 4-bit format makes of the values written into it."""

    def __init__(self, t):
        self.t = t

    def __setitem__(self, key, val):
        self.t[key] = K4.stored(val).to(self.t.dtype)

    def repeat_interleave(self, *a, **k):
        return self.t.repeat_interleave(*a, **k)


def _oracle(cfg, state, kv4):
    o = O.DualAROracle(cfg, state)
    o.setup_caches(1, cfg.max_seq_len)
    if kv4:
        o.kv = [(_Stored(k), _Stored(v)) for k, v in o.kv]
    return o


def _model(cfg, state, max_batch=4):
    from fish_speech_amd.dual_ar import MiDualAR

    m = MiDualAR.from_state_dict(cfg, state, device=DEV, im_end_id=cfg.im_end_id)
    m.setup_caches(max_batch, cfg.max_seq_len, kv_bits=4)
    return m


def _cfg(kind, max_seq):
    from oracle.search_golden import MID

    return O.DualARConfig(**dict(MID if kind == "mid" else {}, max_seq_len=max_seq))


@pytest.mark.parametrize("kind, T", [("tiny", 1), ("tiny", 40), ("mid", 70), ("mid", 700)])
def test_prompt_and_decode_positions_match_the_oracle_with_stored_keys_and_values(kind, T):
    """Logits and hidden state of a prompt and of three teacher-forced positions.  The distance to the oracle that stores
    the same 4-bit values stays well below what storing them changes (a code flips only where a bf16 rounding of the
    projection falls on a border, a fraction of a percent of them), the layer-0 cache agrees but for such flips."""
    cfg = _cfg(kind, 1024 if T > 100 else 256)
    state = O.make_synthetic_state(cfg, seed=8, head_gain=8.0)
    model = _model(cfg, state, 1)
    o4, o16 = _oracle(cfg, state, True), _oracle(cfg, state, False)
    ncb1 = cfg.num_codebooks + 1
    p = O.make_prompt(cfg, T, seed=T, n_semantic=T // 2)
    g = torch.Generator().manual_seed(T)
    frames = torch.zeros(3, ncb1, dtype=torch.int64)
    frames[:, 1:] = torch.randint(0, cfg.codebook_size, (3, cfg.num_codebooks), generator=g)
    frames[:, 0] = frames[:, 1] + cfg.semantic_begin_id
    ids = model._table(1, torch.int32).view(-1).long().cpu()
    calls = [(p.view(1, ncb1, -1), torch.arange(T))] + [(frames[i].view(1, ncb1, 1), torch.tensor([T + i])) for i in range(3)]
    err, effect = 0.0, 0.0
    for x, pos in calls:
        r = model.forward_generate(x.to(DEV), pos.to(DEV))
        w4, w16 = o4.forward_generate(x, pos, math_backend=True), o16.forward_generate(x, pos, math_backend=True)
        for got, a, b in ((r.logits[0, 0].float().cpu()[ids], w4[0][0, 0].float()[ids], w16[0][0, 0].float()[ids]),
                          (r.hidden_states.float().cpu().view(-1), w4[1].float().view(-1), w16[1].float().view(-1))):
            err = max(err, float((got - a).norm() / a.norm()))
            effect = max(effect, float((b - a).norm() / a.norm()))
    print(kind, T, err, effect)
    assert err <= 0.5 * effect, (err, effect)
    k, v = model.read_kv4(0, 0, T + 3)
    for got, want in ((k, o4.kv[0][0].t), (v, o4.kv[0][1].t)):
        same = (got.cpu().float() == want[0, :, :T + 3].transpose(0, 1).float()).float().mean()
        assert same >= 0.98, same


def test_batch_graph_and_eager_agree_bit_for_bit():
    """A ragged batch whose contexts span one to several key ranges equals its single runs, captured and eager."""
    from fish_speech_amd.dual_ar import generate_batch

    cfg = _cfg("mid", 2304)
    state = O.make_peaky_state(cfg, seed=93, emb_gain=2.5, slow_gain=3.0, fast_gain=2.5)
    model = _model(cfg, state, 4)
    lens = [40, 700, 505, 1300]
    prompts = [O.make_prompt(cfg, T, seed=60 + i, n_semantic=T // 3) for i, T in enumerate(lens)]
    kw = dict(max_new_tokens=14, temperature=0.7, top_p=0.7, top_k=30, stop_on_im_end=False)
    seeds = [31, 32, 33, 34]
    batch = generate_batch(model=model, prompts=prompts, seeds=seeds, **kw)
    model.set_graph(False)
    eager = generate_batch(model=model, prompts=prompts, seeds=seeds, **kw)
    model.set_graph(True)
    for i, p in enumerate(prompts):
        assert torch.equal(batch[i], eager[i]), i
        assert torch.equal(generate_batch(model=model, prompts=[p], seeds=[seeds[i]], **kw)[0], batch[i]), i


def test_ragged_prefill_rows_do_not_depend_on_their_batch():
    """Every prompt of a ragged prefill equals its own prefill next to one other prompt.  (Not alone: a call of up to 16 rows
    in all takes the decode GEMV for its projections instead of the tiled GEMM, whose sums have another order, and a
    last-bit difference of a projection can move a stored 4-bit value by a whole step.)"""
    cfg, state, _ = load_dualar_case("mid_peaky")
    model = _model(cfg, state, 5)
    lens = [1, 16, 17, 130, 47]
    prompts = [O.make_prompt(cfg, T, seed=40 + i, n_semantic=T // 3) for i, T in enumerate(lens)]
    samp = [model._sampling(0.7, 0.7, 1, 9, True) for _ in lens]
    model.prefill(list(range(5)), prompts, [4] * 5, samp)
    logits, _, hidden, _ = model.debug_taps(5)
    for i in range(5):
        model.release(i)
    mate = O.make_prompt(cfg, 33, seed=99, n_semantic=3)
    for i, p in enumerate(prompts):
        model.prefill([3, 1], [p, mate], [4, 4], [samp[i], samp[i]])
        l1, _, h1, _ = model.debug_taps(2)
        model.release(3)
        model.release(1)
        assert torch.equal(l1[0], logits[i]) and torch.equal(h1[0], hidden[i]), i


def test_prefix_reuse_equals_full_prefills():
    from fish_speech_amd.dual_ar import generate

    cfg, state, _ = load_dualar_case("mid_peaky")
    model = _model(cfg, state, 1)
    base = O.make_prompt(cfg, 170, seed=3, n_semantic=20)
    seq = [base[:, :40], base[:, :43], base[:, :170], base[:, :9], base[:, :14], base[:, :30], base[:, :30]]
    kw = dict(max_new_tokens=6, temperature=0.7, top_p=0.7, top_k=1, seed=11)
    want = [generate(model=model, prompt=p, **kw) for p in seq]
    got = [generate(model=model, prompt=p, reuse_prefix=True, **kw) for p in seq]
    model.release(0)
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), i
    assert model.reused_rows > 0


def test_finished_slots_leave_other_slots_alone():
    from fish_speech_amd.dual_ar import generate
    from tests.test_dualar_gpu import _run_slots

    cfg, state, _ = load_dualar_case("tiny_peaky")
    model = _model(cfg, state, 3)
    model.set_ignore_eos(True)
    prompts = [O.make_prompt(cfg, 30, seed=21, n_semantic=6), O.make_prompt(cfg, 65, seed=22, n_semantic=9),
               O.make_prompt(cfg, 1, seed=23)]
    max_new, seeds = [150, 64, 100], [5, 6, 7]
    got = _run_slots(model, cfg, prompts, max_new, seeds, extra_frames=9)
    for i, p in enumerate(prompts):
        alone = generate(model=model, prompt=p, max_new_tokens=max_new[i], temperature=0.7, top_p=0.7, top_k=1,
                         seed=seeds[i], stop_on_im_end=False)
        assert torch.equal(got[i][0].t().long(), alone[:, p.shape[1]:]), i


def test_setup_refusals():
    from fish_speech_amd._lib import FishmiError
    from fish_speech_amd.dual_ar import MiDualAR

    cfg, state, _ = load_dualar_case("tiny_peaky")
    model = MiDualAR.from_state_dict(cfg, state, device=DEV, im_end_id=cfg.im_end_id)
    with pytest.raises(ValueError):
        model.setup_caches(1, 64, kv_bits=8)
    model.setup_caches(1, 64, kv_bits=4)
    model.setup_caches(1, 64)                      # keeps what is there
    with pytest.raises(FishmiError, match="already set up"):
        model.setup_caches(1, 64, kv_bits=16)
    with pytest.raises(FishmiError, match="pages"):
        model.read_kv4(0, 0, 1)                    # nothing was prefilled
    with pytest.raises(FishmiError, match="layer"):
        model.read_kv4(99, 0, 0)
    other = MiDualAR.from_state_dict(cfg, state, device=DEV, im_end_id=cfg.im_end_id)
    other.setup_caches(1, 64)
    with pytest.raises(FishmiError, match="not held in 4 bits"):
        other.read_kv4(0, 0, 0)
    assert other.lib.fmi_dualar_set_kv_bits(other._h, 4) == -3
    assert other.lib.fmi_dualar_set_kv_bits(other._h, 7) == -1


def test_cli_and_worker_queue_options(tmp_path, monkeypatch):
    """--kv-bits 4 and launch_thread_safe_queue(kv_bits=4) set the model's cache up in 4 bits; without them it is bf16."""
    import numpy as np
    from click.testing import CliRunner

    from fish_speech_amd import text2semantic as T
    from tests.test_cli_gpu import _s2_checkpoint

    _s2_checkpoint(tmp_path, monkeypatch)
    models = []
    load = T.init_model

    def init_model(*a, **k):
        models.append(load(*a, **k))
        return models[-1]

    monkeypatch.setattr(T, "init_model", init_model)
    args = ["--text", "<|speaker:0|>Hello there.", "--checkpoint-path", str(tmp_path), "--device", DEV, "--max-new-tokens", "9",
            "--seed", "3", "--output-dir"]
    for name, extra, bits in (("a", ["--kv-bits", "4"], 4), ("b", [], 16)):
        r = CliRunner().invoke(T._cli(), args + [str(tmp_path / name)] + extra)
        assert r.exit_code == 0, r.output + repr(r.exception)
        codes = np.load(tmp_path / name / "codes_0.npy")
        assert codes.shape[0] == 10 and 1 <= codes.shape[1] <= 8 and codes.min() >= 0 and codes.max() < 4096
        assert models[-1][0].kv_bits == bits
    assert CliRunner().invoke(T._cli(), args + [str(tmp_path / "c"), "--kv-bits", "8"]).exit_code != 0
    queue = T.launch_thread_safe_queue(str(tmp_path), DEV, kv_bits=4)
    queue.put(None)
    assert models[-1][0].kv_bits == 4


def test_short_and_long_rows_share_the_graph_of_the_long_ones():
    """Two slots, both past the length from which rows are split, then a short one beside a long one: the second call replays
    the first one's graph (the launch count is that of the frame built last: an eager one in between)."""
    cfg = _cfg("mid", 1024)
    state = O.make_synthetic_state(cfg, seed=8, head_gain=8.0)
    model = _model(cfg, state, 3)
    model.set_ignore_eos(True)
    samp = model._sampling(0.7, 0.7, 1, 9, True)
    prompts = [O.make_prompt(cfg, T, seed=T, n_semantic=3) for T in (800, 750, 40)]
    model.prefill([0, 1, 2], prompts, [60] * 3, [samp] * 3)
    model.decode([0, 1], 2)
    split = model.last_decode_stats()[1]
    model.set_graph(False)
    model.decode([2], 1)
    single = model.last_decode_stats()[1]
    assert single < split                                          # no merge launches
    model.set_graph(True)
    model.decode([0, 2], 2)
    assert model.last_decode_stats()[1] == single                  # no frame was built
    model.synchronize()

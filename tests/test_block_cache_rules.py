"""The 8-bit cache's and the rules' host side: policies, page bookkeeping, parameters, batches (no GPU needed)."""
import math

import numpy as np
import pytest
import torch

from inference_engine_rust_b200 import EvictionPolicy, LoadedModel, SamplingError, SamplingParams
from inference_engine_rust_b200.cache import Cache, CacheError, CacheFull, KVRequest, StateRequest, parse_cache_dtype
from inference_engine_rust_b200.cache.blocks import BlockStore
from inference_engine_rust_b200.config.presets import PRESETS, preset
from inference_engine_rust_b200.engine.generate import generate, plan_batches
from inference_engine_rust_b200.sampling.sampler import pack_allowed


def test_cache_dtypes():
    assert parse_cache_dtype(None) is None and parse_cache_dtype("int8") == torch.int8 == parse_cache_dtype(torch.int8)
    assert parse_cache_dtype("float8_e4m3") == parse_cache_dtype("fp8") == torch.float8_e4m3fn
    for bad in ("int4", "bfloat16", torch.bfloat16, 8):
        with pytest.raises(ValueError, match="cache_dtype"):
            parse_cache_dtype(bad)


@pytest.mark.parametrize("kw, says", [(dict(keep=0), "keep"), (dict(keep=40), "multiple of 16"), (dict(keep=-16), "keep"), (dict(keep=32.0), "whole number"),
                                      (dict(keep=True), "whole number"), (dict(keep=32, recent=48), "recent"), (dict(keep=32, recent=8), "recent"),
                                      (dict(keep=32, every=0), "every"), (dict(keep=32, recent=16, every="8"), "whole number")])
def test_policies_that_are_refused(kw, says):
    with pytest.raises(ValueError, match=says):
        EvictionPolicy(**kw)


def test_policy():
    p = EvictionPolicy(128, every=40)
    assert p.recent == 32 and EvictionPolicy(16).recent == 0 and EvictionPolicy(16, 16).recent == 16
    assert not p.due(167, 1000) and not p.due(1000, 39) and p.due(168, 40)
    # nothing ever holds more than most_held says: any prompt, token by token
    for keep, every, prompt in [(128, 40, 1), (128, 40, 500), (16, 1, 3), (16, 100, 60), (64, 7, 130)]:
        p, held, steps, top = EvictionPolicy(keep, 0, every), prompt, 0, prompt
        for _ in range(2000):
            held, steps = held + 1, steps + 1
            top = max(top, held)
            if p.due(held, steps):
                lost = (held // 16 - keep // 16) * 16
                assert lost >= 0
                held, steps = held - lost, 0
        assert top <= p.most_held(prompt) and (every < 16 or held >= keep)


def cache(monkeypatch, policy=EvictionPolicy(64, 16, 32), max_tokens=64 * 6, **kw):
    calls = []
    monkeypatch.setattr(BlockStore, "evict", lambda self, table, slots, held, new, keep, recent, err: calls.append((list(slots), list(held), new.copy(), keep, recent)))
    c = Cache({0: KVRequest(2, 16), 1: KVRequest(2, 16)}, max_tokens=max_tokens, max_seq_len=4096, max_sequences=4, dtype=torch.float32, device="cpu",
              levels=torch.int8, eviction=policy, **kw)
    return c, calls


def grow(c, slot, n):
    c.reserve(slot, int(c.seq_lens[slot]) + n)
    c.advance(slot, n)
    c.steps_since[slot] += n


def test_pages_come_back(monkeypatch):
    c, calls = cache(monkeypatch)
    a, b = c.open_sequence(), c.open_sequence()
    grow(c, a, 150)
    grow(c, b, 40)
    old = c.kv_groups[0].pages_of(a)
    c.evict([a, b], None)
    (slots, held, new, keep, recent), = calls
    assert slots == [a] and held == [150] and keep == 4 and recent == 1 and new.shape == (1, 2)
    assert c.length(a) == 64 + 150 % 16 and c.lost[a] == 150 - c.length(a) and c.steps_since[a] == 0 and c.steps_since[b] == 40
    g = c.kv_groups[0]
    assert g.pages_of(a) == new[0].tolist() == g.table_host[a, :2].tolist() and g.table_host[a, 2] == -1 and not set(new[0]) & set(old)
    c.check()
    grow(c, a, 20)
    c.check()
    assert len(g.pages_of(a)) == 2
    c.close_sequence(a)
    assert c.lost[a] == 0
    c.check()


def test_a_kept_length_that_ends_a_page_gives_the_spare_page_back(monkeypatch):
    c, calls = cache(monkeypatch)
    a = c.open_sequence()
    grow(c, a, 160)
    c.evict([a], None)
    assert c.length(a) == 64 and len(c.kv_groups[0].pages_of(a)) == 1 and calls[0][2].shape == (1, 2)
    c.check()


def test_sequences_share_a_launch_or_go_one_after_another(monkeypatch):
    c, calls = cache(monkeypatch, max_tokens=64 * 12)
    slots = [c.open_sequence() for _ in range(4)]
    for s in slots:
        grow(c, s, 100)
    c.evict(slots, None)
    assert [len(x[0]) for x in calls] == [3, 1]       # six pages free (12 + 2 - 8): three sequences of two, then the fourth
    c.check()
    assert all(c.length(s) == 64 + 100 % 16 for s in slots)


def test_room_for_the_copies_is_kept(monkeypatch):
    c, calls = cache(monkeypatch, max_tokens=64 * 4)
    a, b = c.open_sequence(), c.open_sequence()
    grow(c, a, 128)
    grow(c, b, 128)
    with pytest.raises(CacheFull, match="0 of 4 free"):
        c.reserve(b, 129)
    c.evict([a, b], None)
    assert [len(x[0]) for x in calls] == [1, 1]
    c.check()
    c.reserve(b, 129)


def test_misuse(monkeypatch):
    c, _ = cache(monkeypatch)
    with pytest.raises(CacheError, match="appears twice"):
        c.kv_groups[0].evict([0, 0], [100, 100], None)
    plain = Cache({0: KVRequest(2, 16)}, max_tokens=64, max_seq_len=64, max_sequences=1, dtype=torch.float32, device="cpu", levels=torch.int8)
    with pytest.raises(CacheError, match="without an eviction policy"):
        plain.kv_groups[0].evict([0], [64], None)
    kw = dict(max_tokens=64, max_seq_len=4096, max_sequences=1, dtype=torch.float32, device="cpu")
    for req, more, says in [(KVRequest(2, 16), dict(eviction=EvictionPolicy(16)), "needs an 8-bit cache"),
                            (KVRequest(2, 16, window=32), dict(eviction=EvictionPolicy(16), levels=torch.int8), "have a window"),
                            (KVRequest(2, 16, values=False), dict(levels=torch.int8), "keys and values"),
                            (KVRequest(2, 16, chunk=32), dict(levels=torch.int8), "keys and values"),
                            (KVRequest(2, 16, window=32, keep=4), dict(levels=torch.int8), "keys and values"),
                            (KVRequest(2, 16), dict(levels=torch.int8, page_tokens=24), "multiple of 16")]:
        with pytest.raises(ValueError, match=says):
            Cache({0: req}, **kw, **more)


def test_bytes_of_a_cache_in_8_bits():
    kw = dict(max_tokens=64, max_seq_len=64, max_sequences=1, dtype=torch.bfloat16, device="cpu")
    wide = Cache({0: KVRequest(8, 128)}, **kw).kv_groups[0].bytes_per_token()
    for levels in (torch.int8, torch.float8_e4m3fn):
        g = Cache({0: KVRequest(8, 128)}, levels=levels, **kw).kv_groups[0]
        assert g.bytes_per_token() == 8 * (2 * 128 + 0.5) and g.bytes_per_token() / wide < 0.502


def test_models_that_do_not_run_over_such_a_cache():
    for name in sorted(PRESETS):
        if "sizes" in name or name.startswith(("7b", "nemo")):
            continue
        from inference_engine_rust_b200 import config_from_dict
        model = LoadedModel._build(config_from_dict(preset(name)), "float32", "cpu", False)
        if name in ("tiny-a", "tiny-b"):
            model.check_block_cache(False)
            model.check_block_cache(True)         # (a window is the cache's to refuse)
        else:
            with pytest.raises(ValueError, match="8-bit cache|state per sequence"):
                model.check_block_cache(False) or model.check_block_cache(True)


@pytest.mark.parametrize("kw, says", [(dict(repetition_penalty=0), "repetition_penalty"), (dict(repetition_penalty=-1.0), "positive"),
                                      (dict(repetition_penalty=math.inf), "finite"), (dict(presence_penalty=math.nan), "presence"),
                                      (dict(frequency_penalty="1"), "frequency"), (dict(frequency_penalty=True), "frequency"),
                                      (dict(logit_bias={1: math.nan}), "finite or -infinity"), (dict(logit_bias={1: math.inf}), "finite or -infinity"),
                                      (dict(logit_bias={-1: 1.0}), "must be >= 0"), (dict(logit_bias={"a": 1.0}), "token ids"),
                                      (dict(logit_bias={1.5: 1.0}), "token ids"), (dict(logit_bias=[(1, 2.0), (1, 3.0)]), "appears twice"),
                                      (dict(logit_bias=[3]), "token ids")])
def test_parameters_that_are_refused(kw, says):
    with pytest.raises(SamplingError, match=says):
        SamplingParams(**kw)


def test_parameters():
    assert not SamplingParams().penalized and SamplingParams(frequency_penalty=-0.1).penalized
    p = SamplingParams(logit_bias={3: -math.inf, np.int64(5): 1})
    assert p.logit_bias == ((3, -math.inf), (5, 1.0)) and not p.penalized and hash(p) is not None


def test_masks():
    words = pack_allowed([None, [0, 31, 32, 69], np.arange(70) % 2 == 0, torch.arange(70) == 33, range(2, 4)], 70).view(np.uint32)
    assert words.shape == (5, 3) and (words[0] == 0xFFFFFFFF).all()
    bits = (words[:, :, None] >> np.arange(32, dtype=np.uint32) & 1).reshape(5, -1)
    assert np.flatnonzero(bits[1]).tolist() == [0, 31, 32, 69] and np.flatnonzero(bits[2]).tolist() == list(range(0, 70, 2))
    assert np.flatnonzero(bits[3]).tolist() == [33] and np.flatnonzero(bits[4]).tolist() == [2, 3]
    for bad, says in [([70], "ids in"), ([-1], "ids in"), ([1.5], "ids in"), (np.ones(71, bool), "length"), ([], "no token"), (np.zeros(70, bool), "no token")]:
        with pytest.raises(SamplingError, match=says):
            pack_allowed([bad], 70)


def test_batches_of_sequences_that_lose_positions():
    p = EvictionPolicy(64, 16, 32)
    kw = dict(max_tokens=384, max_sequences=8, max_seq_len=10000, page_tokens=64, most_held=p.most_held, capacity=384)
    assert plan_batches([10, 10, 10, 10], 5000, **kw) == [[0, 1, 2], [3]]             # at most 111 positions each: two pages
    assert plan_batches([10] * 4, 20, **kw) == [[0, 1, 2, 3]]
    assert plan_batches([300, 10], 5000, **kw) == [[0], [1]]
    with pytest.raises(ValueError, match="comes to hold 385"):
        plan_batches([353], 5000, **kw)


class Scripted:
    """An engine that gives a step's rows their number; what the sampler is told is recorded."""

    def __init__(self):
        self.opened = 0

    def open_sequence(self):
        self.opened += 1
        return self.opened

    def close_sequence(self, slot):
        pass

    def step(self, entries, want="last"):
        return len(entries)


def test_allowed_tokens_and_histories_reach_the_sampler():
    began, seen = [], []

    class Choose:
        def begin(self, ids, prompts, new):
            began.append((ids, prompts, new))

        def __call__(self, logits, ids, steps, allowed=None):
            seen.append((ids, steps, allowed))
            return [7 + s for s in steps]
    generate(Scripted(), Choose(), [[1], [2, 3], [4]], 2, max_tokens=128, max_sequences=2, max_seq_len=64, page_tokens=64,
             request_ids=[5, 6, 9], allowed_tokens=lambda r, answer: (r, tuple(answer)))
    assert began == [([5, 6], [[1], [2, 3]], 2), ([9], [[4]], 2)]
    assert seen == [([5, 6], [0, 0], [(5, ()), (6, ())]), ([5, 6], [1, 1], [(5, (7,)), (6, (7,))]), ([9], [0], [(9, ())]), ([9], [1], [(9, (7,))])]


def test_command_line_refusals(capsys):
    from inference_engine_rust_b200 import cli
    for more, says in [(["--repetition-penalty", "0"], "repetition_penalty"), (["--logit-bias", "x:1"], "invalid literal"), (["--logit-bias", "5"], "could not convert"),
                       (["--evict-to", "32"], "--cache-dtype"), (["--evict-recent", "16"], "--evict-to"),
                       (["--cache-dtype", "int8", "--evict-to", "33"], "multiple of 16")]:
        assert cli.main(["--random", "tiny-b", *more, "1 2 3"]) == 2
        assert says in capsys.readouterr().err


def test_state_requests_are_left_alone():
    c = Cache({0: StateRequest((4,)), 1: KVRequest(1, 16)}, max_tokens=64, max_seq_len=64, max_sequences=2, dtype=torch.float32, device="cpu", levels=torch.int8)
    assert c.layer_view(0).state.shape == (2, 4) and c.layer_view(1).blocks is None and c.kv_groups[0].k is None

"""A whole model over the 8-bit cache, with and without eviction, and generation with penalties, biases and masks: through the public
entry points, against plain decoding (tests/plain/block_decoder.py).

Tolerance.  Two runs whose keys differ by a little may put a number on either side of a border between two levels: a difference d
before the rounding to levels of distance s becomes s with probability d / s (d < s), so its mean square grows from d^2 to d s.
In a float32 run d is about 2^-22 of a number x and s up to 2^-3 x (e4m3: three digits of mantissa) or 1/127 of the block's largest, which
is about 2^-5.5 x: the noise is 2^-12.5 x, far below what the bfloat16 rule of helpers.py allows, which serves here.  In a bfloat16
run d is about 2^-8 x, the noise of a key or value 2^-5.75 x (e4m3; s = 2^-3.5 x on average) or 2^-6.7 x (int8) in place of the 2^-8 x that
rule is made for: it is widened by those factors, 4.8 and 2.5."""
import numpy as np
import pytest
import torch

from helpers import TINY_B, TOL, make_folder, plain_weights, prompts_for
from helpers import compare as compare_as
from plain import mistral_plain as P
from plain.block_decoder import BlockDecoder

pytestmark = pytest.mark.gpu

# heads of 64 and 128 (the tensor-core kernel), of 32 (the plain one); a window that ends inside a block
CONFIGS = {
    "d64": dict(TINY_B, hidden_size=64, num_attention_heads=4, num_key_value_heads=2, head_dim=64),
    "d128": dict(TINY_B, hidden_size=96, num_attention_heads=10, num_key_value_heads=1, head_dim=128, num_hidden_layers=2),
    "d32": dict(TINY_B),
    "window": dict(TINY_B, hidden_size=64, num_attention_heads=4, num_key_value_heads=4, head_dim=64, sliding_window=40),
}


WIDER = {"float32": {"int8": 1.0, "float8_e4m3": 1.0}, "bfloat16": {"int8": 2.5, "float8_e4m3": 4.8}}


def compare(got, ref, what="", dtype="float32", fmt="int8"):
    rule = {k: v * WIDER[dtype][fmt] for k, v in TOL["bfloat16"].items()}
    TOL["levels"] = rule
    try:
        compare_as(got, ref, "levels", what)
    finally:
        del TOL["levels"]


def load(tmp_path, cfg, dtype="float32", **kw):
    from inference_engine_rust_b200 import LoadedModel
    folder = make_folder(tmp_path, cfg, seed=2, dtype=dtype)
    return LoadedModel.load(folder, dtype=dtype, **kw), plain_weights(folder)


def rounding(dtype):
    return P.bf16_rounding if dtype == "bfloat16" else P.no_rounding


@pytest.mark.parametrize("fmt", ["int8", "float8_e4m3"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", sorted(CONFIGS))
@pytest.mark.parametrize("graphs", [False, True])
def test_steps_against_plain_decoding(tmp_path, name, dtype, fmt, graphs):
    cfg = CONFIGS[name]
    model, w = load(tmp_path, cfg, dtype)
    session = model.session(max_tokens=64 * 12, cache_dtype=fmt, use_graphs=graphs, poison_cache=True)
    prompts = prompts_for(cfg, [5, 37, 90], seed=1)
    plain = [BlockDecoder(cfg, w, fmt, rounding(dtype)) for _ in prompts]
    compare(session.prefill(prompts), torch.stack([d.prompt(p) for d, p in zip(plain, prompts)]), "prompts", dtype, fmt)
    g = np.random.default_rng(0)
    for i in range(20):
        toks = g.integers(0, cfg["vocab_size"], size=3).tolist()
        compare(session.decode_tokens(toks), torch.stack([d.step(t) for d, t in zip(plain, toks)]), f"step {i}", dtype, fmt)
    session.engine.check_device()
    session.engine.cache.check()


@pytest.mark.parametrize("plain_kernels", [False, True])
def test_the_plain_kernels_too(tmp_path, plain_kernels):
    cfg = CONFIGS["d64"]
    model, w = load(tmp_path, cfg, plain_kernels=plain_kernels)
    session = model.session(max_tokens=64 * 4, cache_dtype="int8")
    d = BlockDecoder(cfg, w, "int8")
    prompt = prompts_for(cfg, [30], seed=3)[0]
    compare(session.prefill([prompt])[0], d.prompt(prompt))
    for t in prompts_for(cfg, [10], seed=4)[0]:
        compare(session.decode_tokens([t])[0], d.step(t))


@pytest.mark.parametrize("name, fmt", [("d64", "int8"), ("d128", "float8_e4m3"), ("d32", "int8")])
@pytest.mark.parametrize("graphs", [False, True])
def test_eviction_against_plain_decoding(tmp_path, name, fmt, graphs):
    """Two conversations, one with a prompt beyond the bound, far past what the cache could hold: every step's logits, what is held,
    pages given back."""
    cfg = CONFIGS[name]
    model, w = load(tmp_path, cfg)
    keep, recent, every = 48, 16, 24
    session = model.session(max_tokens=64 * 5, cache_dtype=fmt, use_graphs=graphs, evict_to=keep, evict_recent=recent, evict_every=every,
                            poison_cache=True)
    engine = session.engine
    prompts = prompts_for(cfg, [100, 7], seed=1)
    plain = [BlockDecoder(cfg, w, fmt) for _ in prompts]
    compare(session.prefill(prompts), torch.stack([d.prompt(p) for d, p in zip(plain, prompts)]), "prompts")
    g = np.random.default_rng(0)
    went_back = 0
    for i in range(150):
        toks = g.integers(0, cfg["vocab_size"], size=2).tolist()
        compare(session.decode_tokens(toks), torch.stack([d.step(t) for d, t in zip(plain, toks)]), f"step {i}")
        went_back += sum(d.evict(keep, recent, every) for d in plain)
        for slot, d in zip(session._slots, plain):
            assert engine.length(slot) == d.held <= max(100, keep + 15) + every and engine.length(slot) + engine.cache.lost[slot] == d.pos
        engine.cache.check()
    assert went_back >= 8
    engine.check_device()
    session.reset()
    engine.cache.check()
    assert engine.cache.kv_groups[0].pages.free_count == engine.cache.kv_groups[0].n_pages
    # a slot that is used again starts afresh
    d = BlockDecoder(cfg, w, fmt)
    p = prompts_for(cfg, [20], seed=5)[0]
    compare(session.prefill([p])[0], d.prompt(p))
    compare(session.decode_tokens([3])[0], d.step(3))


def test_generation_with_eviction_goes_past_the_cache(tmp_path):
    """200 new tokens in a cache of 192 positions; the device ahead of the host or not, alone or beside another request."""
    cfg = CONFIGS["d64"]
    model, _ = load(tmp_path, cfg)
    kw = dict(cache_dtype="int8", evict_to=32, evict_every=32)
    prompts = prompts_for(cfg, [60, 9], seed=2)
    outs = []
    for ahead in (True, False):
        session = model.session(max_tokens=64 * 4, **kw)
        outs.append(session.generate(prompts, max_new_tokens=200, stop_ids=[], run_ahead=ahead))
        assert [len(o) for o in outs[-1]] == [200, 200]
    assert outs[0] == outs[1]
    # the longest a sequence may grow ends it, lost positions included
    res = model.session(max_tokens=64 * 4, max_seq_len=150, **kw).generate(prompts[1:], max_new_tokens=400, stop_ids=[], full=True)[0]
    assert res.finish_reason == "context" and len(res.tokens) == 150 - 9 + 1
    with pytest.raises(ValueError, match="comes to hold"):
        model.session(max_tokens=64, **kw).generate([list(range(60))], max_new_tokens=100)


def test_a_step_beyond_the_model_s_longest_position_is_refused(tmp_path):
    from inference_engine_rust_b200.cache import CacheFull
    cfg = dict(CONFIGS["d64"], max_position_embeddings=100)
    model, _ = load(tmp_path, cfg)
    session = model.session(max_tokens=64 * 3, cache_dtype="int8", evict_to=16, evict_every=16)
    session.prefill([[1] * 40])
    for _ in range(60):
        session.decode_tokens([2])
    with pytest.raises(CacheFull, match="evicted ones included"):
        session.decode_tokens([2])


def test_a_full_pool_leaves_room_for_evictions(tmp_path):
    """Prompts fill every page that the session was made with: evictions still have pages for what is kept."""
    cfg = CONFIGS["d64"]
    model, w = load(tmp_path, cfg)
    session = model.session(max_tokens=64 * 6, cache_dtype="int8", evict_to=64, evict_recent=16, evict_every=20)
    prompts = prompts_for(cfg, [108, 108, 108], seed=3)
    plain = [BlockDecoder(cfg, w, "int8") for _ in prompts]
    session.prefill(prompts)
    for d, p in zip(plain, prompts):
        d.prompt(p)
    for i in range(45):
        compare(session.decode_tokens([i, i + 1, i + 2]), torch.stack([d.step(i + j) for j, d in enumerate(plain)]), f"step {i}")
        for d in plain:
            d.evict(64, 16, 20)
        session.engine.cache.check()
    session.engine.check_device()


# ---------------------------------------------------------------------------------------
# rules on logits in generation


def ruled(logits, prompt, answer, rep, pres, freq, bias, allowed=None):
    x = logits.double().clone()
    for t in set(prompt) | set(answer):
        x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
    for t in set(answer):
        x[t] -= freq * answer.count(t) + pres
    for t, b in bias.items():
        x[t] += b
    if allowed is not None:
        keep = torch.zeros(len(x), dtype=torch.bool)
        keep[list(allowed)] = True
        x[~keep] = float("-inf")
    return x


@pytest.mark.parametrize("ahead", [True, False])
@pytest.mark.parametrize("rules", [dict(repetition_penalty=1.3), dict(presence_penalty=0.7, frequency_penalty=0.4),
                                   dict(repetition_penalty=0.8, presence_penalty=-0.2, frequency_penalty=0.1, logit_bias={3: 1.5, 7: float("-inf"), 250: -2.0})])
def test_generation_with_penalties_and_biases(tmp_path, rules, ahead):
    cfg = CONFIGS["d64"]
    model, _ = load(tmp_path, cfg)
    prompts = prompts_for(cfg, [5, 23, 11], seed=4)
    got = model.session(max_tokens=64 * 6).generate(prompts, max_new_tokens=30, stop_ids=[], run_ahead=ahead, max_batch=2, request_ids=[40, 7, 19], **rules)
    session = model.session(max_tokens=64 * 6)
    for prompt, answer in zip(prompts, got):
        logits, so_far = session.prefill([prompt])[0], []
        for tok in answer:
            x = ruled(logits.cpu(), prompt, so_far, rules.get("repetition_penalty", 1.0), rules.get("presence_penalty", 0.0),
                      rules.get("frequency_penalty", 0.0), rules.get("logit_bias", {}))
            # the best in 64 bits, or as good up to fp32's roundings (and those of a batch of another size)
            assert x[tok] >= x.max() - 2e-4 * max(1.0, float(x[torch.isfinite(x)].abs().max())), (tok, int(x.argmax()))
            so_far.append(tok)
            logits = session.decode_tokens([tok])[0]
        session.reset()


def test_sampled_generation_with_penalties_is_the_same_ahead_and_behind(tmp_path):
    cfg = CONFIGS["d64"]
    model, _ = load(tmp_path, cfg)
    prompts = prompts_for(cfg, [5, 23], seed=4)
    kw = dict(max_new_tokens=40, stop_ids=[], temperature=0.9, seed=3, repetition_penalty=1.2, frequency_penalty=0.3, logit_bias={9: float("-inf")})
    a, b = (model.session(max_tokens=64 * 4).generate(prompts, run_ahead=r, **kw) for r in (True, False))
    alone = [model.session(max_tokens=64 * 4).generate([p], request_ids=[i], **kw)[0] for i, p in enumerate(prompts)]
    assert a == b and [len(x) for x in a] == [40, 40] and all(9 not in x for x in a)
    assert [x[:3] for x in alone] == [x[:3] for x in a]        # (another batch size rounds its logits differently in the long run)


def test_generation_under_a_grammar(tmp_path):
    """Ids in steps of one modulo 5, by a list, a mask and a boolean array in turn; stop ids still end an answer."""
    cfg = CONFIGS["d64"]
    model, _ = load(tmp_path, cfg)
    vocab = cfg["vocab_size"]
    prompts = prompts_for(cfg, [5, 23], seed=4)
    asked = []

    def allowed(request, answer):
        asked.append((request, len(answer)))
        ids = [t for t in range(vocab) if t % 5 == len(answer) % 5]
        if request == 0:
            return ids
        mask = np.zeros(vocab, dtype=bool)
        mask[ids] = True
        return mask if len(answer) % 2 else torch.from_numpy(mask)
    out = model.session(max_tokens=64 * 4).generate(prompts, max_new_tokens=12, stop_ids=[], allowed_tokens=allowed, repetition_penalty=1.1)
    for answer in out:
        assert [t % 5 for t in answer] == [i % 5 for i in range(12)]
    assert (0, 0) in asked and (1, 11) in asked
    only = model.session(max_tokens=64 * 4).generate(prompts[:1], max_new_tokens=6, stop_ids=[17], temperature=0.7,
                                                     allowed_tokens=lambda r, a: [17] if len(a) == 3 else None, full=True)[0]
    assert only.finish_reason == "stop" and len(only.tokens) == 3
    from inference_engine_rust_b200 import SamplingError
    session = model.session(max_tokens=64 * 4)
    with pytest.raises(SamplingError, match="no token is allowed"):
        session.generate(prompts[:1], max_new_tokens=3, allowed_tokens=lambda r, a: [])
    with pytest.raises(SamplingError, match="outside the vocabulary"):
        session.generate(prompts[:1], max_new_tokens=3, logit_bias={vocab: 1.0})
    assert session.generate(prompts[:1], max_new_tokens=3, stop_ids=[]) != []        # nothing is left behind by a refusal


def test_an_answer_where_biases_leave_nothing_is_an_error(tmp_path):
    from inference_engine_rust_b200 import SamplingError
    model, _ = load(tmp_path, CONFIGS["d64"])
    with pytest.raises(SamplingError, match="left no token"):
        model.session(max_tokens=64).generate([[1, 2]], max_new_tokens=2, stop_ids=[], logit_bias={5: float("-inf")},
                                              allowed_tokens=lambda r, a: [5])


def test_the_command_line(capsys):
    from inference_engine_rust_b200 import cli
    base = ["--random", "tiny-b", "--seed", "3", "-n", "80", "--dtype", "float32", "--stop-token", "-1", "1 5 9"]
    assert cli.main(base + ["--cache-dtype", "int8", "--evict-to", "32", "--evict-every", "16", "--repetition-penalty", "1.2", "--logit-bias", "4:-inf"]) == 0
    ids = [int(t) for t in capsys.readouterr().out.split()]
    assert len(ids) == 80 and 4 not in ids
    assert cli.main(["--random", "tiny-a", "-n", "4", "--cache-dtype", "int8", "--evict-to", "32", "1 5 9"]) == 1
    assert "window" in capsys.readouterr().err
    assert cli.main(["--random", "vefulix-tiny", "-n", "4", "--cache-dtype", "int8", "1 5 9"]) == 1
    assert "8-bit cache" in capsys.readouterr().err

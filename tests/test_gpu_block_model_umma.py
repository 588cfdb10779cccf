"""A whole model over int8 levels with heads of 128, four to a key head, as the 7B presets have them: the sizes of the kernel on tcgen05, with the engine's
rotation, replay and eviction, against plain decoding (tolerance: see test_gpu_block_model)."""
import numpy as np
import pytest
import torch

from helpers import TINY_B, prompts_for
from plain.block_decoder import BlockDecoder
from test_gpu_block_model import compare, load, rounding

pytestmark = pytest.mark.gpu

# key heads, prompts, positions that the cache holds (all of which one sequence may take)
FEW = (2, [5, 130], 32_768)                 # few sequences that may become long: CTAs that are no clusters, and a second kernel that adds them up
MANY = (4, [3, 17, 64, 90, 33, 70, 1, 48], 64 * 32)       # clusters, or a CTA for each


def setup(tmp_path, what, dtype, **kw):
    kv_heads, lens, room = what
    cfg = dict(TINY_B, hidden_size=64, num_attention_heads=4 * kv_heads, num_key_value_heads=kv_heads, head_dim=128, num_hidden_layers=2,
               max_position_embeddings=32_768)
    model, w = load(tmp_path, cfg, dtype)
    session = model.session(max_tokens=room, max_sequences=len(lens), cache_dtype="int8", poison_cache=True, **kw)
    group = session.engine.cache.kv_groups[0]
    pairs, reach = len(lens) * kv_heads, group.ring_pages * group.page_tokens
    # the kernel's own rule: fewer pairs of sequence and key head over less are left to the one on mma.sync
    assert pairs > 24 or pairs * reach >= 120_000
    assert (pairs * 9 <= 148 and reach >= 16_384) == (what is FEW)
    prompts = prompts_for(cfg, lens, seed=1)
    return cfg, session, prompts, [BlockDecoder(cfg, w, "int8", rounding(dtype)) for _ in prompts]


@pytest.mark.parametrize("what", [FEW, MANY], ids=["few", "many"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs", [False, True])
def test_steps_against_plain_decoding(tmp_path, what, dtype, graphs):
    cfg, session, prompts, plain = setup(tmp_path, what, dtype, use_graphs=graphs)
    compare(session.prefill(prompts), torch.stack([d.prompt(p) for d, p in zip(plain, prompts)]), "prompts", dtype)
    g = np.random.default_rng(0)
    for i in range(20):
        toks = g.integers(0, cfg["vocab_size"], size=len(prompts)).tolist()
        compare(session.decode_tokens(toks), torch.stack([d.step(t) for d, t in zip(plain, toks)]), f"step {i}", dtype)
    session.engine.check_device()
    session.engine.cache.check()


@pytest.mark.parametrize("what", [FEW, MANY], ids=["few", "many"])
@pytest.mark.parametrize("graphs", [False, True])
def test_eviction_against_plain_decoding(tmp_path, what, graphs):
    keep, recent, every = 48, 16, 24
    cfg, session, prompts, plain = setup(tmp_path, what, "float32", use_graphs=graphs, evict_to=keep, evict_recent=recent, evict_every=every)
    compare(session.prefill(prompts), torch.stack([d.prompt(p) for d, p in zip(plain, prompts)]), "prompts")
    g = np.random.default_rng(0)
    went_back = 0
    for i in range(80):
        toks = g.integers(0, cfg["vocab_size"], size=len(prompts)).tolist()
        compare(session.decode_tokens(toks), torch.stack([d.step(t) for d, t in zip(plain, toks)]), f"step {i}")
        went_back += sum(d.evict(keep, recent, every) for d in plain)
        for slot, d in zip(session._slots, plain):
            assert session.engine.length(slot) == d.held and session.engine.cache.lost[slot] == d.pos - d.held
    assert went_back >= 2 * len(prompts)
    session.engine.check_device()
    session.engine.cache.check()

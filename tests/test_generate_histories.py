"""What the generation loop tells a sampler of a batch: the room its histories need."""
import pytest

from inference_engine_rust_b200.engine.generate import generate
from test_generate_loop import AheadEngine, AheadSampler


class Remembering(AheadSampler):
    """Keeps histories of the room that `begin` was told of: a prompt, the new tokens, and a row that ran in vain behind a stop token."""

    def begin(self, request_ids, prompts, max_new_tokens):
        self.told = max_new_tokens
        self.room = {r: max(map(len, prompts)) + max_new_tokens + 1 - len(p) for r, p in zip(request_ids, prompts)}

    def sample_device(self, logits, request_ids, steps):
        for r in request_ids:
            self.room[r] -= 1
            assert self.room[r] >= 0
        return super().sample_device(logits, request_ids, steps)


@pytest.mark.parametrize("run_ahead", [True, False])
@pytest.mark.parametrize("max_new_tokens", [1, 5, 39, 40, 41, 10 ** 12])
def test_histories_are_no_longer_than_a_sequence_may_grow(max_new_tokens, run_ahead):
    engine = AheadEngine(2)
    sampler = Remembering({0: [9] * 60, 1: [9, 9, 7]}, engine)
    res = generate(engine, sampler, [[1, 2, 3], [4]], max_new_tokens, stop_ids=[7], max_tokens=200, max_sequences=2, max_seq_len=40, page_tokens=20,
                   run_ahead=run_ahead)
    assert len(res[0].tokens) == min(max_new_tokens, 38) and sampler.told <= 41

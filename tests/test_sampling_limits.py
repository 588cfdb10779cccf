"""Penalties that 32 bits cannot hold are refused (no GPU needed)."""
import pytest

from inference_engine_rust_b200 import SamplingError
from inference_engine_rust_b200.sampling import SamplingParams


@pytest.mark.parametrize("kw", [dict(repetition_penalty=1e-46), dict(repetition_penalty=1e39), dict(presence_penalty=1e39), dict(frequency_penalty=-1e39),
                                dict(logit_bias={3: 1e39}), dict(repetition_penalty=10 ** 400)])
def test_penalties_and_biases_beyond_fp32(kw):
    with pytest.raises(SamplingError, match=next(iter(kw))):
        SamplingParams(**kw)


def test_the_largest_and_smallest_are_taken():
    SamplingParams(repetition_penalty=1e-44, presence_penalty=3e38, frequency_penalty=-3e38, logit_bias={1: -3e38, 2: float("-inf"), 3: -1e39})

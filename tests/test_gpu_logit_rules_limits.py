"""Penalties whose results are no numbers to choose among."""
import numpy as np
import pytest
import torch

from test_gpu_logit_rules import B, dev

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def go(x, penalties, mask=None):
    b = B()
    err, chosen = torch.zeros(1, dtype=torch.int32, device=DEV), dev([-1])
    b.logit_rules(x, None, dev([[5, 77, 77, 0]]), dev([3]), dev([0]), None, err, b.stream_ptr(), penalties=dev([penalties], torch.float32), mask=mask,
                  chosen=chosen)
    return err.item(), chosen.item()


@pytest.mark.parametrize("vocab", [640, 641])
@pytest.mark.parametrize("penalties, logit", [((1e-38, 0, 0), 20.0), ((1, -3e38, 0), 2e38), ((1, 0, -1e38), 2e38), ((1e-38, -1e38, 1), 20.0)])
def test_infinite_results_of_penalties_set_the_error_word(vocab, penalties, logit):
    """An id whose logit becomes infinity is a mistake as it is with a bias; where the mask rules it out it is none."""
    x = torch.randn(1, vocab, generator=torch.Generator().manual_seed(1)).to(DEV)
    x[0, 5], x[0, 77] = -1.0, logit
    assert go(x, penalties)[0] == B().ERR_NONFINITE_LOGIT
    mask = torch.full((1, -(-vocab // 32)), -1, dtype=torch.int32, device=DEV)
    mask[0, 77 // 32] &= np.int32(~(1 << 77 % 32)).item()
    assert go(x, penalties, mask)[0] == 0


@pytest.mark.parametrize("penalties", [(0.0, 0, 0), (-1.0, 0, 0), (float("nan"), 0, 0), (float("inf"), 0, 0), (1, float("nan"), 0), (1, float("inf"), 0),
                                       (1, 0, float("nan")), (1, 0, float("-inf")), (1, 0, 2e38)])
def test_penalties_that_are_no_numbers_set_the_error_word(penalties):
    x = torch.randn(1, 640, generator=torch.Generator().manual_seed(1)).to(DEV)
    assert go(x, penalties)[0] == B().ERR_NONFINITE_LOGIT


def test_a_result_of_minus_infinity_is_ruled_out():
    b = B()
    x = torch.zeros(1, 64, device=DEV)
    x[0, 7] = -3e38
    err, chosen = torch.zeros(1, dtype=torch.int32, device=DEV), dev([-1])
    b.logit_rules(x, None, dev([[7, 0]]), dev([1]), dev([0]), None, err, b.stream_ptr(), penalties=dev([[2.0, 0, 0]], torch.float32), chosen=chosen)
    assert err.item() == 0 and chosen.item() == 0

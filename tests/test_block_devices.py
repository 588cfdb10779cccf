"""Memory that a block kernel could not reach is refused before anything is launched (no GPU needed: the meta device stands for another one)."""
import pytest
import torch

from inference_engine_rust_b200.csrc import bindings as B
from test_block_refusals import batch, pools


@pytest.mark.parametrize("name", ["v", "k_scale", "v_scale", "tail_k", "tail_v", "page_table", "weight", "shift"])
def test_a_view_is_of_one_device(name):
    p = dict(pools(), weight=torch.zeros(3, 2, 4), shift=torch.zeros(2, dtype=torch.int32))
    B.block_view(**p)
    p[name] = p[name].to("meta")
    with pytest.raises(B.KernelError, match=f"{name} is on another device than k"):
        B.block_view(**p)


def attention(**kw):
    view = B.block_view(**pools())
    a = dict(qkv=torch.zeros(2, 8 * 16, dtype=torch.bfloat16), out=torch.zeros(2, 64, dtype=torch.bfloat16),
             scratch=torch.zeros(B.block_attention_scratch_floats(2, 4, view)), inv_freq=torch.zeros(8))
    a.update(kw)
    B.block_attention(a["qkv"], a["out"], batch(2, 2), view, 4, 1.0, a["scratch"], torch.zeros(1, dtype=torch.int32), 0,
                      rope=(a["inv_freq"], 16, B.PAIR_HALF, 1.0))


def test_every_tensor_of_a_step_is_looked_at(monkeypatch):
    seen = []

    def look(*tensors):
        seen.extend(tensors)
        raise B.KernelError("looked")
    monkeypatch.setattr(B, "_on_current_device", look)
    inv_freq = torch.zeros(8)
    with pytest.raises(B.KernelError, match="looked"):
        attention(inv_freq=inv_freq)
    assert any(t is inv_freq for t in seen)


@pytest.mark.parametrize("inv_freq", [torch.zeros(7), torch.zeros(8, dtype=torch.float64), torch.zeros(16)[::2]])
def test_frequencies_that_do_not_fit_are_refused(inv_freq):
    with pytest.raises(B.KernelError, match="frequencies must be"):
        attention(inv_freq=inv_freq)


def test_scratch_with_gaps_is_refused():
    """Its count of numbers says nothing of the memory behind its first then."""
    view = B.block_view(**pools())
    with pytest.raises(B.KernelError, match="scratch"):
        attention(scratch=torch.zeros(B.block_attention_scratch_floats(2, 4, view), 2)[:, 0])
    with pytest.raises(B.KernelError, match="scratch"):
        attention(scratch=torch.zeros(1).expand(B.block_attention_scratch_floats(2, 4, view)))

"""Rotary positions and the attention of prompts have no backward pass: a gradient that is asked for is refused, and not lost."""
import pytest
import torch


def _rope():
    import kch_b200
    rope = object.__new__(kch_b200.RotaryPositions)
    rope.c, rope.device, rope._index, rope.sections, rope._axes = 64, torch.device("cuda:0"), 0, (32,), 1
    return rope


@pytest.mark.parametrize("which", ["q", "k"])
def test_a_turn_of_tensors_that_require_a_gradient_is_refused(which):
    x = {n: torch.zeros(3, 2, 64, requires_grad=n == which) for n in "qk"}
    pos = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(NotImplementedError, match="rotate.*forward only"):
        _rope().rotate(x["q"], x["k"], pos)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):      # (the next check)
        _rope().rotate(x["q"], x["k"], pos)
    with pytest.raises(RuntimeError, match="CUDA"):
        _rope().rotate(x["q"].detach(), x["k"].detach(), pos)


@pytest.mark.parametrize("which", ["q", "k", "v", "sink"])
def test_attention_of_tensors_that_require_a_gradient_is_refused(which):
    from kch_b200 import prompt_attention
    x = {n: torch.zeros(3, 2, 64, requires_grad=n == which) for n in "qkv"}
    sink, cu = torch.zeros(2, requires_grad=which == "sink"), torch.tensor([0, 3], dtype=torch.int32)
    with pytest.raises(NotImplementedError, match="prompt_attention.*forward only"):
        prompt_attention(x["q"], x["k"], x["v"], cu, sink_logits=sink)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        prompt_attention(x["q"], x["k"], x["v"], cu, sink_logits=sink)
    with pytest.raises(RuntimeError, match="CUDA"):
        prompt_attention(*(x[n].detach() for n in "qkv"), cu, sink_logits=sink.detach())

"""`AdapterLinear.scaling` is alpha / rank, a constant of 32 bits whatever type the module's parameters are cast to."""
import copy

import pytest
import torch

import scattermoe_b200 as sm


@pytest.mark.parametrize("cast", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.to("cpu", torch.float16),
                                  lambda m: torch.nn.Sequential(m).bfloat16()[0], lambda m: copy.deepcopy(m).half().float()])
def test_scaling_keeps_its_bits(cast):
    m = sm.AdapterLinear(16, 24, 3, 24, bias=True, alpha=16)
    with torch.no_grad():
        m.scaling[1] = 0.1
    want = m.scaling.clone()
    m = cast(m)
    assert m.scaling.dtype == torch.float32 and torch.equal(m.scaling, want)
    assert m.weight.dtype == m.lora_a.dtype == m.bias.dtype
    assert "scaling" in dict(m.named_buffers()) and torch.equal(m.state_dict()["scaling"], want)


def test_other_moves_still_work():
    m = sm.AdapterLinear(16, 24, 3, 24).bfloat16().to("meta")
    assert m.scaling.device.type == "meta" and m.scaling.dtype == torch.float32
    m = m.to_empty(device="cpu")
    m.load_state_dict(sm.AdapterLinear(16, 24, 3, 24, alpha=48).state_dict())
    assert (m.scaling == 2.0).all() and m.weight.dtype == torch.bfloat16
    m.share_memory()
    assert m.scaling.is_shared()

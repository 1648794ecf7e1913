"""A forward-mode derivative is refused, never dropped: a dual tensor does not say `requires_grad`, and an entry point that skips its
autograd function would hand back a result without a tangent. The launchers are replaced, so no kernel runs."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import scattermoe_b200 as sm
from scattermoe_b200 import _lib, adapters, few_token


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    monkeypatch.setattr(_lib, "on_device", lambda t: True)
    monkeypatch.setattr(few_token, "_mlp_impl", lambda x, up, down, *a, **k: x.new_zeros(x.size(0), down.size(2)))
    monkeypatch.setattr(few_token, "_route_impl", lambda x, wr, br, k, *a: (x.new_zeros(x.size(0), k), torch.zeros(x.size(0), k, dtype=torch.int64)))
    monkeypatch.setattr(adapters, "_forward_impl", lambda x, w, *a: (x.new_zeros(x.size(0), w.size(0)), None, None, None))


IDS = torch.zeros(2, 1, dtype=torch.int64)
LAYER = dict(inputs=torch.ones(2, 8), up_weights=torch.ones(3, 8, 8), down_weights=torch.ones(3, 8, 8), gates=torch.ones(2, 1),
             up_biases=torch.ones(3, 8), down_biases=torch.ones(3, 8))
MOE = dict(inputs=torch.ones(2, 8), router_weight=torch.ones(3, 8), up_weights=torch.ones(3, 8, 8), down_weights=torch.ones(3, 8, 8),
           router_bias=torch.ones(3), up_biases=torch.ones(3, 8), down_biases=torch.ones(3, 8))
ADAPTER = dict(inputs=torch.ones(2, 8), weight=torch.ones(4, 8), lora_a=torch.ones(3, 2, 8), lora_b=torch.ones(3, 4, 2), bias=torch.ones(4),
               scaling=torch.ones(3))
CALLS = {"few_token_mlp": (LAYER, lambda **k: sm.few_token_mlp(expert_idxs=IDS, act_layout=0, act=0, **k)),
         "few_token_moe": (MOE, lambda **k: sm.few_token_moe(k=1, act_layout=0, act=0, **k)),
         "adapter_linear": (ADAPTER, lambda **k: sm.adapter_linear(adapter_idxs=IDS[:, 0], **k))}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("entry,name", [(e, n) for e, (args, _) in CALLS.items() for n in args])
def test_a_tangent_is_refused(entry, name, grad):
    """On every operand, and under no_grad as well, which does not switch forward mode off."""
    args, call = CALLS[entry]
    call(**args)
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        call(**args)                     # no operand has a tangent
        with pytest.raises(RuntimeError, match="%s.*forward-mode" % entry):
            call(**{**args, name: fwAD.make_dual(args[name], torch.ones_like(args[name]))})


def test_decode_refuses_a_tangent():
    m = sm.mlp.GLUMLP(8, 8, 3, 1)
    x, p = torch.ones(2, 8), torch.ones(2, 1)
    m.decode(x, p, IDS)
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        m.decode(fwAD.make_dual(x, x), p, IDS)


def test_reverse_mode_is_what_it_was():
    """Gradients of the adapters go through the autograd function; the layer refuses them."""
    x = torch.ones(2, 8, requires_grad=True)
    assert sm.adapter_linear(adapter_idxs=IDS[:, 0], **{**ADAPTER, "inputs": torch.ones(2, 8)}).grad_fn is None
    with pytest.raises(RuntimeError, match="no backward"):
        sm.few_token_mlp(expert_idxs=IDS, act_layout=0, act=0, **{**LAYER, "inputs": x})

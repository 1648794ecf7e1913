"""Refusals of the few-token layer and of the adapters that need no GPU: the C entry points' argument checks and the Python ones."""
import pytest
import torch

import scattermoe_b200 as sm
from scattermoe_b200 import _lib


def mlp_args(**kw):
    """smoe_few_token_mlp's arguments for a small valid call on pointers that are never read."""
    a = dict(X=256, T=4, sxm=64, W1=256, w1e=64 * 128, w1k=1, w1n=64, b1=None, b1e=0, b1n=0, W2=256, w2e=64 * 64, w2k=1, w2n=64,
             b2=None, b2e=0, b2n=0, gates=256, sgt=2, sgk=1, gdt=1, ids=256, sit=2, sik=1, Y=256, sym=64, k=2, d=64, F=64, d_out=64,
             E=4, layout=2, act=0, alpha=1.0, limit=1.0, dtype=1, flags=0, ws=256, ws_bytes=1 << 24, status=None, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize("bad,word", [
    (dict(T=129), "at most 128"), (dict(T=-1), "tokens"), (dict(T=128, k=9), "slots"), (dict(E=0), "E=0"), (dict(E=1025), "E=1025"),
    (dict(dtype=7), "dtype"), (dict(gdt=3), "gates"), (dict(layout=4), "layout"), (dict(act=-1), "function"), (dict(F=0), "F=0"),
    (dict(d=0), "d=0"), (dict(X=None), "null"), (dict(ids=None), "null"), (dict(k=0), "k=0"), (dict(ws=264), "aligned")])
def test_few_token_mlp_refuses(bad, word):
    assert _lib.load().smoe_few_token_mlp(*mlp_args(**bad)) == _lib.SMOE_ERR_BAD_ARG
    assert word in _lib.last_error()


def test_few_token_mlp_workspace():
    lib = _lib.load()
    need = lib.smoe_few_token_workspace_bytes(4, 2, 64, 64)
    assert need > 0 and lib.smoe_few_token_workspace_bytes(-1, 2, 64, 64) == 0
    for kw in (dict(ws=None), dict(ws_bytes=need - 1)):
        assert lib.smoe_few_token_mlp(*mlp_args(**kw)) == 4 and "workspace" in _lib.last_error()
    assert lib.smoe_few_token_mlp(*mlp_args(T=0, X=None, Y=None)) == _lib.SMOE_OK      # nothing to do, nothing launched


@pytest.mark.parametrize("bad,word", [(dict(E=0), "E=0"), (dict(k=5), "k=5"), (dict(k=33, E=64), "k=33"), (dict(mode=2), "mode"),
                                      (dict(dtype=9), "dtype"), (dict(X=None), "null")])
def test_few_token_route_refuses(bad, word):
    a = dict(X=256, T=2, sxm=64, Wr=256, swm=64, br=None, sbn=0, E=4, d=64, k=2, mode=0, renorm=1, ids=256, gates=256, dtype=1, stream=None)
    assert _lib.load().smoe_few_token_route(*{**a, **bad}.values()) == _lib.SMOE_ERR_BAD_ARG
    assert word in _lib.last_error()


@pytest.mark.parametrize("bad,word", [(dict(n=0), "adapters"), (dict(n=4097), "adapters"), (dict(r=0), "rank"), (dict(r=257), "rank"),
                                      (dict(T=-1), "T=-1"), (dict(width=0), "width"), (dict(out=0), "width"), (dict(dtype=3), "dtype"),
                                      (dict(X=None), "null"), (dict(H=None), "null")])
def test_adapter_entry_points_refuse(bad, word):
    lib = _lib.load()
    forward = dict(X=256, T=4, sxm=64, W=256, swo=64, swi=1, bias=None, A=256, saa=512, saj=64, sai=1, B=256, sba=512, sbo=8, sbj=1,
                   ids=256, scaling=None, scale=1.0, Y=256, H=256, sorted_idx=None, offsets=None, n=2, width=64, out=64, r=8, dtype=1,
                   flags=0, ws=None, ws_bytes=0, status=None, stream=None)
    assert lib.smoe_adapter_forward(*{**forward, **bad}.values()) == _lib.SMOE_ERR_BAD_ARG and word in _lib.last_error()
    backward = dict(DY=256, T=4, sdy=64, X=256, sxm=64, W=256, swo=64, swi=1, A=256, saa=512, saj=64, sai=1, B=256, sba=512, sbo=8,
                    sbj=1, ids=256, scaling=None, scale=1.0, H=256, sorted_idx=256, offsets=256, DX=256, DA=256, DB=256, DW=256, Db=256, n=2,
                    width=64, out=64, r=8, dtype=1, flags=0, ws=256, ws_bytes=1 << 24, status=None, stream=None)
    assert lib.smoe_adapter_backward(*{**backward, **bad}.values()) == _lib.SMOE_ERR_BAD_ARG and word in _lib.last_error()


def test_adapter_workspaces_and_lists():
    lib = _lib.load()
    need = lib.smoe_adapter_workspace_bytes(100, 3, 64, 96, 8, 1)
    assert need > 0 and lib.smoe_adapter_workspace_bytes(-1, 3, 64, 96, 8, 1) == 0
    tail = [3, 64, 96, 8, 1, 0]
    head = [256, 100, 64, 256, 64, 1, None, 256, 512, 64, 1, 256, 768, 8, 1, 256, None, 1.0, 256, 256]
    assert lib.smoe_adapter_forward(*head, 256, 256, *tail, 256, need - 1, None, None) == 4 and "workspace" in _lib.last_error()
    assert lib.smoe_adapter_forward(*head, 256, None, *tail, 256, need, None, None) == _lib.SMOE_ERR_BAD_ARG
    head = [256, 100, 96, 256, 64, 256, 64, 1, 256, 512, 64, 1, 256, 768, 8, 1, 256, None, 1.0, 256]
    assert lib.smoe_adapter_backward(*head, 256, 256, 256, 256, 256, 256, 256, *tail, 256, need - 1, None, None) == 4
    assert lib.smoe_adapter_backward(*head, None, None, 256, 256, None, None, None, *tail, 256, need, None, None) == _lib.SMOE_ERR_BAD_ARG
    assert "sorted" in _lib.last_error()


def test_cpu_tensors_fail_loudly():
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        sm.few_token_mlp(x, torch.zeros(2, 8, 8), torch.zeros(2, 8, 8), None, torch.zeros(2, 1, dtype=torch.int64), 0, 0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        sm.few_token_moe(x, torch.zeros(2, 8), torch.zeros(2, 8, 8), torch.zeros(2, 8, 8), 1, 0, 0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        sm.adapter_linear(x, torch.zeros(4, 8), torch.zeros(1, 2, 8), torch.zeros(1, 4, 2), torch.zeros(2, dtype=torch.int64))


def test_shapes_are_checked(monkeypatch):
    """The Python checks come before any launch: run them on stand-in tensors."""
    monkeypatch.setattr(_lib, "on_device", lambda t: True)
    x, ids = torch.zeros(2, 8), torch.zeros(2, 1, dtype=torch.int64)
    up, down = torch.zeros(2, 8, 8), torch.zeros(2, 8, 8)
    ok = dict(gates=None, expert_idxs=ids, act_layout=0, act=0)
    for kw in (dict(expert_idxs=ids[:1]), dict(expert_idxs=ids[:, 0]), dict(gates=torch.zeros(2, 2)), dict(act_layout=2), dict(act=9),
               dict(up_biases=torch.zeros(2, 9)), dict(down_biases=torch.zeros(3, 8))):
        with pytest.raises(AssertionError):
            sm.few_token_mlp(x, up, down, **{**ok, **kw})
    with pytest.raises(AssertionError, match="at most 128"):
        sm.few_token_mlp(torch.zeros(129, 8), up, down, None, torch.zeros(129, 1, dtype=torch.int64), 0, 0)
    with pytest.raises(RuntimeError, match="float64"):
        sm.few_token_mlp(x.double(), up.double(), down.double(), **ok)
    with pytest.raises(RuntimeError, match="tokens are"):
        sm.few_token_mlp(x, up.half(), down, **ok)
    with pytest.raises(RuntimeError, match="not integers"):
        sm.few_token_mlp(x, up, down, **{**ok, "expert_idxs": ids.float()})
    with pytest.raises(RuntimeError, match="no backward"):
        sm.few_token_mlp(x.requires_grad_(), up, down, **ok)
    x = x.detach()
    for kw in (dict(k=3), dict(k=0), dict(mode="nope"), dict(router_weight=torch.zeros(3, 8)), dict(router_bias=torch.zeros(3))):
        with pytest.raises(AssertionError):
            sm.few_token_moe(**{**dict(inputs=x, router_weight=torch.zeros(2, 8), up_weights=up, down_weights=down, k=1, act_layout=0, act=0), **kw})
    a = dict(inputs=x, weight=torch.zeros(4, 8), lora_a=torch.zeros(3, 2, 8), lora_b=torch.zeros(3, 4, 2), adapter_idxs=ids[:, 0])
    for kw in (dict(inputs=torch.zeros(2, 9)), dict(lora_a=torch.zeros(3, 2, 9)), dict(lora_b=torch.zeros(3, 5, 2)),
               dict(lora_b=torch.zeros(2, 4, 2)), dict(adapter_idxs=ids), dict(scaling=torch.ones(2)), dict(bias=torch.zeros(3)),
               dict(lora_a=torch.zeros(3, 300, 8), lora_b=torch.zeros(3, 4, 300))):
        with pytest.raises(AssertionError):
            sm.adapter_linear(**{**a, **kw})
    with pytest.raises(RuntimeError, match="not integers"):
        sm.adapter_linear(**{**a, "adapter_idxs": ids[:, 0].bool()})


def test_modules():
    m = sm.AdapterLinear(16, 24, 3, 4, bias=True, alpha=8)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {
        "weight": (24, 16), "bias": (24,), "lora_a": (3, 4, 16), "lora_b": (3, 24, 4), "scaling": (3,)}
    assert not m.weight.requires_grad and not m.bias.requires_grad and m.lora_a.requires_grad
    assert (m.lora_b == 0).all() and (m.scaling == 2.0).all() and "rank=4" in repr(m)
    with pytest.raises(RuntimeError, match="activation"):
        sm.mlp.MLP(16, 8, 4, 2, activation=torch.tanh).decode(torch.zeros(1, 16), torch.zeros(1, 2), torch.zeros(1, 2, dtype=torch.int64))

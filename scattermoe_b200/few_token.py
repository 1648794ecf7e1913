"""The MoE layer for a few tokens (decoding), forward only.

`expert_mlp` is built for thousands of tokens: its grouped GEMM walks 128-row tiles of one expert. While a server decodes, an
expert has zero to a few dozen rows and the layer is a read of the weights of the experts that occur. The entry points
here are that form:

    few_token_mlp   gates and expert ids given (what `MLP` / `GLUMLP` take): two kernels, the up-projection with the
                    activation and the down-projection with the gate-weighted sum
    few_token_moe   the whole layer from the tokens: router product, top-k and gates in one kernel before those two

At most `max_tokens()` tokens and 1024 slots (tokens x k); the sort into experts happens inside the kernels, so no
`flatten_sort_count` is needed. A slot whose id lies outside [0, E) contributes nothing (a padded batch marks its empty rows
with -1; a row without any expert comes out as zeros, whatever its input holds). Results are bit-equal from call to call.
Nothing is kept for backward: inputs that require gradients are refused while gradients are enabled, forward-mode tangents always.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from . import activation as _act
from .routing import MODES

MAX_SLOTS = 1024
MAX_EXPERTS = 1024


_max_tokens = None


def max_tokens() -> int:
    global _max_tokens
    if _max_tokens is None:
        _max_tokens = _lib.load().smoe_few_token_max_tokens()
    return _max_tokens


def _refuse_grad(what, *tensors):
    _lib.refuse_tangents(what, *tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("%s has no backward pass: call it under torch.no_grad(), or use expert_mlp for training" % what)


def _same(what, x, **tensors):
    """Operands on the tokens' device and, the router's outputs apart, of their dtype."""
    dev, dtype = x.device, x.dtype
    for name, t in tensors.items():
        if t is None:
            continue
        if t.device != dev:
            raise RuntimeError("%s: `%s` is on %s, the tokens are on %s" % (what, name, t.device, dev))
        if t.dtype != dtype and name not in ("gates", "expert_idxs"):
            raise RuntimeError("%s: `%s` is %s, the tokens are %s" % (what, name, t.dtype, dtype))


def _mlp_impl(x: torch.Tensor, up: torch.Tensor, down: torch.Tensor, gates: Optional[torch.Tensor], ids: torch.Tensor,
              act_layout: int, act: int, up_b: Optional[torch.Tensor], down_b: Optional[torch.Tensor], alpha: float,
              limit: float, after_router: bool = False) -> torch.Tensor:
    T, d = x.shape
    E, F, d_out = down.shape
    k = ids.size(1)
    dev = x.device
    lib = _lib.load()
    y = torch.empty((T, d_out), dtype=x.dtype, device=dev)
    ws_bytes = lib.smoe_few_token_workspace_bytes(T, k, F, d_out)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    null = (None, 0, 0)
    with _lib.on_device_of(dev):
        rc = lib.smoe_few_token_mlp(
            x.data_ptr(), T, x.stride(0), up.data_ptr(), *up.stride(),
            *((up_b.data_ptr(), *up_b.stride()) if up_b is not None else null),
            down.data_ptr(), *down.stride(),
            *((down_b.data_ptr(), *down_b.stride()) if down_b is not None else null),
            *((gates.data_ptr(), *gates.stride(), _lib.DTYPE_CODE[gates.dtype]) if gates is not None
              else (None, 0, 0, 0)),
            ids.data_ptr(), *ids.stride(), y.data_ptr(), d_out, k, d, F, d_out, E, act_layout, act,
            alpha, limit, _lib.DTYPE_CODE[x.dtype], _lib.path_flags() | (_lib.FLAG_AFTER_ROUTER if after_router else 0),
            ws.data_ptr(), ws_bytes, _lib.status_ptr(dev), _lib.stream_ptr(dev))
    _lib.check(rc, "smoe_few_token_mlp")
    return y


@torch.library.custom_op("scattermoe_b200::few_token_mlp", mutates_args={})
def few_token_mlp_compileable(x: torch.Tensor, up: torch.Tensor, down: torch.Tensor, gates: Optional[torch.Tensor],
                              ids: torch.Tensor, act_layout: int, act: int, up_b: Optional[torch.Tensor],
                              down_b: Optional[torch.Tensor], alpha: float, limit: float) -> torch.Tensor:
    return _mlp_impl(x, up, down, gates, ids, act_layout, act, up_b, down_b, alpha, limit)


@few_token_mlp_compileable.register_fake
def _(x, up, down, gates, ids, act_layout, act, up_b, down_b, alpha, limit):
    return torch.empty((x.size(0), down.size(2)), dtype=x.dtype, device=x.device)


def _check_mlp(what, x, up, down, act_layout, act, up_b, down_b):
    """Shapes as in `expert_mlp`; returns E."""
    assert x.dim() == 2, "%s: tokens must be (T, d)" % what
    assert up.dim() == 3 and down.dim() == 3, "%s: expert weights must be (E, in, out)" % what
    assert 0 <= act_layout <= 3 and 0 <= act <= 4, "%s: layout %s / function %s" % (what, act_layout, act)
    E, F = down.size(0), down.size(1)
    n_up = F if act_layout == _act.LAYOUT_PLAIN else 2 * F
    assert up.shape == (E, x.size(1), n_up), "%s: up-projection %s, expected %s" % (
        what, tuple(up.shape), (E, x.size(1), n_up))
    assert E <= MAX_EXPERTS, "%s: %d experts, at most %d are taken" % (what, E, MAX_EXPERTS)
    assert up_b is None or tuple(up_b.shape) == (E, n_up), "%s: bias of the up-projection %s" % (what, tuple(up_b.shape))
    assert down_b is None or tuple(down_b.shape) == (E, down.size(2)), "%s: bias of the down-projection %s" % (
        what, tuple(down_b.shape))
    if x.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError("%s: %s is not one of fp32, bf16, fp16" % (what, x.dtype))
    return E


def _check_slots(what, T, k):
    assert T <= max_tokens(), "%s takes at most %d tokens, got %d: use expert_mlp" % (what, max_tokens(), T)
    assert T * k <= MAX_SLOTS, "%s takes at most %d slots (tokens x k), got %d: use expert_mlp" % (what, MAX_SLOTS, T * k)


def _rows(t):
    return t if t.stride(-1) == 1 else t.contiguous()


def _run_mlp(x, up, down, gates, ids, act_layout, act, up_b, down_b, alpha, limit, after_router=False):
    args = (x, up, down, gates, ids, act_layout, act, up_b, down_b, float(alpha), float(limit))
    return few_token_mlp_compileable(*args) if torch.compiler.is_compiling() else _mlp_impl(*args, after_router=after_router)


def few_token_mlp(inputs, up_weights, down_weights, gates, expert_idxs, act_layout, act, up_biases=None, down_biases=None,
                  alpha=1.702, limit=7.0):
    """The expert MLP of one MoE layer for a few tokens: y[t] = sum_j gates[t, j] * (h W2[e] + b2[e]), h = act(x[t] W1[e] + b1[e]),
    e = expert_idxs[t, j].

    inputs (T, d); up_weights (E, d, n_up) and down_weights (E, hidden, d_out) as `expert_mlp` takes them (any strides);
    gates (T, k) in any of the three dtypes, or None for a plain sum; expert_idxs (T, k), ids outside [0, E) contribute
    nothing; layout / function codes as in `scattermoe_b200.activation`. Weights and biases have the tokens' dtype.
    Returns (T, d_out). fp32 accumulation; on the tensor-core path the hidden rows are rounded once to the tokens' dtype.

    The fast path is 16-bit, d and hidden multiples of 8, tokens and weights whose rows start on 16 bytes. fp32 and everything else take
    CUDA-core kernels, exact but not tuned: measured at 0.85 to 6 times the speed of the same layer in elementary torch operations."""
    what = "few_token_mlp"
    _refuse_grad(what, inputs, up_weights, down_weights, gates, up_biases, down_biases)
    _lib.require_cuda(inputs, "inputs")
    _check_mlp(what, inputs, up_weights, down_weights, act_layout, act, up_biases, down_biases)
    assert expert_idxs.dim() == 2 and expert_idxs.size(0) == inputs.size(0) and expert_idxs.size(1) >= 1, \
        "%s: expert_idxs %s for %d tokens" % (what, tuple(expert_idxs.shape), inputs.size(0))
    assert gates is None or gates.shape == expert_idxs.shape, "%s: gates %s, expert_idxs %s" % (
        what, tuple(gates.shape), tuple(expert_idxs.shape))
    _same(what, inputs, up_weights=up_weights, down_weights=down_weights, up_biases=up_biases, down_biases=down_biases,
          gates=gates, expert_idxs=expert_idxs)
    if gates is not None and gates.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError("%s: gates are %s, not one of fp32, bf16, fp16" % (what, gates.dtype))
    if expert_idxs.dtype not in (torch.int64, torch.int32):
        raise RuntimeError("%s: expert_idxs are %s, not integers of 64 or 32 bits" % (what, expert_idxs.dtype))
    _check_slots(what, inputs.size(0), expert_idxs.size(1))
    if inputs.size(0) == 0:
        return inputs.new_empty((0, down_weights.size(2)))
    ids = expert_idxs if expert_idxs.dtype == torch.int64 else expert_idxs.to(torch.int64)
    return _run_mlp(_rows(inputs), up_weights, down_weights, gates, ids, act_layout, act, up_biases, down_biases, alpha, limit)


def _route_impl(x: torch.Tensor, wr: torch.Tensor, br: Optional[torch.Tensor], k: int, mode: int,
                renormalize: bool) -> tuple[torch.Tensor, torch.Tensor]:
    T, d = x.shape
    dev = x.device
    ids = torch.empty((T, k), dtype=torch.int64, device=dev)
    gates = torch.empty((T, k), dtype=torch.float32, device=dev)
    with _lib.on_device_of(dev):
        rc = _lib.load().smoe_few_token_route(
            x.data_ptr(), T, x.stride(0), wr.data_ptr(), wr.stride(0), br.data_ptr() if br is not None else None,
            br.stride(0) if br is not None else 0, wr.size(0), d, k, mode, int(renormalize), ids.data_ptr(), gates.data_ptr(),
            _lib.DTYPE_CODE[x.dtype], _lib.stream_ptr(dev))
    _lib.check(rc, "smoe_few_token_route")
    return gates, ids


@torch.library.custom_op("scattermoe_b200::few_token_route", mutates_args={})
def few_token_route_compileable(x: torch.Tensor, wr: torch.Tensor, br: Optional[torch.Tensor], k: int, mode: int,
                                renormalize: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return _route_impl(x, wr, br, k, mode, renormalize)


@few_token_route_compileable.register_fake
def _(x, wr, br, k, mode, renormalize):
    T = x.size(0)
    return (torch.empty((T, k), dtype=torch.float32, device=x.device), torch.empty((T, k), dtype=torch.int64, device=x.device))


def few_token_moe(inputs, router_weight, up_weights, down_weights, k, act_layout, act, mode="softmax_topk", renormalize=True,
                  router_bias=None, up_biases=None, down_biases=None, alpha=1.702, limit=7.0):
    """A whole MoE layer for a few tokens: router logits x Wr^T + br (fp32, never rounded), the k best experts of each token and
    their gates as `route_topk` defines them (`mode`, `renormalize`; equal logits: the lower expert id first), then
    `few_token_mlp`. router_weight is (E, d) in the tokens' dtype. Returns (y (T, d_out), gates (T, k) fp32,
    expert_idxs (T, k) int64)."""
    what = "few_token_moe"
    _refuse_grad(what, inputs, router_weight, up_weights, down_weights, router_bias, up_biases, down_biases)
    _lib.require_cuda(inputs, "inputs")
    if mode not in MODES:
        raise AssertionError("%s: mode must be one of %s" % (what, sorted(MODES)))
    E = _check_mlp(what, inputs, up_weights, down_weights, act_layout, act, up_biases, down_biases)
    assert tuple(router_weight.shape) == (E, inputs.size(1)), "%s: router weight %s, expected %s" % (
        what, tuple(router_weight.shape), (E, inputs.size(1)))
    assert router_bias is None or tuple(router_bias.shape) == (E,), "%s: router bias %s" % (what, tuple(router_bias.shape))
    assert 1 <= k <= min(E, 32), "%s: k=%d of %d experts (at most 32)" % (what, k, E)
    _same(what, inputs, router_weight=router_weight, router_bias=router_bias, up_weights=up_weights, down_weights=down_weights,
          up_biases=up_biases, down_biases=down_biases)
    T = inputs.size(0)
    _check_slots(what, T, k)
    if T == 0:
        return (inputs.new_empty((0, down_weights.size(2))), inputs.new_empty((0, k), dtype=torch.float32),
                inputs.new_empty((0, k), dtype=torch.int64))
    x = _rows(inputs)
    route = few_token_route_compileable if torch.compiler.is_compiling() else _route_impl
    gates, ids = route(x, _rows(router_weight), router_bias, int(k), MODES[mode], bool(renormalize))
    y = _run_mlp(x, up_weights, down_weights, gates, ids, act_layout, act, up_biases, down_biases, alpha, limit, after_router=True)
    return y, gates, ids

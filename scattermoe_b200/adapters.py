"""Low-rank adapters of many requests beside a shared projection.

    y[t] = W x[t] + b + s_a B_a (A_a x[t]),      a = adapter_idxs[t]

`parallel_linear` lets the id of a row choose its projection; here all rows share one and the id chooses what is added to it. A
batch mixes the tokens of many requests, each with an adapter of its own or none (an id outside [0, n): y = W x + b).
The ids may be in any order; tokens of one request usually stand together, which the kernels use and do not need.

Two launches forward: the shrink into the rank (h = s A x; in 16 bits rounded once, as the tensor cores take it) and the shared product, whose accumulators take up
B h before they are rounded once: the adapted output is never read back. Backward mirrors it (g = s B^T dy, then
dx = W^T dy + A^T g in one launch) and sums the outer products dA_a = sum g x^T, dB_a = sum dy h^T per adapter in a fixed
order. Gradients nobody asked for are not computed; adapters without rows get zeros; `scaling` is a constant. Infinities and NaN
in one adapter, or in one row, stay with the rows they belong to. Forward-mode derivatives are refused.

A training step can be captured into a CUDA graph as any other autograd function: warm up on the capturing side stream, and let go of
eager graphs of the same leaves first (torch ends the process where a captured backward meets one).
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from .parallel_experts import _rowmajor

MAX_RANK = 256
MAX_ADAPTERS = 4096


def _forward_impl(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], lora_a: torch.Tensor, lora_b: torch.Tensor,
                  ids: torch.Tensor, scaling: Optional[torch.Tensor], scale: float, sort: bool) -> tuple[
                      torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, h, sorted_idx, offsets): the output, the rows of the rank, and (empty unless `sort`) the rows sorted by adapter."""
    T, width = x.shape
    out = weight.size(0)
    n, r, _ = lora_a.shape
    dev, dtype = x.device, _lib.DTYPE_CODE[x.dtype]
    lib = _lib.load()
    y = torch.empty((T, out), dtype=x.dtype, device=dev)
    h = torch.empty((T, (r + 7) // 8 * 8), dtype=x.dtype, device=dev)
    lists = torch.empty(T + n if sort else 0, dtype=torch.int64, device=dev)
    sorted_idx, offsets = (lists[:T], lists[T:]) if sort else (lists, lists)
    ws_bytes = lib.smoe_adapter_workspace_bytes(T, n, width, out, r, dtype) if sort else 0
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if sort else None
    with _lib.on_device_of(dev):
        rc = lib.smoe_adapter_forward(
            x.data_ptr(), T, x.stride(0), weight.data_ptr(), *weight.stride(), bias.data_ptr() if bias is not None else None,
            lora_a.data_ptr(), *lora_a.stride(), lora_b.data_ptr(), *lora_b.stride(), ids.data_ptr(),
            scaling.data_ptr() if scaling is not None else None, scale, y.data_ptr(), h.data_ptr(),
            lists.data_ptr() if sort else None, offsets.data_ptr() if sort else None, n, width, out, r, dtype, _lib.path_flags(),
            ws.data_ptr() if sort else None, ws_bytes, _lib.status_ptr(dev), _lib.stream_ptr(dev))
    _lib.check(rc, "smoe_adapter_forward")
    return y, h, sorted_idx, offsets


def _backward_impl(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                   ids: torch.Tensor, scaling: Optional[torch.Tensor], scale: float, h: torch.Tensor, sorted_idx: torch.Tensor,
                   offsets: torch.Tensor, need_x: bool, need_a: bool, need_b: bool, need_w: bool, need_bias: bool) -> tuple[
                       torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(d_x, d_a, d_b, d_weight, d_bias), empty where not needed."""
    T, width = x.shape
    out = weight.size(0)
    n, r, _ = lora_a.shape
    dev, dtype = x.device, _lib.DTYPE_CODE[x.dtype]
    lib = _lib.load()

    def result(wanted, *shape):
        return torch.empty(shape if wanted else (0,), dtype=x.dtype, device=dev)

    d_x, d_a, d_b = result(need_x, T, width), result(need_a, n, r, width), result(need_b, n, out, r)
    d_w, d_bias = result(need_w, out, width), result(need_bias, out)
    ws_bytes = lib.smoe_adapter_workspace_bytes(T, n, width, out, r, dtype)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    with _lib.on_device_of(dev):
        rc = lib.smoe_adapter_backward(
            dy.data_ptr(), T, dy.stride(0), x.data_ptr(), x.stride(0), weight.data_ptr(), *weight.stride(), lora_a.data_ptr(),
            *lora_a.stride(), lora_b.data_ptr(), *lora_b.stride(), ids.data_ptr(), scaling.data_ptr() if scaling is not None else None,
            scale, h.data_ptr(), sorted_idx.data_ptr() or None, offsets.data_ptr() or None, d_x.data_ptr() or None,
            d_a.data_ptr() or None, d_b.data_ptr() or None, d_w.data_ptr() or None, d_bias.data_ptr() or None, n, width, out, r, dtype, _lib.path_flags(),
            ws.data_ptr(), ws_bytes, _lib.status_ptr(dev), _lib.stream_ptr(dev))
    _lib.check(rc, "smoe_adapter_backward")
    return d_x, d_a, d_b, d_w, d_bias


# The registered forms are used while torch.compile traces, as everywhere in this package.
@torch.library.custom_op("scattermoe_b200::adapter_forward", mutates_args={})
def forward_compileable(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], lora_a: torch.Tensor,
                        lora_b: torch.Tensor, ids: torch.Tensor, scaling: Optional[torch.Tensor], scale: float, sort: bool) -> tuple[
                            torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    y, h, sorted_idx, offsets = _forward_impl(x, weight, bias, lora_a, lora_b, ids, scaling, scale, sort)
    return y, h, sorted_idx.clone(), offsets.clone()      # outputs of a registered operator do not share memory


@forward_compileable.register_fake
def _(x, weight, bias, lora_a, lora_b, ids, scaling, scale, sort):
    T, n, r = x.size(0), lora_a.size(0), lora_a.size(1)
    i64 = dict(dtype=torch.int64, device=x.device)
    return (x.new_empty((T, weight.size(0))), x.new_empty((T, (r + 7) // 8 * 8)), torch.empty(T if sort else 0, **i64),
            torch.empty(n if sort else 0, **i64))


@torch.library.custom_op("scattermoe_b200::adapter_backward", mutates_args={})
def backward_compileable(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                         ids: torch.Tensor, scaling: Optional[torch.Tensor], scale: float, h: torch.Tensor,
                         sorted_idx: torch.Tensor, offsets: torch.Tensor, need_x: bool, need_a: bool, need_b: bool, need_w: bool,
                         need_bias: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return _backward_impl(dy, x, weight, lora_a, lora_b, ids, scaling, scale, h, sorted_idx, offsets, need_x, need_a, need_b, need_w,
                          need_bias)


@backward_compileable.register_fake
def _(dy, x, weight, lora_a, lora_b, ids, scaling, scale, h, sorted_idx, offsets, need_x, need_a, need_b, need_w, need_bias):
    return (x.new_empty(x.shape if need_x else (0,)), x.new_empty(lora_a.shape if need_a else (0,)),
            x.new_empty(lora_b.shape if need_b else (0,)), x.new_empty(weight.shape if need_w else (0,)),
            x.new_empty((weight.size(0) if need_bias else 0,)))


class AdapterLinear_(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, lora_a, lora_b, ids, scaling, scale, bias):
        x = _rowmajor(x)
        # the gradients of the adapters need the rows sorted by adapter; the shrinks of both directions profit from it
        sort = ctx.needs_input_grad[2] or ctx.needs_input_grad[3]
        run = forward_compileable if torch.compiler.is_compiling() else _forward_impl
        y, h, sorted_idx, offsets = run(x, weight, bias, lora_a, lora_b, ids, scaling, scale, sort)
        ctx.save_for_backward(x, weight, lora_a, lora_b, ids, scaling, h, sorted_idx, offsets)
        ctx.scale = scale
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, lora_a, lora_b, ids, scaling, h, sorted_idx, offsets = ctx.saved_tensors
        need_x, need_w, need_a, need_b = ctx.needs_input_grad[:4]
        need_bias = ctx.needs_input_grad[7]
        dy = _rowmajor(dy)
        if dy.dtype != x.dtype:
            dy = dy.to(x.dtype)
        run = backward_compileable if torch.compiler.is_compiling() else _backward_impl
        d_x, d_a, d_b, d_w, d_bias = run(dy, x, weight, lora_a, lora_b, ids, scaling, ctx.scale, h, sorted_idx, offsets, need_x, need_a,
                                         need_b, need_w, need_bias)
        return (d_x if need_x else None, d_w if need_w else None, d_a if need_a else None, d_b if need_b else None, None, None, None,
                d_bias if need_bias else None)


def adapter_linear(inputs, weight, lora_a, lora_b, adapter_idxs, scaling=1.0, bias=None):
    """y[t] = weight x[t] + bias + s_a lora_b[a] (lora_a[a] x[t]), a = adapter_idxs[t]; differentiable.

    inputs (..., in); weight (out, in) as nn.Linear stores it; lora_a (n, r, in), lora_b (n, out, r), r <= 256, n <= 4096;
    adapter_idxs of the shape of the leading dimensions, any order, ids outside [0, n) take no adapter; scaling a number or
    one fp32 value per adapter (n,), constant; bias (out,) or None. One dtype (fp32, bf16, fp16), weights in any strides.
    Returns (..., out).

    The fast path is 16-bit with in and out multiples of 8 and rows that start on 16 bytes; it costs more the more adapters meet in 128
    neighbouring rows. fp32 and other widths take CUDA-core kernels, exact but not tuned: measured at 0.5 to 2 times the speed of
    elementary torch operations, worst for a training step of many rows."""
    what = "adapter_linear"
    _lib.require_cuda(inputs, "inputs")
    assert weight.dim() == 2 and lora_a.dim() == 3 and lora_b.dim() == 3, "%s: weight (out, in), lora_a (n, r, in), lora_b (n, out, r)" % what
    out, width = weight.shape
    n, r, _ = lora_a.shape
    assert inputs.dim() >= 1 and inputs.size(-1) == width, "%s: inputs %s for a weight %s" % (what, tuple(inputs.shape), tuple(weight.shape))
    assert lora_a.size(2) == width and tuple(lora_b.shape) == (n, out, r), "%s: lora_a %s, lora_b %s for a weight %s" % (
        what, tuple(lora_a.shape), tuple(lora_b.shape), tuple(weight.shape))
    assert 1 <= r <= MAX_RANK, "%s: rank %d, 1 to %d are taken" % (what, r, MAX_RANK)
    assert 1 <= n <= MAX_ADAPTERS, "%s: %d adapters, 1 to %d are taken" % (what, n, MAX_ADAPTERS)
    assert adapter_idxs.shape == inputs.shape[:-1], "%s: adapter_idxs %s for inputs %s" % (
        what, tuple(adapter_idxs.shape), tuple(inputs.shape))
    assert bias is None or tuple(bias.shape) == (out,), "%s: bias %s" % (what, tuple(bias.shape))
    if inputs.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError("%s: %s is not one of fp32, bf16, fp16" % (what, inputs.dtype))
    dtype, dev = inputs.dtype, inputs.device
    for name, t in (("weight", weight), ("lora_a", lora_a), ("lora_b", lora_b), ("bias", bias)):
        if t is not None:
            if t.dtype != dtype:
                raise RuntimeError("%s: `%s` is %s, the inputs are %s" % (what, name, t.dtype, dtype))
            if t.device != dev:
                raise RuntimeError("%s: `%s` is on %s, the inputs are on %s" % (what, name, t.device, dev))
    if adapter_idxs.device != dev:
        raise RuntimeError("%s: `adapter_idxs` is on %s, the inputs are on %s" % (what, adapter_idxs.device, dev))
    if adapter_idxs.dtype not in (torch.int64, torch.int32):
        raise RuntimeError("%s: adapter_idxs are %s, not integers of 64 or 32 bits" % (what, adapter_idxs.dtype))
    per_adapter = None
    if isinstance(scaling, torch.Tensor):
        assert tuple(scaling.shape) == (n,), "%s: scaling %s for %d adapters" % (what, tuple(scaling.shape), n)
        if scaling.requires_grad:
            raise RuntimeError("%s: `scaling` is a constant, it cannot require a gradient" % what)
        if scaling.device != dev:
            raise RuntimeError("%s: `scaling` is on %s, the inputs are on %s" % (what, scaling.device, dev))
        _lib.refuse_tangents(what, scaling)
        per_adapter, scaling = scaling.float().contiguous(), 1.0
    _lib.refuse_tangents(what, inputs, weight, lora_a, lora_b, bias)
    lead = inputs.shape[:-1]
    x = inputs if inputs.dim() == 2 else inputs.reshape(-1, width)
    ids = adapter_idxs.reshape(-1)
    if ids.dtype != torch.int64:
        ids = ids.to(torch.int64)
    ids = ids.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    leaves = (x, weight, lora_a, lora_b, bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in leaves) or torch.compiler.is_compiling():
        y = AdapterLinear_.apply(x, weight, lora_a, lora_b, ids, per_adapter, float(scaling), bias)
    else:      # no graph to build
        y = _forward_impl(_rowmajor(x), weight, bias, lora_a, lora_b, ids, per_adapter, float(scaling), False)[0]
    return y if len(lead) == 1 else y.view(*lead, out)


class AdapterLinear(nn.Module):
    """A linear layer with `num_adapters` low-rank adapters beside it; each row names its adapter.

    Parameters: weight (out, in) and bias (out,) as nn.Linear, lora_a (n, r, in) ~ N(0, 1/in), lora_b (n, out, r) zeros (a new
    adapter changes nothing). `scaling` (n,) is a buffer, alpha / rank by default, and stays fp32 when
    the module is cast. `freeze_shared=True` (default) trains the adapters alone."""

    def __init__(self, in_features, out_features, num_adapters, rank, bias=False, alpha=None, freeze_shared=True) -> None:
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.num_adapters, self.rank = num_adapters, rank
        self.weight = nn.Parameter(torch.empty(out_features, in_features), requires_grad=not freeze_shared)
        self.bias = nn.Parameter(torch.zeros(out_features), requires_grad=not freeze_shared) if bias else None
        self.lora_a = nn.Parameter(torch.empty(num_adapters, rank, in_features))
        self.lora_b = nn.Parameter(torch.zeros(num_adapters, out_features, rank))
        self.register_buffer("scaling", torch.full((num_adapters,), (alpha if alpha is not None else rank) / rank,
                                                    dtype=torch.float32))
        self.reset_parameters()

    def _apply(self, fn, recurse=True):
        """Casts and moves of a module come through here: `scaling` moves, but keeps its 32 bits (0.1 would be off by 2^-10 of itself in bf16)."""
        scaling = self.scaling
        super()._apply(fn, recurse)
        if self.scaling.dtype != scaling.dtype:
            self.scaling = scaling.to(self.scaling.device)
        return self

    def reset_parameters(self) -> None:
        nn.init.normal_(self.weight, std=0.02)
        nn.init.normal_(self.lora_a, std=self.in_features ** -0.5)
        nn.init.zeros_(self.lora_b)

    def extra_repr(self):
        return 'in_features={}, out_features={}, num_adapters={}, rank={}'.format(
            self.in_features, self.out_features, self.num_adapters, self.rank)

    def forward(self, inputs, adapter_idxs):
        return adapter_linear(inputs, self.weight, self.lora_a, self.lora_b, adapter_idxs, scaling=self.scaling, bias=self.bias)

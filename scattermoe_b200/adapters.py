"""Low-rank adapters of many requests beside a shared projection.

    y[t] = W x[t] + b + s_a B_a (A_a x[t]),      a = adapter_idxs[t]

`parallel_linear` lets the id of a row choose its projection; here all rows share one and the id chooses what is added to it. A
batch mixes the tokens of many requests, each with an adapter of its own or none (an id outside [0, n): y = W x + b).
The ids may be in any order; tokens of one request usually stand together, which the kernels use and do not need.

Two launches forward: the shrink into the rank (h = s A x; in 16 bits rounded once, as the tensor cores take it) and the shared product, whose accumulators take up
B h before they are rounded once: the adapted output is never read back. Backward mirrors it (g = s B^T dy, then
dx = W^T dy + A^T g in one launch) and sums the outer products dA_a = sum g x^T, dB_a = sum dy h^T per adapter in a fixed
order. Gradients nobody asked for are not computed; adapters without rows get zeros; `scaling` is a constant.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from . import kernels
from .parallel_experts import _rowmajor, _sort_count_impl, sort_count_compileable

MAX_RANK = 256
MAX_ADAPTERS = 4096


def _padded(r: int) -> int:
    return (r + 7) // 8 * 8


def _shrink_impl(x: torch.Tensor, m: torch.Tensor, ids: torch.Tensor, scaling: Optional[torch.Tensor], scale: float,
                 sorted_idx: Optional[torch.Tensor], offsets: Optional[torch.Tensor]) -> torch.Tensor:
    """h[t, j] = s sum_c x[t, c] m[ids[t], j, c], (T, r padded to a multiple of 8); zero rows for ids outside [0, n)."""
    T = x.size(0)
    n, r, C = m.shape
    h = torch.empty((T, _padded(r)), dtype=x.dtype, device=x.device)
    with _lib.on_device_of(x.device):
        rc = _lib.load().smoe_adapter_shrink(
            x.data_ptr(), T, x.stride(0), m.data_ptr(), *m.stride(), ids.data_ptr(),
            scaling.data_ptr() if scaling is not None else None, scale, h.data_ptr(), n, C, r, _lib.DTYPE_CODE[x.dtype],
            sorted_idx.data_ptr() if sorted_idx is not None else None, offsets.data_ptr() if offsets is not None else None,
            _lib.stream_ptr(x.device))
    _lib.check(rc, "smoe_adapter_shrink")
    return h


def _linear_impl(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], h: torch.Tensor, m: torch.Tensor,
                 ids: torch.Tensor, after_shrink: bool = False) -> torch.Tensor:
    """y = x w + bias + h m[ids]; w is (C, O), m is (n, r, O), any strides."""
    T, C = x.shape
    O = w.size(1)
    n, r, _ = m.shape
    y = torch.empty((T, O), dtype=x.dtype, device=x.device)
    with _lib.on_device_of(x.device):
        rc = _lib.load().smoe_adapter_linear(
            x.data_ptr(), T, x.stride(0), w.data_ptr(), *w.stride(), bias.data_ptr() if bias is not None else None,
            h.data_ptr(), m.data_ptr(), *m.stride(), ids.data_ptr(), y.data_ptr(), O,
            n, C, O, r, _lib.DTYPE_CODE[x.dtype], _lib.path_flags() | (_lib.FLAG_AFTER_SHRINK if after_shrink else 0),
            _lib.status_word(x.device).data_ptr(), _lib.stream_ptr(x.device))
    _lib.check(rc, "smoe_adapter_linear")
    return y


def _grad_impl(u: torch.Tensor, v: torch.Tensor, r: int, sorted_idx: torch.Tensor, offsets: torch.Tensor,
               transposed: bool) -> torch.Tensor:
    """d[a] = sum over the rows t of adapter a of u[t, :r]^T v[t]: (n, r, C), or its transpose (n, C, r)."""
    n, C = offsets.size(0), v.size(1)
    lib = _lib.load()
    ws_bytes = lib.smoe_adapter_grad_workspace_bytes(u.size(0), C, r)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=v.device)
    d = torch.empty((n, C, r) if transposed else (n, r, C), dtype=v.dtype, device=v.device)
    view = d.transpose(1, 2) if transposed else d
    with _lib.on_device_of(v.device):
        rc = lib.smoe_adapter_grad(
            u.data_ptr(), u.size(0), v.data_ptr(), v.stride(0), sorted_idx.data_ptr(), offsets.data_ptr(), d.data_ptr(),
            view.stride(0), view.stride(1), view.stride(2), n, C, r, _lib.DTYPE_CODE[v.dtype], ws.data_ptr(), ws_bytes,
            _lib.stream_ptr(v.device))
    _lib.check(rc, "smoe_adapter_grad")
    return d


def _column_sum_impl(v: torch.Tensor) -> torch.Tensor:
    T, C = v.shape
    lib = _lib.load()
    out = torch.empty((C,), dtype=v.dtype, device=v.device)
    ws_bytes = lib.smoe_column_sum_workspace_bytes(T, C)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=v.device)
    with _lib.on_device_of(v.device):
        rc = lib.smoe_column_sum(v.data_ptr(), T, v.stride(0), C, out.data_ptr(), _lib.DTYPE_CODE[v.dtype], ws.data_ptr(), ws_bytes,
                                 _lib.stream_ptr(v.device))
    _lib.check(rc, "smoe_column_sum")
    return out


# The registered forms are used while torch.compile traces, as everywhere in this package.
@torch.library.custom_op("scattermoe_b200::adapter_shrink", mutates_args={})
def shrink_compileable(x: torch.Tensor, m: torch.Tensor, ids: torch.Tensor, scaling: Optional[torch.Tensor], scale: float,
                       sorted_idx: Optional[torch.Tensor], offsets: Optional[torch.Tensor]) -> torch.Tensor:
    return _shrink_impl(x, m, ids, scaling, scale, sorted_idx, offsets)


@shrink_compileable.register_fake
def _(x, m, ids, scaling, scale, sorted_idx, offsets):
    return torch.empty((x.size(0), _padded(m.size(1))), dtype=x.dtype, device=x.device)


@torch.library.custom_op("scattermoe_b200::adapter_linear", mutates_args={})
def linear_compileable(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], h: torch.Tensor, m: torch.Tensor,
                       ids: torch.Tensor) -> torch.Tensor:
    return _linear_impl(x, w, bias, h, m, ids)


@linear_compileable.register_fake
def _(x, w, bias, h, m, ids):
    return torch.empty((x.size(0), w.size(1)), dtype=x.dtype, device=x.device)


@torch.library.custom_op("scattermoe_b200::adapter_grad", mutates_args={})
def grad_compileable(u: torch.Tensor, v: torch.Tensor, r: int, sorted_idx: torch.Tensor, offsets: torch.Tensor,
                     transposed: bool) -> torch.Tensor:
    return _grad_impl(u, v, r, sorted_idx, offsets, transposed)


@grad_compileable.register_fake
def _(u, v, r, sorted_idx, offsets, transposed):
    n, C = offsets.size(0), v.size(1)
    return torch.empty((n, C, r) if transposed else (n, r, C), dtype=v.dtype, device=v.device)


@torch.library.custom_op("scattermoe_b200::column_sum", mutates_args={})
def column_sum_compileable(v: torch.Tensor) -> torch.Tensor:
    return _column_sum_impl(v)


@column_sum_compileable.register_fake
def _(v):
    return torch.empty((v.size(1),), dtype=v.dtype, device=v.device)


def _pick(compiled, direct):
    return compiled if torch.compiler.is_compiling() else direct


def _linear(*args, after_shrink):
    return linear_compileable(*args) if torch.compiler.is_compiling() else _linear_impl(*args, after_shrink=after_shrink)


class AdapterLinear_(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, lora_a, lora_b, ids, scaling, scale, bias):
        x = _rowmajor(x)
        # the gradients of the adapters need the rows sorted by adapter; the shrinks of both directions profit from it
        sorted_idx = offsets = None
        if ctx.needs_input_grad[2] or ctx.needs_input_grad[3]:
            _, sorted_idx, offsets = _pick(sort_count_compileable, _sort_count_impl)(ids, lora_a.size(0))
        h = _pick(shrink_compileable, _shrink_impl)(x, lora_a, ids, scaling, scale, sorted_idx, offsets)
        y = _linear(x, weight.t(), bias, h, lora_b.transpose(1, 2), ids, after_shrink=True)
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
        d_x = d_w = d_a = d_b = d_bias = None
        if need_x or need_a:
            g = _pick(shrink_compileable, _shrink_impl)(dy, lora_b.transpose(1, 2), ids, scaling, ctx.scale, sorted_idx, offsets)
        if need_x:
            d_x = _linear(dy, weight, None, g, lora_a, ids, after_shrink=True)
        if need_a or need_b:
            grad = _pick(grad_compileable, _grad_impl)
            if need_a:
                d_a = grad(g, x, lora_a.size(1), sorted_idx, offsets, False)
            if need_b:
                d_b = grad(h, dy, lora_a.size(1), sorted_idx, offsets, True)
        if need_w:
            rows = torch.full((1,), x.size(0), dtype=torch.int64, device=x.device)
            d_w, db = kernels.ops.group_bwd_W(DY=dy, X=x, expert_offsets=rows, E=1, has_bias=need_bias)
            d_w = d_w[0].t()
            if need_bias:
                d_bias = db[0]
        elif need_bias:
            d_bias = _pick(column_sum_compileable, _column_sum_impl)(dy)
        return d_x, d_w, d_a, d_b, None, None, None, d_bias


def adapter_linear(inputs, weight, lora_a, lora_b, adapter_idxs, scaling=1.0, bias=None):
    """y[t] = weight x[t] + bias + s_a lora_b[a] (lora_a[a] x[t]), a = adapter_idxs[t]; differentiable.

    inputs (..., in); weight (out, in) as nn.Linear stores it; lora_a (n, r, in), lora_b (n, out, r), r <= 256, n <= 4096;
    adapter_idxs of the shape of the leading dimensions, any order, ids outside [0, n) take no adapter; scaling a number or
    one fp32 value per adapter (n,), constant; bias (out,) or None. One dtype (fp32, bf16, fp16), weights in any strides.
    Returns (..., out)."""
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
        per_adapter, scaling = scaling.float().contiguous(), 1.0
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
        x = _rowmajor(x)
        h = _shrink_impl(x, lora_a, ids, per_adapter, float(scaling), None, None)
        y = _linear_impl(x, weight.t(), bias, h, lora_b.transpose(1, 2), ids, after_shrink=True)
    return y if len(lead) == 1 else y.view(*lead, out)


class AdapterLinear(nn.Module):
    """A linear layer with `num_adapters` low-rank adapters beside it; each row names its adapter.

    Parameters: weight (out, in) and bias (out,) as nn.Linear, lora_a (n, r, in) ~ N(0, 1/in), lora_b (n, out, r) zeros (a new
    adapter changes nothing). `scaling` (n,) is a buffer, alpha / rank by default. `freeze_shared=True` (default) trains the adapters
    alone."""

    def __init__(self, in_features, out_features, num_adapters, rank, bias=False, alpha=None, freeze_shared=True) -> None:
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.num_adapters, self.rank = num_adapters, rank
        self.weight = nn.Parameter(torch.empty(out_features, in_features), requires_grad=not freeze_shared)
        self.bias = nn.Parameter(torch.zeros(out_features), requires_grad=not freeze_shared) if bias else None
        self.lora_a = nn.Parameter(torch.empty(num_adapters, rank, in_features))
        self.lora_b = nn.Parameter(torch.zeros(num_adapters, out_features, rank))
        self.register_buffer("scaling", torch.full((num_adapters,), (alpha if alpha is not None else rank) / rank))
        self.reset_parameters()

    def reset_parameters(self) -> None:
        nn.init.normal_(self.weight, std=0.02)
        nn.init.normal_(self.lora_a, std=self.in_features ** -0.5)
        nn.init.zeros_(self.lora_b)

    def extra_repr(self):
        return 'in_features={}, out_features={}, num_adapters={}, rank={}'.format(
            self.in_features, self.out_features, self.num_adapters, self.rank)

    def forward(self, inputs, adapter_idxs):
        return adapter_linear(inputs, self.weight, self.lora_a, self.lora_b, adapter_idxs, scaling=self.scaling, bias=self.bias)

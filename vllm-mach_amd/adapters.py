"""Low-rank adapters of many requests beside a shared quantized linear layer.

``LowRankAdapters`` holds the adapters of one prepared layer in slots, ``AdapterBatch`` says which slot each token of a
batch uses; ``MxLinearMethod.apply(layer, x, bias, adapters=, batch=)`` adds them to the layer's output:

    y[t] = layer(x[t]) + scaling[s] * lora_b[s] @ (lora_a[s] @ x[t]),   s the slot of token t

One batch serves every layer of a step.  The adapters see the unquantized bf16 input; their sums are fp32.  Both
``lora_a`` and ``lora_b``, and the input, have gradients, the layer's own weight stays frozen.  No counterpart in the
reference.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import ops
from .linear import _epilogue_bias, _function_bias, _gated_args


class AdapterBatch:
    """The adapter slot of each token of a batch, sorted for the kernels.

    ``ids``: integers [M] on the layers' device; a value outside [0, slots) is a token without an adapter.  ``update``
    takes the next step's ids into the same memory, for graphs that were captured with it.
    """

    def __init__(self, ids: torch.Tensor, slots: int):
        self.slots, self.updates = int(slots), 0
        self.tensors = ops.adapter_batch(ids, self.slots)  # ids, order, offsets, tiles

    def __len__(self) -> int:
        return self.tensors[0].shape[0]

    def update(self, ids: torch.Tensor) -> "AdapterBatch":
        if tuple(ids.shape) != (len(self),) or ids.device != self.tensors[0].device:
            raise ValueError(f"update needs ids of {len(self)} tokens on {self.tensors[0].device}, got {tuple(ids.shape)} on "
                             f"{ids.device}")
        for kept, new in zip(self.tensors, ops.adapter_batch(ids, self.slots)):
            kept.copy_(new)
        self.updates += 1
        return self


class LowRankAdapters(torch.nn.Module):
    """``slots`` adapters of up to ``rank`` (a multiple of 8, at most 256) beside a prepared layer.

    ``lora_a`` bf16 [slots, parts * rank, K]: each merged part of the layer (``layer.logical_widths``) has ``rank`` rows;
    ``lora_b`` bf16 [slots, N, rank]; ``scaling`` fp32 [slots].  All zero at first, so a slot adds nothing until it is
    loaded.  Without gradients until ``requires_grad_()``.
    """

    def __init__(self, layer: torch.nn.Module, slots: int, rank: int, device=None):
        super().__init__()
        if not hasattr(layer, "mxl_shape"):
            raise ValueError("adapters need a layer that process_weights_after_loading has prepared")
        if not 0 < slots <= 2048:
            raise ValueError(f"1 to 2048 slots ({slots})")
        if rank % 8 or not 8 <= rank <= 256:
            raise ValueError(f"ranks of 8 to 256, multiples of 8 ({rank}): pad smaller ones with zeros")
        n, k = layer.mxl_shape
        widths = list(getattr(layer, "logical_widths", None) or [n])
        if sum(widths) != n or len(widths) > 8 or any(w % 16 for w in widths[:-1]) or (len(widths) > 1 and widths[-1] % 16):
            raise ValueError(f"up to 8 merged parts of multiples of 16 columns, {n} together ({widths})")
        device = layer.weight.device if device is None else device
        self.slots, self.rank, self.widths = int(slots), int(rank), widths
        self.cols = [sum(widths[:i]) for i in range(len(widths) + 1)]
        self.lora_a = torch.nn.Parameter(torch.zeros((slots, len(widths) * rank, k), dtype=torch.bfloat16, device=device),
                                         requires_grad=False)
        self.lora_b = torch.nn.Parameter(torch.zeros((slots, n, rank), dtype=torch.bfloat16, device=device),
                                         requires_grad=False)
        self.register_buffer("scaling", torch.zeros(slots, dtype=torch.float32, device=device))

    def _slot(self, slot: int) -> int:
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} of {self.slots}")
        return slot

    @torch.no_grad()
    def load(self, slot: int, a: torch.Tensor, b: torch.Tensor, scaling: float, part: Optional[int] = None) -> None:
        """Put one adapter's a [r, K] and b [columns, r] (r <= rank) into a slot: of the merged part ``part``, or (None) of
        a layer of one part.  ``scaling`` is the slot's (alpha / r by custom), the same for all of its parts."""
        if part is None and len(self.widths) > 1:
            raise ValueError(f"the layer has {len(self.widths)} merged parts: name one")
        p = 0 if part is None else part
        if not 0 <= p < len(self.widths):
            raise ValueError(f"part {p} of {len(self.widths)}")
        r, k = a.shape[0] if a.ndim else 0, self.lora_a.shape[2]
        if a.ndim != 2 or a.shape[1] != k or tuple(b.shape) != (self.widths[p], r) or not 0 < r <= self.rank:
            raise ValueError(f"a {tuple(a.shape)} and b {tuple(b.shape)} are no adapter of rank <= {self.rank} of "
                             f"[{self.widths[p]}, {k}]")
        slot = self._slot(slot)
        to_a = self.lora_a.data[slot, p * self.rank:(p + 1) * self.rank]
        to_b = self.lora_b.data[slot, self.cols[p]:self.cols[p + 1]]
        to_a[:r].copy_(a.clone())  # (the slot's own values may come back, or others of this set)
        to_b[:, :r].copy_(b.clone())
        to_a[r:].zero_()
        to_b[:, r:].zero_()
        self.scaling[slot] = float(scaling)

    @torch.no_grad()
    def clear(self, slot: int) -> None:
        slot = self._slot(slot)
        for t in (self.lora_a.data, self.lora_b.data, self.scaling):
            t[slot].zero_()


def grad_of(layer: torch.nn.Module) -> tuple:
    """What ``ops.input_grad`` takes of a prepared layer: (w, sw, n, k, format, block)."""
    n, k = layer.mxl_shape
    if hasattr(layer, "mxl_block_scale"):
        return layer.weight, layer.mxl_block_scale, n, k, ops.E4M3, True
    return layer.weight, layer.weight_scale, n, k, layer.mxl_format, False


def _versions(*tensors: torch.Tensor) -> Optional[tuple]:
    """The tensors' writes so far (inference tensors count none; traced code has no versions)."""
    if torch.compiler.is_compiling():
        return None
    return tuple([None if t.is_inference() else t._version for t in tensors])


def _check_versions(what: str, versions: Optional[tuple], *tensors: torch.Tensor) -> None:
    if versions is not None and _versions(*tensors) != versions:
        raise RuntimeError(f"{what} has been modified by an inplace operation between this layer's forward and its backward")


# Each of the functions below has a second form whose context is set up apart, which torch.func's transforms ask for and which
# costs a call some 50 us: ``_apply`` takes it under a transform.

def _saved(ctx):
    if torch.compiler.is_compiling():
        return ctx.saved_tensors
    return [torch._C._functorch.unwrap_if_dead(t) for t in ctx.saved_tensors]  # (of a transform that has ended)


def _apply(function, *args):
    if not torch.compiler.is_compiling() and torch._C._functorch.peek_interpreter_stack() is not None:
        return function.transformed.apply(*args)
    return function.apply(*args)


class FrozenLinear(torch.autograd.Function):
    """A prepared layer's product (with a bias in its epilogue) with the gradients of its input and the bias."""

    @staticmethod
    def forward(ctx, x, bias, layer):
        FrozenLinear.hold(ctx, layer)
        return layer.mxl_kernel.apply_weights(layer, x, bias)

    @staticmethod
    def hold(ctx, layer):
        ctx.layer = grad_of(layer)
        ctx.versions = _versions(*ctx.layer[:2])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        w, sw, n, k, fmt, block = ctx.layer
        _check_versions("the layer's weight", ctx.versions, w, sw)
        dy2 = dy.reshape(-1, n)
        dx = ops.input_grad(dy2, w, sw, n, k, fmt, block).reshape(*dy.shape[:-1], k) if ctx.needs_input_grad[0] else None
        return dx, ops.bias_grad(dy2) if ctx.needs_input_grad[1] else None, None


class _FrozenLinear(torch.autograd.Function):
    """``FrozenLinear`` under torch.func's transforms; a batch of inputs is so many rows more."""

    @staticmethod
    def forward(x, bias, layer):
        return layer.mxl_kernel.apply_weights(layer, x, bias)

    @staticmethod
    def setup_context(ctx, inputs, output):
        FrozenLinear.hold(ctx, inputs[2])

    @staticmethod
    def vmap(info, in_dims, x, bias, layer):
        return _FrozenLinear.apply(x.movedim(in_dims[0], 0), bias, layer), 0

    backward = FrozenLinear.backward


FrozenLinear.transformed = _FrozenLinear


class AdapterLinear(torch.autograd.Function):
    """A prepared layer with its adapters: the gradients of the input, the adapters and a bias in the epilogue."""

    @staticmethod
    def forward(ctx, x, a, b, bias, layer, adapters, batch):
        y, v = _forward(layer, x, bias, a, b, adapters.scaling, batch.tensors, adapters.cols)
        AdapterLinear.hold(ctx, x, a, b, v, layer, adapters, batch)
        return y

    @staticmethod
    def hold(ctx, x, a, b, v, layer, adapters, batch):
        ctx.save_for_backward(x, a, b, v)
        of = grad_of(layer)
        ctx.held = of, adapters.scaling, batch, batch.updates, adapters.cols
        ctx.versions = _versions(adapters.scaling, *of[:2])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, *_):
        x, a, b, v = _saved(ctx)
        (w, sw, n, k, fmt, block), scaling, batch, updates, cols = ctx.held
        if batch.updates != updates:
            raise RuntimeError("the batch has been modified by an inplace operation (update) between this layer's forward and "
                               "its backward")
        _check_versions("the adapters' scaling or the layer's weight", ctx.versions, scaling, w, sw)
        need_x, need_a, need_b, need_bias = ctx.needs_input_grad[:4]
        dy2 = dy.reshape(-1, n)
        dx, da, db = ops.adapter_grad(dy2, x.reshape(-1, k), w, sw, fmt, block, a, b, scaling, v, *batch.tensors, cols, need_x,
                                      need_a, need_b)
        return (dx.reshape(x.shape) if need_x else None, da if need_a else None, db if need_b else None,
                ops.bias_grad(dy2) if need_bias else None, None, None, None)


class _AdapterLinear(torch.autograd.Function):
    """``AdapterLinear`` under torch.func's transforms -> (y, v): a context set up apart keeps inputs and outputs only."""

    @staticmethod
    def forward(x, a, b, bias, layer, adapters, batch):
        return _forward(layer, x, bias, a, b, adapters.scaling, batch.tensors, adapters.cols)

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, a, b, _, layer, adapters, batch = inputs
        ctx.mark_non_differentiable(output[1])
        AdapterLinear.hold(ctx, x, a, b, output[1], layer, adapters, batch)

    backward = AdapterLinear.backward


AdapterLinear.transformed = _AdapterLinear


class GatedLinear(torch.autograd.Function):
    """``ops.gated_linear`` with the gradient of its input."""

    @staticmethod
    def forward(ctx, x, layer, act):
        GatedLinear.hold(ctx, x, layer, act)
        return GatedLinear.product(x, layer, act)

    @staticmethod
    def product(x, layer, act):
        args = _gated_args(layer, act)
        return ops.gated_linear(x.reshape(-1, x.shape[-1]), *args).reshape(*x.shape[:-1], args[2])

    @staticmethod
    def hold(ctx, x, layer, act):
        ctx.save_for_backward(x)
        ctx.args = _gated_args(layer, act)
        ctx.versions = _versions(*ctx.args[:2])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x, = _saved(ctx)
        w, sw, i, fmt, act, rule = ctx.args
        _check_versions("the layer's weight", ctx.versions, w, sw)
        k = x.shape[-1]
        both = ops.gated_grad(x.reshape(-1, k), dh.reshape(-1, i), w, sw, i, fmt, act, rule)
        return ops.input_grad(both, w, sw, 2 * i, k, fmt).reshape(x.shape), None, None


class _GatedLinear(torch.autograd.Function):
    """``GatedLinear`` under torch.func's transforms."""

    @staticmethod
    def forward(x, layer, act):
        return GatedLinear.product(x, layer, act)

    @staticmethod
    def setup_context(ctx, inputs, output):
        GatedLinear.hold(ctx, *inputs)

    @staticmethod
    def vmap(info, in_dims, x, layer, act):
        return _GatedLinear.apply(x.movedim(in_dims[0], 0), layer, act), 0

    backward = GatedLinear.backward


GatedLinear.transformed = _GatedLinear


def _forward(layer: torch.nn.Module, x: torch.Tensor, bias: Optional[torch.Tensor], a, b, scaling, batch, cols):
    """(y, v): in one product where the shape has it, else the layer and then the adapters in place.  ``bias``: one that the
    product's epilogue adds, or None."""
    w, sw, n, k, fmt, block = grad_of(layer)
    x2 = x.reshape(-1, k)
    two_limbs = x2.shape[0] in getattr(layer.mxl_kernel, "dual_m", ())  # (the product with adapters has one)
    if not two_limbs and ops.adapter_linear_supported(x2.shape[0], n, k, fmt, block, a.shape[0], len(cols) - 1, b.shape[2]):
        y, v = ops.adapter_linear(x2, w, sw, fmt, block, getattr(layer.mxl_kernel, "act_rule", 0), bias, a, b, scaling, *batch,
                                  cols)
        return y.reshape(*x.shape[:-1], n), v
    y = layer.mxl_kernel.apply_weights(layer, x, bias)
    return y, ops.adapter_apply(y.view(-1, n), x2, a, b, scaling, *batch, cols)


def apply_adapters(layer: torch.nn.Module, x: torch.Tensor, adapters: LowRankAdapters, batch: AdapterBatch,
                   bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A prepared layer's output with the adapters of a batch's tokens added: x bf16 [..., K] of ``len(batch)`` rows."""
    n, k = layer.mxl_shape
    if not isinstance(adapters, LowRankAdapters) or not isinstance(batch, AdapterBatch):
        raise ValueError("adapters and batch go together: LowRankAdapters and AdapterBatch")
    if tuple(adapters.lora_b.shape[:2]) != (adapters.slots, n) or adapters.lora_a.shape[2] != k:
        raise ValueError(f"the adapters are not of this layer, [{n}, {k}]")
    if batch.slots != adapters.slots:
        raise ValueError(f"the batch is of {batch.slots} slots, the adapters of {adapters.slots}")
    if x.dtype != torch.bfloat16 or x.shape[-1] != k or x.numel() != len(batch) * k:
        raise ValueError(f"adapters need bf16 [..., {k}] of the batch's {len(batch)} rows, got {x.dtype} {tuple(x.shape)}")
    a, b = adapters.lora_a, adapters.lora_b
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, a, b, bias)):
        inner = _function_bias(bias, x, n)
        y = _apply(AdapterLinear, x, a, b, inner, layer, adapters, batch)
        y = y[0] if isinstance(y, tuple) else y
        return y if bias is inner else y + bias
    inner = _epilogue_bias(bias, x, n)  # (any other joins the output, as a layer without adapters has it)
    y = _forward(layer, x, inner, a, b, adapters.scaling, batch.tensors, adapters.cols)[0]
    return y if bias is inner else y + bias

"""Decoder-layer operators as graph ops.

The entry points of kernels.py (residual norm with an 8-bit result, rotary positions over several axes, attention with a
sliding window and visible first tokens) registered in the package's operator library npu_graph with shape
functions, and wrapped with gradients: torch.compile keeps them in its graph and autograd passes through them.  The
functions of this module are what a model calls; outside a compilation they call the kernels' entry points without
the dispatcher, unless a tracer, a dispatch mode, a functorch transform or a tensor subclass has to see the call there.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch.autograd import Function, forward_ad
from torch.library import register_autograd

from . import kernels
from .fusion_attention_graph import gpu_lib, meta_lib, npu_def

npu_def.define("add_rmsnorm_quant(Tensor h, Tensor r, Tensor w, float eps=1e-6, int group=0) -> (Tensor, Tensor, Tensor)")
npu_def.define(
    "rotary_axes(Tensor q, Tensor k, Tensor positions, Tensor inv_freq, int[]? sections=None, bool interleaved=False, "
    "bool inverse=False) -> (Tensor, Tensor)"
)
npu_def.define(
    "window_attention(Tensor q, Tensor k, Tensor v, float scale, int window, int sinks=0, Tensor? lengths=None, "
    "bool keep_low=False) -> (Tensor, Tensor, Tensor)"
)
npu_def.define(
    "window_attention_backward(Tensor q, Tensor k, Tensor v, Tensor out, Tensor dout, Tensor lse, float scale, "
    "int window, int sinks=0, Tensor? lengths=None, Tensor? low=None) -> (Tensor, Tensor, Tensor)"
)
npu_def.define(
    "window_attention_decode(Tensor q, Tensor k_cache, Tensor v_cache, Tensor lengths, float scale, int window, "
    "int sinks=0) -> Tensor"
)


def _add_rmsnorm_quant(h, r, w, eps=1e-6, group=0):
    return kernels.run(kernels._NORM, h, r, w, eps, group)


def _rotary_axes(q, k, positions, inv_freq, sections=None, interleaved=False, inverse=False):
    return kernels.run(kernels._ROTARY, q, k, positions, inv_freq, None if sections is None else tuple(sections), interleaved, inverse)


def _window_attention(q, k, v, scale, window, sinks=0, lengths=None, keep_low=False):
    """kernels.window_attention with three outputs in any case: an empty `low` where it is not kept."""
    outputs = kernels.run(kernels._WINDOW, q, k, v, scale, window, sinks, lengths, keep_low)
    return outputs if keep_low else (*outputs, q.new_empty(0))


def _window_attention_backward(q, k, v, out, dout, lse, scale, window, sinks=0, lengths=None, low=None):
    # the address that counts is known here and not where the gradient's call was traced
    return kernels.run(kernels._WINDOW_BACKWARD, q, k, v, out, kernels.placed(dout), lse, scale, window, sinks, lengths, low)


def _window_attention_decode(q, k_cache, v_cache, lengths, scale, window, sinks=0):
    return kernels.run(kernels._DECODE, q, k_cache, v_cache, lengths, scale, window, sinks)


IMPLEMENTATIONS = {
    "add_rmsnorm_quant": _add_rmsnorm_quant, "rotary_axes": _rotary_axes, "window_attention": _window_attention,
    "window_attention_backward": _window_attention_backward, "window_attention_decode": _window_attention_decode,
}
for _name, _implementation in IMPLEMENTATIONS.items():
    gpu_lib.impl(_name, _implementation)


def _refuse_jvp():
    """Under a functorch jvp a registered op would give a result with a tangent of zero."""
    layers = torch._C._functorch.get_interpreter_stack() or ()
    if any(layer.key() == torch._C._functorch.TransformType.Jvp for layer in layers):
        raise NotImplementedError("the decoder operators have no derivative under torch.func.jvp")


# The kernels' entry points as calls of the registered ops, in the order of kernels._NORM ..., without gradients as those are
@torch.no_grad()
def _registered_norm(h, r, w, eps, group):
    _refuse_jvp()
    return torch.ops.npu_graph.add_rmsnorm_quant(h, r, w, float(eps), int(group))


@torch.no_grad()
def _registered_rotary(q, k, positions, inv_freq, sections, interleaved, inverse):
    _refuse_jvp()
    return torch.ops.npu_graph.rotary_axes(q, k, positions, inv_freq, sections, bool(interleaved), bool(inverse))


@torch.no_grad()
def _registered_window(q, k, v, scale, window, sinks, lengths, keep_low):
    _refuse_jvp()
    outputs = torch.ops.npu_graph.window_attention(q, k, v, float(scale), int(window), int(sinks), lengths, bool(keep_low))
    return outputs if keep_low else outputs[:2]


@torch.no_grad()
def _registered_window_backward(q, k, v, out, dout, lse, scale, window, sinks, lengths, low):
    _refuse_jvp()
    return torch.ops.npu_graph.window_attention_backward(q, k, v, out, dout, lse, float(scale), int(window), int(sinks), lengths, low)


@torch.no_grad()
def _registered_decode(q, k_cache, v_cache, lengths, scale, window, sinks):
    _refuse_jvp()
    return torch.ops.npu_graph.window_attention_decode(q, k_cache, v_cache, lengths, float(scale), int(window), int(sinks))


REGISTERED = (_registered_norm, _registered_rotary, _registered_window, _registered_window_backward, _registered_decode)


def registered_window_attention(q, k, v, scale, window, sinks, lengths):
    """kernels.window_attention_with_gradients as a call of the registered op and its gradient."""
    _refuse_jvp()
    return torch.ops.npu_graph.window_attention(q, k, v, float(scale), int(window), int(sinks), lengths, True)[0]


def _add_rmsnorm_quant_meta(h, r, w, eps=1e-6, group=0):
    groups = (h.shape[-1] + 127) // 128 if group else 1
    return (torch.empty(h.shape, dtype=torch.float8_e4m3fn, device=h.device),
            torch.empty(tuple(h.shape[:-1]) + (groups,), dtype=torch.float32, device=h.device),
            torch.empty(h.shape, dtype=h.dtype, device=h.device))


def _rotary_axes_meta(q, k, positions, inv_freq, sections=None, interleaved=False, inverse=False):
    return torch.empty_like(q), torch.empty_like(k)


def _window_attention_meta(q, k, v, scale, window, sinks=0, lengths=None, keep_low=False):
    return (torch.empty_like(q), torch.empty(q.shape[:3], dtype=torch.float32, device=q.device),
            torch.empty_like(q) if keep_low else q.new_empty(0))


def _window_attention_backward_meta(q, k, v, out, dout, lse, scale, window, sinks=0, lengths=None, low=None):
    return torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)


def _window_attention_decode_meta(q, k_cache, v_cache, lengths, scale, window, sinks=0):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


meta_lib.impl("add_rmsnorm_quant", _add_rmsnorm_quant_meta)
meta_lib.impl("rotary_axes", _rotary_axes_meta)
meta_lib.impl("window_attention", _window_attention_meta)
meta_lib.impl("window_attention_backward", _window_attention_backward_meta)
meta_lib.impl("window_attention_decode", _window_attention_decode_meta)


def _needs_grad(*tensors: torch.Tensor) -> bool:
    return torch.is_grad_enabled() and any(t.requires_grad for t in tensors)


def _has_tangent(*tensors: torch.Tensor) -> bool:
    return forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


# Gradients.  A compilation sees those of the registered ops.  Eager calls go through autograd functions over the kernels'
# entry points: the dispatcher's way to a Python kernel and its gradient costs about 40 us of host time more, half of
# what a short text's kernels run.  Rotary's function is here and shares its two steps (what the forward keeps, what
# the backward calls) with the op; window attention's is csrc/mi_ops.cpp's.  Forward-mode derivatives: rotary's function has
# one, everything else refuses operands with a tangent (csrc/mi_ops.cpp).
def _rotary_context(ctx, inputs, output):
    _, _, positions, inv_freq, sections, interleaved, inverse = inputs
    ctx.save_for_backward(positions, inv_freq)
    ctx.form = (sections, interleaved, inverse)


def _columns(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy with contiguous columns (contiguous() returns an empty tensor as it is)."""
    return t if t.stride(-1) == 1 else t.clone(memory_format=torch.contiguous_format)


def _rotary_gradient(ctx, call, dq, dk):
    positions, inv_freq = ctx.saved_tensors
    sections, interleaved, inverse = ctx.form
    # a rotation's gradient is the rotation back
    dq, dk = _columns(dq), _columns(dk)
    return (*call(dq, dk, positions, inv_freq, sections, interleaved, not inverse), None, None, None, None, None)


def _window_context(ctx, inputs, output):
    q, k, v, scale, window, sinks, lengths, keep_low = inputs
    out, lse, low = output
    ctx.save_for_backward(q, k, v, out, lse, low if keep_low else None, lengths)
    ctx.form = (scale, window, sinks)
    ctx.mark_non_differentiable(lse, low)
    ctx.set_materialize_grads(False)


def _window_gradient(ctx, call, dout):
    q, k, v, out, lse, low, lengths = ctx.saved_tensors
    if dout is None:
        return (None,) * 8
    scale, window, sinks = ctx.form
    return (*call(q, k, v, out, dout, lse, scale, window, sinks, lengths, low), None, None, None, None, None)


register_autograd("npu_graph::rotary_axes", lambda ctx, dq, dk: _rotary_gradient(ctx, torch.ops.npu_graph.rotary_axes, dq, dk),
                  setup_context=_rotary_context)
register_autograd("npu_graph::window_attention",
                  lambda ctx, dout, *_: _window_gradient(ctx, torch.ops.npu_graph.window_attention_backward, dout),
                  setup_context=_window_context)


class RotaryFunction(Function):
    @staticmethod
    def forward(ctx, *inputs):
        output = kernels.rotary_axes(*inputs)
        _rotary_context(ctx, inputs, output)
        ctx.save_for_forward(*inputs[:4])
        return output

    @staticmethod
    def backward(ctx, dq, dk):
        return _rotary_gradient(ctx, rotary_axes, dq, dk)  # a gradient of it can be asked for in turn

    @staticmethod
    def jvp(ctx, tq, tk, *rest):
        q, k, positions, inv_freq = ctx.saved_tensors
        # a linear map: tangents turn as their operands do
        tq, tk = (torch.zeros_like(x) if t is None else _columns(t) for t, x in ((tq, q), (tk, k)))
        return rotary_axes(tq, tk, positions, inv_freq, *ctx.form)


def add_rmsnorm_quant(h: torch.Tensor, r: torch.Tensor, w: torch.Tensor, eps: float = 1e-6, group: int = 0):
    """(q, scales, h + r): kernels.add_rmsnorm_quant as a graph op.  Serving only: an 8-bit result has no gradient."""
    if torch.compiler.is_compiling():
        return torch.ops.npu_graph.add_rmsnorm_quant(h, r, w, eps, group)
    return kernels.add_rmsnorm_quant(h, r, w, eps, group)


def rotary_axes(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                sections: Optional[Sequence[int]] = None, interleaved: bool = False, inverse: bool = False):
    """kernels.rotary_axes as a graph op with gradients for q and k, eagerly also in forward mode."""
    if torch.compiler.is_compiling():
        return torch.ops.npu_graph.rotary_axes(q, k, positions, inv_freq, sections, interleaved, inverse)
    if kernels.watched(q, k, positions, inv_freq):
        _refuse_jvp()
        return torch.ops.npu_graph.rotary_axes(q, k, positions, inv_freq, sections, interleaved, inverse)
    if _has_tangent(inv_freq):
        raise NotImplementedError("rotary_axes has no derivative for its frequencies")
    call = RotaryFunction.apply if _needs_grad(q, k) or _has_tangent(q, k) else kernels.rotary_axes
    return call(q, k, positions, inv_freq, sections, interleaved, inverse)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, window: int, sinks: int = 0,
                     lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The output of kernels.window_attention as a graph op with gradients for q, k and v."""
    train = _needs_grad(q, k, v)
    if torch.compiler.is_compiling():
        return torch.ops.npu_graph.window_attention(q, k, v, scale, window, sinks, lengths, train)[0]
    if train:
        return kernels.window_attention_with_gradients(q, k, v, scale, window, sinks, lengths)
    return kernels.window_attention(q, k, v, scale, window, sinks, lengths)[0]


def window_attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor,
                            scale: float, window: int, sinks: int = 0) -> torch.Tensor:
    """kernels.window_attention_decode as a graph op (inference)."""
    if torch.compiler.is_compiling():
        return torch.ops.npu_graph.window_attention_decode(q, k_cache, v_cache, lengths, scale, window, sinks)
    return kernels.window_attention_decode(q, k_cache, v_cache, lengths, scale, window, sinks)

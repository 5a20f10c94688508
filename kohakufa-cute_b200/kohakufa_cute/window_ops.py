"""Autograd and fake implementations for causal attention with a sliding window and sinks.

Like the attention operator (``_ops.py``): eager calls use a ``torch.autograd.Function`` (least host overhead), calls
under ``torch.compile`` the ``kohakufa_cute::window_forward`` / ``window_backward`` custom operators.  Only O is
differentiable, and only once; the two row statistics are saved outputs.  Calls that nobody differentiates keep none
(``kohakufa_cute::window_inference`` under ``torch.compile``): only these reach the decoding kernels, which form none.
"""

from typing import Optional

import torch

from . import native


@torch.library.custom_op("kohakufa_cute::window_forward", mutates_args=())
def forward(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: Optional[torch.Tensor], start: int, window: int,
    sinks: int, scale: float
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return native.window_forward(q, k, v, starts, start, window, sinks, scale)


@forward.register_fake
def _forward_fake(q, k, v, starts, start, window, sinks, scale):
    stats = torch.empty(q.shape[:-1], device=q.device, dtype=torch.float32)
    return torch.empty_like(q), stats, torch.empty_like(stats)


@torch.library.custom_op("kohakufa_cute::window_inference", mutates_args=())
def inference(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: Optional[torch.Tensor], start: int, window: int,
    sinks: int, scale: float
) -> torch.Tensor:
    return native.window_forward(q, k, v, starts, start, window, sinks, scale, statistics=False)[0]


@inference.register_fake
def _inference_fake(q, k, v, starts, start, window, sinks, scale):
    return torch.empty_like(q)


@torch.library.custom_op("kohakufa_cute::window_backward", mutates_args=())
def backward(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, maximum: torch.Tensor,
    logsum: torch.Tensor, dout: torch.Tensor, start: int, window: int, sinks: int, scale: float
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return native.window_backward(q, k, v, out, maximum, logsum, dout, start, window, sinks, scale)


@backward.register_fake
def _backward_fake(q, k, v, out, maximum, logsum, dout, start, window, sinks, scale):
    return torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)


def _setup_context(ctx, inputs, output):
    q, k, v, _, *ctx.parameters = inputs
    out, maximum, logsum = output
    ctx.save_for_backward(q, k, v, out, maximum, logsum)
    ctx.mark_non_differentiable(maximum, logsum)


def _autograd_backward(ctx, dout, dmaximum, dlogsum):
    return *backward(*ctx.saved_tensors, dout, *ctx.parameters), None, None, None, None, None


forward.register_autograd(_autograd_backward, setup_context=_setup_context)


class _EagerWindow(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, start, window, sinks, scale):
        out, maximum, logsum = native.window_forward(q, k, v, None, start, window, sinks, scale)
        ctx.parameters = start, window, sinks, scale
        ctx.save_for_backward(q, k, v, out, maximum, logsum)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, maximum, logsum = ctx.saved_tensors
        grads = native.window_backward(q, k, v, out, maximum, logsum, dout, *ctx.parameters)
        if torch.is_grad_enabled():  # create_graph: gradients that raise when they are differentiated, not constants
            twice = torch._C._functions.DelayedError("sliding_window_attention cannot be differentiated twice", 3)
            grads = twice(*(grad.detach().requires_grad_() for grad in grads))
        return *grads, None, None, None, None


def attention(q, k, v, starts, start, window, sinks, scale):
    differentiated = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if starts is None:
        # keys behind the last query's position are seen by nobody: leave them out (and their gradients zero)
        end = start + q.shape[2]
        if end < k.shape[2]:
            k, v = k[:, :, :end], v[:, :, :end]
    elif differentiated:
        raise ValueError("sliding_window_attention: gradients need one query_start (an int) for the whole batch.")
    if torch.compiler.is_compiling():
        if not differentiated:
            return inference(q, k, v, starts, start, window, sinks, scale)
        return forward(q, k, v, starts, start, window, sinks, scale)[0]
    if not differentiated:
        return native.window_forward(q, k, v, starts, start, window, sinks, scale, statistics=False)[0]
    return _EagerWindow.apply(q, k, v, start, window, sinks, scale)

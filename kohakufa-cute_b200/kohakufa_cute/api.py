"""Public attention API: strict CUDA attention, SDPA-style wrappers and neighbourhood attention.

Signatures, argument meaning and error behaviour follow the reference package
(src/kohakufa_cute/api.py:76-225 of the reference project):

* ``attention(q, k, v, *, mask, causal, scale, center_keys)`` - implicit grouped-query heads,
  boolean mask and causal visibility may be combined;
* ``scaled_dot_product_attention`` - PyTorch SDPA argument convention, strict (raises on
  anything unsupported); causal together with a mask is rejected, differing head counts need
  ``enable_gqa=True``;
* ``automatic_scaled_dot_product_attention`` - the same kernels when the call is supported,
  PyTorch's native SDPA otherwise (CPU, FP32, additive masks, dropout, ...); an error raised by
  a selected kernel is never hidden behind the native path;
* ``neighborhood_attention`` / ``neighborhood_attention_3d`` - shifted-window attention, head dim 64.

Validation errors are ``ValueError``; kernel or library errors propagate unchanged.
"""

from functools import lru_cache
from math import isfinite, prod

import torch
from torch.autograd import forward_ad

from . import native

_native_sdpa = torch.nn.functional.scaled_dot_product_attention
_HALF_TYPES = (torch.float16, torch.bfloat16)
_SUPPORTED_CAPABILITY = (10, 0)
_LONGEST = 2**40  # positions end at 2^32


def _device_supported(device):
    if torch.compiler.is_compiling():
        return torch.cuda.get_device_capability(device) == _SUPPORTED_CAPABILITY
    return _device_supported_once(device)


@lru_cache(maxsize=None)
def _device_supported_once(device):
    supported = torch.cuda.get_device_capability(device) == _SUPPORTED_CAPABILITY
    if supported and native.fast is not None and device.index is not None:
        native.fast.allow(device.index)
    return supported


def _check_arguments(q, k, v, mask, dropout, causal, gqa, *, combined_mask=False):
    """Raises ``ValueError`` for everything the strict operator does not accept."""
    if dropout != 0.0:
        raise ValueError("CuTe attention does not support dropout.")
    if any(getattr(t, "ndim", None) != 4 for t in (q, k, v)):
        raise ValueError("CuTe attention requires 4D [batch, heads, sequence, dim] Q/K/V.")
    if q.device.type != "cuda" or k.device != q.device or v.device != q.device:
        raise ValueError("CuTe attention requires Q/K/V on the same CUDA device.")
    if q.dtype not in _HALF_TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("CuTe attention requires matching FP16/BF16 Q/K/V; FP32 attention is unsupported.")
    if 0 in q.shape or 0 in k.shape or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError("CuTe attention requires nonempty matching batch/head dimensions and equal K/V shapes.")
    if q.shape[1] % k.shape[1] or not 1 <= q.shape[3] <= 512:
        raise ValueError("CuTe attention requires head dimensions 1..512 and query heads divisible by K/V heads.")
    if not gqa and q.shape[1] != k.shape[1]:
        raise ValueError("CuTe SDPA requires enable_gqa=True for differing Q and K/V head counts.")
    if mask is not None:
        if mask.dtype != torch.bool or mask.device != q.device:
            raise ValueError("CuTe attention requires a boolean mask on the Q/K/V device.")
        if causal and not combined_mask:
            raise ValueError("CuTe attention requires causal visibility folded into the boolean mask.")
    if not _device_supported(q.device):
        raise ValueError("This build of CuTe attention requires an sm_100 (B200) device.")


def _supported(q, k, v, mask, dropout, causal, gqa):
    """Non-raising twin of ``_check_arguments`` used by the automatic entry point."""
    try:
        tensors = (q, k, v)
        return (
            dropout == 0.0
            and all(t.ndim == 4 for t in tensors)
            and q.device.type == "cuda"
            and k.device == q.device == v.device
            and q.dtype in _HALF_TYPES
            and k.dtype == q.dtype == v.dtype
            and 0 not in q.shape
            and 0 not in k.shape
            and k.shape == v.shape
            and q.shape[0] == k.shape[0]
            and q.shape[3] == k.shape[3]
            and q.shape[3] <= 512
            and q.shape[1] % k.shape[1] == 0
            and (gqa or q.shape[1] == k.shape[1])
            and (mask is None or (mask.dtype == torch.bool and mask.device == q.device and not causal))
            and _device_supported(q.device)
        )
    except (AttributeError, TypeError):
        return False


def _center_keys(k):
    """Subtract each (batch, head)'s mean key in FP32 and round once to the input dtype."""
    if k.device.type == "cuda":
        from . import _ops

        return _ops.center_keys(k)
    keys = k.float()
    return (keys - keys.mean(dim=-2, keepdim=True)).to(k.dtype)


def attention(q, k, v, *, mask=None, causal=False, scale=None, center_keys=False):
    """Strict CUDA attention; Q is ``[B, Hq, Sq, D]``, K/V are ``[B, Hkv, Sk, D]`` with ``Hq % Hkv == 0``.

    ``mask`` is a boolean tensor broadcastable to ``[B, Hq, Sq, Sk]`` (True = visible) and may be
    combined with ``causal`` (key ``c`` visible to query ``r`` iff ``c <= r``).  ``center_keys``
    subtracts the per-(batch, K/V head) mean key in FP32 before one rounding to the input dtype;
    softmax is invariant to that shift and autograd projects the key gradient back.
    """
    _check_arguments(q, k, v, mask, 0.0, causal, True, combined_mask=True)
    if center_keys:
        k = _center_keys(k)
    from . import _ops

    return _ops.attention(q, k, v, mask=mask, causal=causal, scale=scale)


def scaled_dot_product_attention(
    query, key, value, attn_mask=None, dropout_p=0.0, is_causal=False, scale=None, enable_gqa=False
):
    """Strict implementation with the PyTorch SDPA argument convention."""
    _check_arguments(query, key, value, attn_mask, dropout_p, is_causal, enable_gqa)
    from . import _ops

    return _ops.attention(query, key, value, mask=attn_mask, causal=is_causal, scale=scale)


def automatic_scaled_dot_product_attention(
    query, key, value, attn_mask=None, dropout_p=0.0, is_causal=False, scale=None, enable_gqa=False
):
    """Uses the CUDA kernels for supported calls and PyTorch's native SDPA for everything else."""
    if getattr(query, "device", None) is not None and query.device.type == "cuda":
        if _supported(query, key, value, attn_mask, dropout_p, is_causal, enable_gqa):
            return scaled_dot_product_attention(query, key, value, attn_mask, dropout_p, is_causal, scale, enable_gqa)
    return _native_sdpa(query, key, value, attn_mask, dropout_p, is_causal, scale=scale, enable_gqa=enable_gqa)


def _window_arguments(name, batch, device, window, sinks, query_start):
    """``(starts, start)`` of checked window arguments: a tensor of positions per sequence, or ``None`` and one int."""
    if not isinstance(window, int) or isinstance(window, bool) or window < 1:
        raise ValueError(f"{name}: window must be a positive integer.")
    if not isinstance(sinks, int) or isinstance(sinks, bool) or sinks < 0:
        raise ValueError(f"{name}: sinks must be a nonnegative integer.")
    if isinstance(query_start, torch.Tensor):
        if query_start.dtype != torch.int32 or query_start.shape != (batch,) or query_start.device != device:
            raise ValueError(f"{name}: a query_start tensor must be int32 [batch] on the Q device.")
        return query_start.contiguous(), 0
    if not isinstance(query_start, int) or isinstance(query_start, bool) or not 0 <= query_start < 2**31:
        raise ValueError(f"{name}: query_start must be a nonnegative 32-bit integer or an int32 [batch] tensor.")
    return None, query_start


def _no_tangent(name, *tensors):
    """Raises ``ValueError`` for operands with forward-mode tangents: the kernels would drop them."""
    if torch.compiler.is_compiling():
        return
    if any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):  # (none outside a dual level)
        raise ValueError(f"{name}: forward-mode differentiation is not supported.")


def _in_64_bits(window, sinks):
    """The two as the library takes them: beyond every position, longer is the same (an integer may have any length)."""
    return min(window, _LONGEST), min(sinks, _LONGEST)


def _resolved_scale(name, scale, head_dim):
    scale = head_dim**-0.5 if scale is None else float(scale)
    if not isfinite(scale) or abs(scale) > torch.finfo(torch.float32).max:
        raise ValueError(f"{name}: scale must be a finite FP32 number.")
    return scale


def sliding_window_attention(q, k, v, *, window, sinks=0, query_start=0, scale=None):
    """Causal attention with a sliding window and a few first tokens (sinks) that stay visible.

    Q is ``[B, Hq, Sq, D]``, K/V are ``[B, Hkv, Sk, D]`` with ``Hq % Hkv == 0``.  Query row ``r`` stands at position
    ``p = query_start + r`` of its key sequence and sees key ``c`` iff ``c <= p`` and (``c > p - window`` or
    ``c < sinks``); a row that sees no key is zero.  ``query_start`` is an int (0: queries and keys start together, as
    in training), or an int32 ``[B]`` CUDA tensor with one position per sequence, read by the kernels (a captured
    graph can be replayed with new positions; any value is allowed).  Keys and values behind a sequence's last position
    may hold anything; up to there they have to be finite, also where no row sees them.  Differentiable (once, in reverse mode) with respect to Q, K and V when ``query_start`` is an int.
    """
    if native.fast is not None and not torch.compiler.is_compiling():
        out = native.fast.window_attention(q, k, v, window, sinks, query_start, scale)
        if out is not None:
            return out
    _check_arguments(q, k, v, None, 0.0, False, True)
    _no_tangent("sliding_window_attention", q, k, v)
    starts, start = _window_arguments("sliding_window_attention", q.shape[0], q.device, window, sinks, query_start)
    scale = _resolved_scale("sliding_window_attention", scale, q.shape[-1])
    from . import window_ops

    return window_ops.attention(q, k, v, starts, start, *_in_64_bits(window, sinks), scale)


def neighborhood_attention(q, k, v, *, spatial_shape, window_size, scale=None):
    """Non-causal 2-D/3-D neighbourhood attention, stride and dilation one, head dim 64.

    Q/K/V: matching FP16/BF16 CUDA tensors ``[B, heads, prod(spatial_shape), 64]``.
    ``spatial_shape`` is ``(height, width)`` or ``(depth, height, width)``; ``window_size`` is an
    int or a matching tuple and each window must fit its axis.  On each axis the window starts at
    ``clamp(query - window // 2, 0, extent - window)`` (shifted at the borders, also for even
    windows), so every query sees exactly ``prod(window_size)`` keys.
    """
    if (
        not isinstance(spatial_shape, (tuple, list))
        or len(spatial_shape) not in (2, 3)
        or any(type(n) is not int or n <= 0 for n in spatial_shape)
    ):
        raise ValueError("spatial_shape must contain two or three positive integers.")
    if type(window_size) is int:
        window_size = (window_size,) * len(spatial_shape)
    if (
        not isinstance(window_size, (tuple, list))
        or len(window_size) != len(spatial_shape)
        or any(type(n) is not int or n <= 0 or n > extent for n, extent in zip(window_size, spatial_shape))
    ):
        raise ValueError("window_size must contain positive integers no larger than spatial_shape.")
    _check_arguments(q, k, v, None, 0, False, False)
    if q.shape != k.shape or q.shape[-1] != 64 or q.shape[2] != prod(spatial_shape):
        raise ValueError("Neighborhood attention requires matching [B, heads, prod(spatial_shape), 64] Q/K/V.")
    scale = 0.125 if scale is None else float(scale)
    if not isfinite(scale) or abs(scale) > torch.finfo(torch.float32).max:
        raise ValueError("Neighborhood attention requires a finite FP32 scale.")
    from .neighborhood_ops import forward

    # The library reads physical storage: resolve lazy conj/neg flags while autograd can still
    # map the logical operands back to their bases.
    q, k, v = (t.resolve_conj().resolve_neg() for t in (q, k, v))
    return forward(q, k, v, list(spatial_shape), list(window_size), scale)[0]


def neighborhood_attention_3d(q, k, v, kernel_size, is_causal=None, scale=None):
    """Video-latent layout adapter: ``[B, T, H, W, heads, 64]`` in and out, non-causal.

    Windows larger than an axis are clipped to it (an 11-frame window on one frame is legal here,
    unlike in the flattened API).  Pass ``scale=1.0`` when Q already carries the scale.
    """
    if any(getattr(t, "ndim", None) != 6 for t in (q, k, v)) or q.shape != k.shape or q.shape != v.shape:
        raise ValueError("3D neighborhood attention requires matching [B, T, H, W, heads, 64] Q/K/V.")
    causal = (False,) * 3 if is_causal is None else ((is_causal,) * 3 if type(is_causal) is bool else is_causal)
    if not isinstance(causal, (tuple, list)) or len(causal) != 3 or any(flag is not False for flag in causal):
        raise ValueError("3D neighborhood attention supports only noncausal windows.")
    window = (kernel_size,) * 3 if type(kernel_size) is int else kernel_size
    if not isinstance(window, (tuple, list)) or len(window) != 3 or any(type(n) is not int or n <= 0 for n in window):
        raise ValueError("kernel_size must be a positive integer or three positive integers.")
    spatial = tuple(int(n) for n in q.shape[1:4])
    window = tuple(min(n, extent) for n, extent in zip(window, spatial))
    flat = [t.flatten(1, 3).transpose(1, 2) for t in (q, k, v)]
    out = neighborhood_attention(*flat, spatial_shape=spatial, window_size=window, scale=scale)
    return out.transpose(1, 2).reshape(q.shape)

"""Key/value cache held in 4 bits: written, read back and attended to.

Each token's row of ``D`` channels is held in groups of 64: a scale and a zero in the model's 16-bit type and a 4-bit
code per channel, 36 bytes instead of 128.  ``scale = round16((max - min) / 15)``, ``zero = min``,
``code = round_half_even((x - zero) / scale)``; the value a code stands for is ``zero + scale * code``, at most half a
``scale`` from ``x`` (plus 15 times the rounding of the scale at the group's maximum).  Inference only.
"""

from typing import NamedTuple, Optional

import torch

from . import native
from .api import _HALF_TYPES, _device_supported, _in_64_bits, _no_tangent, _resolved_scale, _window_arguments

GROUP = 64


class QuantizedCache(NamedTuple):
    """The four tensors of a cache: codes ``uint8 [B, H, capacity, D / 2]`` (byte ``i`` holds channels ``2i`` in its low
    and ``2i + 1`` in its high half) and params ``[B, H, capacity, D / 64, 2]`` (scale, zero) in the model's type."""

    k_codes: torch.Tensor
    k_params: torch.Tensor
    v_codes: torch.Tensor
    v_params: torch.Tensor


def quantized_cache(batch, heads, capacity, head_dim, *, dtype=torch.bfloat16, device="cuda"):
    """An empty (zero) cache for ``capacity`` tokens of ``batch`` sequences; ``head_dim`` a multiple of 64 up to 512."""
    if any(not isinstance(n, int) or isinstance(n, bool) or n < 1 for n in (batch, heads, capacity, head_dim)):
        raise ValueError("quantized_cache: batch, heads, capacity and head_dim must be positive integers.")
    if head_dim % GROUP or head_dim > 512:
        raise ValueError("quantized_cache: head_dim must be a multiple of 64 up to 512.")
    if dtype not in _HALF_TYPES:
        raise ValueError("quantized_cache: dtype must be FP16 or BF16.")
    codes = [torch.zeros((batch, heads, capacity, head_dim // 2), dtype=torch.uint8, device=device) for _ in range(2)]
    params = [torch.zeros((batch, heads, capacity, head_dim // GROUP, 2), dtype=dtype, device=device) for _ in range(2)]
    return QuantizedCache(codes[0], params[0], codes[1], params[1])


def _check_cache(name, cache):
    """Raises ``ValueError`` unless ``cache`` is a quantised cache this library can address."""
    if not isinstance(cache, tuple) or len(cache) != 4 or any(not isinstance(t, torch.Tensor) for t in cache):
        raise ValueError(f"{name}: cache must be a QuantizedCache.")
    kc, kp, vc, vp = cache
    shape, pair, device = kc.shape, kp.shape, kc.device
    if kc.dtype != torch.uint8 or len(shape) != 4 or 0 in shape or shape[3] % 32 or shape[3] > 256:
        raise ValueError(f"{name}: cache codes must be uint8 [B, H, capacity, D / 2], D a multiple of 64 up to 512.")
    if kp.dtype not in _HALF_TYPES or pair != (*shape[:3], shape[3] // 32, 2):
        raise ValueError(f"{name}: cache params must be FP16/BF16 [B, H, capacity, D / 64, 2].")
    if vc.dtype != kc.dtype or vc.shape != shape or vp.dtype != kp.dtype or vp.shape != pair:
        raise ValueError(f"{name}: the cache's key and value tensors must match.")
    if device.type != "cuda" or kp.device != device or vc.device != device or vp.device != device:
        raise ValueError(f"{name}: the cache must live on one CUDA device.")
    if not _device_supported(device):
        raise ValueError("This build of CuTe attention requires an sm_100 (B200) device.")


def _may_overlap(t):
    """Whether two elements of ``t`` may share memory: an axis whose stride does not clear what the axes of smaller
    strides reach.  An axis of one element has no stride that matters."""
    reach = 0
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if size > 1:
            if stride <= reach:
                return True
            reach += stride * (size - 1)
    return False


def _positions(name, what, value, batch, device):
    """``(tensor, int)`` of a position argument: one int for all sequences or an int32 ``[batch]`` tensor."""
    if isinstance(value, torch.Tensor):
        if value.dtype != torch.int32 or value.shape != (batch,) or value.device != device:
            raise ValueError(f"{name}: a {what} tensor must be int32 [batch] on the cache's device.")
        return value.contiguous(), 0
    if not isinstance(value, int) or isinstance(value, bool) or not 0 <= value < 2**31:
        raise ValueError(f"{name}: {what} must be a nonnegative 32-bit integer or an int32 [batch] tensor.")
    return None, value


def _no_gradient(name, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError(f"{name}: inference only; the operands must not require gradients.")
    _no_tangent(name, *tensors)


@torch.library.custom_op("kohakufa_cute::quantized_cache_write",
                         mutates_args=("k_codes", "k_params", "v_codes", "v_params"))
def _write_op(k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor,
              v_params: torch.Tensor, starts: Optional[torch.Tensor], lengths: Optional[torch.Tensor],
              start: int) -> None:
    native.cache_write(k, v, k_codes, k_params, v_codes, v_params, starts, lengths, start)


@_write_op.register_fake
def _write_fake(k, v, k_codes, k_params, v_codes, v_params, starts, lengths, start):
    return None


@torch.library.custom_op("kohakufa_cute::quantized_cache_read", mutates_args=())
def _read_op(k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor, v_params: torch.Tensor,
             starts: Optional[torch.Tensor], start: int, length: int) -> tuple[torch.Tensor, torch.Tensor]:
    return native.cache_read(k_codes, k_params, v_codes, v_params, starts, start, length)


@_read_op.register_fake
def _read_fake(k_codes, k_params, v_codes, v_params, starts, start, length):
    shape = (k_codes.shape[0], k_codes.shape[1], length, 2 * k_codes.shape[3])
    k = torch.empty(shape, device=k_codes.device, dtype=k_params.dtype)
    return k, torch.empty_like(k)


@torch.library.custom_op("kohakufa_cute::quantized_cache_attention", mutates_args=())
def _attention_op(q: torch.Tensor, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor,
                  v_params: torch.Tensor, starts: Optional[torch.Tensor], start: int, window: int, sinks: int,
                  scale: float) -> torch.Tensor:
    return native.cache_attention(q, k_codes, k_params, v_codes, v_params, starts, start, window, sinks, scale)


@_attention_op.register_fake
def _attention_fake(q, k_codes, k_params, v_codes, v_params, starts, start, window, sinks, scale):
    return torch.empty_like(q)


def quantized_cache_write(cache, k, v, *, start=0, lengths=None):
    """Quantises the rows of ``k`` and ``v`` (``[B, H, n, D]``) into ``cache`` in place.

    Row ``r`` of sequence ``b`` goes to position ``start_b + r``; ``start`` is an int or an int32 ``[B]`` tensor.
    ``lengths`` (int32 ``[B]``) limits each sequence to its first rows (a padded batch of prompts).  Everything else in
    the cache stays as it was: rows at or behind a sequence's length, and rows whose position lies outside the cache
    (an int ``start`` that would write past the end is refused).  A group of channels with a value that is not finite, or
    with values further apart than FP32 holds (near the ends of BF16's range), reads back as NaN.  The cache's tensors,
    and the rows of each, must not overlap in memory.
    """
    if native.fast is not None and not torch.compiler.is_compiling():
        if native.fast.cache_write(cache, k, v, start, lengths):
            return
    name = "quantized_cache_write"
    _check_cache(name, cache)
    kc, kp = cache[0], cache[1]
    if any(getattr(t, "ndim", None) != 4 for t in (k, v)) or k.shape != v.shape or 0 in k.shape:
        raise ValueError(f"{name}: K and V must be nonempty [B, H, n, D] tensors of one shape.")
    if k.device != kc.device or v.device != kc.device or k.dtype != kp.dtype or v.dtype != kp.dtype:
        raise ValueError(f"{name}: K and V must have the cache's device and type.")
    if (k.shape[0], k.shape[1], k.shape[3]) != (kc.shape[0], kc.shape[1], 2 * kc.shape[3]):
        raise ValueError(f"{name}: K and V must match the cache's batch, heads and channels.")
    if any(not t.is_contiguous() and _may_overlap(t) for t in cache):
        raise ValueError(f"{name}: the cache's rows overlap in memory (an expanded view can only be read).")
    _no_gradient(name, k, v, kp, cache[3])
    starts, at = _positions(name, "start", start, kc.shape[0], kc.device)
    if starts is None and at + k.shape[2] > kc.shape[2]:
        raise ValueError(f"{name}: rows {at}..{at + k.shape[2]} do not fit a cache of {kc.shape[2]} tokens.")
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor):
            raise ValueError(f"{name}: lengths must be an int32 [batch] tensor.")
        lengths = _positions(name, "lengths", lengths, kc.shape[0], kc.device)[0]
    if torch.compiler.is_compiling():
        _write_op(k, v, *cache, starts, lengths, at)
    else:
        native.cache_write(k, v, *cache, starts, lengths, at)
        for t in cache:  # a change in place, for what autograd may have saved (inference tensors keep no count)
            if not t.is_inference():
                torch.autograd.graph.increment_version(t)


def quantized_cache_read(cache, *, start=0, length=None):
    """``(k, v)``: the values of ``length`` rows of every sequence from position ``start`` (an int or an int32 ``[B]``
    tensor) on, ``[B, H, length, D]`` in the cache's type, rounded once (at most the type's largest value).  ``length``
    defaults to the rest of the cache behind an int ``start``; rows outside the cache (possible with a tensor) read as
    zeros.  Inference only."""
    if native.fast is not None and not torch.compiler.is_compiling():
        rows = native.fast.cache_read(cache, start, length)
        if rows is not None:
            return rows
    name = "quantized_cache_read"
    _check_cache(name, cache)
    kc = cache[0]
    _no_gradient(name, cache[1], cache[3])
    starts, at = _positions(name, "start", start, kc.shape[0], kc.device)
    if length is None:
        if starts is not None:
            raise ValueError(f"{name}: a start per sequence needs a length.")
        length = kc.shape[2] - at
    if not isinstance(length, int) or isinstance(length, bool) or length < 1:
        raise ValueError(f"{name}: length must be a positive integer.")
    if starts is None and at + length > kc.shape[2]:
        raise ValueError(f"{name}: rows {at}..{at + length} lie outside a cache of {kc.shape[2]} tokens.")
    if torch.compiler.is_compiling():
        return _read_op(*cache, starts, at, length)
    return native.cache_read(*cache, starts, at, length)


def quantized_cache_attention(q, cache, *, query_start, window=None, sinks=0, scale=None):
    """Causal attention of a few new tokens to a 4-bit cache that already holds their keys and values.

    Q is ``[B, Hq, Sq, D]`` with ``D`` 64 or 128 and ``Hq`` a multiple of the cache's heads.  Query row ``r`` stands at
    position ``p = query_start + r`` (an int, or an int32 ``[B]`` tensor read by the kernels) and sees key ``c`` iff
    ``c <= p``; with a ``window`` only ``c > p - window`` or ``c < sinks`` of these, as in
    ``sliding_window_attention``.  A row that sees no key is zero; what lies behind a sequence's last position may hold
    anything.  Inference only.
    """
    if native.fast is not None and not torch.compiler.is_compiling():
        out = native.fast.cache_attention(q, cache, query_start, window, sinks, scale)
        if out is not None:
            return out
    name = "quantized_cache_attention"
    _check_cache(name, cache)
    kc, kp = cache[0], cache[1]
    if getattr(q, "ndim", None) != 4 or 0 in q.shape:
        raise ValueError(f"{name}: Q must be a nonempty [B, Hq, Sq, D] tensor.")
    if q.device != kc.device or q.dtype != kp.dtype:
        raise ValueError(f"{name}: Q must have the cache's device and type.")
    if q.shape[0] != kc.shape[0] or q.shape[1] % kc.shape[1] or q.shape[3] != 2 * kc.shape[3]:
        raise ValueError(f"{name}: Q must match the cache's batch and channels, its heads a multiple of the cache's.")
    if q.shape[3] not in (64, 128):
        raise ValueError(f"{name}: head dimensions 64 and 128 are supported.")
    _no_gradient(name, q, kp, cache[3])
    if window is None and sinks != 0:
        raise ValueError(f"{name}: sinks need a window.")
    starts, at = _window_arguments(name, q.shape[0], q.device, 1 if window is None else window, sinks, query_start)
    scale = _resolved_scale(name, scale, q.shape[3])
    arguments = (q, *cache, starts, at, *_in_64_bits(0 if window is None else window, sinks), scale)
    if torch.compiler.is_compiling():
        return _attention_op(*arguments)
    return native.cache_attention(*arguments)

"""Rotary positions of queries and keys, forward and backward (``csrc/kernels/rotary.cu``).

Pair ``i`` of a head's values turns by ``position * freqs[i]`` radians. ``rotary_frequencies`` makes the frequencies, also for contexts longer
than the model was trained on; any others do as well. Angles are formed in 64 bits, values turned in fp32 and rounded once.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from .._lib import C
from .act8 import _DTYPES, check, launch_stream

_POSITIONS = {torch.int64: False, torch.int32: True}
_NO_HEADS = (0,) * 9


def rotary_frequencies(dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                       trained_length: Optional[int] = None, fast: float = 32.0, slow: float = 1.0,
                       device=None) -> Tuple[torch.Tensor, float]:
    """``(freqs, scale)`` for heads of which ``dim`` values turn: ``dim / 2`` angles per position (fp64, radians), ``base^(-2i/dim)``, and the
    factor that :func:`rotary` takes with them.

    ``scaling``, for contexts ``factor`` times as long as ``trained_length``: "linear" divides all frequencies by ``factor``; "ntk" raises
    the base so that the slowest pair is divided by it and the fastest stays; "yarn" (Peng, Quesnelle, Fan, Shippole, 2023) leaves pairs that
    turn ``fast`` times or more over ``trained_length``, divides those below ``slow`` turns, goes linearly in the number of turns in between, as
    that paper has it, and has ``scale`` = 0.1 ln(factor) + 1. (A model that was trained with a ramp that is linear in the number of the pair has other
    frequencies in between: :func:`rotary` takes any.)"""
    what = "rotary_frequencies"
    if dim <= 0 or dim % 2:
        raise ValueError(f"{what}: dim is even and positive, not {dim}")
    if not base > 0 or not factor >= 1:
        raise ValueError(f"{what}: base is positive and factor at least 1, not {base!r} and {factor!r}")
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    scale = 1.0
    if scaling == "ntk" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    freqs = base ** (-i / dim)
    if scaling == "linear" or (scaling == "ntk" and dim == 2):
        freqs = freqs / factor
    elif scaling == "yarn":
        if trained_length is None or trained_length <= 0 or not fast > slow:
            raise ValueError(f"{what}: yarn needs trained_length, and fast above slow")
        kept = ((freqs * trained_length / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        freqs = freqs * kept + freqs / factor * (1 - kept)
        scale = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "none", "ntk"):
        raise ValueError(f"{what}: scaling is None, 'linear', 'ntk' or 'yarn', not {scaling!r}")
    return freqs.to(device if device is not None else torch.device("cuda", torch.cuda.current_device())), scale


def _misfit(x, out, shape, dtype, dev, what, name):
    """Which argument does not fit (off the path of calls that do)."""
    if len(x.shape) not in (3, 4):
        raise ValueError(f"{what}: {name} is [tokens, heads, dim] or [batch, tokens, heads, dim], not {tuple(x.shape)}")
    if x.shape[:-2] != shape[:-2] or x.shape[-1] != shape[-1] or x.dtype != dtype or x.get_device() != dev:
        raise ValueError(f"{what}: {name} of {tuple(x.shape)} {x.dtype} on {x.device} does not go with q of {tuple(shape)} {dtype} on cuda:{dev}")
    raise ValueError(f"{what}: out of {name} must be like it ({tuple(x.shape)} of {dtype} on cuda:{dev}), the values of a head side by side and no two "
                     f"at one place, got {tuple(out.shape)} of {out.dtype} on {out.device} with strides {out.stride()}")


def _heads(x, own, out, shape, dtype, dev, what, name):
    """(result, arguments of the native call, what to hold) of queries or keys ``x`` of shape ``own``; ``shape``, ``dtype`` and ``dev`` are q's."""
    st = x.stride()
    if st[-1] != 1 and own[-1] > 1:
        x = x.contiguous()
        st = x.stride()
    if out is None:
        out = torch.empty_like(x)
        to = out.stride()
        if to[-1] != 1 and own[-1] > 1:   # (heads that share memory: a stride of 1 that is not the last)
            out = torch.empty(own, dtype=dtype, device=x.device)
            to = out.stride()
    else:
        to = out.stride()
        if out.shape != own or out.dtype is not dtype or out.get_device() != dev or (to[-1] != 1 and own[-1] > 1) or (
                0 in to and any(n > 1 and d == 0 for n, d in zip(own, to))):
            _misfit(x, out, shape, dtype, dev, what, name)
    if len(own) == 4:
        return out, (x.data_ptr(), st[0], st[1], st[2], out.data_ptr(), to[0], to[1], to[2], own[2]), x
    return out, (x.data_ptr(), 0, st[0], st[1], out.data_ptr(), 0, to[0], to[1], own[1]), x


def _rotary(q, k, freqs, positions, offset, interleaved, scale, out_q, out_k, backward, what):
    dtype, shape, s, dev = q.dtype, q.shape, launch_stream(q), q.get_device()
    dt = _DTYPES.get(dtype)
    if dt is None:
        raise ValueError(f"{what}: bf16 or fp32, not {dtype}")
    if len(shape) == 4:
        batch, tokens, _, dim = shape
    elif len(shape) == 3:
        (tokens, _, dim), batch = shape, 1
    else:
        _misfit(q, out_q, shape, dtype, dev, what, "q")
    out_q, q_args, _held = _heads(q, shape, out_q, shape, dtype, dev, what, "q")
    k_args = _NO_HEADS
    if k is not None:
        own = k.shape
        if len(own) != len(shape) or own[-1] != dim or own[-3] != tokens or (own[0] != batch and len(own) == 4) or k.dtype is not dtype or k.get_device() != dev:
            _misfit(k, out_k, shape, dtype, dev, what, "k")
        out_k, k_args, _held_k = _heads(k, own, out_k, shape, dtype, dev, what, "k")
    elif out_k is not None:
        raise ValueError(f"{what}: out_k without k")
    pairs = freqs.numel()
    if freqs.dtype is not torch.float64 or freqs.dim() != 1 or freqs.get_device() != dev or 2 * pairs > dim or not freqs.is_contiguous():
        raise ValueError(f"{what}: freqs must be at most {dim // 2} contiguous fp64 values on {q.device}, got {tuple(freqs.shape)} of {freqs.dtype} on {freqs.device}")
    at, narrow, pb, pt = 0, False, 0, 0
    if positions is not None:
        narrow, places, st = _POSITIONS.get(positions.dtype), positions.shape, positions.stride()
        dims = len(places)
        if narrow is None or positions.get_device() != dev or not 1 <= dims <= 2 or places[-1] != tokens or (dims == 2 and places[0] != batch and places[0] != 1):
            raise ValueError(f"{what}: positions must be int64 or int32, [{tokens}] or [{batch}, {tokens}], on {q.device}, "
                             f"got {tuple(places)} of {positions.dtype} on {positions.device}")
        at, pt = positions.data_ptr(), st[-1]
        if dims == 2 and places[0] > 1:
            pb = st[0]
    rc = C.rotary(dt, q_args, k_args, batch, tokens, dim, pairs, interleaved, freqs.data_ptr(), at, narrow, pb, pt, offset, scale, backward, s)
    if rc != 0:
        check(rc, what)
    return out_q if k is None else (out_q, out_k)


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], freqs: torch.Tensor, positions: Optional[torch.Tensor] = None, *, offset: int = 0,
           interleaved: bool = False, scale: float = 1.0, out_q: Optional[torch.Tensor] = None, out_k: Optional[torch.Tensor] = None):
    """``(q, k)`` with the first ``2 * len(freqs)`` values of every head turned, times ``scale``, and the others as they are.

    ``q`` and ``k`` (which may be None; its result is left out then): ``[batch, tokens, heads, dim]`` or ``[tokens, heads, dim]`` with any
    strides but the last (heads ahead of tokens: ``x.transpose(1, 2)``; heads of a packed QKV product: slices of its view), bf16 or fp32, with heads in any
    number each. ``freqs``: fp64, one angle per position of each pair. ``positions``: int64 or int32, ``[tokens]`` or ``[batch, tokens]``, any
    sign; without them a token's place in its row. ``offset`` is added to them. ``interleaved``: a pair is two neighbours, otherwise value
    ``i`` and value ``i + len(freqs)``. ``out_q`` and ``out_k`` may be ``q`` and ``k`` themselves (the values that do not turn are left alone then), and must
    not overlap them otherwise, nor have heads that share memory. Angles are as exact as a product in 64 bits (1.5e-6 radians at position 2^31 times one radian), up to 2^51 radians."""
    return _rotary(q, k, freqs, positions, offset, interleaved, scale, out_q, out_k, False, "rotary")


def rotary_backward(dq: torch.Tensor, dk: Optional[torch.Tensor], freqs: torch.Tensor, positions: Optional[torch.Tensor] = None, *, offset: int = 0,
                    interleaved: bool = False, scale: float = 1.0, out_q: Optional[torch.Tensor] = None, out_k: Optional[torch.Tensor] = None):
    """The gradients that reach ``q`` and ``k`` of :func:`rotary` with the same ``freqs``, ``positions`` and options: turned back, times ``scale``."""
    return _rotary(dq, dk, freqs, positions, offset, interleaved, scale, out_q, out_k, True, "rotary_backward")

"""Rotary positions of queries and keys: turned by where their tokens stand, for training (forwards and backwards) and on the way into
the 4-bit attention cache.

No counterpart exists in the reference, which has no models.  Everything runs on the GPU through libqtensor_hip.so, on torch's current
stream.

    rotary = Rotary(head_dim)                                   # or part of a head: Rotary(dims)
    q, k = rotary.turn(q, k, positions)                         # [.., tokens, heads, head_dim]; has a gradient
    q = cache.write_turned(rotary, q, k, v, table, lengths)     # QTensorCache: turned and encoded in one launch

Pair p of the first `dims` elements of a head -- neighbours (2 p, 2 p + 1) if interleaved, else (p, p + dims / 2) -- turns by the angle
position * frequencies[p]: (a, b) becomes (a c - b s, b c + a s), c and s the fp32 numbers nearest to magnitude * cos and magnitude * sin of
the angle, which is worked out in 64 bits (in fp32 a position of 10^5 leaves it two digits).  Products and their sum are rounded to fp32, the
result to its type; the elements behind `dims` stay as they are.
"""
import copy
import ctypes as ct
import math
from typing import Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

import qtensor.functional as F

_MOST = 1024                                        # elements of a head


class _Rotary(ct.Structure):
    _fields_ = [("frequencies", ct.c_void_p), ("magnitude", ct.c_double), ("dims", ct.c_int), ("interleaved", ct.c_int), ("back", ct.c_int)]


class _Part(ct.Structure):
    _fields_ = [("from_", ct.c_void_p), ("to", ct.c_void_p)] + [(n, ct.c_longlong) for n in ("from_batch", "from_token", "from_head", "to_batch", "to_token",
                                                                                             "to_head")] + [("heads", ct.c_int)]


class _Call(ct.Structure):
    _fields_ = [("part", _Part * 2), ("parts", ct.c_int), ("head_dim", ct.c_int), ("is_bf16", ct.c_int), ("long_positions", ct.c_int),
                ("batch", ct.c_longlong), ("tokens", ct.c_longlong), ("position_batch", ct.c_longlong), ("positions", ct.c_void_p)]


if F.lib is not None:
    F.lib.qtensor_hip_rotary_turn.restype = None
    F.lib.qtensor_hip_rotary_turn.argtypes = [ct.POINTER(_Rotary), ct.POINTER(_Call), ct.c_void_p]


def frequencies(dims: int, base: float = 10000.0, factor: float = 1.0, stretch: str = "all", original: Optional[int] = None, slow: float = 1.0,
                fast: float = 32.0) -> list:
    """base^(-2 p / dims) for the pairs p of `dims` elements, for a context `factor` times the one a model was trained on:
      "all"    every frequency over factor (positions as if they were that much closer)
      "base"   of a base that is larger by factor^(dims / (dims - 2)): the fastest as it was, the slowest over factor
      "parts"  pairs that turn more than `fast` times in `original` positions as they were, those that turn less than `slow` times over
               factor, in between in proportion."""
    if dims < 2 or dims % 2:
        raise ValueError(f"{dims} elements are not pairs.")
    if not (base > 0 and math.isfinite(base) and factor > 0 and math.isfinite(factor)):
        raise ValueError(f"base {base} and factor {factor} must be positive numbers.")
    if stretch not in ("all", "base", "parts"):
        raise ValueError(f"stretch {stretch!r} is not one of 'all', 'base', 'parts'.")
    if stretch == "base":
        base = base * factor ** (dims / max(1, dims - 2))
    speed = [base ** (-2.0 * p / dims) for p in range(dims // 2)]
    if stretch == "all":
        return [f / factor for f in speed]
    if stretch == "parts":
        if original is None or original < 1 or not 0 <= slow < fast:
            raise ValueError("stretch 'parts' needs the number of positions that a model was trained on, and 0 <= slow < fast.")
        kept = [min(1.0, max(0.0, (original * f / (2 * math.pi) - slow) / (fast - slow))) for f in speed]
        return [f * k + f / factor * (1.0 - k) for f, k in zip(speed, kept)]
    return speed


class Rotary:
    """The angles of one kind of layer: `dims` elements of a head turn (an even number), as pairs of neighbours if interleaved, else of both
    halves.  frequencies: dims / 2 numbers, angles per position (default: frequencies(dims, base))."""

    def __init__(self, dims: int, base: float = 10000.0, frequencies: Union[None, Tensor, Sequence[float]] = None, magnitude: float = 1.0,
                 interleaved: bool = False, device="cuda"):
        if dims < 2 or dims % 2 or dims > _MOST:
            raise ValueError(f"need an even number of elements, 2 to {_MOST} (got {dims})")
        if not math.isfinite(magnitude):
            raise ValueError(f"magnitude {magnitude} is not finite")
        if frequencies is None:
            frequencies = globals()["frequencies"](dims, base)
        speed = torch.as_tensor(frequencies, dtype=torch.float64).detach().flatten()
        if speed.numel() != dims // 2 or not bool(torch.isfinite(speed).all()):
            raise ValueError(f"need {dims // 2} finite frequencies for {dims} elements (got {speed.numel()})")
        self.dims, self.magnitude, self.interleaved = dims, float(magnitude), bool(interleaved)
        self.frequencies = speed.to(device).contiguous()

    def turn(self, q: Tensor, k: Optional[Tensor], positions: Tensor) -> Tuple[Tensor, Optional[Tensor]]:
        """(q, k) turned: [.., tokens, heads, head_dim] with at most one dimension in front (fp32 or bf16, the last dimension contiguous),
        heads of both may differ in number; k may be None.  positions: int32 or int64 [tokens] or [batch, tokens], any values.  The
        gradients of q and k are theirs turned back, in reverse mode and of every order; forward mode, torch.func's transformations and batched
        gradients (is_grads_batched) raise."""
        if F._direct is not None:
            done = F._direct.rotary_turn(self.frequencies, self.magnitude, self.dims, self.interleaved, q, k, positions)
            if done is not None:
                return done
        return _Turn.apply(self, False, q, k, positions)

    def _turned(self, back, tensors, positions):
        """The tensors of a list (one or two) turned, as new ones."""
        F._require_gpu(self.frequencies, "Rotary.turn")
        first = tensors[0]
        F._dtype_slot(first.dtype, "q")
        device = self.frequencies.device
        for t, name in zip(tensors, "qk"):
            if t.device != device:
                raise ValueError(f"{name} must live on the frequencies' device ({t.device} vs {device}).")
            if t.dtype != first.dtype:
                raise ValueError(f"{name} has dtype {t.dtype}, expected {first.dtype}.")
            if t.dim() not in (3, 4) or t.dim() != first.dim() or t.shape[:-2] != first.shape[:-2] or t.shape[-1] != first.shape[-1]:
                raise ValueError(f"{name} has shape {tuple(t.shape)}, expected [tokens, heads, head_dim] or [batch, tokens, heads, head_dim], alike but for heads.")
            if not self.dims <= t.shape[-1] <= _MOST:
                raise ValueError(f"{name} has heads of {t.shape[-1]} elements, expected {self.dims} to {_MOST}.")
            if not 1 <= t.shape[-2] <= 32767:
                raise ValueError(f"{name} has {t.shape[-2]} heads, expected 1 to 32767.")
            if t.stride(-1) != 1:
                raise ValueError(f"the last dimension of {name} must be contiguous.")
        batch, tokens = (first.shape[0], first.shape[1]) if first.dim() == 4 else (1, first.shape[0])
        _check_positions(positions, device, ((tokens,), (batch, tokens)) if first.dim() == 4 else ((tokens,),))
        if positions.shape[-1] > 1 and positions.stride(-1) != 1:
            raise ValueError("the last dimension of positions must be contiguous.")
        out = [torch.empty(t.shape, dtype=t.dtype, device=device) for t in tensors]
        parts = [_Part(t.data_ptr(), y.data_ptr(), *_strides(t), *_strides(y), t.shape[-2]) for t, y in zip(tensors, out)]
        call = _Call((_Part * 2)(*parts), len(parts), first.shape[-1], first.dtype == torch.bfloat16, positions.dtype == torch.int64, batch, tokens,
                     positions.stride(0) if positions.dim() == 2 else 0, positions.data_ptr())
        F._call(F.lib.qtensor_hip_rotary_turn, device, self._ref(back), call)
        return out

    def _ref(self, back=False):
        # (the kernels go by dims, whatever has taken the tensor's place)
        speed = self.frequencies
        if speed.dtype != torch.float64 or tuple(speed.shape) != (self.dims // 2,) or not speed.is_contiguous():
            raise ValueError(f"frequencies are {speed.dtype} {tuple(speed.shape)}, not contiguous {torch.float64} {(self.dims // 2,)}.")
        return _Rotary(speed.data_ptr(), self.magnitude, self.dims, self.interleaved, back)


def _strides(t: Tensor):
    return (t.stride(0) if t.dim() == 4 else 0, t.stride(-3), t.stride(-2))


def _check_positions(positions: Tensor, device, shapes) -> None:
    if positions.device != device:
        raise ValueError(f"positions must live on the same device as the data ({positions.device} vs {device}).")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions have dtype {positions.dtype}, expected torch.int32 or torch.int64.")
    if tuple(positions.shape) not in shapes:
        raise ValueError(f"positions have shape {tuple(positions.shape)}, expected {' or '.join(map(str, shapes))}.")


class _Turn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rotary, back, q, k, positions):
        # (its angles are kept as they are now, frequencies by torch, or where they were made in inference mode, which it does not save, as a copy)
        speed = rotary.frequencies
        ctx.rotary, ctx.back = copy.copy(rotary), back
        ctx.rotary.frequencies = speed.clone() if speed.is_inference() else None
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, *([] if speed.is_inference() else [speed]))
        out = rotary._turned(back, [q] if k is None else [q, k], positions)
        return out[0], out[1] if k is not None else None

    @staticmethod
    def backward(ctx, dq, dk):
        rotary = copy.copy(ctx.rotary)
        positions, *frequencies = ctx.saved_tensors
        if frequencies:
            rotary.frequencies, = frequencies
        wanted = [d if d is not None and need else None for d, need in zip((dq, dk), ctx.needs_input_grad[2:4])]
        given = [d if d.stride(-1) == 1 else d.contiguous() for d in wanted if d is not None]
        if not given:
            return None, None, None, None, None
        turned = list(_Turn.apply(rotary, not ctx.back, given[0], given[1] if len(given) > 1 else None, positions))
        return None, None, *(turned.pop(0) if d is not None else None for d in wanted), None

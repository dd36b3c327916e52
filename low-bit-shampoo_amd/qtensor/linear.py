"""Projections whose weights are held in 4 bits, and their products with tokens.

No counterpart exists in the reference, whose low-bit tensors are the state of an optimizer; this is the attention cache's format
(qtensor.cache) for the weights that a trained model generates with: segments of inputs, an fp32 scale each, 4 bits per weight.
A step of generation is bound by reading its weights, and reads 0.56 bytes of each here; products are exact and summed in fp32, so
beside the weights' 4 bits and the result's rounding there are only the roundings of these sums, 2^-24 of the products' magnitudes added up for each step
in them.  Everything runs on the GPU through libqtensor_hip.so, on
torch's current stream.

    weights = QTensorLinear(inputs, outputs)
    weights.quantize(layer.weight)                   # [outputs, inputs], as torch.nn.Linear has it
    y = weights.product(x, layer.bias)               # [.., inputs] -> [.., outputs]
"""
import ctypes as ct
from typing import Optional

import torch
from torch import Tensor

import qtensor.functional as F

_BLOCKSIZES = (64, 128, 256)
_MOST = 2 ** 24                                     # inputs or outputs


class _Linear(ct.Structure):
    _fields_ = [("codes", ct.c_void_p), ("scales", ct.c_void_p), ("inputs", ct.c_int), ("outputs", ct.c_int), ("blocksize", ct.c_int)]


class _Call(ct.Structure):
    _fields_ = [("x", ct.c_void_p), ("bias", ct.c_void_p), ("out", ct.c_void_p), ("x_stride", ct.c_longlong), ("out_stride", ct.c_longlong),
                ("tokens", ct.c_longlong), ("is_bf16", ct.c_int), ("bias_is_bf16", ct.c_int)]


if F.lib is not None:
    for _name in ("qtensor_hip_linear_quantize", "qtensor_hip_linear_dequantize"):
        getattr(F.lib, _name).restype = None
        getattr(F.lib, _name).argtypes = [ct.POINTER(_Linear), ct.c_void_p, ct.c_int, ct.c_longlong, ct.c_void_p]
    F.lib.qtensor_hip_linear_product.restype = None
    F.lib.qtensor_hip_linear_product.argtypes = [ct.POINTER(_Linear), ct.POINTER(_Call), ct.c_void_p]


class QTensorLinear:
    """Weights [outputs, inputs] of a projection.  A row is held in segments of `blocksize` (64, 128 or 256) inputs: an fp32 scale, the
    largest magnitude over 6, and the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 with a sign for every weight over the scale (ties to the even
    code).  A segment that holds a NaN or an infinity stands for NaN.  It begins as zeros."""

    def __init__(self, inputs: int, outputs: int, blocksize: int = 64, device="cuda"):
        if blocksize not in _BLOCKSIZES:
            raise ValueError(f"blocksize {blocksize} is not one of {_BLOCKSIZES}")
        if not 1 <= inputs <= _MOST or not 1 <= outputs <= _MOST:
            raise ValueError(f"need 1 to {_MOST} inputs and outputs (got {inputs}, {outputs})")
        self.inputs, self.outputs, self.blocksize = inputs, outputs, blocksize
        # (in the order of the matrix instructions' operands: csrc/qt_linear.h)
        self.codes = torch.zeros(-(-outputs // 16), -(-inputs // 128), 1024, dtype=torch.uint8, device=device)
        self.scales = torch.zeros(-(-outputs // 16), -(-inputs // blocksize), 16, dtype=torch.float32, device=device)

    # ---- flat checkpoint form, as the holders of qtensor.utils have it
    def state_dict(self):
        """Tensors and numbers only."""
        return {"inputs": self.inputs, "outputs": self.outputs, "blocksize": self.blocksize, "codes": self.codes, "scales": self.scales}

    def load_state_dict(self, sd):
        """Takes what state_dict() wrote into weights constructed with the same arguments."""
        for name in ("inputs", "outputs", "blocksize"):
            if int(sd[name]) != getattr(self, name):
                raise ValueError(f"checkpointed weights have {name} {int(sd[name])}, these {getattr(self, name)}")
        for name in ("codes", "scales"):
            here, there = getattr(self, name), sd[name]
            if there.shape != here.shape or there.dtype != here.dtype:
                raise ValueError(f"checkpointed {name} are {there.dtype} {tuple(there.shape)}, expected {here.dtype} {tuple(here.shape)}")
        for name in ("codes", "scales"):
            getattr(self, name).copy_(sd[name])

    # ---- the calls
    def quantize(self, weight: Tensor) -> "QTensorLinear":
        """Encodes a weight matrix [outputs, inputs] (fp32 or bf16, rows contiguous); returns self.  A parameter may be given as it is: what is
        held of it has no gradient."""
        F._require_gpu(self.codes, "QTensorLinear.quantize")
        F._dtype_slot(weight.dtype, "weight")
        self._check(weight, "weight", (self.outputs, self.inputs), weight.dtype)
        F._call(F.lib.qtensor_hip_linear_quantize, self.codes.device, self._ref(), weight.data_ptr(), weight.dtype == torch.bfloat16, weight.stride(0))
        return self

    def dequantize(self, dtype: torch.dtype = torch.float32) -> Tensor:
        """The weights [outputs, inputs] as they are held."""
        F._require_gpu(self.codes, "QTensorLinear.dequantize")
        F._dtype_slot(dtype, "the result")
        out = torch.empty(self.outputs, self.inputs, dtype=dtype, device=self.codes.device)
        F._call(F.lib.qtensor_hip_linear_dequantize, self.codes.device, self._ref(), out.data_ptr(), dtype == torch.bfloat16, self.inputs)
        return out

    def product(self, x: Tensor, bias: Optional[Tensor] = None, out: Optional[Tensor] = None) -> Tensor:
        """W x + bias for every token: x [.., inputs] (fp32 or bf16) -> [.., outputs] of its type; bias [outputs] of fp32 or x's type.  Products are
        exact and summed in fp32, the result is rounded once.  out: optional result, contiguous, that shares no memory with x or bias.  Up to
        2^31 - 256 tokens; sums in front of the scales, so up to 768 of x's largest magnitude, have to stay below 2^128, and
        what an fp32 x has of bits below 2^-133 is cut off."""
        if F._direct is not None:
            done = F._direct.linear_product(self.codes, self.scales, self.inputs, self.outputs, self.blocksize, x, bias, out)
            if done is not None:
                return done
        F._require_gpu(self.codes, "QTensorLinear.product")
        F._dtype_slot(x.dtype, "x")
        if x.dim() < 1 or x.shape[-1] != self.inputs:
            raise ValueError(f"x has shape {tuple(x.shape)}, expected [.., {self.inputs}].")
        F._check_derivatives("weights", x=x, bias=bias, out=out)
        rows = x if x.dim() == 2 else x.reshape(-1, self.inputs)
        self._check(rows, "x", (rows.shape[0], self.inputs), x.dtype)
        if bias is not None:
            if bias.dtype not in (torch.float32, x.dtype):
                raise ValueError(f"bias has dtype {bias.dtype}, expected torch.float32 or {x.dtype}.")
            F._check_buffer(bias, "bias", self.outputs, bias.dtype, self.codes.device)
        shape = (*x.shape[:-1], self.outputs)
        if out is None:
            out = torch.empty(shape, dtype=x.dtype, device=x.device)
        else:
            if tuple(out.shape) != shape:
                raise ValueError(f"out has shape {tuple(out.shape)}, expected {shape}.")
            F._check_buffer(out, "out", rows.shape[0] * self.outputs, x.dtype, self.codes.device)
            if F._overlap(out, rows) or (bias is not None and F._overlap(out, bias)):
                raise ValueError("out shares memory with x or bias, which are read while it is written.")
        F._call(F.lib.qtensor_hip_linear_product, self.codes.device, self._ref(),
                _Call(rows.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), rows.stride(0), self.outputs, rows.shape[0],
                      x.dtype == torch.bfloat16, bias is not None and bias.dtype == torch.bfloat16))
        return out

    # ---- checks and descriptions
    def _ref(self):
        # (what they were made as: the kernels go by the numbers below, whatever has taken the tensors' place)
        codes, scales = self.codes, self.scales
        tiles = -(-self.outputs // 16)
        for name, t, dtype, shape in (("codes", codes, torch.uint8, (tiles, -(-self.inputs // 128), 1024)),
                                      ("scales", scales, torch.float32, (tiles, -(-self.inputs // self.blocksize), 16))):
            if t.device != codes.device or t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"the weights' {name} are {t.dtype} {tuple(t.shape)} on {t.device}, not contiguous {dtype} {shape} on {codes.device}.")
        return _Linear(codes.data_ptr(), scales.data_ptr(), self.inputs, self.outputs, self.blocksize)

    def _check(self, t: Tensor, name: str, shape, dtype: torch.dtype) -> None:
        if t.device != self.codes.device:
            raise ValueError(f"{name} must live on the weights' device ({t.device} vs {self.codes.device}).")
        if t.dtype != dtype:
            raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}.")
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}.")
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise ValueError(f"the last dimension of {name} must be contiguous.")

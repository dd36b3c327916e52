"""Keys and values of a model's attention held in 4 bits, and the attention that reads them as they are.

No counterpart exists in the reference, whose low-bit tensors are the state of an optimizer; this is the same idea for the
state a trained transformer generates with: segments of a few dozen elements, an fp32 scale each, 4 bits per element.  The
numbers are the 4-bit floating ones that MI355X's matrix instructions multiply directly, so attention never expands the
cache.  Everything runs on the GPU through libqtensor_hip.so, on torch's current stream.

    cache = QTensorCache(pages, kv_heads, head_dim)            # one per layer
    cache.write(keys, values, table, lengths, starts)          # new tokens, after `lengths` has counted them
    q = cache.write_turned(rotary, q, keys, values, table, lengths, starts)    # the same with rotary positions (qtensor.rotary)
    out = cache.attend(q, table, lengths, starts)              # every new token sees its sequence up to itself
    cache.weigh(totals, q, table, lengths, starts)             # adds up the weights that tokens are given (totals = cache.totals(table))
    shorter = cache.evict(totals, table, lengths, keep)        # those with the largest sums stay

`table` int32 [batch, n]: the pages of every sequence in order; `lengths` int32 [batch]: its tokens, the new ones included;
`starts` int32 [batch + 1]: where the new tokens of each sequence begin in the packed tensors (the first 0, the last their
number), or None where every sequence has one.  All three live on the GPU and no call waits for it, so a step of generation can be
captured in a graph and replayed with other contents; tensors may have room for more tokens than starts says: those are of no
sequence, are not written, read as zeros and get zeros from `attend`.  A token of a negative position or without a page (beyond the table, or a
number that is not a page of the cache) is not written, reads as zeros and is not seen: pages that a window has left behind may
be handed back and marked -1.
"""
import ctypes as ct
import math
from typing import Optional, Tuple

import torch
from torch import Tensor

import qtensor.functional as F
from qtensor.rotary import Rotary, _check_positions, _Rotary

_BLOCKSIZES = (64, 128, 256)
_MOST = 2 ** 31 - 1                                 # of anything that is counted: the library's numbers have 32 bits


class _Cache(ct.Structure):
    _fields_ = [("codes", ct.c_void_p * 2), ("scales", ct.c_void_p * 2), ("pages", ct.c_int), ("page_size", ct.c_int),
                ("kv_heads", ct.c_int), ("head_dim", ct.c_int), ("blocksize", ct.c_int)]


class _Places(ct.Structure):
    _fields_ = [("table", ct.c_void_p), ("lengths", ct.c_void_p), ("starts", ct.c_void_p), ("table_stride", ct.c_longlong),
                ("table_pages", ct.c_int), ("batch", ct.c_int), ("tokens", ct.c_int)]


class _Vectors(ct.Structure):
    _fields_ = [("base", ct.c_void_p), ("is_bf16", ct.c_int), ("token_stride", ct.c_longlong), ("head_stride", ct.c_longlong)]


if F.lib is not None:
    for _name in ("qtensor_hip_cache_write", "qtensor_hip_cache_read"):
        getattr(F.lib, _name).restype = None
        getattr(F.lib, _name).argtypes = [ct.POINTER(_Cache), ct.POINTER(_Places), ct.POINTER(_Vectors), ct.POINTER(_Vectors), ct.c_void_p]
    F.lib.qtensor_hip_cache_write_turned.restype = None
    F.lib.qtensor_hip_cache_write_turned.argtypes = [ct.POINTER(_Cache), ct.POINTER(_Places), ct.POINTER(_Rotary), ct.POINTER(_Vectors), ct.POINTER(_Vectors),
                                                     ct.c_int, ct.POINTER(_Vectors), ct.POINTER(_Vectors), ct.c_void_p, ct.c_int, ct.c_void_p]
    F.lib.qtensor_hip_cache_attend.restype = None
    F.lib.qtensor_hip_cache_attend.argtypes = [ct.POINTER(_Cache), ct.POINTER(_Places), ct.POINTER(_Vectors), ct.POINTER(_Vectors), ct.c_int,
                                               ct.c_float, ct.c_int, ct.c_int, ct.c_void_p, ct.c_longlong, ct.c_void_p]
    F.lib.qtensor_hip_cache_attend_workspace.restype = ct.c_longlong
    F.lib.qtensor_hip_cache_attend_workspace.argtypes = [ct.POINTER(_Cache), ct.c_int, ct.c_int, ct.c_int]

    F.lib.qtensor_hip_cache_weigh_workspace.restype = F.lib.qtensor_hip_cache_evict_workspace.restype = ct.c_longlong
    F.lib.qtensor_hip_cache_weigh_workspace.argtypes = [ct.POINTER(_Cache), ct.POINTER(_Places), ct.c_int]
    F.lib.qtensor_hip_cache_evict_workspace.argtypes = [ct.POINTER(_Cache), ct.POINTER(_Places), ct.c_longlong]
    F.lib.qtensor_hip_cache_weigh.restype = F.lib.qtensor_hip_cache_evict.restype = None
    F.lib.qtensor_hip_cache_weigh.argtypes = [ct.POINTER(_Cache), ct.POINTER(_Places), ct.POINTER(_Vectors), ct.c_int, ct.c_float, ct.c_int, ct.c_int, ct.c_void_p,
                                              ct.c_longlong, ct.c_longlong, ct.c_void_p, ct.c_longlong, ct.c_void_p]
    F.lib.qtensor_hip_cache_evict.argtypes = [ct.POINTER(_Cache), ct.POINTER(_Places), ct.c_void_p] + [ct.c_longlong] * 5 + [ct.c_void_p, ct.c_void_p,
                                              ct.c_longlong, ct.c_void_p]

    # the same calls with their host side in native code (csrc/direct_call.cpp): what it does not take goes the way below
    _native = F._direct
    if _native is not None:
        _native.bind_cache([ct.cast(getattr(F.lib, "qtensor_hip_cache_" + n), ct.c_void_p).value
                            for n in ("write", "read", "attend", "attend_workspace")])
else:
    _native = None


class QTensorCache:
    """The cache of one layer: `pages` pages of `page_size` tokens (a power of two from 16 to 4096), kv_heads heads of head_dim
    (1 to 256) elements.  A vector of a head is held in segments of `blocksize` (64, 128 or 256) elements: an fp32 scale, the
    largest magnitude over 6, and the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 with a sign for every element over the scale
    (ties to the even code).  blocksize 64 keeps most and costs 4.5 bits per element; one segment per vector is fastest."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, blocksize: int = 64, device="cuda"):
        if blocksize not in _BLOCKSIZES:
            raise ValueError(f"blocksize {blocksize} is not one of {_BLOCKSIZES}")
        if page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError(f"page_size {page_size} is not a power of two from 16 to 4096")
        if not 1 <= head_dim <= 256 or not 1 <= kv_heads <= 32767 or pages < 1:
            raise ValueError(f"need 1 to 256 elements per head, 1 to 32767 heads and a page (got {head_dim}, {kv_heads}, {pages})")
        self.pages, self.kv_heads, self.head_dim, self.page_size, self.blocksize = pages, kv_heads, head_dim, page_size, blocksize
        self.segments = -(-head_dim // blocksize)
        # (a cache begins as zeros: what a page has not been written holds stands for something all the same)
        self.codes = torch.zeros(2, pages, kv_heads, page_size, 16 * (-(-head_dim // 32)), dtype=torch.uint8, device=device)
        self.scales = torch.zeros(2, pages, kv_heads, self.segments, page_size, dtype=torch.float32, device=device)

    # ---- flat checkpoint form, as the holders of qtensor.utils have it
    def state_dict(self):
        """Tensors and numbers only."""
        return {"page_size": self.page_size, "blocksize": self.blocksize, "head_dim": self.head_dim, "codes": self.codes,
                "scales": self.scales}

    def load_state_dict(self, sd):
        """Takes what state_dict() wrote into a cache constructed with the same arguments."""
        for name in ("page_size", "blocksize", "head_dim"):
            if int(sd[name]) != getattr(self, name):
                raise ValueError(f"checkpointed cache has {name} {int(sd[name])}, this one {getattr(self, name)}")
        for name in ("codes", "scales"):
            here, there = getattr(self, name), sd[name]
            if there.shape != here.shape or there.dtype != here.dtype:
                raise ValueError(f"checkpointed {name} are {there.dtype} {tuple(there.shape)}, expected {here.dtype} {tuple(here.shape)}")
        for name in ("codes", "scales"):
            getattr(self, name).copy_(sd[name])

    # ---- the calls
    def write(self, keys: Tensor, values: Tensor, table: Tensor, lengths: Tensor, starts: Optional[Tensor] = None) -> None:
        """Encodes keys and values [tokens, kv_heads, head_dim] (fp32 or bf16, the last dimension contiguous) of the new tokens."""
        if _native is not None and _native.cache_write(self.codes, self.scales, self.page_size, self.kv_heads, self.head_dim, self.blocksize,
                                                       keys, values, table, lengths, starts):
            return
        F._require_gpu(self.codes, "QTensorCache.write")
        F._dtype_slot(keys.dtype, "keys")
        tokens = keys.shape[0] if keys.dim() == 3 else -1
        self._check_vectors(keys, "keys", (tokens, self.kv_heads, self.head_dim), keys.dtype)
        self._check_vectors(values, "values", (tokens, self.kv_heads, self.head_dim), keys.dtype)
        places = self._places(table, lengths, starts, tokens)
        F._call(F.lib.qtensor_hip_cache_write, self.codes.device, self._ref(), places, _vectors(keys), _vectors(values))

    def write_turned(self, rotary: Rotary, q: Tensor, keys: Tensor, values: Tensor, table: Tensor, lengths: Tensor, starts: Optional[Tensor] = None,
                     positions: Optional[Tensor] = None, out: Optional[Tensor] = None) -> Tensor:
        """Rotary positions on the way into the cache, in one launch: the queries q [tokens, heads, head_dim] turned; keys turned and encoded,
        values encoded, as `write` does with what rotary.turn gives.  positions: int32 or int64 [tokens], or None: a token's
        place in its sequence (which is another where tokens have been evicted).  Queries of tokens that are of no sequence or of a
        negative place become zeros.  out: optional result of the shape and type of q that shares no memory with q, keys or values."""
        if _native is not None:
            done = _native.cache_write_turned(self.codes, self.scales, self.page_size, self.kv_heads, self.head_dim, self.blocksize, rotary.frequencies,
                                              rotary.magnitude, rotary.dims, rotary.interleaved, q, keys, values, table, lengths, starts, positions, out)
            if done is not None:
                return done
        F._require_gpu(self.codes, "QTensorCache.write_turned")
        F._dtype_slot(q.dtype, "q")
        tokens, heads = (q.shape[0], q.shape[1]) if q.dim() == 3 else (-1, -1)
        self._check_vectors(q, "q", (tokens, heads, self.head_dim), q.dtype)
        if not 1 <= heads <= 32767:
            raise ValueError(f"need 1 to 32767 query heads (got {heads}).")
        self._check_vectors(keys, "keys", (tokens, self.kv_heads, self.head_dim), q.dtype)
        self._check_vectors(values, "values", (tokens, self.kv_heads, self.head_dim), q.dtype)
        if rotary.dims > self.head_dim or rotary.frequencies.device != self.codes.device:
            raise ValueError(f"{rotary.dims} elements on {rotary.frequencies.device} cannot turn in heads of {self.head_dim} on {self.codes.device}.")
        if positions is not None:
            _check_positions(positions, self.codes.device, ((tokens,),))
            if not positions.is_contiguous():
                raise ValueError("positions must be contiguous.")
        if out is None:
            out = torch.empty(tokens, heads, self.head_dim, dtype=q.dtype, device=q.device)
        else:
            self._check_vectors(out, "out", (tokens, heads, self.head_dim), q.dtype)
            if any(F._overlap(out, t) for t in (q, keys, values)):
                raise ValueError("out shares memory with q, keys or values, which are read while it is written.")
            by_stride = sorted((s, n) for s, n in zip(out.stride()[:2], out.shape[:2]) if n > 1)
            for (stride, _), least in zip(by_stride, [self.head_dim] + [s * (n - 1) + self.head_dim for s, n in by_stride]):
                if stride < least and out.numel():
                    raise ValueError("out has elements that share memory with each other.")
        places = self._places(table, lengths, starts, tokens)
        F._call(F.lib.qtensor_hip_cache_write_turned, self.codes.device, self._ref(), places, rotary._ref(), _vectors(q), _vectors(out), heads, _vectors(keys),
                _vectors(values), None if positions is None else positions.data_ptr(), positions is not None and positions.dtype == torch.int64)
        return out

    def read(self, table: Tensor, lengths: Tensor, starts: Optional[Tensor] = None, tokens: Optional[int] = None,
             dtype: torch.dtype = torch.float32) -> Tuple[Tensor, Tensor]:
        """(keys, values) [tokens, kv_heads, head_dim] as the cache holds them, of the same tokens that `write` would take; with
        starts up to the lengths of whole sequences, everything.  tokens: how many (starts[-1], which only the GPU knows);
        one of each sequence without starts."""
        if tokens is None:
            if starts is not None:
                raise ValueError("read with starts needs the number of tokens")
            tokens = lengths.numel()
        if _native is not None:
            done = _native.cache_read(self.codes, self.scales, self.page_size, self.kv_heads, self.head_dim, self.blocksize, table, lengths,
                                      starts, tokens, dtype)
            if done is not None:
                return done
        F._require_gpu(self.codes, "QTensorCache.read")
        F._dtype_slot(dtype, "the result")
        places = self._places(table, lengths, starts, tokens)
        keys, values = (torch.empty(tokens, self.kv_heads, self.head_dim, dtype=dtype, device=self.codes.device) for _ in range(2))
        F._call(F.lib.qtensor_hip_cache_read, self.codes.device, self._ref(), places, _vectors(keys), _vectors(values))
        return keys, values

    def attend(self, q: Tensor, table: Tensor, lengths: Tensor, starts: Optional[Tensor] = None, scale: Optional[float] = None,
               window: Optional[int] = None, sinks: int = 0, out: Optional[Tensor] = None) -> Tensor:
        """softmax(scale q k) v for the queries q [tokens, heads, head_dim] (fp32 or bf16) of the new tokens, which the cache
        must have already.  heads is a multiple of kv_heads: query head h reads head h // (heads // kv_heads).  A token sees its
        sequence up to itself; with a window only the last `window` tokens of that, itself included, and the first `sinks`
        of the sequence.  scale: 1 / sqrt(head_dim) unless given.  A token that sees nothing gets zeros.  out: optional result of the
        shape and type of q.  Many bf16 queries of a sequence are computed in fp16 (errors of 2^-12 in keys, values and weights); what fp16 does
        not hold, as queries and keys of thousands or values 2^16 below the largest of their head, is computed in fp32 and far slower."""
        if _native is not None:
            done = _native.cache_attend(self.codes, self.scales, self.page_size, self.kv_heads, self.head_dim, self.blocksize, q, table, lengths,
                                        starts, scale, window, sinks, out)
            if done is not None:
                return done
        F._require_gpu(self.codes, "QTensorCache.attend")
        tokens, heads, scale = self._check_queries(q, scale, window, sinks)
        if out is None:
            out = torch.empty(tokens, heads, self.head_dim, dtype=q.dtype, device=q.device)
        else:
            self._check_vectors(out, "out", (tokens, heads, self.head_dim), q.dtype)
        places = self._places(table, lengths, starts, tokens)
        # scratch for the pieces of long sequences: taken for the call, as that of the products is
        with torch.cuda.device(q.device):
            size = F.lib.qtensor_hip_cache_attend_workspace(self._ref(), heads, q.dtype == torch.bfloat16, starts is not None)
        scratch = torch.empty(size, dtype=torch.uint8, device=q.device)
        F._call(F.lib.qtensor_hip_cache_attend, q.device, self._ref(), places, _vectors(q), _vectors(out), heads, scale,
                min(window or 0, _MOST), min(sinks, _MOST), scratch.data_ptr(), size)
        return out

    # ---- what is kept, by the attention it is given
    def totals(self, table: Tensor) -> Tensor:
        """Zeros for `weigh` to add to: fp32 [batch, kv_heads, tokens that the table has room for]."""
        return torch.zeros(table.shape[0], self.kv_heads, table.shape[1] * self.page_size, dtype=torch.float32, device=self.codes.device)

    def weigh(self, totals: Tensor, q: Tensor, table: Tensor, lengths: Tensor, starts: Optional[Tensor] = None, scale: Optional[float] = None,
              window: Optional[int] = None, sinks: int = 0) -> Tensor:
        """Adds to totals (fp32 [batch, kv_heads, n], n at least what the table has room for) the weights softmax(scale q k) that `attend`, called with the
        same arguments, multiplies values with: for every token of a sequence and head of the cache the sum over the call's queries and over the query
        heads that read the head.  Sums are in fp32, in one order; six times a query's elements, added up, have to stay below 2^128, and what an fp32 query
        has of bits below 2^-133 is cut off.  Returns totals."""
        if _native is not None:
            done = _native.cache_weigh(self.codes, self.scales, self.page_size, self.kv_heads, self.head_dim, self.blocksize, totals, q, table, lengths,
                                       starts, scale, window, sinks)
            if done is not None:
                return done
        F._require_gpu(self.codes, "QTensorCache.weigh")
        tokens, heads, scale = self._check_queries(q, scale, window, sinks)
        places = self._places(table, lengths, starts, tokens)
        self._check_totals(totals, places)
        if tokens * (heads // self.kv_heads) >= 2 ** 27 or places.batch > 65535:
            raise ValueError(f"{tokens} tokens of {heads} heads in {places.batch} sequences are too many for one call.")
        if F._overlap(totals, q):
            raise ValueError("totals share memory with q, which is read while they are written.")
        cache = self._ref()
        with torch.cuda.device(q.device):
            size = F.lib.qtensor_hip_cache_weigh_workspace(cache, places, heads)
        scratch = torch.empty(size, dtype=torch.uint8, device=q.device)
        F._call(F.lib.qtensor_hip_cache_weigh, q.device, cache, places, _vectors(q), heads, scale, min(window or 0, _MOST), min(sinks, _MOST), totals.data_ptr(),
                totals.stride(0), totals.stride(1), scratch.data_ptr(), size)
        return totals

    def evict(self, totals: Tensor, table: Tensor, lengths: Tensor, keep: int, recent: int = 0, sinks: int = 0) -> Tensor:
        """Of every sequence and head, `keep` tokens stay: the first `sinks` and the last `recent` of the sequence, then those with the largest totals (NaN
        above all, ties to the earlier one); all of them where there are no more.  In their order they move to the front, keys, values and
        totals, and what lies behind is left as it was.  Returns the new lengths, as a tensor of its own: layers with caches of their own share
        `lengths`, so copy them there once all caches are done, set the totals behind them to zero before tokens are written there, and hand the
        pages behind back.  A position that a token was turned by stays its own: give write_turned positions from now on.  Tokens without a
        page are no candidates, and their places stay empty.  No page may be twice in the call, in one sequence or in two."""
        if _native is not None:
            done = _native.cache_evict(self.codes, self.scales, self.page_size, self.kv_heads, self.head_dim, self.blocksize, totals, table, lengths,
                                       keep, recent, sinks)
            if done is not None:
                return done
        F._require_gpu(self.codes, "QTensorCache.evict")
        if keep < 1 or recent < 0 or sinks < 0 or recent + sinks > keep:
            raise ValueError(f"need a token to keep, and no more first and last ones than are kept (got {keep}, {sinks} and {recent}).")
        places = self._places(table, lengths, None, lengths.numel())
        self._check_totals(totals, places)
        if places.batch > 65535:
            raise ValueError(f"{places.batch} sequences are too many for one call.")
        keep, recent, sinks = (min(n, 2 ** 62) for n in (keep, recent, sinks))
        cache = self._ref()
        with torch.cuda.device(totals.device):
            size = F.lib.qtensor_hip_cache_evict_workspace(cache, places, keep)
        scratch = torch.empty(size, dtype=torch.uint8, device=totals.device)
        out = torch.empty(places.batch, dtype=torch.int32, device=totals.device)
        F._call(F.lib.qtensor_hip_cache_evict, totals.device, cache, places, totals.data_ptr(), totals.stride(0), totals.stride(1), keep, recent, sinks,
                out.data_ptr(), scratch.data_ptr(), size)
        return out

    # ---- checks and descriptions
    def _check_queries(self, q: Tensor, scale: Optional[float], window: Optional[int], sinks: int):
        """(tokens, heads, scale) of queries and of what they see."""
        F._dtype_slot(q.dtype, "q")
        tokens, heads = (q.shape[0], q.shape[1]) if q.dim() == 3 else (-1, -1)
        self._check_vectors(q, "q", (tokens, heads, self.head_dim), q.dtype)
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"{heads} query heads are not a multiple of the cache's {self.kv_heads}.")
        if window is not None and window < 1:
            raise ValueError(f"window {window} is not positive.")
        if sinks < 0 or (sinks and window is None):
            raise ValueError("sinks are the first tokens that stay visible beside a window.")
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else float(scale)
        if not math.isfinite(scale):
            raise ValueError(f"scale {scale} is not finite.")
        return tokens, heads, scale

    def _check_totals(self, totals: Tensor, places: _Places) -> None:
        if totals.device != self.codes.device or totals.dtype != torch.float32:
            raise ValueError(f"totals are {totals.dtype} on {totals.device}, expected {torch.float32} on {self.codes.device}.")
        room = places.table_pages * self.page_size
        if totals.dim() != 3 or tuple(totals.shape[:2]) != (places.batch, self.kv_heads) or totals.shape[2] < room or not totals.is_contiguous():
            raise ValueError(f"totals have shape {tuple(totals.shape)}, expected contiguous ({places.batch}, {self.kv_heads}, {room} or more).")

    def _ref(self):
        # (what they were made as: the kernels go by the numbers below, whatever has taken the tensors' place)
        codes, scales = self.codes, self.scales
        for name, t, dtype, shape in (("codes", codes, torch.uint8, (self.kv_heads, self.page_size, 16 * (-(-self.head_dim // 32)))),
                                      ("scales", scales, torch.float32, (self.kv_heads, self.segments, self.page_size))):
            if t.device != codes.device or t.dtype != dtype or tuple(t.shape) != (2, self.pages, *shape) or not t.is_contiguous():
                raise ValueError(f"the cache's {name} are {t.dtype} {tuple(t.shape)} on {t.device}, not contiguous {dtype} {(2, self.pages, *shape)} on {codes.device}.")
        return _Cache((codes.data_ptr(), codes.data_ptr() + codes.stride(0)), (scales.data_ptr(), scales.data_ptr() + 4 * scales.stride(0)),
                      self.pages, self.page_size, self.kv_heads, self.head_dim, self.blocksize)

    def _check_vectors(self, t: Tensor, name: str, shape, dtype: torch.dtype) -> None:
        if t.device != self.codes.device:
            raise ValueError(f"{name} must live on the cache's device ({t.device} vs {self.codes.device}).")
        if t.dtype != dtype:
            raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}.")
        if tuple(t.shape) != shape or min(shape) < 0:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected [tokens, heads, {self.head_dim}]"
                             + (f" = {shape}." if min(shape) >= 0 else "."))
        if t.shape[2] > 1 and t.stride(2) != 1:
            raise ValueError(f"the last dimension of {name} must be contiguous.")
        F._check_derivatives("a cache", **{name: t})

    def _places(self, table: Tensor, lengths: Tensor, starts: Optional[Tensor], tokens: int) -> _Places:
        batch = lengths.numel()
        F._check_buffer(lengths, "lengths", batch, torch.int32, self.codes.device)
        if table.device != lengths.device or table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != batch:
            raise ValueError("table must be int32 [batch, pages of the longest sequence] on the cache's device, with a row per entry of lengths.")
        if table.shape[1] > 1 and table.stride(1) != 1:
            raise ValueError("the rows of table must be contiguous.")
        if batch < 1 or table.shape[1] < 1:
            raise ValueError("need at least one sequence and one page in the table.")
        if tokens > _MOST:
            raise ValueError(f"{tokens} tokens are too many for one call.")
        if starts is not None:
            F._check_buffer(starts, "starts", batch + 1, torch.int32, self.codes.device)
        elif tokens != batch:
            raise ValueError(f"without starts there is one token for each of {batch} sequences, not {tokens}.")
        return _Places(table.data_ptr(), lengths.data_ptr(), None if starts is None else starts.data_ptr(), table.stride(0), table.shape[1],
                       batch, tokens)


def _vectors(t: Tensor) -> _Vectors:
    return _Vectors(t.data_ptr(), t.dtype == torch.bfloat16, t.stride(0), t.stride(1))

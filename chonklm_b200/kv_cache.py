"""Quantised paged key-value cache (ck_kv_*) for torch tensors.

`QuantKvCache` holds one layer's pages: keys in 8 bits, values in 8 or 4, one
fp16 scale for each 32 values of a head.  The caller keeps the block table
([sequences][blocks] int32, on the device) and hands out the blocks.

    cache = QuantKvCache(heads=16, kv_heads=8, head_dim=128, n_blocks=512)
    q = cache.store(q, k, v, seq, pos, table, inv_freq=f)   # q rotated, k and v into their pages
    o = cache.attend_prompt(q, cu, length, table)           # the prompts' tokens, causal
    o = cache.attend(q, length, table)                      # one new token per sequence
    k, v = cache.load(seq, pos, table)                      # what the cache holds

Every call enqueues its kernel on `stream` (a cudaStream_t as an integer) or,
by default, on torch's current stream of the cache's device, and returns
without waiting; calls on one cache have to be ordered among themselves.  An
output that a call makes itself is memory of the stream that the call runs on.
A tensor that is used on another stream than its own is the caller's to keep
alive (`Tensor.record_stream`).  A wrong argument raises ValueError or
CkError, and so does a tensor that requires a gradient while gradients are
recorded (there is no backward); what only the device can see (a sequence,
position, block or row out of range) is skipped there and raised by `check()`.
There is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional, Tuple

import torch

from . import _lib

_I32 = torch.int32
_raw_stream = torch._C._cuda_getCurrentRawStream   # torch.cuda.current_stream(device).cuda_stream without its object
_DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

# the C argument structs (include/chonk_b200.h), packed by hand: a call is on
# the path of every token
_ROWS = "Pqqii"
_TABLE = "Pii"
_STORE = struct.Struct("@" + 4 * _ROWS + _TABLE + "PPPPPfiii")
_LOAD = struct.Struct("@" + 2 * _ROWS + _TABLE + "PPii")
_ATTEND = struct.Struct("@" + 2 * _ROWS + _TABLE + "PPiifi")
_NO_ROWS = (0, 0, 0, 1, 0)
_NO_NUMBER = (struct.error, OverflowError)   # a window, scale or eps that its field cannot hold


class QuantKvCache:
    """One layer's pages and the operators on them."""

    def __init__(self, heads: int, kv_heads: int, head_dim: int, n_blocks: int, block: int = 16, v_bits: int = 8,
                 device: int = 0):
        self._L = _lib.lib()
        self.heads, self.kv_heads, self.head_dim = int(heads), int(kv_heads), int(head_dim)
        self.n_blocks, self.block, self.v_bits = int(n_blocks), int(block), int(v_bits)
        self.device = int(device)
        cfg = (ctypes.c_int32 * 6)(self.heads, self.kv_heads, self.head_dim, self.block, self.v_bits, self.n_blocks)
        self.h = None
        h = ctypes.c_void_p()
        _lib._check(self._L.ck_kv_create(cfg, self.device, ctypes.byref(h)))
        self.h = h
        self._dev = torch.device("cuda", self.device)
        self._scale = 1.0 / math.sqrt(self.head_dim)

    # -- argument checks (each call is on the path of every token: plain comparisons, no helper objects) --
    def _rows(self, name: str, t, n: int, heads: int, f32: bool = True) -> tuple:
        dt = _DT.get(t.dtype, -1)
        if dt < 0 or (dt == 0 and not f32):
            raise ValueError(f"{name}: {t.dtype}, expected {'float32, ' if f32 else ''}float16 or bfloat16")
        if t.shape != (n, heads, self.head_dim):
            raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {(n, heads, self.head_dim)}")
        if t.get_device() != self.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {self._dev}")
        st, sh, sd = t.stride()
        if sd != 1:
            raise ValueError(f"{name}: the elements of a head are not contiguous")
        if t.requires_grad:
            self._no_grad(name)
        return t.data_ptr(), st, sh, dt, 0

    def _ints(self, name: str, t, n: int) -> int:
        if t.dtype is not _I32 or t.shape != (n,) or t.get_device() != self.device or not t.is_contiguous():
            raise ValueError(f"{name}: expected a contiguous int32 vector of {n} on {self._dev}")
        return t.data_ptr()

    def _table(self, t) -> tuple:
        if t.dtype is not _I32 or t.dim() != 2 or t.get_device() != self.device or not t.is_contiguous():
            raise ValueError(f"table: expected a contiguous int32 matrix on {self._dev}")
        return t.data_ptr(), *t.shape

    def _vector(self, name: str, t, n: int) -> int:
        if t is None:
            return 0
        if t.dtype is not torch.float32 or t.shape != (n,) or t.get_device() != self.device or not t.is_contiguous():
            raise ValueError(f"{name}: expected a contiguous float32 vector of {n} on {self._dev}")
        if t.requires_grad:
            self._no_grad(name)
        return t.data_ptr()

    @staticmethod
    def _no_grad(name: str) -> None:
        if torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient, and the cache's operators have none: call them under "
                             "torch.no_grad() or on detached tensors")

    def _stream(self, stream: Optional[int]) -> int:
        return _raw_stream(self.device) if stream is None else stream

    def _make(self, stream: int, empty, *args, **kw):
        """An output in memory of the stream that writes it: what is still pending elsewhere does not write there."""
        s = torch.cuda.ExternalStream(stream, self._dev) if stream else torch.cuda.default_stream(self._dev)
        with torch.cuda.stream(s):
            return empty(*args, **kw)

    def _like(self, t, stream: Optional[int]):
        return torch.empty_like(t) if stream is None else self._make(stream, torch.empty_like, t)

    def _check(self, rc: int) -> None:
        if rc:
            raise _lib.CkError(rc, (self._L.ck_kv_last_error(self.h) or b"").decode("utf-8", "replace"))

    # -- operators ----------------------------------------------------------
    def store(self, q, k, v, seq, pos, table, inv_freq=None, q_norm=None, k_norm=None, eps: float = 1e-6,
              interleaved: bool = False, out=None, stream: Optional[int] = None):
        """q [n, heads, head_dim] (or None), k and v [n, kv_heads, head_dim] of n tokens, token i of sequence seq[i] at
        position pos[i] (seq < 0: padding).  q and k are normed per head with q_norm / k_norm [head_dim] where given,
        rotated by pos * inv_freq [head_dim / 2] where given; k and v go into the cache.  Returns q in 16 bits (in
        `out`; of q's type, float16 for float32) or None."""
        n = k.shape[0]
        if q is not None:
            if out is None:
                if q.dtype is not torch.float32:
                    out = self._like(q, stream)
                elif stream is None:
                    out = torch.empty_like(q, dtype=torch.float16)
                else:
                    out = self._make(stream, torch.empty_like, q, dtype=torch.float16)
            qa, oa = self._rows("q", q, n, self.heads), self._rows("out", out, n, self.heads, False)
        else:
            if out is not None:
                raise ValueError("out without q")
            qa = oa = _NO_ROWS
        try:
            a = _STORE.pack(*qa, *self._rows("k", k, n, self.kv_heads), *self._rows("v", v, n, self.kv_heads), *oa,
                            *self._table(table), self._ints("seq", seq, n), self._ints("pos", pos, n),
                            self._vector("q_norm", q_norm, self.head_dim), self._vector("k_norm", k_norm, self.head_dim),
                            self._vector("inv_freq", inv_freq, self.head_dim // 2), eps, 1 if interleaved else 0, n, 0)
        except _NO_NUMBER as e:
            raise ValueError(str(e)) from None
        self._check(self._L.ck_kv_store(self.h, a, self._stream(stream)))
        return out

    def load(self, seq, pos, table, dtype=torch.float16, out: Optional[Tuple] = None, stream: Optional[int] = None):
        """(k, v) [n, kv_heads, head_dim] of the tokens (seq[i], pos[i]) as the cache holds them."""
        n = seq.shape[0]
        if out is None:
            shape = n, self.kv_heads, self.head_dim
            if stream is None:
                first = torch.empty(shape, dtype=dtype, device=self._dev)
            else:
                first = self._make(stream, torch.empty, shape, dtype=dtype, device=self._dev)
            out = first, self._like(first, stream)
        a = _LOAD.pack(*self._rows("k", out[0], n, self.kv_heads), *self._rows("v", out[1], n, self.kv_heads),
                       *self._table(table), self._ints("seq", seq, n), self._ints("pos", pos, n), n, 0)
        self._check(self._L.ck_kv_load(self.h, a, self._stream(stream)))
        return out

    def attend(self, q, length, table, scale: Optional[float] = None, window: int = 0, seq=None, out=None,
               stream: Optional[int] = None):
        """Attention of one new token per query: q [n, heads, head_dim] over the last `window` (0: all) of its length[i]
        cached positions, the new one among them; sequence i of the table, or seq[i].  scale: 1 / sqrt(head_dim)."""
        n = q.shape[0]
        if out is None:
            out = self._like(q, stream)
        try:
            a = _ATTEND.pack(*self._rows("q", q, n, self.heads, False), *self._rows("out", out, n, self.heads, False),
                             *self._table(table), self._ints("length", length, n), 0 if seq is None else self._ints("seq", seq, n),
                             n, window, self._scale if scale is None else scale, 0)
        except _NO_NUMBER as e:
            raise ValueError(str(e)) from None
        self._check(self._L.ck_kv_attend(self.h, a, self._stream(stream)))
        return out

    def attend_prompt(self, q, cu, length, table, scale: Optional[float] = None, window: int = 0, out=None,
                      stream: Optional[int] = None):
        """Causal attention of several new tokens per sequence: rows cu[i] .. cu[i + 1] of q are the last tokens of
        sequence i's length[i] cached positions (row i of the table).  Rows of no sequence are zero."""
        n = q.shape[0]
        if out is None:
            out = self._like(q, stream)
        s = cu.numel() - 1
        if s < 0:
            raise ValueError("cu: expected one entry more than sequences")
        cua = self._ints("cu", cu, s + 1)
        try:
            a = _ATTEND.pack(*self._rows("q", q, n, self.heads, False), *self._rows("out", out, n, self.heads, False),
                             *self._table(table), self._ints("length", length, s), 0, s, window,
                             self._scale if scale is None else scale, 0)
        except _NO_NUMBER as e:
            raise ValueError(str(e)) from None
        self._check(self._L.ck_kv_attend_prompt(self.h, a, cua, n, self._stream(stream)))
        return out

    def check(self, stream: Optional[int] = None) -> None:
        """Wait for the stream; raise if a kernel met a sequence, position, block or row out of range."""
        self._check(self._L.ck_kv_check(self.h, self._stream(stream)))

    @property
    def nbytes(self) -> int:
        n = ctypes.c_size_t()
        self._check(self._L.ck_kv_bytes(self.h, ctypes.byref(n)))
        return n.value

    def close(self) -> None:
        if getattr(self, "h", None):
            self._L.ck_kv_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

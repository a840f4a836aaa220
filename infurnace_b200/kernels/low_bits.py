"""Serving in few bits: matrices in microscaled 4-bit floating point and the products with them; pages of keys and values in
8 bits, the store into them and the attention that reads them.

:class:`Mx4Matrix` and :class:`Kv8Pages` are the data, :class:`LowBitKernels` the calls (a part of the kernel set).  Elements,
scales and layouts are defined at the heads of ``csrc/mx4.cu`` and ``csrc/kv8.cu``.
"""
from __future__ import annotations

from ctypes import c_char_p, c_int, c_longlong, c_void_p

import struct
import threading

import torch

from ..errors import KernelError
from .build import load_library

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
if _raw_stream is None:                       # an older torch: the public, slower way
    def _raw_stream(device_index):
        return torch.cuda.current_stream(device_index).cuda_stream
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)
_KV8_CALL = struct.Struct("=26qd").pack       # csrc/kv8_attention.cuh: Kv8Call

MX4_BLOCK = 32         # elements of a row that share a scale
_CODES = {torch.float32: 0, torch.bfloat16: 1}


class Mx4Matrix:
    """``rows`` x ``k`` numbers of 4 bits with a scale (a power of two) for each 32 of a row, ``k`` a multiple of 32.

    ``codes`` uint8 [rows, k / 2], element 2 i in the low half of a byte; ``scales`` uint8, in tiles of 128 rows x 128 of k as
    the tensor core takes them.  ``gated``: the rows are pairs (gate row i, up row i) of a matrix that had all gate rows before
    all up rows, which is the order that the gated epilogues of a product want.

    A product asks for its matrix before the kernel ahead of it in the stream has ended.  ``mx4_quantize`` and ``from_parts`` take care
    of that; who writes ``codes`` or ``scales`` in another way calls :meth:`written` on that stream before the next product.

    ``room``: None, or a uint8 tensor beside the codes for the rows that a product with the matrix rounds first (``row_bytes`` of
    them), in place of memory kept per stream (and, within a recording, of the graph's own pool for each graph).  Several matrices may
    have one room, as an engine's have, if the products with them, and the replays of recorded ones, follow one another."""

    _room, _room_at = None, (0, 0)

    def __init__(self, codes, scales, rows, k, gated=False):
        if codes.dtype != torch.uint8 or codes.shape != (rows, k // 2) or not codes.is_contiguous() or codes.data_ptr() % 16:
            raise KernelError("Mx4Matrix: codes are uint8 [rows, k / 2], contiguous, on 16 bytes")
        if scales.dtype != torch.uint8 or scales.numel() != self.scale_bytes(rows, k) or not scales.is_contiguous() \
                or scales.data_ptr() % 16 or scales.device != codes.device:
            raise KernelError("Mx4Matrix: scales are uint8, scale_bytes(rows, k) of them, contiguous, on 16 bytes, beside the codes")
        self.codes, self.scales, self.rows, self.k, self.gated = codes, scales, rows, k, bool(gated)
        self._at = (codes.data_ptr(), scales.data_ptr())
        self._index = codes.get_device()          # -1: not on a CUDA device

    @staticmethod
    def scale_bytes(rows, k):
        """Bytes of the scales: rows to a multiple of 256, k to a multiple of 128."""
        if rows < 1 or k < MX4_BLOCK or k % MX4_BLOCK:
            raise KernelError(f"Mx4Matrix: {rows} rows of {k}: rows are positive and k is a multiple of {MX4_BLOCK}")
        return -(-rows // 256) * 2 * -(-k // 128) * 512

    @property
    def room(self):
        return self._room

    @room.setter
    def room(self, room):
        if room is not None and (room.dtype != torch.uint8 or room.dim() != 1 or not room.is_contiguous() or room.data_ptr() % 256
                                 or room.device != self.codes.device):
            raise KernelError("Mx4Matrix: a room is uint8 [bytes], contiguous, on 256 bytes, beside the codes")
        self._room, self._room_at = room, (0, 0) if room is None else (room.data_ptr(), room.numel())

    @classmethod
    def row_bytes(cls, rows, k):
        """Bytes of a room for ``rows`` rows of ``k`` numbers: codes to a multiple of 256 bytes, then scales."""
        return -(-rows * k // 512) * 256 + cls.scale_bytes(rows, k)

    @classmethod
    def empty(cls, rows, k, device="cuda", gated=False):
        """Room for a matrix (``mx4_quantize`` fills it)."""
        scales = torch.zeros(cls.scale_bytes(rows, k), dtype=torch.uint8, device=device)
        return cls(torch.empty((rows, k // 2), dtype=torch.uint8, device=device), scales, rows, k, gated)

    @classmethod
    def from_parts(cls, codes, scales, gated=False):
        """From codes [rows, k / 2] and scales [rows, k / 32] in the order of the rows (a gated matrix: gate rows, then up
        rows), as a checkpoint keeps them."""
        rows, k = codes.shape[0], 2 * codes.shape[1]
        if scales.shape != (rows, k // MX4_BLOCK) or scales.dtype != torch.uint8 or codes.dtype != torch.uint8 or (gated and rows % 2):
            raise KernelError("Mx4Matrix.from_parts: codes are uint8 [rows, k / 2] and scales uint8 [rows, k / 32]; gated: of an even number of rows")
        size = cls.scale_bytes(rows, k)
        if gated:
            pairs = torch.arange(rows, device=codes.device).view(2, rows // 2).t().reshape(-1)
            codes, scales = codes[pairs], scales[pairs]
        rt, kt = -(-rows // 256) * 2, -(-k // 128)
        padded = torch.zeros((rt * 128, kt * 4), dtype=torch.uint8, device=codes.device)
        padded[:rows, :k // MX4_BLOCK] = scales
        tiles = padded.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).contiguous().view(size)
        return cls(codes.contiguous(), tiles, rows, k, gated).written()

    def written(self):
        """What the current stream has written so far into ``codes`` and ``scales`` is there before a product of that stream asks
        for it.  Returns the matrix."""
        if self._index >= 0:
            lib = load_library("mx4")
            lib.ifb_mx4_written.argtypes = [c_void_p]
            status = lib.ifb_mx4_written(_raw_stream(self._index))
            if status:
                LowBitKernels._low_bit_status(status, "Mx4Matrix.written")
        return self

    def parts(self):
        """(codes [rows, k / 2], scales [rows, k / 32]) in the order of the rows: what ``from_parts`` takes."""
        rt, kt = -(-self.rows // 256) * 2, -(-self.k // 128)
        scales = self.scales.view(rt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)[:self.rows, :self.k // MX4_BLOCK]
        codes = self.codes
        if self.gated:
            back = torch.arange(self.rows, device=codes.device).view(self.rows // 2, 2).t().reshape(-1)
            codes, scales = codes[back], scales[back]
        return codes.contiguous(), scales.contiguous()

    @property
    def shape(self):
        return (self.rows, self.k)

    @property
    def dtype(self):
        return torch.uint8

    @property
    def device(self):
        return self.codes.device

    def numel(self):
        return self.rows * self.k

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel()


class Kv8Pages:
    """Pages of keys and values of 8 bits: ``codes`` int8 [pages, 2, kv_heads, page_size, head_dim] and ``exponents`` uint8
    [pages, 2, kv_heads], one for the keys (or values) of a page and head.

    A number is (code + 1/2) step with step = 2^(exponent - 133); ``exponent`` is the exponent field of the block's largest
    number as a float32, 0 where all are zero (the values are then 0), 255 where one is infinite or NaN (the values are NaN).

    ``room``: None, or a uint8 tensor beside the codes in which ``kv8_attention`` lays out the pages that it expands, in place of
    memory of the allocator's for each call (and, within a recording, of the graph's own pool for each graph).  Several ``Kv8Pages``
    may have one room, as an engine's layers have, if the calls over them, and the replays of recorded ones, follow one another.
    A call that would need more than the room takes another form.  ``shared``: whether a page may be in the tables of two requests, or
    twice in one; where none is (False), there are no more pages to expand than the pool has."""

    room, shared = None, True

    def __init__(self, codes, exponents):
        if codes.dtype != torch.int8 or codes.dim() != 5 or codes.shape[1] != 2 or not codes.is_contiguous() or codes.data_ptr() % 16:
            raise KernelError("Kv8Pages: codes are int8 [pages, 2, kv_heads, page_size, head_dim], contiguous, on 16 bytes")
        if exponents.dtype != torch.uint8 or exponents.shape != codes.shape[:3] or not exponents.is_contiguous() \
                or exponents.device != codes.device:
            raise KernelError("Kv8Pages: exponents are uint8 [pages, 2, kv_heads], contiguous, beside the codes")
        self.codes, self.exponents = codes, exponents
        self._shape = codes.shape
        self.pages, _, self.kv_heads, self.page_size, self.head_dim = codes.shape
        if self.page_size % 16 or self.head_dim % 16 or not 16 <= self.head_dim <= 256 or not 16 <= self.page_size <= 4096:
            raise KernelError("Kv8Pages: page_size is a multiple of 16 up to 4,096, head_dim one up to 256")
        self._at = (codes.data_ptr(), exponents.data_ptr())
        self._index = codes.get_device()          # -1: not on a CUDA device

    @classmethod
    def empty(cls, pages, kv_heads, page_size, head_dim, device="cuda"):
        return cls(torch.zeros((pages, 2, kv_heads, page_size, head_dim), dtype=torch.int8, device=device),
                   torch.zeros((pages, 2, kv_heads), dtype=torch.uint8, device=device))


KV8_EXPAND_BYTES = 4 << 30       # room for expanded pages that a call takes at most


def kv8_room_bytes(pages, requests, pages_each, kv_heads, page_size, head_dim, dtype):
    """Bytes of a room (``Kv8Pages.room``) with which no call over a pool of ``pages`` pages, none of which two requests share, is
    short of it: for so many requests of so many pages at most.  0 where no call expands pages of these sizes."""
    if dtype != torch.bfloat16 or head_dim > 128 or page_size not in (16, 32, 64):
        return 0
    return min(KV8_EXPAND_BYTES, _expanded_bytes(pages, requests * pages_each, kv_heads, page_size, head_dim))


def _expanded_bytes(pages, entries, kv_heads, page_size, head_dim):
    return pages * 4 * kv_heads * page_size * head_dim + -(-entries // 64) * 256


class LowBitKernels:
    """The calls over 4-bit matrices; mixed into the kernel set, which gives streams, counters and the error word."""

    # Held by a call of several launches over one room, or of memory kept per stream, until the last is launched: the library's calls let
    # other threads run, and one on the same stream would write the room in between.
    _low_bit_lock = threading.RLock()
    _mx4 = None

    def _mx4_lib(self):
        if self._mx4 is None:
            lib = load_library("mx4", progress=self._progress)
            lib.ifb_mx4_quantize.argtypes = [c_void_p, c_int, c_longlong, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p]
            lib.ifb_mx4_values.argtypes = [c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p]
            lib.ifb_mx4_linear.argtypes = [c_void_p, c_int, c_longlong, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int,
                                           c_int, c_int, c_int, c_int, c_void_p, c_void_p]
            self._mx4_round_rows = {code: int(lib.ifb_mx4_round_rows(code)) for code in _CODES.values()}
            self._mx4 = lib
        return self._mx4

    @staticmethod
    def _low_bit_status(status, what):
        if status:
            from .cuda import _check
            _check(status, what)

    def mx4_quantize(self, x, matrix):
        """Rows of ``x`` (bfloat16 or float32 [rows, k], rows may lie apart) rounded to 4 bits into ``matrix``; for a gated
        matrix ``x`` has its gate rows, then its up rows.  Returns ``matrix``."""
        code = _CODES.get(x.dtype)
        index = matrix._index
        if code is None or x.shape != (matrix.rows, matrix.k) or x.stride(1) != 1 or x.get_device() != index or index < 0:
            raise KernelError(f"mx4_quantize: x is bfloat16 or float32 [{matrix.rows}, {matrix.k}] with unit stride along k, on the "
                              f"matrix's device; got {x.dtype} {tuple(x.shape)} on {x.device}")
        self.launches += 1
        status = self._mx4_lib().ifb_mx4_quantize(x.data_ptr(), code, x.stride(0) if matrix.rows > 1 else matrix.k, *matrix._at, matrix.rows, matrix.k, matrix.gated,
                                                  _raw_stream(index))
        if status:
            self._low_bit_status(status, "mx4_quantize")
        return matrix

    def mx4_values(self, matrix, out):
        """The numbers that ``matrix`` stands for, as bfloat16 (which holds them exactly) or float32 [rows, k]; a gated
        matrix's gate rows come before its up rows."""
        code = _CODES.get(out.dtype)
        index = matrix._index
        if code is None or out.shape != (matrix.rows, matrix.k) or not out.is_contiguous() or out.get_device() != index or index < 0:
            raise KernelError(f"mx4_values: out is bfloat16 or float32 [{matrix.rows}, {matrix.k}], contiguous, on the matrix's device")
        self.launches += 1
        status = self._mx4_lib().ifb_mx4_values(*matrix._at, out.data_ptr(), code, matrix.rows, matrix.k, matrix.gated, _raw_stream(index))
        if status:
            self._low_bit_status(status, "mx4_values")
        return out

    def mx4_matrix(self, w, gated=False):
        """A weight matrix rounded to 4 bits (``w`` [rows, k]; ``gated``: gate rows, then up rows)."""
        if w.dim() != 2 or (gated and w.shape[0] % 2):
            raise KernelError("mx4_matrix: w is [rows, k], a gated one of an even number of rows")
        return self.mx4_quantize(w, Mx4Matrix.empty(w.shape[0], w.shape[1], w.device, gated))

    def _mx4_room(self, w, stream, size):
        """Address of room for rounded rows: the matrix's, if it suffices; else of a stream each, whose launches follow one another, and
        memory of its own in a recording."""
        at, held = w._room_at
        if held >= size:
            return at
        device = w.codes.device
        if _capturing():
            held = self._mx4_recorded = torch.empty(size, dtype=torch.uint8, device=device)      # the graph's own pool keeps it for its replays
            return held.data_ptr()
        rooms = self.__dict__.setdefault("_mx4_rooms", {})
        held = rooms.get(stream)
        if held is None or held[0] < size:
            size = max(size, 1 << 20)
            room = torch.empty(size, dtype=torch.uint8, device=device)
            held = rooms[stream] = (size, room.data_ptr(), room)
        return held[1]

    def mx4_linear(self, x, w, out, epilogue="none", nt=0, splits=0):
        """out = Q(x) w^T with the epilogue (a key of ``EPILOGUES``), ``w`` an :class:`Mx4Matrix` and Q(x) the rows of ``x``
        rounded to 4 bits as ``mx4_quantize`` rounds them; ``x`` bfloat16 or float32 [n, k], or an :class:`Mx4Matrix` that
        has been rounded already.  ``out`` bfloat16 or float32 [n, features].  The gated epilogues want a gated ``w``.  ``nt`` and
        ``splits`` (for measurements): tokens of a tile and CTAs that share its k range, where the rule's choice is not wanted."""
        epi = self._epilogues.get(epilogue)
        if epi is None:
            raise KernelError(f"mx4_linear: unknown epilogue {epilogue!r}; known: {', '.join(self._epilogues)}")
        if len(x.shape) != 2:
            raise KernelError(f"mx4_linear: x is [n, k]; got {tuple(x.shape)}")
        n, k = x.shape
        code = _CODES.get(out.dtype)
        if k != w.k or (epi & 1 != 0) != w.gated or out.shape != (n, w.rows >> (epi & 1)):
            raise KernelError(f"mx4_linear: x {tuple(x.shape)}, w {w.shape} ({'gated' if w.gated else 'plain'}), out {tuple(out.shape)} "
                              f"and epilogue {epilogue!r} do not match")
        index = w._index
        if code is None or out.get_device() != index or not out.is_contiguous() or index < 0:
            raise KernelError("mx4_linear: out is bfloat16 or float32, contiguous, and all is on the matrix's device")
        if n == 0:
            return out
        lib, stream, launches, lock = self._mx4_lib(), _raw_stream(index), 1, None
        if isinstance(x, Mx4Matrix):
            if x.gated or x._index != index:
                raise KernelError("mx4_linear: x is a plain matrix on w's device")
            rows = (0, -1, 0, *x._at)
        else:
            x_code = _CODES.get(x.dtype)
            pitch, unit = x.stride()
            if x_code is None or unit != 1 or x.get_device() != index:
                raise KernelError("mx4_linear: x is bfloat16 or float32 with unit stride along k on w's device, or an Mx4Matrix")
            rows = (x.data_ptr(), x_code, pitch if n > 1 else k, 0, 0)      # (one row's pitch leads nowhere)
            if n > self._mx4_round_rows[x_code]:
                launches, lock = 2, self._low_bit_lock
        if lock is not None:
            lock.acquire()
        try:
            if lock is not None:
                codes = -(-n * k // 512) * 256                             # half a byte an element, to a multiple of 256
                room = self._mx4_room(w, stream, codes + Mx4Matrix.scale_bytes(n, k))
                rows = (*rows[:3], room, room + codes)
            self.launches += launches
            self._err_armed = True
            status = lib.ifb_mx4_linear(*rows, *w._at, out.data_ptr(), code, n, k, w.rows, epi, nt, splits, self._dev_err_at, stream)
        finally:
            if lock is not None:
                lock.release()
        if status:
            self._low_bit_status(status, "mx4_linear")
        return out

    # ------------------------------------------------------------------ keys and values of 8 bits
    _kv8 = None

    def _kv8_lib(self):
        if self._kv8 is None:
            lib = load_library("kv8", progress=self._progress)
            lib.ifb_kv8_store.argtypes = [c_void_p, c_void_p, c_int, c_longlong, c_longlong, c_void_p, c_void_p, c_void_p, c_int, c_int,
                                          c_int, c_int, c_void_p]
            lib.ifb_kv8_values.argtypes = [c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_int, c_void_p]
            lib.ifb_kv8_expand.argtypes = [c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p] + [c_int] * 9 + [c_void_p]
            self._kv8 = lib
        return self._kv8

    def kv8_store(self, k, v, slot_mapping, pages):
        """The step's keys and values (bfloat16 or float32 [tokens, kv_heads, head_dim], views with rows of their own pitch) into
        ``pages`` at ``slot_mapping`` (int32, page * page_size + offset; negative: not stored).  A page's tokens are adjacent
        rows in ascending order, as the step function lays them out; a token at offset 0 begins its page anew."""
        code = _CODES.get(k.dtype)
        heads, dim, index = pages.kv_heads, pages.head_dim, pages._index
        shape, pitch, v_pitch = k.shape, k.stride(), v.stride()
        n = shape[0] if len(shape) == 3 else -1
        if code is None or v.dtype != k.dtype or shape != (n, heads, dim) or v.shape != shape:
            raise KernelError(f"kv8_store: k and v are bfloat16 or float32 [tokens, {heads}, {dim}]; got {k.dtype} {tuple(k.shape)} and "
                              f"{v.dtype} {tuple(v.shape)}")
        if pitch[2] != 1 or v_pitch[2] != 1 or (heads > 1 and (pitch[1] != dim or v_pitch[1] != dim)):
            raise KernelError("kv8_store: the heads of a token lie one after the other")
        if slot_mapping.dtype != torch.int32 or slot_mapping.shape != (n,) or not slot_mapping.is_contiguous():
            raise KernelError("kv8_store: slot_mapping is int32, one per token, contiguous")
        if index < 0 or k.get_device() != index or v.get_device() != index or slot_mapping.get_device() != index:
            raise KernelError("kv8_store: k, v and slot_mapping are on the pages' device")
        if n == 0:
            return
        self.launches += 1
        k_row, v_row = (pitch[0], v_pitch[0]) if n > 1 else (heads * dim, heads * dim)
        status = self._kv8_lib().ifb_kv8_store(k.data_ptr(), v.data_ptr(), code, k_row, v_row, slot_mapping.data_ptr(), *pages._at, n, heads,
                                               pages.page_size, dim, _raw_stream(index))
        if status:
            self._low_bit_status(status, "kv8_store")

    def kv8_values(self, pages, out):
        """The numbers that the bits of all pages stand for, as bfloat16 or float32 (both hold them exactly) of the codes' shape."""
        code = _CODES.get(out.dtype)
        index = pages._index
        if code is None or out.shape != pages._shape or not out.is_contiguous() or out.get_device() != index or index < 0:
            raise KernelError("kv8_values: out is bfloat16 or float32 of the codes' shape, contiguous, on the pages' device")
        self.launches += 1
        status = self._kv8_lib().ifb_kv8_values(*pages._at, out.data_ptr(), code, pages.pages, pages.kv_heads, pages.page_size, pages.head_dim,
                                                _raw_stream(index))
        if status:
            self._low_bit_status(status, "kv8_values")
        return out

    def _kv8_attention_lib(self, dim, dtype):
        libs = self.__dict__.setdefault("_kv8_attention", {})
        lib = libs.get((dim, dtype))
        if lib is None:
            lib = load_library("kv8_attention" if dtype == torch.bfloat16 else "kv8_attention_f32", {"HEAD_DIM": dim}, progress=self._progress)
            lib.ifb_kv8_attention.argtypes = [c_char_p]
            lib.ifb_kv8_attention_scratch.restype = c_longlong
            lib.ifb_kv8_attention_scratch.argtypes = [c_int]
            floats = [int(lib.ifb_kv8_attention_scratch(nt)) for nt in range(1, lib.ifb_kv8_attention_tiles() + 1)]
            if min(floats) < 0:
                raise KernelError(f"kv8_attention: the device cannot be asked for its size (error {min(floats)})")
            lib.most_floats = max(floats)
            libs[(dim, dtype)] = lib
        return lib

    def _kv8_scratch(self, stream, floats, counters):
        """Addresses of (sums, counters) of the split form: of a stream each, and one pair for recorded graphs, whose replays follow
        one another.  The counters are zero between launches; a recording could not clear new ones, so what it uses is made
        before, with the first call outside of one; what an older recording uses is kept when room grows.  The counters' number goes by
        powers of two: new ones make recorded steps stale."""
        held = self.__dict__.setdefault("_kv8_held", {})
        capturing = _capturing()
        for key in (("graph",) if capturing else (stream, "graph")):
            have = held.get(key)
            if have is None or have[0] < floats or have[1] < counters:
                if capturing:
                    raise KernelError("kv8_attention: run the call once before it is recorded into a graph")
                floats_, counters_ = max(floats, have[0] if have else 0), max(1 << (counters - 1).bit_length(), have[1] if have else 4096)
                sums = torch.empty(floats_, dtype=torch.float32, device="cuda")
                zeros = torch.zeros(counters_, dtype=torch.int32, device="cuda")
                held[key] = (floats_, counters_, sums.data_ptr(), zeros.data_ptr(), sums, zeros)
                if key == "graph":
                    self.__dict__.setdefault("_kv8_recorded", []).append(have)
                    torch.cuda.current_stream().synchronize()            # cleared before a graph on another stream can use them
                    self.scratch_generation += 1
        return held["graph" if capturing else stream][2:4]

    kv8_expand_bytes = KV8_EXPAND_BYTES
    # Which form attends to requests of more than 16 score rows (queries x query heads of a key head) in bfloat16.  The split form's time
    # grows with the rows, 3.5 ns for 1,000 keys and row in all (heads of 128).  The tcgen05 kernel has a tile of 128 rows per SM: 10.7 ns
    # for a key and round of tiles, and the pages' expansion, 0.12 ns for a key and key head.  So up to 24 rows of an SM in
    # every round of tiles, and 32 of every request's key head, the split form is the shorter.  Measured, split and tcgen05, 32 query and
    # 8 key heads of 128: a request of 16 queries over 5,000 and 16,000 keys 22 and 60, 36 and 172 us; of 64 queries 43 and 61, 110 and 173; of
    # 128 queries 69 and 62, 201 and 175; 16 requests of 8 and of 32 queries over 1,200 keys 23 and 42, 71 and 44 us.
    kv8_split_rows = (24, 32)
    # Where that kernel does not fit (float32, heads wider than 128, other pages) all requests run split, but those of more than 64 rows
    # whole where the device has plenty of rows and the keys are few, so that an item's beginning and end count.  Measured, split and whole,
    # float32, 8 key heads of 128: 8 requests of 64 queries over 300 keys 50 and 37 us, of 1,024 over 1,200 keys 1,122 and 1,009, of 256 over
    # 5,000 keys 1,416 and 1,805; one of 64 over 300 keys 18 and 29.
    kv8_whole_rows, kv8_whole_keys = 64, 2048      # rows of an SM from which, keys up to which

    def _kv8_room_size(self, pages):
        """Bytes that the pages which a call expands may take."""
        room = pages.room
        if room is None:
            return self.kv8_expand_bytes
        if room.dtype != torch.uint8 or room.dim() != 1 or not room.is_contiguous() or room.data_ptr() % 128 or room.get_device() != pages._index:
            raise KernelError("kv8_attention: a room is uint8 [bytes], contiguous, on 128 bytes, on the pages' device")
        return room.numel()

    def _kv8_expand(self, pages, block_tables, cu_q, seq_lens, window, r, group, most, room, stream):
        """The pages of the requests with more than 16 score rows as bfloat16 (exact), and tables of them."""
        kv_heads, ps, dim = pages.kv_heads, pages.page_size, pages.head_dim
        held = pages.room
        if held is None:
            wide = torch.empty((room, 2, kv_heads, ps, dim), dtype=torch.bfloat16, device=pages.codes.device)
            tables = torch.empty((r, most), dtype=torch.int32, device=pages.codes.device)
        else:
            split = room * 4 * kv_heads * ps * dim
            wide = held[:split].view(torch.bfloat16).view(room, 2, kv_heads, ps, dim)
            tables = held[split:split + 4 * r * most].view(torch.int32).view(r, most)
        self.launches += 1
        status = self._kv8_lib().ifb_kv8_expand(*pages._at, block_tables.data_ptr(), block_tables.stride(0), cu_q.data_ptr(), seq_lens.data_ptr(),
                                                wide.data_ptr(), tables.data_ptr(), room, r, most, kv_heads, group, ps, dim, window, 16, stream)
        if status:
            self._low_bit_status(status, "kv8_attention")
        return wide, tables

    def kv8_attention(self, q, pages, block_tables, cu_q, seq_lens, out, scale, window, max_q_len, max_seq_len, min_q_len=1,
                      exact_lens=False):
        """Causal attention of a step's queries over 8-bit pages: ``q`` and ``out`` bfloat16 or float32 [tokens, heads, head_dim] (the
        rows of ``q`` may lie apart, those of ``out`` not); the query at position p sees positions max(0, p - window + 1) .. p
        (``window`` 0: from 0); request r has the rows cu_q[r] .. cu_q[r + 1] - 1 and ``seq_lens[r]`` keys, these queries' own
        among them.  A row that sees no key becomes zero.  No request has more than ``max_q_len`` queries or ``max_seq_len``
        keys, none fewer than ``min_q_len`` queries; ``exact_lens``: some request has ``max_q_len``, and ``q`` no other rows than
        theirs, which bounds how many are long.  Numbers of queries, keys and values are below 2^100 in size, or infinite or NaN
        (which the rows that see them become): sums of larger ones may overflow.  Recorded calls share memory for the split form's sums:
        run the call once before a recording, and let replays follow one another."""
        code = _CODES.get(q.dtype)
        shape, pitch, index = q.shape, q.stride(), pages._index
        n, heads, dim = shape if len(shape) == 3 else (0, 0, 0)
        kv_heads = pages.kv_heads
        if code is None or out.dtype != q.dtype or out.shape != shape or dim != pages.head_dim or heads % kv_heads:
            raise KernelError(f"kv8_attention: q and out are bfloat16 or float32 [tokens, a multiple of {kv_heads}, {pages.head_dim}]; got "
                              f"{q.dtype} {tuple(q.shape)} and {out.dtype} {tuple(out.shape)}")
        if pitch[2] != 1 or (heads > 1 and pitch[1] != dim) or not out.is_contiguous():
            raise KernelError("kv8_attention: the heads of a query lie one after the other, and out is contiguous")
        r = seq_lens.numel()
        table_shape, table_pitch = block_tables.shape, block_tables.stride()
        if cu_q.dtype != torch.int32 or seq_lens.dtype != torch.int32 or block_tables.dtype != torch.int32 or cu_q.numel() != r + 1 \
                or len(table_shape) != 2 or table_shape[0] < r or (table_pitch[1] != 1 and table_shape[1] > 1) or not cu_q.is_contiguous() or not seq_lens.is_contiguous():
            raise KernelError("kv8_attention: cu_q, seq_lens and block_tables are int32 for the same requests, dense along their last axis")
        if table_shape[1] * pages.page_size < max_seq_len:
            raise KernelError(f"kv8_attention: block tables of {table_shape[1]} pages do not hold {max_seq_len} keys")
        if index < 0 or q.get_device() != index or out.get_device() != index or cu_q.get_device() != index or seq_lens.get_device() != index \
                or block_tables.get_device() != index:
            raise KernelError("kv8_attention: all tensors are on the pages' device")
        if n == 0 or r == 0:
            return out
        if window < 0 or max_q_len < 1 or not 1 <= min_q_len <= max_q_len:
            raise KernelError("kv8_attention: window is not negative, and 1 <= min_q_len <= max_q_len")
        lib, stream, group = self._kv8_attention_lib(dim, q.dtype), _raw_stream(index), heads // kv_heads
        q_row = pitch[0] if n > 1 else heads * dim
        rows, least = max_q_len * group, min_q_len * group
        tc = False
        if rows > 16 and q.dtype == torch.bfloat16 and dim <= 128 and group <= 128 and pages.page_size in (16, 32, 64) and self.attention_tc:
            per_round, per_head = self.kv8_split_rows
            long = min(r, -(-n // max_q_len)) * kv_heads
            rounds = -(-long * -(-max_q_len // (128 // group)) // self.sm_count)
            if n * heads > per_round * self.sm_count * rounds + per_head * long:
                # (a long request has more than 16 score rows)
                most = -(-max_seq_len // pages.page_size)
                room = most * (self.long_requests(n, r, group, max_q_len, min_q_len) if exact_lens else min(r, n // (16 // group + 1)))
                if not pages.shared:
                    room = min(room, pages.pages)
                tc = _expanded_bytes(room, r * most, kv_heads, pages.page_size, dim) <= self._kv8_room_size(pages)
        with self._low_bit_lock:
            if tc:
                wide, wide_tables = self._kv8_expand(pages, block_tables, cu_q, seq_lens, window, r, group, most, room, stream)
                rows = 16
            # score rows up to which a request runs split
            limit = min(rows, 64) if n * heads > self.kv8_whole_rows * self.sm_count and max_seq_len <= self.kv8_whole_keys else rows
            nt = 1 if rows <= 8 or dim > 128 or tc and group <= 8 else 2      # (beside prompts the short requests decode)
            fixed = (q.data_ptr(), code, q_row, *pages._at, block_tables.data_ptr(), table_pitch[0], cu_q.data_ptr(), seq_lens.data_ptr(),
                     out.data_ptr())
            sizes = (r, heads, kv_heads, pages.page_size, dim, window, max_q_len)
            status = 0
            if least <= limit:
                tiles = -(-limit // (8 * nt))
                items = min(r * tiles, r + n * group // (8 * nt)) * kv_heads
                self.launches += 1
                status = lib.ifb_kv8_attention(_KV8_CALL(*fixed, *self._kv8_scratch(stream, lib.most_floats, r * tiles * kv_heads), *sizes, 0, limit,
                                                         tiles, nt, 0, items, stream, scale))
            if rows > limit and not status:
                self.launches += 1
                status = lib.ifb_kv8_attention(_KV8_CALL(*fixed, 0, 0, *sizes, limit + 1, (1 << 31) - 1, 1, 1, 1, 0, stream, scale))
            if status:
                self._low_bit_status(status, "kv8_attention")
            if tc:
                at, step, block = wide.data_ptr(), wide.stride(0), 2 * kv_heads * pages.page_size * dim
                self._attention_tc_streams(q.as_strided((n, heads * dim), (q_row, 1)), heads, kv_heads, 1, dim, dim, (at, step, pages.page_size),
                                           (at + block, step, pages.page_size), room, wide_tables, cu_q, seq_lens, out, scale, window, max_q_len, n, r,
                                           2, None, None, kind=0)
        return out

"""Serving in few bits: matrices in microscaled 4-bit floating point and the products with them.

:class:`Mx4Matrix` is the data, :class:`LowBitKernels` the calls (a part of the kernel set).  Elements, scales and layout are
defined at the head of ``csrc/mx4.cu``.
"""
from __future__ import annotations

from ctypes import c_int, c_longlong, c_void_p

import torch

from ..errors import KernelError
from .build import load_library

MX4_BLOCK = 32         # elements of a row that share a scale
_CODES = {torch.float32: 0, torch.bfloat16: 1}


class Mx4Matrix:
    """``rows`` x ``k`` numbers of 4 bits with a scale (a power of two) for each 32 of a row, ``k`` a multiple of 32.

    ``codes`` uint8 [rows, k / 2], element 2 i in the low half of a byte; ``scales`` uint8, in tiles of 128 rows x 128 of k as
    the tensor core takes them.  ``gated``: the rows are pairs (gate row i, up row i) of a matrix that had all gate rows before
    all up rows, which is the order that the gated epilogues of a product want."""

    def __init__(self, codes, scales, rows, k, gated=False):
        if codes.dtype != torch.uint8 or codes.shape != (rows, k // 2) or not codes.is_contiguous() or codes.data_ptr() % 16:
            raise KernelError("Mx4Matrix: codes are uint8 [rows, k / 2], contiguous, on 16 bytes")
        if scales.dtype != torch.uint8 or scales.numel() != self.scale_bytes(rows, k) or not scales.is_contiguous() \
                or scales.data_ptr() % 16 or scales.device != codes.device:
            raise KernelError("Mx4Matrix: scales are uint8, scale_bytes(rows, k) of them, contiguous, on 16 bytes, beside the codes")
        self.codes, self.scales, self.rows, self.k, self.gated = codes, scales, rows, k, bool(gated)
        self._at = (codes.data_ptr(), scales.data_ptr())

    @staticmethod
    def scale_bytes(rows, k):
        """Bytes of the scales: rows to a multiple of 256, k to a multiple of 128."""
        if rows < 1 or k < MX4_BLOCK or k % MX4_BLOCK:
            raise KernelError(f"Mx4Matrix: {rows} rows of {k}: rows are positive and k is a multiple of {MX4_BLOCK}")
        return -(-rows // 256) * 2 * -(-k // 128) * 512

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
        return cls(codes.contiguous(), tiles, rows, k, gated)

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
    number as a float32, 0 where all are zero (the values are then 0), 255 where one is infinite or NaN (the values are NaN)."""

    def __init__(self, codes, exponents):
        if codes.dtype != torch.int8 or codes.dim() != 5 or codes.shape[1] != 2 or not codes.is_contiguous() or codes.data_ptr() % 16:
            raise KernelError("Kv8Pages: codes are int8 [pages, 2, kv_heads, page_size, head_dim], contiguous, on 16 bytes")
        if exponents.dtype != torch.uint8 or exponents.shape != codes.shape[:3] or not exponents.is_contiguous() \
                or exponents.device != codes.device:
            raise KernelError("Kv8Pages: exponents are uint8 [pages, 2, kv_heads], contiguous, beside the codes")
        self.codes, self.exponents = codes, exponents
        self.pages, _, self.kv_heads, self.page_size, self.head_dim = codes.shape
        self._at = (codes.data_ptr(), exponents.data_ptr())

    @classmethod
    def empty(cls, pages, kv_heads, page_size, head_dim, device="cuda"):
        return cls(torch.zeros((pages, 2, kv_heads, page_size, head_dim), dtype=torch.int8, device=device),
                   torch.zeros((pages, 2, kv_heads), dtype=torch.uint8, device=device))


class LowBitKernels:
    """The calls over 4-bit matrices; mixed into the kernel set, which gives streams, counters and the error word."""

    _mx4 = None

    def _mx4_lib(self):
        if self._mx4 is None:
            lib = load_library("mx4", progress=self._progress)
            lib.ifb_mx4_quantize.argtypes = [c_void_p, c_int, c_longlong, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p]
            lib.ifb_mx4_values.argtypes = [c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p]
            lib.ifb_mx4_linear.argtypes = [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_int,
                                           c_void_p, c_void_p]
            self._mx4_scratch = {}
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
        if code is None or not x.is_cuda or x.dim() != 2 or x.shape != (matrix.rows, matrix.k) or x.stride(1) != 1 \
                or x.device != matrix.codes.device:
            raise KernelError(f"mx4_quantize: x is bfloat16 or float32 [{matrix.rows}, {matrix.k}] with unit stride along k, on the "
                              f"matrix's device; got {x.dtype} {tuple(x.shape)} on {x.device}")
        self.launches += 1
        self._low_bit_status(self._mx4_lib().ifb_mx4_quantize(x.data_ptr(), code, x.stride(0), *matrix._at, matrix.rows, matrix.k,
                                                              matrix.gated, self._stream()), "mx4_quantize")
        return matrix

    def mx4_values(self, matrix, out):
        """The numbers that ``matrix`` stands for, as bfloat16 (which holds them exactly) or float32 [rows, k]; a gated
        matrix's gate rows come before its up rows."""
        code = _CODES.get(out.dtype)
        if code is None or not out.is_cuda or out.shape != (matrix.rows, matrix.k) or not out.is_contiguous() \
                or out.device != matrix.codes.device:
            raise KernelError(f"mx4_values: out is bfloat16 or float32 [{matrix.rows}, {matrix.k}], contiguous, on the matrix's device")
        self.launches += 1
        self._low_bit_status(self._mx4_lib().ifb_mx4_values(*matrix._at, out.data_ptr(), code, matrix.rows, matrix.k, matrix.gated,
                                                            self._stream()), "mx4_values")
        return out

    def mx4_matrix(self, w, gated=False):
        """A weight matrix rounded to 4 bits (``w`` [rows, k]; ``gated``: gate rows, then up rows)."""
        if w.dim() != 2 or (gated and w.shape[0] % 2):
            raise KernelError("mx4_matrix: w is [rows, k], a gated one of an even number of rows")
        return self.mx4_quantize(w, Mx4Matrix.empty(w.shape[0], w.shape[1], w.device, gated))

    def mx4_linear(self, x, w, out, epilogue="none"):
        """out = Q(x) w^T with the epilogue (a key of ``EPILOGUES``), ``w`` an :class:`Mx4Matrix` and Q(x) the rows of ``x``
        rounded to 4 bits as ``mx4_quantize`` rounds them; ``x`` bfloat16 or float32 [n, k], or an :class:`Mx4Matrix` that
        has been rounded already.  ``out`` bfloat16 or float32 [n, features].  The gated epilogues want a gated ``w``."""
        from .cuda import EPILOGUES
        epi = EPILOGUES.get(epilogue)
        if epi is None:
            raise KernelError(f"mx4_linear: unknown epilogue {epilogue!r}; known: {', '.join(EPILOGUES)}")
        n, k = x.shape
        code = _CODES.get(out.dtype)
        features = w.rows // 2 if epi & 1 else w.rows
        if k != w.k or bool(epi & 1) != w.gated or out.shape != (n, features):
            raise KernelError(f"mx4_linear: x {tuple(x.shape)}, w {w.shape} ({'gated' if w.gated else 'plain'}), out {tuple(out.shape)} "
                              f"and epilogue {epilogue!r} do not match")
        if code is None or not out.is_cuda or not out.is_contiguous() or out.device != w.codes.device:
            raise KernelError("mx4_linear: out is bfloat16 or float32, contiguous, on the matrix's device")
        lib, stream = self._mx4_lib(), self._stream()
        if not isinstance(x, Mx4Matrix):
            held = self._mx4_scratch.get((stream, k))
            if held is None or held.codes.shape[0] < n:
                held = self._mx4_scratch[(stream, k)] = Mx4Matrix.empty(max(n, 256), k, w.codes.device)
                self.scratch_generation += 1
            x = self.mx4_quantize(x, Mx4Matrix(held.codes[:n], held.scales[:Mx4Matrix.scale_bytes(n, k)], n, k))
        elif x.gated or x.codes.device != w.codes.device:
            raise KernelError("mx4_linear: x is a plain matrix on w's device")
        self.launches += 1
        self._err_armed = True
        self._low_bit_status(lib.ifb_mx4_linear(*x._at, *w._at, out.data_ptr(), code, n, k, w.rows, epi, self._dev_err.data_ptr(),
                                                stream), "mx4_linear")
        return out

"""Several answers to one prompt: drawing tokens under top-k, top-p and min-p, the log probabilities of tokens, and attention over
pages that requests share.

:class:`AnswerKernels` is the calls (a part of the kernel set).  What is drawn, and how, is defined at the head of ``csrc/sampling.cu``, how
attention is cut into pieces at the head of ``csrc/attention_shared.cuh``.
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_longlong, c_void_p

import torch

from ..errors import KernelError
from .build import load_library

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
if _raw_stream is None:                       # an older torch: the public, slower way
    def _raw_stream(device_index):
        return torch.cuda.current_stream(device_index).cuda_stream
_CODES = {torch.float32: 0, torch.bfloat16: 1}


def _status(status, what):
    if status:
        from .cuda import _check
        _check(status, what)


def _logit_rows(logits, what):
    """(dtype code, rows, vocabulary, elements between rows, device) of a call's logits."""
    code = _CODES.get(logits.dtype)
    shape = logits.shape
    if code is None or len(shape) != 2 or shape[1] < 1 or (shape[1] > 1 and logits.stride(1) != 1):
        raise KernelError(f"{what}: logits are float32 or bfloat16 [rows, vocabulary] with unit stride along the vocabulary; got {logits.dtype} "
                          f"{tuple(shape)} of strides {logits.stride()}")
    index = logits.get_device()
    if index < 0:
        raise KernelError(f"{what}: logits are not on a CUDA device")
    rows, vocab = shape
    pitch = logits.stride(0) if rows > 1 else vocab          # (one row's pitch leads nowhere)
    return code, rows, vocab, pitch, index


def _one_per_row(t, dtype, rows, index, what, name, optional=False):
    """The address of a tensor with one number for each row (0: absent)."""
    if t is None and optional:
        return 0
    if t.dtype != dtype or t.shape != (rows,) or (rows > 1 and t.stride(0) != 1) or t.get_device() != index:
        raise KernelError(f"{what}: {name} is {dtype} [{rows}], contiguous, on the logits' device; got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


class AnswerKernels:
    """Mixed into the kernel set, which gives counters and the error word."""

    _sampling = None

    def _sampling_lib(self):
        if self._sampling is None:
            lib = load_library("sampling", progress=self._progress)
            lib.ifb_sample_cut.argtypes = [c_void_p, c_int, c_longlong, c_int, c_int] + [c_void_p] * 8
            lib.ifb_token_logprobs.argtypes = [c_void_p, c_int, c_longlong, c_int, c_int] + [c_void_p] * 4
            self._sampling_max_vocab = int(lib.ifb_sample_cut_max_vocab())
            self._sampling = lib
        return self._sampling

    def sample_filtered(self, logits, temperature, uniform, out, top_k=None, top_p=None, min_p=None, logprobs=None):
        """A token for each row of ``logits`` (float32 or bfloat16 [rows, vocabulary]; rows may lie apart) from softmax(logits / temperature) cut by
        top-k, then top-p, then min-p, each off where it is None.  All others have one number a row: ``temperature`` (float32; 0: the
        largest logit), ``uniform`` (float32 in [0, 1)), ``top_k`` (int32; below 1: off), ``top_p`` (float32; from 1 on: off; at least the best
        token stays), ``min_p`` (float32; a token stays whose probability is at least this times the best one's), ``out`` (int32) and
        ``logprobs`` (float32: the drawn token's log probability under what the cuts left, 0 at temperature 0).

        Among equal logits the lower index is the better; the draw is by inverse CDF in the order of indices.  NaN counts as -inf,
        which is never drawn; of infinities each is as likely as the other.  A row without a number above -inf gives token 0 and NaN.  A
        row's token depends on that row alone, and on its weights to 2^-44 of the largest."""
        code, rows, vocab, pitch, index = _logit_rows(logits, "sample_filtered")
        args = (_one_per_row(temperature, torch.float32, rows, index, "sample_filtered", "temperature"),
                _one_per_row(uniform, torch.float32, rows, index, "sample_filtered", "uniform"),
                _one_per_row(top_k, torch.int32, rows, index, "sample_filtered", "top_k", True),
                _one_per_row(top_p, torch.float32, rows, index, "sample_filtered", "top_p", True),
                _one_per_row(min_p, torch.float32, rows, index, "sample_filtered", "min_p", True),
                _one_per_row(out, torch.int32, rows, index, "sample_filtered", "out"),
                _one_per_row(logprobs, torch.float32, rows, index, "sample_filtered", "logprobs", True))
        lib = self._sampling_lib()
        if vocab > self._sampling_max_vocab:
            raise KernelError(f"sample_filtered: a vocabulary of {vocab}; at most {self._sampling_max_vocab}")
        if rows == 0:
            return out
        with torch.cuda.device(index):
            self.launches += 1
            _status(lib.ifb_sample_cut(logits.data_ptr(), code, pitch, rows, vocab, *args, _raw_stream(index)), "sample_filtered")
        return out

    def token_logprobs(self, logits, tokens, out, ranks=None):
        """The log probability of token ``tokens[r]`` under softmax(logits[r]) into ``out`` (float32), and the number of tokens that come before it by
        falling logit, equal ones by rising index, into ``ranks`` (int32).  ``logits`` float32 or bfloat16 [rows, vocabulary], rows may
        lie apart; ``tokens`` int32, one a row.  A token outside the vocabulary (padding) gives NaN and -1; a row with a NaN
        or +inf, or with no number above -inf, NaN."""
        code, rows, vocab, pitch, index = _logit_rows(logits, "token_logprobs")
        args = (_one_per_row(tokens, torch.int32, rows, index, "token_logprobs", "tokens"),
                _one_per_row(out, torch.float32, rows, index, "token_logprobs", "out"),
                _one_per_row(ranks, torch.int32, rows, index, "token_logprobs", "ranks", True))
        if rows == 0:
            return out
        with torch.cuda.device(index):
            self.launches += 1
            _status(self._sampling_lib().ifb_token_logprobs(logits.data_ptr(), code, pitch, rows, vocab, *args, _raw_stream(index)), "token_logprobs")
        return out

    # ------------------------------------------------------------------ attention over shared pages
    def _shared_lib(self, dtype, dim):
        """(call, size of its room) for a type and head size."""
        libs = self.__dict__.setdefault("_shared", {})
        held = libs.get((dtype, dim))
        if held is None:
            if dtype == torch.float32:
                lib = load_library("attention_shared", progress=self._progress)
                call, room = lib.ifb_attention_shared, lib.ifb_attention_shared_room
            else:
                lib = load_library("attention_shared_bf16", {"HEAD_DIM": dim}, progress=self._progress)
                call, room = lib.ifb_attention_shared_bf16, lib.ifb_attention_shared_bf16_room
            call.argtypes = [c_void_p, c_longlong, c_void_p, c_longlong, c_longlong, c_void_p, c_longlong, c_int] + [c_void_p] * 7 + [c_int] * 7 + [
                c_float, c_int, c_void_p]
            room.argtypes, room.restype = [c_int] * (6 if dtype == torch.float32 else 5), c_longlong
            held = libs[(dtype, dim)] = (call, room)
        return held

    def shared_prefix_room(self, tokens, requests, groups, heads, kv_heads, head_dim, dtype):
        """Bytes of the room that ``shared_prefix_attention`` takes for a step of so many tokens, requests and groups."""
        sizes = (tokens, requests, groups, kv_heads, heads // kv_heads)
        return int(self._shared_lib(dtype, head_dim)[1](*sizes, *((head_dim,) if dtype == torch.float32 else ())))

    def shared_prefix_attention(self, q, kv_pages, block_tables, cu_q, seq_lens, cu_groups, shared_lens, out, scale, window, max_q_len, max_seq_len,
                                room=None):
        """``paged_attention`` for requests whose block tables share leading pages, which are then read once for all of them: answers to one
        prompt, questions to one document, conversations behind one system prompt.

        ``q`` and ``out`` are bfloat16 or float32 [tokens, heads, head_dim] (the rows of ``q`` may lie apart, those of ``out`` not), ``kv_pages`` [pages, 2,
        kv_heads, page_size, head_dim] of the same type.  Request r has the rows cu_q[r] .. cu_q[r + 1] - 1 and ``seq_lens[r]`` keys, these
        queries' own among them, in the pages of ``block_tables[r]``; the query at position p sees positions max(0, p - window + 1) .. p
        (``window`` 0: from 0).  Group g is the requests cu_groups[g] .. cu_groups[g + 1] - 1, the first ``shared_lens[g]`` keys of which are the same: they are
        read through the table of its first request.  (Any number of keys; beyond them each request's own table counts, also within
        a page.)  Requests of no group share nothing.  A row that sees no key becomes zero; rows behind the last request stay as they are.
        ``cu_q``, ``seq_lens``, ``block_tables``, ``cu_groups`` [groups + 1] and ``shared_lens`` [groups] are int32 on the device.  No request has more than
        ``max_q_len`` queries or ``max_seq_len`` keys.  An entry of a table that is read and is no page of the pool counts as zeros and is recorded in the
        kernels' error word.

        ``room``: None, or a uint8 tensor of at least ``shared_prefix_room`` bytes for the pieces' sums, in place of memory of the allocator's (within
        a recording: of the graph's own pool); calls that share one follow one another."""
        code = _CODES.get(q.dtype)
        shape, index = q.shape, q.get_device()
        n, heads, dim = shape if len(shape) == 3 else (0, 0, 0)
        pool = kv_pages.shape
        if code is None or out.dtype != q.dtype or out.shape != shape or kv_pages.dtype != q.dtype or len(pool) != 5 or pool[1] != 2 \
                or pool[4] != dim or pool[2] < 1 or heads % pool[2] or heads == 0:
            raise KernelError(f"shared_prefix_attention: q and out are bfloat16 or float32 [tokens, heads, head_dim] and kv_pages [pages, 2, kv_heads, page_size, "
                              f"head_dim] of one type, heads a multiple of kv_heads; got {q.dtype} {tuple(shape)}, {out.dtype} {tuple(out.shape)} and "
                              f"{kv_pages.dtype} {tuple(pool)}")
        pages, _, kv_heads, page_size, _ = pool
        group = heads // kv_heads
        if dim % 16 or not 16 <= dim <= 256 or group > 64:
            raise KernelError(f"shared_prefix_attention: head_dim is a multiple of 16 up to 256, with up to 64 query heads for a key head; got {dim} and {group}")
        if q.stride(2) != 1 or (heads > 1 and q.stride(1) != dim) or not out.is_contiguous():
            raise KernelError("shared_prefix_attention: the heads of a query lie one after the other, and out is contiguous")
        block = 2 * kv_heads * page_size * dim
        page_stride = kv_pages.stride(0) if pages > 1 else block
        if pages < 1 or not kv_pages[0].is_contiguous() or page_stride < block:
            raise KernelError("shared_prefix_attention: the numbers of a page lie one after the other")
        r, groups = seq_lens.numel(), shared_lens.numel()
        table = block_tables.shape
        for t, name, count in ((cu_q, "cu_q", r + 1), (seq_lens, "seq_lens", r), (cu_groups, "cu_groups", groups + 1), (shared_lens, "shared_lens", groups)):
            if t.dtype != torch.int32 or t.shape != (count,) or not t.is_contiguous():
                raise KernelError(f"shared_prefix_attention: {name} is int32 [{count}], contiguous; got {t.dtype} {tuple(t.shape)}")
        if block_tables.dtype != torch.int32 or len(table) != 2 or table[0] < r or (table[1] > 1 and block_tables.stride(1) != 1):
            raise KernelError("shared_prefix_attention: block_tables is int32 [requests, pages] with unit stride along pages")
        if index < 0 or any(t.get_device() != index for t in (kv_pages, out, block_tables, cu_q, seq_lens, cu_groups, shared_lens)):
            raise KernelError("shared_prefix_attention: all tensors are on one CUDA device")
        if window < 0 or max_q_len < 1 or max_seq_len < 0:
            raise KernelError("shared_prefix_attention: window and max_seq_len are not negative, max_q_len is positive")
        if table[1] * page_size < max_seq_len:
            raise KernelError(f"shared_prefix_attention: block tables of {table[1]} pages do not hold {max_seq_len} keys")
        if r + groups > 2048:
            raise KernelError(f"shared_prefix_attention: {r} requests and {groups} groups; at most 2,048 together")
        if n == 0 or r == 0:
            return out
        q_row = q.stride(0) if n > 1 else heads * dim
        with torch.cuda.device(index):
            call, room_of = self._shared_lib(q.dtype, dim)
            size = room_of(n, r, groups, kv_heads, group, dim) if q.dtype == torch.float32 else room_of(n, r, groups, kv_heads, group)
            if room is None:
                room = torch.empty(size, dtype=torch.uint8, device=q.device)
            elif room.dtype != torch.uint8 or room.dim() != 1 or not room.is_contiguous() or room.numel() < size or room.data_ptr() % 256 \
                    or room.get_device() != index:
                raise KernelError(f"shared_prefix_attention: a room is uint8 [{size} or more], contiguous, on 256 bytes, on the same device")
            self.launches += 2 if q.dtype == torch.float32 or group > 16 or n * group <= 16 else 3
            self._err_armed = True
            status = call(q.data_ptr(), q_row, kv_pages.data_ptr(), page_stride, pages, block_tables.data_ptr(), block_tables.stride(0), table[1],
                          cu_q.data_ptr(), seq_lens.data_ptr(), cu_groups.data_ptr(), shared_lens.data_ptr(), out.data_ptr(), room.data_ptr(),
                          self._dev_err_at, n, r, groups, heads, kv_heads, dim, page_size, scale, window, _raw_stream(index))
            _status(status, "shared_prefix_attention")
        return out

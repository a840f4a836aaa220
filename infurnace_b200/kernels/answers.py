"""Several answers to one prompt: drawing tokens under top-k, top-p and min-p, the log probabilities of tokens, and attention over
pages that requests share.

:class:`AnswerKernels` is the calls (a part of the kernel set).  What is drawn, and how, is defined at the head of ``csrc/sampling.cu``, how
attention is cut into pieces at the head of ``csrc/attention_shared.cuh``.
"""
from __future__ import annotations

from ctypes import c_char_p, c_int, c_longlong

import struct

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
    shape, pitch, index = logits.shape, logits.stride(), logits.get_device()
    if code is None or len(shape) != 2 or shape[1] < 1 or (pitch[1] != 1 and shape[1] > 1):
        raise KernelError(f"{what}: logits are float32 or bfloat16 [rows, vocabulary] with unit stride along the vocabulary; got {logits.dtype} "
                          f"{tuple(shape)} of strides {pitch}")
    if index < 0:
        raise KernelError(f"{what}: logits are not on a CUDA device")
    rows, vocab = shape
    return code, rows, vocab, pitch[0] if rows > 1 else vocab, index          # (one row's pitch leads nowhere)


def _one_per_row(t, dtype, rows, index, what, name):
    """The address of a tensor with one number for each row."""
    if t.dtype is not dtype or t.shape != (rows,) or not t.is_contiguous() or t.get_device() != index:
        raise KernelError(f"{what}: {name} is {dtype} [{rows}], contiguous, on the logits' device; got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _device_of(index):
    """The device that calls launch on, for the time of a call; None: it is the current one."""
    return None if torch._C._cuda_getDevice() == index else torch.cuda.device(index)


_CUT_CALL = struct.Struct("=10q4i").pack            # csrc/sampling.cu: CutPacked
_LOGPROB_CALL = struct.Struct("=6q4i").pack         # csrc/sampling.cu: LpPacked
_SHARED_CALL = struct.Struct("=15qd10i").pack       # csrc/attention_shared.cuh: Packed


class AnswerKernels:
    """Mixed into the kernel set, which gives counters and the error word."""

    _sampling = None
    sample_max_vocab = 8 * 46080      # the largest vocabulary that sample_filtered takes (csrc/sampling.cu: SURE_CLUSTER CTAs with SLICE logits each)

    def _sampling_lib(self):
        if self._sampling is None:
            lib = load_library("sampling", progress=self._progress)
            lib.ifb_sample_cut.argtypes = [c_char_p]
            lib.ifb_token_logprobs.argtypes = [c_char_p]
            self._sampling_max_vocab = int(lib.ifb_sample_cut_max_vocab())
            self._sampling = lib
        return self._sampling

    def sample_filtered(self, logits, temperature, uniform, out, top_k=None, top_p=None, min_p=None, logprobs=None):
        """A token for each row of ``logits`` (float32 or bfloat16 [rows, vocabulary]; rows may lie apart) from softmax(logits / temperature) cut by
        top-k, then top-p, then min-p, each off where it is None.  All others have one number a row: ``temperature`` (float32; 0: the
        largest logit; NaN: the row is not drawn, its outputs stay as they are), ``uniform`` (float32 in [0, 1)), ``top_k`` (int32; below 1: off), ``top_p`` (float32; from 1 on: off; at least the best
        token stays), ``min_p`` (float32; a token stays whose probability is at least this times the best one's), ``out`` (int32) and
        ``logprobs`` (float32: the drawn token's log probability under what the cuts left, 0 at temperature 0).

        Among equal logits the lower index is the better; the draw is by inverse CDF in the order of indices.  NaN counts as -inf,
        which is never drawn; of infinities each is as likely as the other.  A row without a number above -inf gives token 0 and NaN.  A
        row's token depends on that row alone, and on its weights to 2^-44 of the largest."""
        what, f32 = "sample_filtered", torch.float32
        code, rows, vocab, pitch, index = _logit_rows(logits, what)
        args = (logits.data_ptr(), _one_per_row(temperature, f32, rows, index, what, "temperature"),
                _one_per_row(uniform, f32, rows, index, what, "uniform"),
                0 if top_k is None else _one_per_row(top_k, torch.int32, rows, index, what, "top_k"),
                0 if top_p is None else _one_per_row(top_p, f32, rows, index, what, "top_p"),
                0 if min_p is None else _one_per_row(min_p, f32, rows, index, what, "min_p"),
                _one_per_row(out, torch.int32, rows, index, what, "out"),
                0 if logprobs is None else _one_per_row(logprobs, f32, rows, index, what, "logprobs"))
        lib = self._sampling or self._sampling_lib()
        if vocab > self._sampling_max_vocab:
            raise KernelError(f"sample_filtered: a vocabulary of {vocab}; at most {self._sampling_max_vocab}")
        if rows == 0:
            return out
        self.launches += 1
        call = _CUT_CALL(*args, _raw_stream(index), pitch, code, rows, vocab, 0)
        other = _device_of(index)
        if other is None:
            status = lib.ifb_sample_cut(call)
        else:
            with other:
                status = lib.ifb_sample_cut(call)
        if status:
            _status(status, what)
        return out

    def token_logprobs(self, logits, tokens, out, ranks=None):
        """The log probability of token ``tokens[r]`` under softmax(logits[r]) into ``out`` (float32), and the number of tokens that come before it by
        falling logit, equal ones by rising index, into ``ranks`` (int32).  ``logits`` float32 or bfloat16 [rows, vocabulary], rows may
        lie apart; ``tokens`` int32, one a row.  A token outside the vocabulary (padding) gives NaN and -1; a row with a NaN
        or +inf, or with no number above -inf, NaN.  Sums are float32: a row's last bits may differ with the number of rows and
        with where in memory it begins."""
        what = "token_logprobs"
        code, rows, vocab, pitch, index = _logit_rows(logits, what)
        args = (logits.data_ptr(), _one_per_row(tokens, torch.int32, rows, index, what, "tokens"), _one_per_row(out, torch.float32, rows, index, what, "out"),
                0 if ranks is None else _one_per_row(ranks, torch.int32, rows, index, what, "ranks"))
        if rows == 0:
            return out
        self.launches += 1
        lib = self._sampling or self._sampling_lib()
        call = _LOGPROB_CALL(*args, _raw_stream(index), pitch, code, rows, vocab, 0)
        other = _device_of(index)
        if other is None:
            status = lib.ifb_token_logprobs(call)
        else:
            with other:
                status = lib.ifb_token_logprobs(call)
        if status:
            _status(status, what)
        return out

    # ------------------------------------------------------------------ attention over shared pages
    @property
    def _shared_sizes(self):
        return self.__dict__.setdefault("_shared_sizes_held", {})

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
            call.argtypes = [c_char_p]
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

        ``q`` and ``out`` are bfloat16 or float32 [tokens, heads, head_dim] (the rows of ``q`` may lie apart, those of ``out`` not, and share no memory; both begin on 16
        bytes), ``kv_pages`` [pages, 2,
        kv_heads, page_size, head_dim] of the same type.  Request r has the rows cu_q[r] .. cu_q[r + 1] - 1 and ``seq_lens[r]`` keys, these
        queries' own among them, in the pages of ``block_tables[r]``; the query at position p sees positions max(0, p - window + 1) .. p
        (``window`` 0: from 0).  Group g is the requests cu_groups[g] .. cu_groups[g + 1] - 1, the first ``shared_lens[g]`` keys of which are the same: they are
        read through the table of its first request.  (Any number of keys; beyond them each request's own table counts, also within
        a page.)  Requests of no group share nothing.  A row that sees no key becomes zero; rows behind the last request stay as they are.
        ``cu_q``, ``seq_lens``, ``block_tables``, ``cu_groups`` [groups + 1] and ``shared_lens`` [groups] are int32 on the device.  No request has more than
        ``max_q_len`` queries or ``max_seq_len`` keys.  An entry of a table that is read and is no page of the pool counts as zeros and is recorded in the
        kernels' error word.  What a row does not see may be anything, infinities and NaN too.

        Worth it where many requests share many keys.  ``paged_attention`` over tables that name the shared pages for every request gives the same (in
        bfloat16 with weights of 8 bits in place of 16), reads what is shared once for each from L2, and has one launch in place of two or three: with 32 on 8 heads
        of 128 in bfloat16 this call is the faster one from 8 answers to 8,000 shared keys, 32 to 2,000 and more than 64 to 500 on, in
        float32 from two answers to any of these (but 32 and more to 500); for requests of many queries, whose tiles are full without it, it is not.

        ``room``: None, or a uint8 tensor of at least ``shared_prefix_room`` bytes for the pieces' sums, in place of memory of the allocator's (within
        a recording: of the graph's own pool); calls that share one follow one another."""
        dtype, shape, pitch, index = q.dtype, q.shape, q.stride(), q.get_device()
        pool, block = kv_pages.shape, kv_pages.stride()
        n, heads, dim = shape if len(shape) == 3 else (0, 0, 0)
        if dtype not in _CODES or out.dtype is not dtype or out.shape != shape or kv_pages.dtype is not dtype or len(pool) != 5 or pool[1] != 2 \
                or pool[4] != dim or pool[0] < 1 or pool[2] < 1 or pool[3] < 1 or heads % pool[2] or heads == 0:
            raise KernelError(f"shared_prefix_attention: q and out are bfloat16 or float32 [tokens, heads, head_dim] and kv_pages [pages, 2, kv_heads, page_size, "
                              f"head_dim] of one type, heads a multiple of kv_heads; got {dtype} {tuple(shape)}, {out.dtype} {tuple(out.shape)} and "
                              f"{kv_pages.dtype} {tuple(pool)}")
        pages, _, kv_heads, page_size, _ = pool
        group = heads // kv_heads
        if dim % 16 or not 16 <= dim <= 256 or group > 64:
            raise KernelError(f"shared_prefix_attention: head_dim is a multiple of 16 up to 256, with up to 64 query heads for a key head; got {dim} and {group}")
        if pitch[2] != 1 or (heads > 1 and pitch[1] != dim) or not out.is_contiguous():
            raise KernelError("shared_prefix_attention: the heads of a query lie one after the other, and out is contiguous")
        inner = page_size * dim
        page_stride = block[0] if pages > 1 else 2 * kv_heads * inner
        if block[4] != 1 or (page_size > 1 and block[3] != dim) or (kv_heads > 1 and block[2] != inner) or block[1] != kv_heads * inner \
                or page_stride < 2 * kv_heads * inner:
            raise KernelError("shared_prefix_attention: the numbers of a page lie one after the other")
        r, groups = seq_lens.numel(), shared_lens.numel()
        for t, count in ((cu_q, r + 1), (seq_lens, r), (cu_groups, groups + 1), (shared_lens, groups)):
            if t.dtype is not torch.int32 or t.dim() != 1 or t.numel() != count or not t.is_contiguous() or t.get_device() != index:
                raise KernelError(f"shared_prefix_attention: cu_q [requests + 1], seq_lens [requests], cu_groups [groups + 1] and shared_lens [groups] are int32, "
                                  f"contiguous, on q's device; got {t.dtype} {tuple(t.shape)} on {t.device} for {count}")
        table, table_pitch = block_tables.shape, block_tables.stride()
        if block_tables.dtype is not torch.int32 or len(table) != 2 or table[0] < r or (table[1] > 1 and table_pitch[1] != 1):
            raise KernelError("shared_prefix_attention: block_tables is int32 [requests, pages] with unit stride along pages")
        if index < 0 or kv_pages.get_device() != index or out.get_device() != index or block_tables.get_device() != index:
            raise KernelError("shared_prefix_attention: all tensors are on one CUDA device")
        q_row = pitch[0] if n > 1 else heads * dim
        lines = 4 if dtype is torch.float32 else 8          # elements of 16 bytes
        if q.data_ptr() % 16 or kv_pages.data_ptr() % 16 or out.data_ptr() % 16 or q_row % lines or page_stride % lines:
            raise KernelError("shared_prefix_attention: q's rows, the pages and out begin on 16 bytes")
        if window < 0 or max_q_len < 1 or max_seq_len < 0:
            raise KernelError("shared_prefix_attention: window and max_seq_len are not negative, max_q_len is positive")
        if table[1] * page_size < max_seq_len:
            raise KernelError(f"shared_prefix_attention: block tables of {table[1]} pages do not hold {max_seq_len} keys")
        if r + groups > (2048 if dim <= 128 else 512):
            raise KernelError(f"shared_prefix_attention: {r} requests and {groups} groups; at most 2,048 together (512 for heads over 128)")
        if n == 0 or r == 0:
            return out
        call, room_of = self._shared_lib(dtype, dim)
        key = (n, r, groups, kv_heads, group, dim, dtype)
        size = self._shared_sizes.get(key)
        if size is None:
            if len(self._shared_sizes) > 4096:
                self._shared_sizes.clear()
            size = self._shared_sizes[key] = self.shared_prefix_room(n, r, groups, heads, kv_heads, dim, dtype)
        if room is None:
            room = torch.empty(size, dtype=torch.uint8, device=q.device)
        elif room.dtype is not torch.uint8 or room.dim() != 1 or not room.is_contiguous() or room.numel() < size or room.data_ptr() % 256 \
                or room.get_device() != index:
            raise KernelError(f"shared_prefix_attention: a room is uint8 [{size} or more], contiguous, on 256 bytes, on the same device")
        self.launches += 3 if dtype is not torch.float32 and group <= 16 < n * group and dim <= 128 and page_size in (16, 32, 64) else 2
        self._err_armed = True
        packed = _SHARED_CALL(q.data_ptr(), kv_pages.data_ptr(), block_tables.data_ptr(), cu_q.data_ptr(), seq_lens.data_ptr(), cu_groups.data_ptr(),
                              shared_lens.data_ptr(), out.data_ptr(), room.data_ptr(), self._dev_err_at, _raw_stream(index), q_row, page_stride, pages,
                              table_pitch[0], scale, table[1], n, r, groups, heads, kv_heads, dim, page_size, window, 0)
        other = _device_of(index)
        if other is None:
            status = call(packed)
        else:
            with other:
                status = call(packed)
        if status:
            _status(status, "shared_prefix_attention")
        return out

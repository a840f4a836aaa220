"""Several answers to one prompt: drawing tokens under top-k, top-p and min-p, and the log probabilities of tokens.

:class:`AnswerKernels` is the calls (a part of the kernel set).  What is drawn, and how, is defined at the head of ``csrc/sampling.cu``.
"""
from __future__ import annotations

from ctypes import c_int, c_longlong, c_void_p

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

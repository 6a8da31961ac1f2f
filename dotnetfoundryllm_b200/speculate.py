"""Verification of drafted tokens on the device over torch tensors
(``fl_verify_device``): the acceptance tests and the draw of speculative
decoding, next to ``CudaForwardPass.sample`` for one token.  What is accepted
and drawn is stated in ``include/foundry_cuda.h``; as in ``sample``, the random
numbers are the caller's (``runtime.XoshiroRandom``).  The reference has no
speculative decoding.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct

import torch

from . import _native as N
from .paged import _cuda_tensor, _enqueue, _int32, _raw, _row_type
from .runtime import ArgumentError, check


# fl_verify_desc, as _native.FlVerifyDesc
_DESC = struct.Struct("=6iQqQq9Q")
assert _DESC.size == C.sizeof(N.FlVerifyDesc)


@functools.lru_cache(maxsize=None)
def _entry():
    return _raw("fl_verify_device", C.c_char_p, C.c_void_p)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(rows: int, n: int, vocab: int) -> int:
    need = C.c_uint64()
    check(N.cuda().fl_verify_workspace(rows, n, vocab, C.byref(need)), "fl_verify_workspace")
    return need.value


def _floats(name: str, t: torch.Tensor, n: int, device: torch.device) -> None:
    _cuda_tensor(name, t, device)
    if t.dtype != torch.float32 or tuple(t.shape) != (n,) or not t.is_contiguous():
        raise ArgumentError(f"{name} must be a contiguous float32 tensor of shape {(n,)}, not {t.dtype} {tuple(t.shape)}")


def verify_drafts(logits: torch.Tensor, row_start: torch.Tensor, draft: torch.Tensor, temperature: torch.Tensor,
                  u_accept: torch.Tensor, u_sample: torch.Tensor, draft_probs: torch.Tensor | None = None,
                  tokens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Accepts or replaces the drafted tokens of each sequence.

    logits [rows, vocab] (float32, float16 or bfloat16, rows may be strided):
    the target's, sequence b in rows row_start[b] .. row_start[b+1]-1, one row
    per drafted token and one more.  draft [rows] int32, temperature [n_seqs],
    u_accept [rows], u_sample [n_seqs] float32; draft_probs [rows, vocab]
    float32, the distributions the drafts were drawn from, or None when each
    was certain.  Returns tokens [rows] int32 (the accepted drafts, the token
    after them, then -1) and accepted [n_seqs] int32.  Entries of ``tokens``
    behind the last sequence are left as they were (undefined when new); it may
    not share memory with ``draft``."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dim() != 2:
        raise ArgumentError("logits must be a [rows, vocab] CUDA tensor")
    device = logits.device
    rows, vocab = logits.shape
    rt = _row_type("logits", logits.dtype)
    if logits.stride(1) != 1 and vocab > 1:
        raise ArgumentError("the logits of a row must be dense")
    _cuda_tensor("row_start", row_start, device)
    n = row_start.numel() - 1
    if n < 0:
        raise ArgumentError("row_start needs n_seqs + 1 entries")
    _int32("row_start", row_start, (n + 1,), device)
    _int32("draft", draft, (rows,), device)
    _floats("temperature", temperature, n, device)
    _floats("u_accept", u_accept, rows, device)
    _floats("u_sample", u_sample, n, device)
    if draft_probs is not None:
        _cuda_tensor("draft_probs", draft_probs, device)
        if draft_probs.dtype != torch.float32 or draft_probs.shape != logits.shape or (draft_probs.stride(1) != 1 and vocab > 1):
            raise ArgumentError(f"draft_probs must be a float32 tensor of shape {tuple(logits.shape)} with dense rows")
    if tokens is None:
        tokens = torch.empty(rows, dtype=torch.int32, device=device)
    else:
        _int32("tokens", tokens, (rows,), device)
    accepted = torch.empty(n, dtype=torch.int32, device=device)
    need = _workspace_bytes(rows, n, vocab)
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    d = _DESC.pack(_DESC.size, rt, rows, n, vocab, 0, logits.data_ptr(), logits.stride(0),
                   draft_probs.data_ptr() if draft_probs is not None else 0,
                   draft_probs.stride(0) if draft_probs is not None else 0, row_start.data_ptr(), draft.data_ptr(),
                   temperature.data_ptr(), u_accept.data_ptr(), u_sample.data_ptr(), tokens.data_ptr(), accepted.data_ptr(),
                   ws.data_ptr(), need)
    _enqueue(device, "fl_verify_device", _entry(), d)
    return tokens, accepted

"""Verification of drafted blocks on the GPU: which drafted tokens the target's distributions accept,
and the token that follows them.

The caller of the reference verifies greedily on the host (generate.py:614-728); this judges sampled
tokens (``sample``, ``DFlashDraftModel.set_sampling``) so that what is kept is distributed as the
target alone would draw it, whatever the draft proposes.  A speculative step of several sequences::

    ids = block ids [n]                                  # each sequence's anchor, then drafted ids
    logits = target(ids, ...)                            # [n, V], row t behind token t
    v = verify_draft(logits, ids, step.starts, torch.rand(n, device="cuda"), temperature=T,
                     draft_logits=draft_logits)          # None for a greedy draft
    kept = base + v.accepted + 1                         # rows that the caches keep
    anchors = v.next_ids                                 # the next blocks' first tokens

No call reads anything back, and every call can be captured into a HIP graph.
"""

from __future__ import annotations

import contextlib
import ctypes
from typing import NamedTuple

from . import _lib

__all__ = ["verify_draft", "Verdict"]

_NOTHING = contextlib.nullcontext()


class Verdict(NamedTuple):
    """``accepted`` [n_seq] int32: drafted tokens accepted, one after another; ``next_ids`` [n_seq]
    int32: the token drawn behind them; ``chances`` [n] fp32: with which chance each row's token is
    accepted (1 for a sequence's first row)."""

    accepted: "torch.Tensor"
    next_ids: "torch.Tensor"
    chances: "torch.Tensor"


_CODES: dict = {}


def _codes():
    if not _CODES:
        import torch
        _CODES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    return _CODES


def _logits(t, what):
    if t.dim() != 2 or t.shape[1] < 1:
        raise ValueError(f"{what} must be [n, vocab], got {tuple(t.shape)}")
    if t.dtype not in _codes():
        raise ValueError(f"{what} must be fp32, fp16 or bf16, got {t.dtype}")
    if not t.is_contiguous() and (t.stride(1) != 1 and t.shape[1] > 1 or t.stride(0) < t.shape[1]):
        t = t.contiguous()   # (the kernels read rows of values next to each other)
    return t


def _ints(t, n, what, device):
    """An int32 tensor [n] (any length if n is None) on the logits' device."""
    import torch
    if (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.dim() == 1 and t.device == device and
            t.is_contiguous() and (n is None or t.shape[0] == n)):
        return t
    if not isinstance(t, torch.Tensor):
        t = torch.as_tensor(t)
        if t.numel() == 0:
            t = t.to(torch.int32)
    if t.dtype in (torch.uint16, torch.uint32):
        t = t.to(torch.int64)
    if t.dtype not in (torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64):
        raise ValueError(f"{what} must be integers, got {t.dtype}")
    if t.dim() != 1 or (n is not None and t.shape[0] != n):
        raise ValueError(f"{what} must be [{'n' if n is None else n}], got {tuple(t.shape)}")
    if t.is_cuda and t.device != device:
        raise ValueError(f"{what} is on {t.device}, the logits on {device}")
    if t.dtype == torch.int64:   # (what 32 bits do not hold stays out of range)
        t = t.clamp(-2**31, 2**31 - 1)
    return t.to(device, torch.int32).contiguous()


def _numbers(t, n, what, device):
    """An fp32 tensor [n] on the logits' device."""
    import torch
    if (isinstance(t, torch.Tensor) and t.dtype is torch.float32 and t.dim() == 1 and t.shape[0] == n and
            t.device == device and t.is_contiguous()):
        return t
    t = torch.as_tensor(t)
    if t.dim() != 1 or t.shape[0] != n or not t.dtype.is_floating_point:
        raise ValueError(f"{what} must be [{n}] numbers, got {t.dtype} {tuple(t.shape)}")
    if t.is_cuda and t.device != device:
        raise ValueError(f"{what} is on {t.device}, the logits on {device}")
    return t


def _temps(t, n_seq, what, device):
    """(one number for all, None) or (0, a device tensor [n_seq])."""
    import torch
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 0:   # (not read back)
        if t.is_complex():
            raise ValueError(f"{what} must be a number, got {t.dtype}")
        t = t.to(torch.float32).expand(n_seq)
    if isinstance(t, torch.Tensor) and t.dim() == 1:
        t = _numbers(t, n_seq, what, device)
        if not t.is_cuda and not all(0.0 <= x <= 3.4e38 for x in t.tolist()):
            raise ValueError(f"{what} must be finite and not negative, got {t.tolist()}")
        return 0.0, t.to(device, torch.float32).contiguous()
    t = float(t)
    if not 0.0 <= t <= 3.4e38:
        raise ValueError(f"{what} must be finite and not negative, got {t}")
    return t, None


def verify_draft(target_logits, ids, starts, uniforms, temperature=1.0, draft_logits=None,
                 draft_temperature=None) -> Verdict:
    """Judge drafted blocks by given uniform numbers.

    ``target_logits`` [n, vocab] (fp32, fp16 or bf16, any row stride) are the target's logits behind
    each row's token, ``ids`` [n] the blocks: rows ``starts[s] .. starts[s + 1] - 1`` are sequence
    s's, the first of them its last verified token, the others drafted.  ``draft_logits`` [n, vocab]
    (any of the types) are the logits that the drafted tokens were drawn from (``draft(...,
    return_logits=True)``; a sequence's first row does not count), None for tokens that were chosen
    otherwise (the largest logit, a lookup).  ``temperature`` is a number, a tensor of one (no
    dimension) or a tensor [n_seq], finite and not negative, 0 for the largest logit alone;
    ``draft_temperature`` alike (default: ``temperature``).  Numbers on the GPU are not read back:
    one that is no temperature leaves its sequences' rows without a distribution (below).

    With p and q the softmax of the target's and the draft's rows (without draft logits all of q's
    weight is on the drafted token), row t's token x is accepted if ``uniforms[t] * q(x) < p(x)``,
    p of row t - 1.  ``uniforms`` [n] are independent numbers of [0, 1); a sequence's first one
    draws its next token: from max(p - q, 0) behind a rejection, from p behind a block that is
    accepted whole.  Kept tokens are then distributed as draws from the target, and for
    temperature 0 they are the target's own choices.

    A logit of -infinity masks its token.  A row that holds a NaN or +infinity, or nothing above
    -infinity, has no distribution: its token is rejected, and -1 is drawn from it.  A sequence
    without rows has 0 accepted and -1.  Rows of no sequence have any ``chances``."""
    import torch
    target_logits = _logits(target_logits, "target_logits")
    n, vocab = target_logits.shape
    dev = target_logits.device
    if dev.type != "cuda":
        raise ValueError(f"target_logits must be on a GPU, not on {dev}")
    if draft_logits is not None:
        draft_logits = _logits(draft_logits, "draft_logits")
        if draft_logits.shape != target_logits.shape or draft_logits.device != dev:
            raise ValueError("draft_logits must have the shape and device of target_logits")
    L = _lib.load()
    with _NOTHING if torch.cuda.current_device() == dev.index else torch.cuda.device(dev):
        starts = _ints(starts, None, "starts", dev)
        n_seq = starts.shape[0] - 1
        if n_seq < 1:
            raise ValueError("starts must hold at least one sequence (two numbers)")
        ids = _ints(ids, n, "ids", dev)
        uniforms = _numbers(uniforms, n, "uniforms", dev)
        if uniforms.dtype is torch.float64:   # (the nearest number below 1 stays below it)
            uniforms = uniforms.clamp(max=1.0 - 2.0 ** -24)
        uniforms = uniforms.to(dev, torch.float32).contiguous()
        temp, temps = _temps(temperature, n_seq, "temperature", dev)
        draft_temp, draft_temps = temp, temps
        if draft_temperature is not None:
            draft_temp, draft_temps = _temps(draft_temperature, n_seq, "draft_temperature", dev)
        accepted, next_ids = torch.empty((2, n_seq), dtype=torch.int32, device=dev).unbind(0)
        chances = torch.empty(n, dtype=torch.float32, device=dev)
        codes = _codes()
        if draft_logits is None:
            draft, draft_row, draft_code = None, 0, 0
        else:
            draft, draft_row, draft_code = (draft_logits.data_ptr(), draft_logits.stride(0),
                                            codes[draft_logits.dtype])
        a = _lib.DflVerify(   # (in the order of its fields: names cost 3 us)
            target_logits.data_ptr(), draft, target_logits.stride(0), draft_row,
            codes[target_logits.dtype], draft_code, n, vocab, n_seq, temp, draft_temp,
            ids.data_ptr(), starts.data_ptr(), uniforms.data_ptr(), _lib.ptr(temps),
            _lib.ptr(draft_temps), accepted.data_ptr(), next_ids.data_ptr(), chances.data_ptr())
        at = ctypes.byref(a)
        a.ws_bytes = L.dfl_verify_ws(at)
        ws = torch.empty(a.ws_bytes, dtype=torch.uint8, device=dev)
        a.ws = ws.data_ptr()
        _lib.check(L.dfl_verify(at, torch._C._cuda_getCurrentRawStream(dev.index)), "dfl_verify")
    return Verdict(accepted, next_ids, chances)

"""Key/value cache of many sequences in 4 bits: pages of one pool, 68 bytes a row, head and half
(K or V) where the draft's fp16 cache (``DFlashKVCache``) takes 256.

For programs that draft for more or longer sequences than fp16 caches of a fixed capacity hold.
A step of such a program is::

    cache = KV4Cache(n_kv_heads=8, n_pages=4096, max_seqs=64, max_len=32768, n_layers=5)
    step = cache.step(grow=new, keep=kept, max_rows=n)       # once: pages, slots, positions
    for layer in range(5):                                   # q, k, v: [n, heads, 128], roped at
        cache.append(k, v, step.slots, layer)                # step.positions
        o = cache.attend(q, step.starts, layer)              # every row sees its whole sequence

``keep`` is what the last step's rows come down to (a rejected block's rows are dropped by the
step that drafts the next one), ``grow`` the rows that follow; a finished sequence keeps 0.  All
lengths stay on the GPU: no call reads them back, and every call can be captured into a HIP graph.

A group of 32 values shares a power of two, each value is a 4-bit float (include/dflash_hip.h has
the format).  A cached row differs from its fp16 row by about a tenth of its norm: a draft's
acceptance feels it, the verified output does not.
"""

from __future__ import annotations

import contextlib
import ctypes
from typing import NamedTuple, Optional

from . import _lib

__all__ = ["KV4Cache", "KV4Step"]

_NOTHING = contextlib.nullcontext()
HEAD_DIM = 128
BLOCK_ROWS, BLOCK_BYTES = 32, 4352

# error bits of the device word (errors())
ERR_LENGTH, ERR_POOL, ERR_ROWS, ERR_SLOT, ERR_PAGE = 8, 16, 32, 64, 128


class KV4Step(NamedTuple):
    """New rows of a step: those of sequence s are starts[s] .. starts[s + 1] - 1 (int32
    [max_seqs + 1]); slots and positions (int32 [max_rows]) are -1 past the last of them."""

    starts: "torch.Tensor"
    slots: "torch.Tensor"
    positions: "torch.Tensor"


class KV4Cache:
    """Paged 4-bit cache of ``max_seqs`` sequences of up to ``max_len`` rows each, sharing
    ``n_pages`` pages of ``page`` rows (32, 64, 128 or 256), for ``n_layers`` layers with one
    block table.  Heads are 128 wide.

    State (int32 tensors on the device, updated in place by ``step``): ``lens`` [max_seqs],
    ``table`` [max_seqs, ceil(max_len / page)] (-1 past a sequence's pages), ``free`` [n_pages] and
    ``n_free`` [1] (a stack of free pages).  ``pool`` holds the codes.

    Calls enqueue work on the current stream of the cache's device; calls that use one cache's
    state from several streams are the caller's to order.  Lengths and pages that do not fit are
    found on the device: such a step changes nothing, such rows are skipped, and ``errors()``
    tells."""

    def __init__(self, n_kv_heads: int, n_pages: int, max_seqs: int, max_len: int, page: int = 64,
                 n_layers: int = 1, device=None):
        import torch
        if page not in (32, 64, 128, 256):
            raise ValueError(f"page must be 32, 64, 128 or 256 rows, got {page}")
        if n_kv_heads < 1 or n_pages < 1 or max_seqs < 1 or max_len < 1 or n_layers < 1:
            raise ValueError("n_kv_heads, n_pages, max_seqs, max_len and n_layers must be positive")
        if n_pages * page > 2**31 - 1 or max_seqs > 65536:
            raise ValueError("at most 2^31 - 1 rows in the pool and 65536 sequences")
        self.n_kv_heads, self.n_pages, self.page = int(n_kv_heads), int(n_pages), int(page)
        self.max_seqs, self.n_layers = int(max_seqs), int(n_layers)
        self.width = -(-int(max_len) // self.page)
        dev = torch.device(device if device is not None else "cuda")
        if dev.type != "cuda":
            raise ValueError(f"the cache lives on a GPU, not on {dev}")
        self._L = _lib.load()
        if dev.index is None:
            dev = torch.device(dev.type, torch.cuda.current_device())
        self.device = dev
        ints = dict(dtype=torch.int32, device=dev)
        self.pool = torch.zeros((self.n_layers, self.n_pages, self.n_kv_heads,
                                 self.page // BLOCK_ROWS, BLOCK_BYTES), dtype=torch.uint8, device=dev)
        self.lens = torch.zeros(self.max_seqs, **ints)
        self.table = torch.full((self.max_seqs, self.width), -1, **ints)
        self.free = torch.arange(self.n_pages - 1, -1, -1, **ints)   # page 0 is taken first
        self.n_free = torch.full((1,), self.n_pages, **ints)
        self._err = torch.zeros(1, **ints)
        self._scratch = self._L.dfl_kv4_step_scratch(self.max_seqs)
        # (the handle alone: torch.cuda.current_stream() makes an object of it, 2 us a call)
        self._raw_stream = torch._C._cuda_getCurrentRawStream
        self._codes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

    # ------------------------------------------------------------------ checks
    def _stream(self):
        return self._raw_stream(self.device.index)

    def _guard(self):
        """Makes the cache's device the current one, if it is not."""
        import torch
        if torch.cuda.current_device() == self.device.index:
            return _NOTHING
        return torch.cuda.device(self.device)

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} outside [0, {self.n_layers})")
        return self.pool.data_ptr() + layer * self.pool.stride(0)

    @staticmethod
    def _integers(t, what: str):
        """A tensor of integers as they are given (a list's as 64 bits)."""
        import torch
        if not isinstance(t, torch.Tensor):
            t = torch.as_tensor(t)
            if t.numel() == 0:
                t = t.to(torch.int32)
        if t.dtype in (torch.uint16, torch.uint32):
            t = t.to(torch.int64)
        if t.dtype not in (torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64):
            raise ValueError(f"{what} must be integers, got {t.dtype}")
        return t

    def _ints(self, t, n: Optional[int], what: str):
        """An int32 tensor [n] (any length if n is None) on the cache's device."""
        import torch
        if (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.dim() == 1 and
                t.device == self.device and t.is_contiguous() and (n is None or t.shape[0] == n)):
            return t
        t = self._integers(t, what)
        if t.dim() != 1 or (n is not None and t.shape[0] != n):
            raise ValueError(f"{what} must be [{'n' if n is None else n}], got {tuple(t.shape)}")
        if t.is_cuda and t.device != self.device:
            raise ValueError(f"{what} is on {t.device}, the cache on {self.device}")
        if t.dtype == torch.int64:   # (what 32 bits do not hold stays out of range)
            t = t.clamp(-2**31, 2**31 - 1)
        return t.to(self.device, torch.int32).contiguous()

    def _rows(self, t, heads: Optional[int], what: str):
        """Rows [n, heads, 128] on the cache's device with strides that the kernels read in place
        (copied otherwise)."""
        if t.dim() != 3 or t.shape[2] != HEAD_DIM or (heads is not None and t.shape[1] != heads):
            raise ValueError(f"{what} must be [n, {'heads' if heads is None else heads}, {HEAD_DIM}], "
                             f"got {tuple(t.shape)}")
        if t.device != self.device:
            raise ValueError(f"{what} is on {t.device}, the cache on {self.device}")
        if t.dtype not in self._codes:
            raise ValueError(f"{what} must be fp32, fp16 or bf16, got {t.dtype}")
        s = t.stride()
        if s[2] != 1 or s[0] % 8 or s[1] % 8 or t.data_ptr() % 16:
            import torch
            t = t.clone(memory_format=torch.contiguous_format)
        return t

    # ------------------------------------------------------------------ the operators
    def step(self, grow=None, keep=None, max_rows: Optional[int] = None) -> KV4Step:
        """Bring every sequence to ``keep[s] + grow[s]`` rows: its first ``keep[s]`` (default: all
        it has) stay, pages past them are put back, pages for ``grow[s]`` new rows (default: none)
        are taken.  ``max_rows`` is the size of the slot map (default: the sum of a ``grow`` given
        on the host); rows past the last new one get slot -1, which ``append`` skips, so a
        captured graph can use one size for all its steps.  If the lengths are out of range, the
        pages do not suffice or the new rows exceed ``max_rows``, nothing changes and there are no
        new rows (``errors()``)."""
        import torch
        if max_rows is None:
            if isinstance(grow, torch.Tensor) and grow.is_cuda:
                raise ValueError("max_rows is needed with lengths on the device")
            if grow is not None:
                grow = self._integers(grow, "grow")
            max_rows = 0 if grow is None else max(0, int(grow.sum()))
        if not 0 <= max_rows < 2**31:
            raise ValueError(f"max_rows {max_rows} out of range")
        n = self.max_seqs
        with self._guard():
            grow = None if grow is None else self._ints(grow, n, "grow")
            keep = None if keep is None else self._ints(keep, n, "keep")
            buf = torch.empty(n + 1 + 2 * max_rows + self._scratch, dtype=torch.int32,
                              device=self.device)
            starts, slots, positions, _ = buf.split_with_sizes((n + 1, max_rows, max_rows,
                                                                self._scratch))
            at = buf.data_ptr()
            _lib.check(self._L.dfl_kv4_step(
                n, self.page, self.width, self.n_pages, _lib.ptr(keep), _lib.ptr(grow),
                self.lens.data_ptr(), self.table.data_ptr(), self.free.data_ptr(),
                self.n_free.data_ptr(), max_rows, at, at + 4 * (n + 1), at + 4 * (n + 1 + max_rows),
                at + 4 * (n + 1 + 2 * max_rows), self._err.data_ptr(), self._stream()),
                "dfl_kv4_step")
        return KV4Step(starts, slots, positions)

    def append(self, k, v, slots, layer: int = 0) -> None:
        """Quantise rows ``k``, ``v`` [n, n_kv_heads, 128] (fp32, fp16 or bf16, any row and head
        strides) into ``slots`` [n].  Slot -1 skips its row; the others must differ."""
        k, v = self._rows(k, self.n_kv_heads, "k"), self._rows(v, self.n_kv_heads, "v")
        if v.dtype != k.dtype or v.shape[0] != k.shape[0]:
            raise ValueError("k and v differ in dtype or row count")
        with self._guard():
            slots = self._ints(slots, k.shape[0], "slots")
            _lib.check(self._L.dfl_kv4_append(
                k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                self._codes[k.dtype], k.shape[0], self.n_kv_heads, self.page, self.n_pages,
                slots.data_ptr(), self._layer(layer), self._err.data_ptr(), self._stream()),
                "dfl_kv4_append")

    def read(self, slots, layer: int = 0, dtype=None):
        """The values held at ``slots`` [n]: (k, v), each [n, n_kv_heads, 128] of ``dtype`` (fp32,
        fp16 or bf16; default fp16).  Zeros for slot -1."""
        import torch
        dtype = torch.float16 if dtype is None else dtype
        if dtype not in self._codes:
            raise ValueError(f"dtype must be fp32, fp16 or bf16, got {dtype}")
        with self._guard():
            slots = self._ints(slots, None, "slots")
            n = slots.shape[0]
            kv = torch.empty((2, n, self.n_kv_heads, HEAD_DIM), dtype=dtype, device=self.device)
            k, v = kv.unbind(0)
            _lib.check(self._L.dfl_kv4_read(
                slots.data_ptr(), n, self.n_kv_heads, self.page, self.n_pages, self._layer(layer),
                self._codes[dtype], k.data_ptr(), v.data_ptr(), self._err.data_ptr(),
                self._stream()), "dfl_kv4_read")
        return k, v

    def attend(self, q, starts, layer: int = 0, causal: bool = False, scale: Optional[float] = None,
               return_lse: bool = False, out=None):
        """Attention of query rows ``q`` [n, heads, 128] (fp16 or bf16; ``heads`` a multiple of
        n_kv_heads, head h reads kv head h // (heads // n_kv_heads)) over the cached rows: rows
        ``starts[s] .. starts[s + 1] - 1`` ([max_seqs + 1]) are sequence s's.  Each sees all
        ``lens[s]`` rows of its sequence (a draft block), or with ``causal`` row t of m the first
        ``lens[s] - m + t + 1`` (tokens, prompts).  ``scale`` defaults to 128^-0.5.

        Returns [n, heads, 128] (``out`` if given: contiguous, same dtype; q itself, or memory that
        does not overlap it), with ``return_lse`` also the fp32 log of the sum of exponentials
        [n, heads], by which results over different keys can be joined.  A row that sees no key
        gives zeros and -inf.  Rows that belong to no sequence are not written (what ``out`` held,
        else anything)."""
        import torch
        q = self._rows(q, None, "q")
        n, heads = q.shape[0], q.shape[1]
        if q.dtype == torch.float32:
            raise ValueError("q must be fp16 or bf16")
        if heads < 1 or heads % self.n_kv_heads:
            raise ValueError(f"{heads} query heads are no multiple of {self.n_kv_heads} kv heads")
        if out is not None and (out.shape != q.shape or out.dtype != q.dtype or
                                out.device != self.device or not out.is_contiguous()):
            raise ValueError("out must be contiguous, of q's shape, dtype and device")
        if out is not None and not (out.data_ptr() == q.data_ptr() and q.is_contiguous()):
            at, size = q.data_ptr(), q.element_size()
            past = at + size * (1 + sum((n - 1) * s for n, s in zip(q.shape, q.stride())))
            if n and out.data_ptr() < past and at < out.data_ptr() + size * out.numel():
                raise ValueError("out overlaps q (it may be q itself)")
        with self._guard():
            starts = self._ints(starts, self.max_seqs + 1, "starts")
            if out is None:
                out = torch.empty((n, heads, HEAD_DIM), dtype=q.dtype, device=self.device)
            lse = torch.empty((n, heads), dtype=torch.float32, device=self.device) if return_lse else None
            ws_bytes = self._L.dfl_kv4_attend_ws(n, heads, self.n_kv_heads, self.max_seqs)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=self.device)
            a = _lib.DflKv4Attn(   # (in the order of its fields: names cost 3 us)
                q.data_ptr(), out.data_ptr(), _lib.ptr(lse), q.stride(0), q.stride(1),
                self._codes[q.dtype], n, heads, self.n_kv_heads, self.max_seqs, bool(causal),
                HEAD_DIM ** -0.5 if scale is None else float(scale), starts.data_ptr(),
                self.lens.data_ptr(), self.table.data_ptr(), self.width, self.page, self.n_pages,
                self._layer(layer), ws.data_ptr(), ws_bytes, self._err.data_ptr())
            _lib.check(self._L.dfl_kv4_attend(ctypes.byref(a), self._stream()), "dfl_kv4_attend")
        return (out, lse) if return_lse else out

    def errors(self) -> int:
        """Error bits since the last call (waits for the device, all its streams): ERR_LENGTH a
        length out of range, ERR_POOL too few free pages, ERR_ROWS more new rows than max_rows,
        ERR_SLOT a slot outside the pool, ERR_PAGE pages, lengths or row ranges that do not fit each
        other."""
        import torch
        torch.cuda.synchronize(self.device)
        e = int(self._err.item())
        if e:
            self._err.zero_()
            torch.cuda.synchronize(self.device)   # (before the bits of a later call on any stream)
        return e

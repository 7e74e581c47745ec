"""Serving over a paged KV cache: appending rotated keys and values, attention over the pages, the pages' bookkeeping.

The reference's cache is one static tensor per layer in which all sequences stand at one position
(examples/run_qwen.py:132-147).  Here the rows of a sequence lie in pages of ``page_size`` rows that
are handed out as it grows, every sequence has a length of its own, and a step takes any number of
new tokens of each: decoding sequences, pieces of prompts and whole prompts in one batch.

``paged_append`` and ``paged_attention`` are the library's calls on torch tensors (CUDA, or host
memory under the test stand-in); ``PagedKVCache`` owns pages and makes the index tensors of a step.
Work is enqueued on the current stream of the tensors' device.
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import numpy as np
import torch

from cuda_runtime import native

_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_S2, _S3 = C.c_int64 * 2, C.c_int64 * 3


def _call(device: torch.device, what: str, name: str, *args) -> None:
    """The library's call on the current stream of ``device``, with that device current."""
    fn = getattr(native.load(), name)
    if device.type != "cuda":
        return native.check(fn(*args, 0), what)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return native.check(fn(*args, torch.cuda.current_stream(device).cuda_stream), what)
    return native.check(fn(*args, torch.cuda.current_stream(device).cuda_stream), what)


def _same(what: str, device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{what}: {name} is on {t.device}, not on {device}")


def _heads(what: str, name: str, x: torch.Tensor, dtype, tokens: int | None = None) -> None:
    if x.dim() != 3 or x.dtype != dtype or (x.shape[2] > 1 and x.stride(2) != 1) or (tokens is not None and x.shape[0] != tokens):
        raise ValueError(f"{what}: {name} must be [tokens, heads, head_dim] of {dtype} with head_dim contiguous, got {tuple(x.shape)} {x.dtype} "
                         f"strides {x.stride()}" + (f" for {tokens} tokens" if tokens is not None else ""))


def _pages(what: str, k_pages: torch.Tensor, v_pages: torch.Tensor, dtype, dim: int) -> None:
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.stride() != v_pages.stride() or k_pages.dtype != dtype or v_pages.dtype != dtype or \
            k_pages.shape[3] != dim or k_pages.stride(3) != 1:
        raise ValueError(f"{what}: pages must be [pages, heads, page_size, {dim}] of {dtype}, keys and values alike with head_dim contiguous, got "
                         f"{tuple(k_pages.shape)} {k_pages.dtype} and {tuple(v_pages.shape)} {v_pages.dtype}")


def _index(what: str, name: str, x: torch.Tensor, dtype, *shape) -> None:
    if x.dtype != dtype or tuple(x.shape) != shape or not x.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous {dtype} tensor of shape {shape}, got {tuple(x.shape)} {x.dtype}")


def paged_append(q, k, v, cos, sin, k_pages, v_pages, slots, q_out=None):
    """Rotate ``q`` and ``k`` by the tables and write ``k`` and ``v`` into rows ``slots`` of the pages; returns the rotated queries.

    ``q`` ``[N, Hq, D]`` (or None), ``k``, ``v`` ``[N, Hkv, D]``: any strides over tokens and heads (columns of a merged projection); ``cos``, ``sin``
    ``[N, D]`` in fp32 or the activation type (both None: no rotation); ``k_pages``, ``v_pages`` ``[pages, Hkv, page_size, D]``; ``slots`` int64 ``[N]``
    (page * page_size + row, negative: written nowhere).  ``q_out`` may be a dense ``q`` itself."""
    what = "paged_append"
    N, Hkv, D = k.shape if k.dim() == 3 else (0, 0, 0)
    _heads(what, "k", k, k.dtype)
    _heads(what, "v", v, k.dtype, N)
    _pages(what, k_pages, v_pages, k.dtype, D)
    if v.shape != k.shape or k_pages.shape[1] != Hkv:
        raise ValueError(f"{what}: k {tuple(k.shape)}, v {tuple(v.shape)} and pages of {k_pages.shape[1]} heads do not belong together")
    if k.dtype not in _CODES:
        raise ValueError(f"{what}: {k.dtype} is not supported")
    _index(what, "slots", slots, torch.int64, N)
    Hq, qs = 0, None
    if q is not None:
        _heads(what, "q", q, k.dtype, N)
        Hq, qs = q.shape[1], _S2(q.stride(0), q.stride(1))
        if q.shape[2] != D:
            raise ValueError(f"{what}: queries of {q.shape[2]} dims, keys of {D}")
        if q_out is None:
            q_out = torch.empty(N, Hq, D, dtype=q.dtype, device=q.device)
        elif q_out.shape != q.shape or q_out.dtype != q.dtype or not q_out.is_contiguous():
            raise ValueError(f"{what}: q_out must be a contiguous {tuple(q.shape)} tensor of {q.dtype}")
    if (cos is None) != (sin is None):
        raise ValueError(f"{what}: cos and sin come together")
    table = 0
    if cos is not None:
        _index(what, "cos", cos, cos.dtype, N, D)
        _index(what, "sin", sin, cos.dtype, N, D)
        if cos.dtype not in _CODES:
            raise ValueError(f"{what}: tables of {cos.dtype} are not supported")
        table = _CODES[cos.dtype]
    _same(what, k.device, q=q, v=v, cos=cos, sin=sin, k_pages=k_pages, v_pages=v_pages, slots=slots, q_out=q_out)
    p = lambda t: None if t is None else t.data_ptr()
    if N:
        _call(k.device, what, "b200_paged_append", p(q), k.data_ptr(), v.data_ptr(), p(cos), p(sin), p(q_out), k_pages.data_ptr(), v_pages.data_ptr(),
              slots.data_ptr(), N, Hq, Hkv, D, k_pages.shape[0], k_pages.shape[2], qs, _S2(k.stride(0), k.stride(1)), _S2(v.stride(0), v.stride(1)),
              _S3(*k_pages.stride()[:3]), table, _CODES[k.dtype])
    return q_out


def paged_attention(q, k_pages, v_pages, q_start, kv_len, page_table, max_q, scale=None, window=0, out=None):
    """Attention of each sequence's new tokens over its pages; returns ``[N, Hq, D]``.

    ``q`` ``[N, Hq, D]`` (any strides over tokens and heads); ``q_start`` int32 ``[B + 1]``: sequence b has the tokens ``q_start[b]`` up to
    ``q_start[b + 1]``, at most ``max_q`` of them; ``kv_len`` int32 ``[B]``: its keys, the new tokens' among them; ``page_table`` int32 ``[B, n]``: its pages.
    A token sees the keys up to its own, with ``window`` > 0 the last ``window`` of them.  ``scale``: 1 / sqrt(D) unless given.  Rows of ``out`` behind
    the last sequence are left as they were (as they come, where ``out`` is made here)."""
    what = "paged_attention"
    _heads(what, "q", q, q.dtype)
    N, Hq, D = q.shape
    _pages(what, k_pages, v_pages, q.dtype, D)
    if q.dtype not in _CODES:
        raise ValueError(f"{what}: {q.dtype} is not supported")
    n_pages, Hkv, page, _ = k_pages.shape
    B = kv_len.shape[0] if kv_len.dim() == 1 else -1
    _index(what, "kv_len", kv_len, torch.int32, B)
    _index(what, "q_start", q_start, torch.int32, B + 1)
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != B or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError(f"{what}: page_table must be int32 [{B}, pages] with contiguous rows, got {tuple(page_table.shape)} {page_table.dtype}")
    if page_table.shape[0] > 1 and page_table.stride(0) != page_table.shape[1]:
        raise ValueError(f"{what}: page_table must be dense")
    if out is None:
        out = torch.empty(N, Hq, D, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError(f"{what}: out must be a contiguous {tuple(q.shape)} tensor of {q.dtype}")
    _same(what, q.device, k_pages=k_pages, v_pages=v_pages, q_start=q_start, kv_len=kv_len, page_table=page_table, out=out)
    if N == 0 or B == 0:
        return out
    # from the allocator on every call: a captured graph gets a workspace of its own, calls on other streams theirs
    need = native.load().b200_attn_paged_workspace_bytes(max_q, Hq, Hkv, D)
    space = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _call(q.device, what, "b200_attn_paged", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(),
          page_table.data_ptr(), B, N, max_q, Hq, Hkv, D, n_pages, page, page_table.shape[1], _S2(q.stride(0), q.stride(1)), _S3(*k_pages.stride()[:3]),
          window, D ** -0.5 if scale is None else scale, _CODES[q.dtype], space.data_ptr() if need else None, need)
    return out


@dataclass
class PagedStep:
    """The index tensors of one step (the same for all layers) and what the host knows of it."""

    seqs: list[int]
    max_q: int
    n_tokens: int
    q_start: torch.Tensor     # int32 [B + 1]
    kv_len: torch.Tensor      # int32 [B], new tokens included
    page_table: torch.Tensor  # int32 [B, pages]
    slots: torch.Tensor       # int64 [n_tokens]
    positions: torch.Tensor   # int64 [n_tokens], for the rotary tables
    last: torch.Tensor        # int64 [B], each sequence's last token of the step


class PagedKVCache:
    """Pages of keys and values for the layers of a model, shared by sequences that come and go."""

    def __init__(self, num_pages: int, page_size: int, num_layers: int, num_kv_heads: int, head_dim: int = 128, dtype: torch.dtype = torch.bfloat16,
                 device_id: int = 0):
        if num_pages < 1 or page_size < 16 or page_size % 16 or num_layers < 1 or num_kv_heads < 1 or head_dim not in (64, 128) or \
                dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"PagedKVCache: {num_pages} pages of {page_size} rows (a multiple of 16), {num_layers} layers, {num_kv_heads} heads of {head_dim} "
                             f"(64 or 128) in {dtype} (16 bits) cannot be")
        self.device = torch.device(native.device_string(device_id))
        self.page_size, self.num_pages = page_size, num_pages
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        self.k = [torch.empty(shape, dtype=dtype, device=self.device) for _ in range(num_layers)]
        self.v = [torch.empty(shape, dtype=dtype, device=self.device) for _ in range(num_layers)]
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._length: dict[int, int] = {}
        self._next = 0

    def open(self) -> int:
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._length[seq] = [], 0
        return seq

    def close(self, seq: int) -> None:
        """Give a sequence's pages back."""
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._length[seq]

    def length(self, seq: int) -> int:
        return self._length[seq]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def step(self, seqs: list[int], new_tokens: list[int]) -> PagedStep:
        """Makes room for ``new_tokens[i]`` more rows of sequence ``seqs[i]`` and returns the step's index tensors.  A step that does not fit
        raises ``RuntimeError`` and changes nothing."""
        if len(seqs) != len(new_tokens) or not seqs or len(set(seqs)) != len(seqs) or min(new_tokens) < 1:
            raise ValueError("PagedKVCache.step: one number of new tokens, at least 1, for each of some different sequences")
        if unknown := [s for s in seqs if s not in self._pages]:
            raise ValueError(f"PagedKVCache.step: no such sequence: {unknown}")
        P = self.page_size
        lengths = [self._length[s] + t for s, t in zip(seqs, new_tokens)]
        more = [-(-n // P) - len(self._pages[s]) for s, n in zip(seqs, lengths)]
        if sum(more) > len(self._free):
            raise RuntimeError(f"the KV cache has {len(self._free)} free pages of {self.num_pages}; the step needs {sum(more)}")
        for s, n, m in zip(seqs, lengths, more):
            self._pages[s].extend(self._free.pop() for _ in range(m))
            self._length[s] = n
        table = np.zeros((len(seqs), max(len(self._pages[s]) for s in seqs)), np.int32)
        for row, s in zip(table, seqs):
            row[:len(self._pages[s])] = self._pages[s]
        start = np.concatenate([[0], np.cumsum(new_tokens)])
        pos = np.concatenate([np.arange(n - t, n, dtype=np.int64) for n, t in zip(lengths, new_tokens)])
        owner = np.repeat(np.arange(len(seqs)), new_tokens)
        slots = table[owner, pos // P].astype(np.int64) * P + pos % P
        up = lambda a, dt: torch.from_numpy(np.ascontiguousarray(a, dtype=dt)).to(self.device)
        return PagedStep(list(seqs), max(new_tokens), int(start[-1]), up(start, np.int32), up(lengths, np.int32), up(table, np.int32), up(slots, np.int64),
                         up(pos, np.int64), up(start[1:] - 1, np.int64))

    def append(self, layer: int, step: PagedStep, q, k, v, cos, sin, q_out=None):
        """``paged_append`` into the pages of ``layer``; returns the rotated queries."""
        return paged_append(q, k, v, cos, sin, self.k[layer], self.v[layer], step.slots, q_out)

    def attend(self, layer: int, step: PagedStep, q, scale=None, window=0, out=None):
        """``paged_attention`` over the pages of ``layer``."""
        return paged_attention(q, self.k[layer], self.v[layer], step.q_start, step.kv_len, step.page_table, step.max_q, scale, window, out)

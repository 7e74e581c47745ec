"""Serving over a paged KV cache: appending rotated keys and values, attention over the pages, the pages' bookkeeping.

The reference's cache is one static tensor per layer in which all sequences stand at one position
(examples/run_qwen.py:132-147).  Here the rows of a sequence lie in pages of ``page_size`` rows that
are handed out as it grows, every sequence has a length of its own, and a step takes any number of
new tokens of each: decoding sequences, pieces of prompts and whole prompts in one batch.

``paged_append`` and ``paged_attention`` are the library's calls on torch tensors (CUDA, or host
memory under the test stand-in); ``PagedKVCache`` owns pages and makes the index tensors of a step.
Work is enqueued on the current stream of the tensors' device.  For serving: no gradients are recorded.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np
import torch

from cuda_runtime import native


def _failed(what: str, rc: int, needs: str, **tensors):
    """The call was not made (rc 1: the tensors do not fit) or refused by the library."""
    if rc != 1:
        native.check(rc, what)
    raise ValueError(f"{what}: {needs}; got " + ", ".join(
        f"{n} {tuple(t.shape)} {str(t.dtype)[6:]} strides {t.stride()} on {t.device}" if isinstance(t, torch.Tensor) else f"{n} {t}" for n, t in tensors.items()))


def paged_append(q, k, v, cos, sin, k_pages, v_pages, slots, q_out=None):
    """Rotate ``q`` and ``k`` by the tables and write ``k`` and ``v`` into rows ``slots`` of the pages; returns the rotated queries.

    ``q`` ``[N, Hq, D]`` (or None), ``k``, ``v`` ``[N, Hkv, D]``: any strides over tokens and heads (columns of a merged projection); ``cos``, ``sin``
    ``[N, D]`` in fp32 or the activation type (both None: no rotation); ``k_pages``, ``v_pages`` ``[pages, Hkv, page_size, D]``; ``slots`` int64 ``[N]``
    (page * page_size + row, negative: written nowhere).  ``q_out`` may be a dense ``q`` itself."""
    out = native.torch_calls().paged_append(native.entry("b200_paged_append"), q, k, v, cos, sin, k_pages, v_pages, slots, q_out)
    if out.__class__ is int:
        _failed("paged_append", out, "q [N, Hq, D] or None, k and v [N, Hkv, D] of one type with contiguous rows, cos and sin dense [N, D] in fp32 or that type "
                "or both None, k_pages and v_pages alike [pages, Hkv, page_size, D], slots dense int64 [N], q_out dense like q, all on one CUDA device",
                q=q, k=k, v=v, cos=cos, sin=sin, k_pages=k_pages, v_pages=v_pages, slots=slots, q_out=q_out)
    return out


def paged_attention(q, k_pages, v_pages, q_start, kv_len, page_table, max_q, scale=None, window=0, out=None):
    """Attention of each sequence's new tokens over its pages; returns ``[N, Hq, D]``.

    ``q`` ``[N, Hq, D]`` (any strides over tokens and heads); ``q_start`` int32 ``[B + 1]``: sequence b has the tokens ``q_start[b]`` up to
    ``q_start[b + 1]``, at most ``max_q`` of them (it chooses the kernel: with a bound that is too small the call is right, but slower);
    ``kv_len`` int32 ``[B]``: its keys, the new tokens' among them; ``page_table`` int32 ``[B, n]``: its pages.
    A token sees the keys up to its own, with ``window`` > 0 the last ``window`` of them.  ``scale``: 1 / sqrt(D) unless given.  Rows of ``out`` behind
    the last sequence are left as they were (as they come, where ``out`` is made here)."""
    got = native.torch_calls().paged_attention(native.entry("b200_attn_paged"), native.entry("b200_attn_paged_workspace_bytes"), q, k_pages, v_pages, q_start, kv_len,
                                               page_table, max_q, math.nan if scale is None else scale, window, out)
    if got.__class__ is int:
        _failed("paged_attention", got, "q [N, Hq, D] with contiguous rows, k_pages and v_pages alike [pages, Hkv, page_size, D] of its type, q_start [B + 1], kv_len "
                "[B] and page_table [B, n] dense int32, out dense like q, all on one CUDA device", q=q, k_pages=k_pages, v_pages=v_pages, q_start=q_start,
                kv_len=kv_len, page_table=page_table, out=out)
    return got


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

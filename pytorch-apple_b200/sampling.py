"""Drawing tokens from logits: temperature, top-k, top-p, min-p.

The reference generates greedily on the host (benchmarks/benchmark_qwen.py); the device arg-max stands for that, and
``sample_rows`` is the library's draw beside it.  Random numbers are the caller's; ``Sampler`` keeps a generator for them.
"""

from __future__ import annotations

import torch

from cuda_runtime import native


def sample_rows(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, out=None):
    """One token id per row of ``logits`` ``[rows, cols]`` (fp32, fp16 or bf16, any row stride); int64 ``[rows]``.

    ``uniform`` fp32 ``[rows]`` in [0, 1): the random numbers.  ``temperature`` (<= 0: the arg-max), ``top_p`` (>= 1: off), ``min_p`` (<= 0: off) fp32
    and ``top_k`` int32 (<= 0: off), each ``[rows]`` or None.  Filters apply in the order top-k, top-p (of what top-k leaves), min-p (relative to the
    likeliest token); the draw goes through what is kept in the order of the token ids.  Enqueued on the current stream of the logits' device."""
    got = native.torch_calls().sample_rows(native.entry("b200_sample_rows"), logits, uniform, temperature, top_k, top_p, min_p, out)
    if got.__class__ is int:
        if got != 1:
            native.check(got, "sample_rows")
        raise ValueError("sample_rows: logits [rows, cols] of a float type with contiguous columns; uniform and, where given, temperature, top_p, min_p dense fp32 and "
                         "top_k dense int32 [rows]; out dense int64 [rows]; all on one CUDA device; got " +
                         ", ".join(f"{n} {tuple(t.shape)} {t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else f"{n} {t}" for n, t in
                                   (("logits", logits), ("uniform", uniform), ("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p), ("out", out))))
    return got


class Sampler:
    """Settings of the draw, for all rows alike or one number per row (as they are when the sampler is made), and the generators of its
    random numbers, one per device.  For calls that are captured into a graph take ``sample_rows`` and numbers of your own."""

    def __init__(self, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, seed: int = 0):
        self.settings = {name: torch.as_tensor(value).detach().to("cpu", dtype, copy=True) for name, value, dtype in (
            ("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32))}
        self.seed = seed
        self._generators: dict[torch.device, torch.Generator] = {}
        self._on: dict[tuple, dict] = {}
        self._last: tuple = (None, {})   # the rows that were drawn for last, and their settings

    def _rows(self, rows: int, device) -> dict:
        last = self._last   # (one thread's own: another may be drawing for another batch)
        if last[0] != (rows, device):
            for name, t in self.settings.items():
                if t.dim() > 1 or (t.dim() == 1 and t.shape[0] != rows):
                    raise ValueError(f"Sampler: {name} must be one number or one for each of the {rows} rows, got shape {tuple(t.shape)}")
            # Kept for the next power of two and cut: a batch that grows and shrinks leaves no more than twice the largest behind.  (Nothing is given
            # back, so no stream can still be reading what another one is given.)
            room = rows if any(t.dim() for t in self.settings.values()) else 1 << max(rows - 1, 0).bit_length()
            if (room, device) not in self._on:
                self._on[room, device] = {name: t.expand(room).contiguous().to(device) for name, t in self.settings.items()}
            last = self._last = (rows, device), {name: t[:rows] for name, t in self._on[room, device].items()}
        return last[1]

    def __call__(self, logits):
        """Token ids ``[rows]`` for logits ``[rows, cols]``."""
        if logits.device not in self._generators:
            self._generators[logits.device] = torch.Generator(device=logits.device).manual_seed(self.seed)
        uniform = torch.rand(logits.shape[0], generator=self._generators[logits.device], device=logits.device)
        return sample_rows(logits, uniform, **self._rows(logits.shape[0], logits.device))

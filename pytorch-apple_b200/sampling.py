"""Drawing tokens from logits: temperature, top-k, top-p, min-p.

The reference generates greedily on the host (benchmarks/benchmark_qwen.py); the device arg-max stands for that, and
``sample_rows`` is the library's draw beside it.  Random numbers are the caller's; ``Sampler`` keeps a generator for them.
"""

from __future__ import annotations

import torch

from cuda_runtime import native

_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def sample_rows(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, out=None):
    """One token id per row of ``logits`` ``[rows, cols]`` (fp32, fp16 or bf16, any row stride); int64 ``[rows]``.

    ``uniform`` fp32 ``[rows]`` in [0, 1): the random numbers.  ``temperature`` (<= 0: the arg-max), ``top_p`` (>= 1: off), ``min_p`` (<= 0: off) fp32
    and ``top_k`` int32 (<= 0: off), each ``[rows]`` or None.  Filters apply in the order top-k, top-p (of what top-k leaves), min-p (relative to the
    likeliest token); the draw goes through what is kept in the order of the token ids.  Enqueued on the current stream of the logits' device."""
    if logits.dim() != 2 or logits.dtype not in _CODES or (logits.shape[1] > 1 and logits.stride(1) != 1) or logits.shape[1] < 1:
        raise ValueError(f"sample_rows: logits must be [rows, cols] of a float type with contiguous columns, got {tuple(logits.shape)} {logits.dtype} "
                         f"strides {logits.stride()}")
    rows, cols = logits.shape
    given = {"uniform": (uniform, torch.float32), "temperature": (temperature, torch.float32), "top_k": (top_k, torch.int32),
             "top_p": (top_p, torch.float32), "min_p": (min_p, torch.float32)}
    if uniform is None:
        raise ValueError("sample_rows: uniform is needed")
    for name, (t, dtype) in given.items():
        if t is not None and (t.dtype != dtype or t.dim() != 1 or t.shape[0] != rows or not t.is_contiguous() or t.device != logits.device):
            raise ValueError(f"sample_rows: {name} must be a contiguous {dtype} tensor of {rows} numbers on {logits.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    elif out.dtype != torch.int64 or tuple(out.shape) != (rows,) or not out.is_contiguous() or out.device != logits.device:
        raise ValueError(f"sample_rows: out must be a contiguous int64 tensor of {rows} on {logits.device}")
    if rows == 0:
        return out
    p = lambda t: None if t is None else t.data_ptr()
    args = (logits.data_ptr(), out.data_ptr(), rows, cols, logits.stride(0), p(temperature), p(top_k), p(top_p), p(min_p), p(uniform), _CODES[logits.dtype])
    lib, dev = native.load(), logits.device
    if dev.type != "cuda":
        native.check(lib.b200_sample_rows(*args, 0), "sample_rows")
    elif dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            native.check(lib.b200_sample_rows(*args, torch.cuda.current_stream(dev).cuda_stream), "sample_rows")
    else:
        native.check(lib.b200_sample_rows(*args, torch.cuda.current_stream(dev).cuda_stream), "sample_rows")
    return out


class Sampler:
    """Settings of the draw, for all rows alike or one number per row, and the generator of its random numbers."""

    def __init__(self, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, seed: int = 0):
        self.settings = {"temperature": (temperature, torch.float32), "top_k": (top_k, torch.int32), "top_p": (top_p, torch.float32),
                         "min_p": (min_p, torch.float32)}
        self.seed = seed
        self._generator = None
        self._on: dict[tuple, dict] = {}

    def _rows(self, rows: int, device) -> dict:
        key = (rows, device)
        if key not in self._on:
            made = {}
            for name, (value, dtype) in self.settings.items():
                t = torch.as_tensor(value, dtype=dtype)
                if t.dim() > 1 or (t.dim() == 1 and t.shape[0] != rows):
                    raise ValueError(f"Sampler: {name} must be one number or one for each of the {rows} rows, got shape {tuple(t.shape)}")
                made[name] = t.expand(rows).contiguous().to(device)
            self._on[key] = made
        return self._on[key]

    def __call__(self, logits):
        """Token ids ``[rows]`` for logits ``[rows, cols]``."""
        if self._generator is None or self._generator.device != logits.device:
            self._generator = torch.Generator(device=logits.device).manual_seed(self.seed)
        uniform = torch.rand(logits.shape[0], generator=self._generator, device=logits.device)
        return sample_rows(logits, uniform, **self._rows(logits.shape[0], logits.device))

"""Operators for drawing several readings of one window, on torch CUDA tensors.

``BatchDecoder`` decodes each slot greedily, as the reference does.  These are
the two operators that several sampled readings of the same audio need next to
it, in the engine's own kernels (``libs2r.so``):

* ``sample`` draws a token per row with temperature, top-k, top-p and min-p
  under the grammar mask and the mode bias, from uniforms the caller gives,
  and returns its log-probability, to rank readings by (``s2r_sample``).

Every call is asynchronous on the current stream of its tensors' device, which
need not be the current device.  Arguments are checked on the host and raise
``ValueError``; there is no CPU path.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.S2R_F32, torch.bfloat16: _lib.S2R_BF16, torch.float16: _lib.S2R_F16}


def _on_device(name: str, t: torch.Tensor, device: torch.device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return t


def _call(fn, args, device: torch.device) -> None:
    """Run a C entry point with the tensors' device current and its current stream."""

    stream = C.c_void_p(torch.cuda.current_stream(device).cuda_stream)
    if torch.cuda.current_device() == device.index:
        _lib.check(fn(C.byref(args), stream))
    else:
        with torch.cuda.device(device):
            _lib.check(fn(C.byref(args), stream))


def _vector(name: str, t: torch.Tensor, rows: int, dtype: torch.dtype, device: torch.device) -> int:
    _on_device(name, t, device)
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != rows or (rows > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {rows} values")
    return t.data_ptr()


def _matrix(name: str, t: torch.Tensor, rows: int, cols: int, device: torch.device) -> tuple[int, int]:
    """Address and row stride (elements) of a [rows, cols] tensor whose rows are contiguous."""

    _on_device(name, t, device)
    if t.dim() == 1:
        t = t.unsqueeze(0).expand(rows, -1)
    if t.dim() != 2 or tuple(t.shape) != (rows, cols) or (cols > 1 and t.stride(1) != 1):
        raise ValueError(f"{name} must be [{rows}, {cols}] with contiguous rows")
    return t.data_ptr(), t.stride(0) if rows > 1 else 0


def sample(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
           bias: torch.Tensor | None = None, allowed: torch.Tensor | None = None, out: torch.Tensor | None = None,
           logprobs: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Draw one token per row; returns ``(tokens [rows] int64, logprobs [rows] float32)``.

    ``logits`` ``[rows, vocab]`` (float32, bfloat16 or float16; rows may be
    strided), ``uniforms`` ``[rows]`` float32 in [0, 1).  ``temperature``,
    ``top_k``, ``top_p`` and ``min_p`` are numbers or per-row tensors (float32;
    int32 for ``top_k``); 0, 0, 1 and 0 mean greedy, no limit, no limit, no
    limit.  ``bias`` ``[vocab]`` float32 is added to every row (the mode bias),
    ``allowed`` ``[rows, vocab]`` or ``[vocab]`` (uint8 or bool) is the grammar
    mask.  ``out`` and ``logprobs`` receive the results if given.

    The order of the filters, what ties and empty rows give and the definition
    of ``logprobs`` are in ``include/s2r.h`` (``s2r_sample``).  A row with
    nothing allowed gives token 0 and ``-inf``.
    """

    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dim() != 2:
        raise ValueError("logits must be a [rows, vocab] CUDA tensor")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits of {logits.dtype}: float32, bfloat16 or float16 expected")
    lib = _lib.load()
    device = logits.device
    rows, vocab = logits.shape
    if rows < 1 or vocab < 1:
        raise ValueError("logits must have at least one row and one token")
    a = _lib.SampleArgs(logits_dtype=_DTYPES[logits.dtype], rows=rows, vocab=vocab)
    a.logits, a.logits_stride = _matrix("logits", logits, rows, vocab, device)
    a.uniforms = _vector("uniforms", uniforms, rows, torch.float32, device)
    if bias is not None:
        a.bias = _vector("bias", bias, vocab, torch.float32, device)
    if allowed is not None:
        if not isinstance(allowed, torch.Tensor) or allowed.dtype not in (torch.uint8, torch.bool):
            raise ValueError("allowed must be a uint8 or bool tensor")
        a.allowed, a.allowed_stride = _matrix("allowed", allowed, rows, vocab, device)
    for name, value, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                               ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if isinstance(value, torch.Tensor):
            setattr(a, name, _vector(name, value, rows, dtype, device))
        elif dtype == torch.int32:
            a.top_k_all = max(-1, min(int(value), 2**31 - 1))
        else:
            setattr(a, name + "_all", value)
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=device)
    if logprobs is None:
        logprobs = torch.empty(rows, dtype=torch.float32, device=device)
    a.tokens = _vector("out", out, rows, torch.int64, device)
    a.logprobs = _vector("logprobs", logprobs, rows, torch.float32, device)
    _call(lib.s2r_sample, a, device)
    return out, logprobs

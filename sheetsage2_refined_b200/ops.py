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
_MASKS = (torch.uint8, torch.bool)


def _bad(name: str, t, dtype, shape, device) -> ValueError:
    """The error for an argument that is not a ``dtype`` tensor of ``shape`` on ``device`` with contiguous rows."""

    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        return ValueError(f"{name} must be a CUDA tensor")
    if t.device != device:
        return ValueError(f"{name} is on {t.device}, expected {device}")
    return ValueError(f"{name} must be a {dtype} tensor of shape {list(shape)} with contiguous rows, "
                      f"not {t.dtype} {list(t.shape)} with strides {t.stride()}")


def _vector(name: str, t: torch.Tensor, n: int, dtype: torch.dtype, device: torch.device) -> int:
    """Address of a contiguous ``[n]`` tensor."""

    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device or t.shape != (n,) or not (
            n == 1 or t.stride(0) == 1):
        raise _bad(name, t, dtype, (n,), device)
    return t.data_ptr()


def _call(fn, args, device: torch.device) -> None:
    """Run a C entry point with the tensors' device current and its current stream."""

    index = device.index
    if torch.cuda.current_device() == index:
        code = fn(C.byref(args), torch.cuda.current_stream(index).cuda_stream)
    else:
        with torch.cuda.device(index):
            code = fn(C.byref(args), torch.cuda.current_stream(index).cuda_stream)
    if code:
        _lib.check(code)


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
    device = logits.device
    rows, vocab = logits.shape
    if rows < 1 or vocab < 1:
        raise ValueError("logits must have at least one row and one token")
    row_stride, stride = logits.stride()
    if vocab > 1 and stride != 1:
        raise _bad("logits", logits, logits.dtype, (rows, vocab), device)
    mask = mask_stride = None
    if allowed is not None:
        if not isinstance(allowed, torch.Tensor) or allowed.dtype not in _MASKS or allowed.device != device or (
                allowed.shape not in ((rows, vocab), (vocab,))) or (vocab > 1 and allowed.stride(-1) != 1):
            raise _bad("allowed", allowed, "uint8 or bool", (rows, vocab), device)
        mask, mask_stride = allowed.data_ptr(), allowed.stride(0) if allowed.dim() == 2 else 0
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=device)
    if logprobs is None:
        logprobs = torch.empty(rows, dtype=torch.float32, device=device)
    each, values = [], []
    for name, value, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                               ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if isinstance(value, torch.Tensor):
            each.append(_vector(name, value, rows, dtype, device))
            values.append(0)
        else:
            each.append(None)
            values.append(value if name != "top_k" else max(-1, min(int(value), 2**31 - 1)))
    lib = _lib.load()
    _call(lib.s2r_sample, _lib.SampleArgs(
        logits.data_ptr(), row_stride if rows > 1 else 0, _DTYPES[logits.dtype], rows, vocab,
        None if bias is None else _vector("bias", bias, vocab, torch.float32, device), mask, mask_stride or 0,
        _vector("uniforms", uniforms, rows, torch.float32, device), *each, *values,
        _vector("out", out, rows, torch.int64, device), _vector("logprobs", logprobs, rows, torch.float32, device)),
        device)
    return out, logprobs

"""Operators for drawing several readings of one window, on torch CUDA tensors.

``BatchDecoder`` decodes each slot greedily, as the reference does.  These are
the two operators that several sampled readings of the same audio need next to
it, in the engine's own kernels (``libs2r.so``):

* ``sample`` draws a token per row with temperature, top-k, top-p and min-p
  under the grammar mask and the mode bias, from uniforms the caller gives,
  and returns its log-probability, to rank readings by (``s2r_sample``);
* ``shared_attention`` lets many rows attend over one K/V that is read once for
  all of them (a window's cross K/V, a common prompt's K/V) and over each row's
  own pages (``s2r_shared_attention``).

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
_NO_OWN = (None, None, 0, 0, None, 0, None)
_workspace: dict = {}  # bytes by (device, sizes)


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


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the same without a Stream object, where this torch has it (a few microseconds a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


def _call(fn, args, device: torch.device) -> None:
    """Run a C entry point with the tensors' device current and its current stream."""

    index = device.index
    if torch.cuda.current_device() == index:
        code = fn(C.byref(args), _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = fn(C.byref(args), _raw_stream(index))
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
    each_t = each_k = each_p = each_m = None  # per-row parameters
    if isinstance(temperature, torch.Tensor):
        each_t, temperature = _vector("temperature", temperature, rows, torch.float32, device), 0.0
    if isinstance(top_k, torch.Tensor):
        each_k, top_k = _vector("top_k", top_k, rows, torch.int32, device), 0
    if isinstance(top_p, torch.Tensor):
        each_p, top_p = _vector("top_p", top_p, rows, torch.float32, device), 0.0
    if isinstance(min_p, torch.Tensor):
        each_m, min_p = _vector("min_p", min_p, rows, torch.float32, device), 0.0
    lib = _lib.load()
    _call(lib.s2r_sample, _lib.SampleArgs(
        logits.data_ptr(), row_stride if rows > 1 else 0, _DTYPES[logits.dtype], rows, vocab,
        None if bias is None else _vector("bias", bias, vocab, torch.float32, device), mask, mask_stride or 0,
        _vector("uniforms", uniforms, rows, torch.float32, device), each_t, each_k, each_p, each_m, temperature,
        max(-1, min(int(top_k), 2**31 - 1)), top_p, min_p,
        _vector("out", out, rows, torch.int64, device), _vector("logprobs", logprobs, rows, torch.float32, device)),
        device)
    return out, logprobs


def shared_attention(q: torch.Tensor, shared_k: torch.Tensor, shared_v: torch.Tensor, *,
                     own_k: torch.Tensor | None = None, own_v: torch.Tensor | None = None,
                     page_table: torch.Tensor | None = None, own_len: torch.Tensor | None = None,
                     scale: float | None = None, shared_len: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                     error: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of single query tokens over one shared K/V and each row's own pages.

    ``q`` ``[rows, heads, dim]``; ``shared_k`` / ``shared_v`` ``[tokens,
    kv_heads, dim]`` (any strides that are multiples of 8 elements: a
    ``[kv_heads, tokens, dim]`` buffer is passed transposed), bfloat16 or
    float16, ``dim`` 64 or 128, ``heads`` a multiple of ``kv_heads``.  Row r
    sees every shared token (the first ``shared_len`` of them, an int32 tensor
    of one value, if given) and then the first ``own_len[r]`` tokens of the
    pages ``page_table[r]`` names in the pools ``own_k`` / ``own_v``
    ``[pages, kv_heads, 64, dim]`` (contiguous); ``page_table`` ``[rows,
    pages]`` and ``own_len`` ``[rows]`` are int32.  ``scale`` defaults to
    ``dim ** -0.5``.

    Returns ``(out, lse)``: ``out`` like ``q`` (it may be ``q`` itself), ``lse`` ``[rows, heads]``
    float32, the log of the sum of exponentials of the scaled scores.  A row
    without keys gives 0 and ``-inf``; a row whose pages are broken gives NaN
    and sets ``error`` (an int32 tensor of one value) if given.
    """

    if not isinstance(q, torch.Tensor) or not q.is_cuda or q.dim() != 3:
        raise ValueError("q must be a [rows, heads, dim] CUDA tensor")
    dtype, device = q.dtype, q.device
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError(f"q of {dtype}: bfloat16 or float16 expected")
    shape = q.shape
    rows, heads, dim = shape
    q_row, q_head, one = q.stride()
    if one != 1:
        raise _bad("q", q, dtype, shape, device)
    shared = getattr(shared_k, "shape", ())
    for name, t in (("shared_k", shared_k), ("shared_v", shared_v)):
        if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device or t.shape != shared or (
                len(shared) != 3 or shared[2] != dim or t.stride(2) != 1):
            raise _bad(name, t, dtype, ("tokens", "kv_heads", dim), device)
    tokens, kv_heads, _ = shared
    k_token, k_head, _ = shared_k.stride()
    v_token, v_head, _ = shared_v.stride()
    own_args, pages = _NO_OWN, 0
    if own_k is not None or own_v is not None or page_table is not None or own_len is not None:
        if own_k is None or own_v is None or page_table is None or own_len is None:
            raise ValueError("own_k, own_v, page_table and own_len go together")
        pool = (own_k.shape[0] if isinstance(own_k, torch.Tensor) and own_k.dim() else 0, kv_heads,
                _lib.S2R_PAGE_TOKENS, dim)
        for name, t in (("own_k", own_k), ("own_v", own_v)):
            if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.device != device or t.shape != pool or (
                    not t.is_contiguous()):
                raise _bad(name, t, dtype, pool, device)
        if not isinstance(page_table, torch.Tensor) or page_table.dtype is not torch.int32 or (
                page_table.device != device or page_table.dim() != 2 or page_table.shape[0] != rows or (
                    page_table.shape[1] > 1 and page_table.stride(1) != 1)):
            raise _bad("page_table", page_table, torch.int32, (rows, "pages"), device)
        pages = page_table.shape[1]
        own_args = (own_k.data_ptr(), own_v.data_ptr(), pool[0], pages, page_table.data_ptr(),
                    page_table.stride(0) if rows > 1 else 0, _vector("own_len", own_len, rows, torch.int32, device))
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(shape, dtype=dtype, device=device)
    elif not isinstance(out, torch.Tensor) or out.dtype is not dtype or out.device != device or (
            out.shape != shape or out.stride(2) != 1):
        raise _bad("out", out, dtype, shape, device)
    if lse is None:
        lse = torch.empty((rows, heads), dtype=torch.float32, device=device)
    elif not isinstance(lse, torch.Tensor) or lse.dtype is not torch.float32 or lse.device != device or (
            lse.shape != (rows, heads) or not lse.is_contiguous()):
        raise _bad("lse", lse, torch.float32, (rows, heads), device)
    out_row, out_head, _ = out.stride()
    args = _lib.SharedAttentionArgs(
        _DTYPES[dtype], rows, heads, kv_heads, dim, dim**-0.5 if scale is None else scale, q.data_ptr(), q_row, q_head,
        shared_k.data_ptr(), shared_v.data_ptr(), k_token, k_head, v_token, v_head, tokens,
        None if shared_len is None else _vector("shared_len", shared_len, 1, torch.int32, device), *own_args,
        out.data_ptr(), out_row, out_head, lse.data_ptr(), None, 0,
        None if error is None else _vector("error", error, 1, torch.int32, device))
    lib = _lib.load()
    # the workspace a call needs is a function of its sizes: asked for once
    sizes = (device.index, rows, heads, kv_heads, dim, tokens, pages)
    need = _workspace.get(sizes)
    if need is None:
        count = C.c_int64()
        with torch.cuda.device(device):
            _lib.check(lib.s2r_shared_attention_workspace(C.byref(args), C.byref(count)))
        if len(_workspace) >= 4096:
            _workspace.clear()
        need = _workspace[sizes] = count.value
    if need:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), need
    _call(lib.s2r_shared_attention, args, device)
    return out, lse

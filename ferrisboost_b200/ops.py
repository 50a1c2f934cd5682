"""Operators on a model's leaves and class scores, on tensors in GPU memory.

A trained model gives each row's leaf in every tree (``predict(pred_leaf=True)``)
and, for multiclass objectives, a score for each class.  ``embed`` looks up and
sums a vector for each leaf (or categorical code), ``embed_grad`` is its
gradient for the table, ``dropout`` drops elements by a seed and their index,
and ``sample`` draws a class from a row of scores.

The functions take torch CUDA tensors (float32, float16 or bfloat16) and return
new ones, or fill ``out``.  Like torch's own operations they are enqueued on the
current stream of the tensors' device and do not wait for it; a tensor made on
another stream needs the usual ``wait_stream`` / ``record_stream``.  They can be
captured into a CUDA graph.  They do not record gradients: a training step calls
the backward operators itself (examples/leaf_head.py).  A tensor that asks for a
gradient is refused while torch records gradients (pass ``t.detach()``, or call
under ``torch.no_grad()``), and what is written to ``out`` counts as an in-place
change of it.  Wrong arguments raise ValueError before anything is enqueued.  The
kernels are ``fbgpu_embed``, ``fbgpu_embed_grad``,
``fbgpu_dropout`` and ``fbgpu_sample`` of include/fbgpu.h, which has the exact
definitions; there is no CPU path.
"""
from __future__ import annotations

import ctypes as C
from operator import index
from typing import Any

import torch

from . import _lib

__all__ = ["embed", "embed_grad", "dropout", "sample"]

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # FBGPU_F32, FBGPU_F16, FBGPU_BF16
_F32 = {torch.float32: 0}
_TOKENS = {torch.int32: 0, torch.int64: 1}                        # FBGPU_I32, FBGPU_I64


_entry = _lib.load()
_device, _stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _lost_gradient(name: str, t: torch.Tensor) -> None:
    """Refuses a tensor that requires a gradient where that would be lost without a word."""
    if torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, and no gradient is recorded here: pass it detached, or call under "
                         "torch.no_grad()")


def _type(name: str, t: Any, dims: int | None, types: dict) -> int:
    """The type code of a CUDA tensor, with its dimensions checked."""
    if isinstance(t, torch.Tensor):
        code = types.get(t.dtype)
        if code is not None and t.is_cuda and (dims is None or t.dim() == dims):
            if t.requires_grad:
                _lost_gradient(name, t)
            return code
        if not t.is_cuda:
            raise ValueError(f"{name} must be on a CUDA device, it is on {t.device}")
        if dims is not None and t.dim() != dims:
            raise ValueError(f"{name} must have {dims} dimension(s), got shape {tuple(t.shape)}")
        raise ValueError(f"{name} must be one of {', '.join(str(k) for k in types)}, got {t.dtype}")
    raise ValueError(f"{name} must be a torch tensor, got {type(t).__name__}")


def _rows(name: str, t: torch.Tensor) -> int:
    """The row stride of a 2-D tensor whose rows are contiguous."""
    row, col = t.stride()
    if col != 1 and t.shape[1] > 1:
        raise ValueError(f"{name} must have contiguous rows, its strides are {(row, col)}")
    return row


def _same_device(name: str, t: torch.Tensor, device: int) -> None:
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors are on cuda:{device}")


def _out(out: Any, shape: tuple, like: torch.Tensor) -> torch.Tensor:
    if not isinstance(out, torch.Tensor) or tuple(out.shape) != shape or out.dtype != like.dtype:
        raise ValueError(f"out must be a {like.dtype} tensor of shape {shape}")
    _same_device("out", out, like.get_device())
    if out.requires_grad:
        _lost_gradient("out", out)
    return out


def _call(device: int, f: Any, *args: Any) -> None:
    """Calls the entry point on the device, with its current stream as the last argument."""
    if device == _device():
        status = f(*args, _stream(device))
    else:
        with torch.cuda.device(device):
            status = f(*args, _stream(device))
    if status:
        message = (_entry.fbgpu_last_error(None) or b"").decode()
        raise (ValueError if status == 1 else RuntimeError)(message)


# Counts a write to a caller's tensor, so that autograd sees a change of one that it has saved.
_wrote = torch.autograd.graph.increment_version


def _token_shape(tokens: torch.Tensor) -> tuple:
    """(token code, rows, tokens per row, row stride, column stride)"""
    code = _type("tokens", tokens, None, _TOKENS)
    dims = tokens.dim()
    if dims == 1:
        return code, tokens.shape[0], 1, tokens.stride(0), 1
    if dims == 2:
        n, k = tokens.shape
        return (code, n, k, *tokens.stride())
    raise ValueError(f"tokens must have 1 or 2 dimensions, got shape {tuple(tokens.shape)}")


def _count(dim: int, k: int) -> None:
    """The entry points take 32-bit row lengths."""
    if dim >= 1 << 32 or k >= 1 << 32:
        raise ValueError(f"rows of {dim} elements and {k} tokens: both must be below 2**32")


def embed(table: torch.Tensor, tokens: torch.Tensor, *, scale: float = 1.0,
          out: torch.Tensor | None = None) -> torch.Tensor:
    """``scale`` times the sum of the table rows that each row's tokens name.

    ``table`` is vocab x dim; ``tokens`` (int32 or int64, any strides) is n, or
    n x k for k tokens a row, such as a row's leaf in each of k trees with the
    tree's first node added.  A token outside [0, vocab) stands for a missing
    value and adds nothing.  The sum is taken in float32 and rounded once.
    Returns n x dim in the table's type."""
    code = _type("table", table, 2, _TYPES)
    tcode, n, k, trow, tcol = _token_shape(tokens)
    device = table.get_device()
    _same_device("tokens", tokens, device)
    vocab, dim = table.shape
    _count(dim, k)
    given = out
    out = table.new_empty((n, dim)) if out is None else _out(out, (n, dim), table)
    _call(device, _entry.fbgpu_embed, table.data_ptr(), code, vocab, dim, _rows("table", table), tokens.data_ptr(), tcode, n,
          k, trow, tcol, scale, out.data_ptr(), _rows("out", out))
    if given is not None:
        _wrote(given)
    return out


def embed_grad(grad: torch.Tensor, tokens: torch.Tensor, vocab: int, *, scale: float = 1.0,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of ``embed`` for its table, vocab x dim in grad's type.

    ``grad`` (n x dim) is the gradient of ``embed``'s result for the same
    ``tokens`` and ``scale``.  Row v is ``scale`` times the float32 sum of
    grad[r] over the places (r, j) with token v, zero where there is none.
    The same inputs give the same bits: the places are sorted by token and no
    atomic adds are used.  n * k and vocab are at most 2**31 - 2."""
    code = _type("grad", grad, 2, _TYPES)
    tcode, n, k, trow, tcol = _token_shape(tokens)
    device = grad.get_device()
    _same_device("tokens", tokens, device)
    vocab = int(vocab)
    if vocab < 0:
        raise ValueError(f"vocab must not be negative, got {vocab}")
    if grad.shape[0] != n:
        raise ValueError(f"grad has {grad.shape[0]} rows, tokens has {n}")
    dim = grad.shape[1]
    _count(dim, k)
    given = out
    out = grad.new_empty((vocab, dim)) if out is None else _out(out, (vocab, dim), grad)
    size = _entry.fbgpu_embed_grad_workspace(n, k, vocab, dim)
    space = grad.new_empty(size, dtype=torch.uint8)
    _call(device, _entry.fbgpu_embed_grad, grad.data_ptr(), code, n, k, dim, _rows("grad", grad), tokens.data_ptr(), tcode,
          trow, tcol, vocab, scale, out.data_ptr(), _rows("out", out), space.data_ptr(), size)
    if given is not None:
        _wrote(given)
    return out


def dropout(x: torch.Tensor, p: float, seed: int, offset: int = 0, *,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """x / (1 - p) where an element is kept, else 0.

    Whether element i (in row-major order) is kept follows from ``seed`` and
    ``offset + i`` alone, not from x's strides, so no mask is stored:
    ``dropout(grad, p, seed, offset)`` is the backward pass.  Steps that must
    differ take another seed, or an offset that is further by the number of
    elements.  ``x`` has any shape if it is contiguous, else two dimensions with
    contiguous rows.  ``out=x`` works in place."""
    code = _type("x", x, None, _TYPES)
    p = float(p)
    given = out
    out = x.new_empty(x.shape) if out is None else _out(out, tuple(x.shape), x)
    if x.is_contiguous() and out.is_contiguous():
        n, dim = 1, x.numel()
        xs = os = dim
    elif x.dim() == 2:
        n, dim = x.shape
        xs, os = _rows("x", x), _rows("out", out)
    else:
        raise ValueError(f"x and out must be contiguous, or 2-D with contiguous rows; x has shape {tuple(x.shape)} "
                         f"and strides {x.stride()}")
    _call(x.get_device(), _entry.fbgpu_dropout, x.data_ptr(), code, n, dim, xs, p,
          index(seed) & 0xFFFFFFFFFFFFFFFF, index(offset) & 0xFFFFFFFFFFFFFFFF, out.data_ptr(), os)
    if given is not None:
        _wrote(given)
    return out


def _limit(name: str, value: Any, scores: torch.Tensor, dtype: torch.dtype) -> tuple:
    """(scalar, pointer) of a limit given as a number or as a tensor with a value for each row."""
    if not isinstance(value, torch.Tensor):
        return value, None
    if value.dtype != dtype or value.shape != scores.shape[:1] or not value.is_contiguous():
        raise ValueError(f"{name} must be a number or a contiguous {dtype} tensor of {scores.shape[0]} values")
    _same_device(name, value, scores.get_device())
    if value.requires_grad:
        _lost_gradient(name, value)
    return 0, value.data_ptr()


def _result(name: str, t: Any, u: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != u.shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {u.shape[0]} values")
    _same_device(name, t, u.get_device())
    if t.requires_grad:
        _lost_gradient(name, t)
    return t


def sample(scores: torch.Tensor, u: torch.Tensor, *, temperature: Any = 1.0, top_k: Any = 0, top_p: Any = 1.0,
           min_p: Any = 0.0, classes: torch.Tensor | None = None,
           probs: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Draws a class from each row of scores; returns (classes, probs).

    ``scores`` is n x K (2 <= K <= 2**20): margins or logits, in which -inf and
    NaN rule a class out.  ``u`` has a float32 random number in [0, 1) for each
    row.  The softmax of scores / ``temperature`` is limited to the ``top_k``
    largest (0: no limit), then to the shortest beginning of the falling order
    that holds ``top_p`` of their total, then to classes at least ``min_p``
    times as probable as the first; equal scores are ordered by class.  The
    class drawn (int32) is the first, by class, at which the running sum of
    what is left passes u times its total, and ``probs`` (float32) is its share.
    ``temperature`` 0 gives the first maximum.  A row with every class ruled out
    gives class -1 and share 0.  Each limit is a number or a tensor with a
    value for each row (float32; ``top_k`` int32).  Weights are whole multiples
    of 2**-40 of the first class's, so a draw does not depend on the order of
    sums; classes below that are never drawn."""
    code = _type("scores", scores, 2, _TYPES)
    n, k = scores.shape
    _type("u", u, 1, _F32)
    if u.shape[0] != n or not u.is_contiguous():
        raise ValueError(f"u must be contiguous with {n} values, got shape {tuple(u.shape)}")
    device = scores.get_device()
    _same_device("u", u, device)
    t, ts = _limit("temperature", temperature, scores, torch.float32)
    tk, tks = _limit("top_k", top_k, scores, torch.int32)
    tp, tps = _limit("top_p", top_p, scores, torch.float32)
    mp, mps = _limit("min_p", min_p, scores, torch.float32)
    if tks is None and (not 0 <= tk < 1 << 31 or tk != int(tk)):
        raise ValueError(f"top_k must be a whole number in 0..2**31 - 1, got {tk}")
    if k > 1 << 20:
        raise ValueError(f"classes must be in 2..1048576, got {k}")
    given = [t for t in (classes, probs) if t is not None]
    classes = u.new_empty(n, dtype=torch.int32) if classes is None else _result("classes", classes, u, torch.int32)
    probs = u.new_empty(n) if probs is None else _result("probs", probs, u, torch.float32)
    params = _lib.FbgpuSampleParams(t, int(tk), tp, mp, ts, tks, tps, mps)
    _call(device, _entry.fbgpu_sample, scores.data_ptr(), code, n, k, _rows("scores", scores), u.data_ptr(),
          C.byref(params), classes.data_ptr(), probs.data_ptr())
    if given:
        _wrote(given)
    return classes, probs

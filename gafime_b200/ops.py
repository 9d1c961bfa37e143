"""Operators of a linear softmax head on torch CUDA tensors: cross entropy over many classes
without keeping the logits, with its gradients, and the gradients' global norm with clipping.

They are what ``GafimeEngine``'s joint fit runs on, and the step of any head trained on the
features and interactions a selector leaves.  Everything is queued on torch's current stream of
the tensors' device; nothing waits, and calls can be captured into a CUDA graph.  Scratch memory
comes from torch's allocator.  The kernels are those of ``gafime_xent_*`` and
``gafime_grad_norm`` in libgafime_cuda.so; there is no other path.
"""
from __future__ import annotations

import array
import ctypes
import functools
import operator
from typing import NamedTuple, Optional, Sequence

import torch
from torch.autograd import forward_ad

from . import _native

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_DX, _DW, _DBIAS, _GRADIENT = 1, 2, 4, 8
# over lists of hundreds of tensors, without a Python frame for each
_numel, _pointer, _device = torch.Tensor.numel, torch.Tensor.data_ptr, torch.Tensor.get_device
_contiguous = torch.Tensor.is_contiguous
_dtype = operator.attrgetter("dtype")


def _address(values: array.array) -> int:
    return values.buffer_info()[0]


class XentGrad(NamedTuple):
    """Result of softmax_xent_grad."""

    loss: torch.Tensor                  # (n,) float32
    lse: torch.Tensor                   # (n,) float32
    dx: Optional[torch.Tensor]          # (n, d), x's type and order
    dw: Optional[torch.Tensor]          # (c, d), w's type
    dbias: Optional[torch.Tensor]       # (c,) float32


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(device: int, type_id: int, x_off: int, xr: int, xk: int, w_off: int, wr: int, wk: int,
                     n: int, d: int, c: int, want: int) -> int:
    """Of sizes, strides and alignments alone (x_off, w_off: addresses modulo 16)."""
    out = ctypes.c_size_t(0)
    lib = _native.load(require_gpu=False)
    with torch.cuda.device(device):      # the plan follows from the device's SM count
        _native.check("gafime_xent_workspace", lib.gafime_xent_workspace(
            type_id, 256 + x_off, xr, xk, 256 + w_off, wr, wk, n, d, c, want, ctypes.byref(out)))
    return out.value


def _check(x, w, labels, bias, row_weight):
    if not isinstance(x, torch.Tensor) or not isinstance(w, torch.Tensor) or not isinstance(labels, torch.Tensor):
        raise TypeError("x, w and labels must be torch tensors")
    if x.dim() != 2 or w.dim() != 2 or labels.dim() != 1:
        raise ValueError("x must be (n, d), w (c, d) and labels (n,)")
    n, d = x.shape
    c = w.shape[0]
    if w.shape[1] != d or labels.shape[0] != n:
        raise ValueError(f"shapes do not fit: x {tuple(x.shape)}, w {tuple(w.shape)}, labels {tuple(labels.shape)}")
    if d < 1 or c < 1:
        raise ValueError("at least one feature and one class are needed")
    if x.dtype not in TYPES or w.dtype != x.dtype:
        raise TypeError(f"x and w must both be float32, float16 or bfloat16, got {x.dtype} and {w.dtype}")
    if labels.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"labels must be int64 or int32, got {labels.dtype}")
    if bias is not None and (bias.shape != (c,) or bias.dtype != torch.float32):
        raise ValueError(f"bias must be a float32 ({c},) tensor")
    if row_weight is not None and (row_weight.shape != (n,) or row_weight.dtype != torch.float32):
        raise ValueError(f"row_weight must be a float32 ({n},) tensor")
    index = x.get_device()
    if index < 0 or w.get_device() != index or labels.get_device() != index or (
            bias is not None and bias.get_device() != index) or (
            row_weight is not None and row_weight.get_device() != index):
        raise ValueError("x, w, labels, bias and row_weight must be on one GPU (there is no CPU path)")
    return n, d, c


def _plain(t: torch.Tensor) -> torch.Tensor:
    """Memory that holds the values themselves (a conjugate's imaginary part holds the other sign)."""
    return t.resolve_neg() if t.is_neg() else t


def _on_device(index: int, name: str, fn, args) -> None:
    """fn(*args, stream) on torch's current stream of device `index`."""
    if torch.cuda.current_device() == index:
        code = fn(*args, torch.cuda.current_stream(index).cuda_stream)
    else:
        with torch.cuda.device(index):
            code = fn(*args, torch.cuda.current_stream(index).cuda_stream)
    if code:
        _native.check(name, code)


def _call(x, w, labels, bias, n, d, c, want, row_weight=None, scale=1.0, loss=None, lse=None, dx=None, dw=None,
          dbias=None):
    """One library call on the current stream of x's device; loss and lse given: read, not written."""
    x, w = _plain(x), _plain(w)
    bias, row_weight = bias if bias is None else _plain(bias), row_weight if row_weight is None else _plain(row_weight)
    lib = _native.load()
    type_id, device, index = TYPES[x.dtype], x.device, x.get_device()
    xp, wp = x.data_ptr(), w.data_ptr()
    xr, xk = x.stride()
    wr, wk = w.stride()
    have = loss is not None
    if labels.dtype != torch.int64 or (n > 1 and labels.stride(0) != 1):
        labels = labels.to(torch.int64).contiguous()
    if bias is not None and c > 1 and bias.stride(0) != 1:
        bias = bias.contiguous()
    size = _workspace_bytes(index, type_id, xp % 16, xr, xk, wp % 16, wr, wk, n, d, c, want)
    ws = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    if not have:
        loss = torch.empty(n, dtype=torch.float32, device=device)
        lse = torch.empty(n, dtype=torch.float32, device=device)
    args = (type_id, xp, xr, xk, wp, wr, wk, None if bias is None else bias.data_ptr(), labels.data_ptr(), n, d, c)
    end = (None if ws is None else ws.data_ptr(), size)
    if want == 0:
        args += (loss.data_ptr(), lse.data_ptr())
        _on_device(index, "gafime_xent_forward", lib.gafime_xent_forward, args + end)
    else:
        args += (None, 0) if row_weight is None else (row_weight.data_ptr(), row_weight.stride(0))
        args += (scale, int(have), loss.data_ptr(), lse.data_ptr())
        args += (None, 0, 0) if dx is None else (dx.data_ptr(), dx.stride(0), dx.stride(1))
        args += (None if dw is None else dw.data_ptr(), None if dbias is None else dbias.data_ptr())
        _on_device(index, "gafime_xent_gradient", lib.gafime_xent_gradient, args + end)
    return loss, lse


def _gradients(x, w, labels, bias, n, d, c, row_weight, scale, need_dx, need_dw, need_dbias, loss=None, lse=None):
    dx = dw = dbias = None
    if need_dx:
        # x's order: a table held column by column gets its gradient column by column
        if x.stride(0) == 1 and x.stride(1) != 1:
            dx = torch.empty((d, n), dtype=x.dtype, device=x.device).t()
        else:
            dx = torch.empty((n, d), dtype=x.dtype, device=x.device)
    if need_dw:
        dw = torch.empty((c, d), dtype=w.dtype, device=w.device)
    if need_dbias:
        dbias = torch.empty(c, dtype=torch.float32, device=x.device)
    want = _GRADIENT | (_DX if need_dx else 0) | (_DW if need_dw else 0) | (_DBIAS if need_dbias else 0)
    loss, lse = _call(x, w, labels, bias, n, d, c, want, row_weight, scale, loss, lse, dx, dw, dbias)
    return XentGrad(loss, lse, dx, dw, dbias)


class _SoftmaxXent(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, labels, bias):
        n, d, c = x.shape[0], x.shape[1], w.shape[0]
        loss, lse = _call(x, w, labels, bias, n, d, c, 0)
        ctx.save_for_backward(x, w, labels, bias, loss, lse)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        x, w, labels, bias, loss, lse = ctx.saved_tensors
        need_x, need_w, _, need_b = ctx.needs_input_grad
        if grad_loss.dtype != torch.float32:
            grad_loss = grad_loss.float()
        g = _gradients(x, w, labels, bias, x.shape[0], x.shape[1], w.shape[0], grad_loss, 1.0, need_x, need_w,
                       need_b and bias is not None, loss, lse)
        return g.dx, g.dw, None, g.dbias


def softmax_xent(x: torch.Tensor, w: torch.Tensor, labels: torch.Tensor,
                 bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Per-row softmax cross entropy of ``x @ w.T + bias``, (n,) float32, without keeping the
    logits; differentiable in x, w and bias.

    x (n, d) and w (c, d): float32, float16 or bfloat16 alike, any strides (a bucket's columns
    as they are); labels (n,) int64 or int32; bias (c,) float32, -inf excludes a class.  A row
    with a negative label is left out: loss 0, no part in any gradient, whatever its features
    hold.  A label >= c makes the row's loss, and the gradients it enters, NaN.  Reverse mode and
    first order only: tensors with forward-mode tangents are refused.

    To capture a backward pass into a CUDA graph, let go of eager graphs of the same leaves
    first (torch's autograd waits for the stream on which they were made), or capture
    softmax_xent_grad, which needs no autograd."""
    _check(x, w, labels, bias, None)
    # (the level is -1 outside of forward mode)
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (x, w, bias)):
        raise RuntimeError("softmax_xent has no forward-mode derivative")
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or (bias is not None and bias.requires_grad)):
        return _SoftmaxXent.apply(x, w, labels, bias)
    return _call(x, w, labels, bias, x.shape[0], x.shape[1], w.shape[0], 0)[0]


def softmax_xent_grad(x: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, bias: Optional[torch.Tensor] = None,
                      row_weight: Optional[torch.Tensor] = None, scale: float = 1.0, need_dx: bool = True,
                      need_dw: bool = True) -> XentGrad:
    """Losses, and the gradients of ``sum_i scale * row_weight[i] * loss[i]``, in one call: the
    step of a fit whose row weights are known beforehand (1 / n for the mean).  With few classes
    and need_dx=False that is one pass over x.  The gradient of a bias that is None is None.
    The losses are detached, like the gradients: for a loss to differentiate take softmax_xent.
    Arguments as softmax_xent; row_weight (n,) float32, None for ones."""
    n, d, c = _check(x, w, labels, bias, row_weight)
    return _gradients(x, w, labels, bias, n, d, c, row_weight, float(scale), need_dx, need_dw, bias is not None)


def _whole(t: torch.Tensor) -> bool:
    """The elements are, in some order of the dimensions, those of a whole storage: a transposed or
    channels-last tensor (a slice of one is not)."""
    if t.storage_offset() or t.untyped_storage().nbytes() != t.numel() * t.element_size():
        return False
    step = 1
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if size != 1:
            if stride != step:
                return False
            step *= size
    return True


def _dense(tensors: list) -> bool:
    return all(t.is_contiguous() or _whole(t) for t in tensors)


def _alike(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Elements in the same order: both contiguous, or of the same shape and strides."""
    return (a.is_contiguous() and b.is_contiguous()) or (a.shape == b.shape and a.stride() == b.stride())


def _grad_norm(tensors: list, out, max_norm: float) -> torch.Tensor:
    count = len(tensors)
    if count == 0:
        raise ValueError("at least one tensor is needed")
    device = tensors[0].device
    if device.type != "cuda":
        raise ValueError(f"the tensors must be on one GPU, got {device}")
    index = device.index
    # whole lists at C speed: 64-bit arrays that the library reads in place
    sizes = array.array("q", map(_numel, tensors))
    dtypes = list(map(_dtype, tensors))
    if not set(dtypes) <= TYPES.keys():
        raise TypeError(f"tensors must be float32, float16 or bfloat16, got {set(dtypes) - TYPES.keys()}")
    plain = all(map(_contiguous, tensors))
    if set(map(_device, tensors)) != {index} or not (plain or _dense(tensors)):
        raise ValueError("the tensors must be on one GPU, and contiguous or a whole storage in another order")
    lib = _native.load()
    outs = written = None
    ptrs = array.array("q", map(_pointer, tensors))
    if out is tensors:
        outs, written = ptrs, tensors
    elif out is not None:
        written = out = list(out)
        if len(out) != count:
            raise ValueError(f"{count} tensors, but {len(out)} outs")
        if (list(map(_dtype, out)) != dtypes or array.array("q", map(_numel, out)) != sizes
                or set(map(_device, out)) != {index}
                or not (plain and all(map(_contiguous, out)) or _dense(out) and all(map(_alike, tensors, out)))):
            raise ValueError("every out must have its tensor's size, type, device and order of elements")
        # (a dense view that negates has one element: imaginary parts lie two apart)
        if 1 in sizes and any(t.is_neg() != o.is_neg() for t, o, m in zip(tensors, out, sizes) if m == 1):
            raise ValueError("a view that negates can be clipped in place only")
        outs = array.array("q", map(_pointer, out))
    size = _norm_workspace(count)
    ws = torch.empty(size, dtype=torch.uint8, device=device)
    norm = torch.empty((), dtype=torch.float32, device=device)
    types = array.array("i", map(TYPES.__getitem__, dtypes))
    args = (_address(ptrs), _address(sizes), _address(types), count, None if outs is None else _address(outs), max_norm,
            norm.data_ptr(), ws.data_ptr(), size)
    _on_device(index, "gafime_grad_norm", lib.gafime_grad_norm, args)
    if written:
        # torch does not see the writes: a tensor that autograd saved before has to be noticed
        torch.autograd.graph.increment_version(written)
    return norm


@functools.lru_cache(maxsize=1024)
def _norm_workspace(count: int) -> int:
    out = ctypes.c_size_t(0)
    _native.check("gafime_grad_norm_workspace",
                  _native.load(require_gpu=False).gafime_grad_norm_workspace(count, ctypes.byref(out)))
    return out.value


@torch.no_grad()
def grad_norm(tensors: Sequence[torch.Tensor]) -> torch.Tensor:
    """2-norm over all elements of the tensors together, a float32 scalar on their GPU, detached.
    The tensors are contiguous, or hold a whole storage in another order of their dimensions (a
    transposed dx, channels last); float32, float16 or bfloat16 in any mix.  Squares are summed in
    fp64."""
    return _grad_norm(list(tensors), None, 0.0)


@torch.no_grad()
def clip_grad_norm(tensors: Sequence[torch.Tensor], max_norm: float,
                   out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scale the tensors by min(1, max_norm / norm) of their norm together, in place or into
    ``out`` (one tensor each, alike in size, type and order of elements, apart from one another
    and from the tensors), and return the norm before it, detached.  Tensors as grad_norm.  A norm
    that is not finite leaves the values as they are: the caller sees it in the result and skips the
    step."""
    max_norm = float(max_norm)
    if not 0.0 <= max_norm <= 3.4028234663852886e38:
        raise ValueError(f"max_norm must be a finite number >= 0, got {max_norm}")
    tensors = list(tensors)
    return _grad_norm(tensors, tensors if out is None else out, max_norm)

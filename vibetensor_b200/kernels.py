"""Row ops and gather / scatter_add with the call signatures of the reference's
``vibe_kernels.*.vbt_native`` modules, served by plain CUDA in libvbt_b200.so instead of
Triton kernels compiled at run time:

* ``softmax`` / ``log_softmax``  -- vibe_kernels/softmax/vbt_native.py:193-328
* ``rmsnorm``                    -- vibe_kernels/rmsnorm/vbt_native.py:340-406
* ``rmsnorm_backward``           -- vibe_kernels/rmsnorm/vbt_native.py:409-492
* ``softmax_backward`` / ``log_softmax_backward``
                                 -- vibe_kernels/softmax/impl/cutedsl_softmax/softmax.py:992-1017
* ``gather`` / ``scatter_add``   -- vibe_kernels/indexing/vbt_native.py:197-280, :490-580

Same argument meaning and the same exception classes for the same misuse (RuntimeError for a
non-CUDA tensor, TypeError for a dtype, NotImplementedError for an unsupported dim); float16
and bfloat16 inputs are accepted in addition to the reference's float32.

Around a transformer block's matrix products, in the same manner (no counterpart in the reference):

* ``residual_norm``              -- a branch joined with the residual stream between two norms
* ``checkpoint8`` and its users  -- activations kept in 8 bits for the backward pass
* ``silu_mul``                   -- the gated activation
* ``rotary``                     -- rotary positions with several axes
"""
from __future__ import annotations

import builtins
import ctypes
import functools
from typing import Optional

import torch

from . import ops as _ops
from ._lib import Q8_FORMATS as _Q8_FORMATS, Q8_GROUP, check, dtype_code, lib, stream_ptr

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _row_stride(x: torch.Tensor) -> Optional[int]:
    """The one stride onto which x's leading dims collapse, that of the innermost with more than one
    index (a row's length with none); None if they do not.  A dim of one index has no say: whatever
    stride it carries is never taken."""
    step, rows = None, 1
    for n, st in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
        if n == 1:
            continue
        if step is None:
            step = st
        elif st != step * rows:
            return None
        rows *= n
    return x.shape[-1] if step is None else step


def _rows_view(x: torch.Tensor, what: str):
    """(rows, cols, row_stride) of x seen as a stack of last-dim rows, the reference's 2-D
    view (rows = product of leading dims, row stride = strides[-2])."""
    if not x.is_cuda:
        raise RuntimeError(f"{what} requires CUDA tensors")
    if x.dtype not in _FLOATS:
        raise TypeError(f"{what} requires float32, float16 or bfloat16")
    if x.dim() == 0:
        return x.reshape(1, 1), 1, 1, 1
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    if cols and x.is_contiguous():
        return x, rows, cols, cols
    row_stride = _row_stride(x)
    if row_stride is None or (x.stride(-1) != 1 and cols > 1):
        x, row_stride = _ops.contiguous(x), cols
    return x, rows, cols, row_stride


def _softmax(x: torch.Tensor, dim: int, log: bool) -> torch.Tensor:
    what = "log_softmax" if log else "softmax"
    nd = x.dim()
    d = dim + nd if dim < 0 else dim
    if nd and d != nd - 1:
        raise NotImplementedError(f"{what} currently only supports dim=-1 (last dimension)")
    xv, rows, cols, rs = _rows_view(x, what)
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if rows == 0 or cols == 0:
        return out
    check(lib().vbt_b200_softmax(ctypes.c_void_p(out.data_ptr()), ctypes.c_void_p(xv.data_ptr()),
                                 dtype_code(x.dtype), rows, cols, rs, int(log), stream_ptr(x)))
    return out


def softmax(x: torch.Tensor, dim: int = -1) -> torch.Tensor:
    return _softmax(x, dim, False)


def log_softmax(x: torch.Tensor, dim: int = -1) -> torch.Tensor:
    return _softmax(x, dim, True)


def rmsnorm(x: torch.Tensor, gamma: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """Returns (out, inv_rms): out has x's shape and dtype, inv_rms is float32 [rows]."""
    xv, rows, cols, rs = _rows_view(x, "rmsnorm")
    if gamma is not None:
        if not gamma.is_cuda:
            raise RuntimeError("rmsnorm requires CUDA tensors")
        if gamma.dtype != torch.float32 or gamma.numel() != cols:
            raise TypeError("gamma must be float32 of shape [hidden_size]")
        gamma = gamma.contiguous()
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    inv = torch.empty((rows,), dtype=torch.float32, device=x.device)
    if rows == 0 or cols == 0:
        return out, inv
    check(lib().vbt_b200_rmsnorm(ctypes.c_void_p(out.data_ptr()), ctypes.c_void_p(inv.data_ptr()),
                                 ctypes.c_void_p(xv.data_ptr()),
                                 ctypes.c_void_p(gamma.data_ptr()) if gamma is not None else None,
                                 dtype_code(x.dtype), rows, cols, rs, float(eps), stream_ptr(x)))
    return out, inv


def _softmax_backward(dy: torch.Tensor, y: torch.Tensor, log: bool) -> torch.Tensor:
    what = "log_softmax_backward" if log else "softmax_backward"
    if dy.shape != y.shape:
        raise ValueError(f"{what}: dy and y must have the same shape")
    if dy.dtype != y.dtype:
        raise TypeError(f"{what}: dy and y must have the same dtype")
    dyv, rows, cols, rs_dy = _rows_view(dy, what)
    yv, _, _, rs_y = _rows_view(y, what)
    dx = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    if rows == 0 or cols == 0:
        return dx
    check(lib().vbt_b200_softmax_backward(ctypes.c_void_p(dx.data_ptr()), ctypes.c_void_p(dyv.data_ptr()),
                                          ctypes.c_void_p(yv.data_ptr()), dtype_code(y.dtype), rows, cols,
                                          rs_dy, rs_y, int(log), stream_ptr(y)))
    return dx


def softmax_backward(dy: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """dx of y = softmax(x, -1): y * (dy - sum(dy * y))."""
    return _softmax_backward(dy, y, False)


def log_softmax_backward(dy: torch.Tensor, log_y: torch.Tensor) -> torch.Tensor:
    """dx of log_y = log_softmax(x, -1): dy - exp(log_y) * sum(dy)."""
    return _softmax_backward(dy, log_y, True)


def rmsnorm_backward(grad_output: torch.Tensor, x, inv_rms: torch.Tensor,
                     gamma: Optional[torch.Tensor] = None):
    """Returns (grad_input, grad_gamma); grad_gamma is None when gamma is None, float32
    [hidden_size] otherwise.  inv_rms is the second result of ``rmsnorm``.  x may be the
    ``Checkpoint8`` that ``rmsnorm_checkpoint8`` kept in its place."""
    what = "rmsnorm_backward"
    if isinstance(x, Checkpoint8):
        return _rmsnorm_backward8(grad_output, x, inv_rms, gamma)
    if grad_output.shape != x.shape:
        raise ValueError(f"{what}: grad_output and x must have the same shape")
    if grad_output.dtype != x.dtype:
        raise TypeError(f"{what}: grad_output and x must have the same dtype")
    xv, rows, cols, rs_x = _rows_view(x, what)
    gv, _, _, rs_g = _rows_view(grad_output, what)
    if not inv_rms.is_cuda:
        raise RuntimeError(f"{what} requires CUDA tensors")
    if inv_rms.dtype != torch.float32 or inv_rms.numel() != rows:
        raise TypeError("inv_rms must be float32 of shape [rows]")
    inv_rms = inv_rms.contiguous()
    if gamma is not None:
        if not gamma.is_cuda:
            raise RuntimeError(f"{what} requires CUDA tensors")
        if gamma.dtype != torch.float32 or gamma.numel() != cols:
            raise TypeError("gamma must be float32 of shape [hidden_size]")
        gamma = gamma.contiguous()
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dgamma = torch.empty((cols,), dtype=torch.float32, device=x.device) if gamma is not None else None
    ws, ws_bytes = None, 0
    if dgamma is not None and cols:
        need = ctypes.c_size_t()
        check(lib().vbt_b200_rmsnorm_backward_workspace_bytes(rows, cols, dtype_code(x.dtype), x.device.index,
                                                              ctypes.byref(need)))
        # the dgamma partial rows live in the general scratch buffer of this (device, stream)
        ws = _ops._workspace(max(need.value, 16), x.device)
        ws_bytes = ws.numel()
    if cols == 0:
        return dx, dgamma
    check(lib().vbt_b200_rmsnorm_backward(
        ctypes.c_void_p(dx.data_ptr()), ctypes.c_void_p(dgamma.data_ptr()) if dgamma is not None else None,
        ctypes.c_void_p(gv.data_ptr()), ctypes.c_void_p(xv.data_ptr()), ctypes.c_void_p(inv_rms.data_ptr()),
        ctypes.c_void_p(gamma.data_ptr()) if gamma is not None else None, dtype_code(x.dtype), rows, cols,
        rs_g, rs_x, ctypes.c_void_p(ws.data_ptr()) if ws is not None else None, ws_bytes, stream_ptr(x)))
    return dx, dgamma


def _check_gather_args(src, dim, index, what):
    if not src.is_cuda:
        raise RuntimeError(f"{what} requires CUDA tensors")
    if not index.is_cuda:
        raise RuntimeError("index must be on CUDA")
    if index.dtype != torch.int64:
        raise TypeError("index must be int64")
    nd = src.dim()
    d = dim + nd if dim < 0 else dim
    if d != 0:
        raise NotImplementedError(f"{what} currently only supports dim=0")
    if index.dim() != 1:
        raise NotImplementedError(f"{what} currently only supports 1D index")


def gather(src: torch.Tensor, dim: int, index: torch.Tensor, status=None) -> torch.Tensor:
    """out[i, ...] = src[index[i], ...] (dim 0, 1-D int64 index).  The Triton kernel reads
    whatever an out-of-range index points at; here such a row comes back as zeros and is
    counted in ``status`` (an ops.IndexStatus) when one is given."""
    _check_gather_args(src, dim, index, "gather")
    src2 = src.reshape(src.shape[0], -1) if src.dim() != 2 else src
    out = _ops.index_rows(src2, index, policy=_ops.INDEX_STRICT, status=status, eager_check=False)
    return out.reshape((index.numel(),) + tuple(src.shape[1:]))


def scatter_add(out: torch.Tensor, dim: int, index: torch.Tensor, src: torch.Tensor, status=None):
    """out[index[i], ...] += src[i, ...] in place (dim 0, 1-D int64 index); indices are
    clamped into range as the Triton kernel does (vibe_kernels/indexing/kernels.py:79-80)."""
    _check_gather_args(out, dim, index, "scatter_add")
    if out.dtype != src.dtype:
        raise TypeError("out and src must have the same dtype")
    out2 = out.view(out.shape[0], -1) if out.dim() != 2 else out
    src2 = src.reshape(index.numel(), -1)
    _ops.index_put_rows_(out2, index, src2, accumulate=True, policy=_ops.INDEX_CLAMP, status=status,
                         eager_check=False)
    return out


# --------------------------------------------------------------------------------------
# around a transformer block's matrix products
# --------------------------------------------------------------------------------------
_F32 = torch.float32


def _ptr(t: Optional[torch.Tensor]):
    return t if t is None else t.data_ptr()


def _same_device(what: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    device = first.get_device()
    for t in others:
        if t is not None and t.get_device() != device:
            if not t.is_cuda:
                raise RuntimeError(f"{what} requires CUDA tensors")
            raise ValueError(f"{what}: operands on {first.device} and {t.device}")


# Allocations on the host path: sizes as plain integers and no device argument parse in 1.4 us where a
# tuple takes 2.3 and a device 3.3.
def _dense_like(x: torch.Tensor) -> torch.Tensor:
    if x.is_contiguous():
        return torch.empty_like(x)
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _floats(x: torch.Tensor, n: int) -> torch.Tensor:
    return x.new_empty(n, dtype=_F32)


def _like(what: str, name: str, t: torch.Tensor, x: torch.Tensor) -> None:
    if t is x:
        return
    if t.shape != x.shape:
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected {tuple(x.shape)}")
    if t.dtype != x.dtype:
        raise TypeError(f"{what}: {name} is {t.dtype}, expected {x.dtype}")


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(entry: str, *sizes: int) -> int:
    """What a ``*_workspace_bytes`` entry answers, a function of its arguments alone."""
    need = ctypes.c_size_t()
    check(getattr(lib(), entry)(*sizes, ctypes.byref(need)))
    return need.value


def _gamma(name: str, g: Optional[torch.Tensor], cols: int) -> Optional[torch.Tensor]:
    if g is None:
        return None
    if g.dtype != _F32 or g.numel() != cols:
        raise TypeError(f"{name} must be float32 of shape [hidden_size]")
    return g if g.is_contiguous() else g.contiguous()


def _row_scalars(name: str, t: Optional[torch.Tensor], rows: int) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != rows:
        raise TypeError(f"{name} must be float32 of shape [rows]")
    return t.contiguous()


def _gate_rows(what: str, gate: Optional[torch.Tensor], x: torch.Tensor, rows: int):
    """(gate, row stride, rows of x per gate row) of a gate that broadcasts to x over its inner
    leading dims: [hidden], x.shape[:k] + (1, ..., 1, hidden), or x's own shape."""
    if gate is None:
        return None, 0, max(rows, 1)
    if gate.dtype != x.dtype:
        raise TypeError(f"{what}: gate is {gate.dtype}, expected {x.dtype}")
    lead, g = tuple(x.shape[:-1]), tuple(gate.shape[:-1])
    if gate.dim() == 0 or gate.shape[-1] != x.shape[-1] or (gate.dim() != 1 and gate.dim() != x.dim()):
        raise ValueError(f"{what}: gate of shape {tuple(gate.shape)} does not broadcast to {tuple(x.shape)}")
    k = 0
    while k < len(g) and g[k] == lead[k]:
        k += 1
    if any(n != 1 for n in g[k:]):
        raise ValueError(f"{what}: gate of shape {tuple(gate.shape)} does not broadcast to the last leading dims of "
                         f"{tuple(x.shape)}")
    gv, grows, _, stride = _rows_view(gate, what)
    return gv, stride, max(rows // max(grows, 1), 1)


def residual_norm(x: torch.Tensor, y: torch.Tensor, gamma_post: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None, gamma_pre: Optional[torch.Tensor] = None, eps: float = 1e-6, *,
                  post_norm: bool = True, pre_norm: bool = True, residual_scale: float = 1.0,
                  branch_scale: float = 1.0):
    """The join of a branch's output y with the residual stream x, and the norm in front of the next
    block, in one pass over the rows:

        v = y * inv_post * gamma_post           (post_norm; v = y without)
        r = residual_scale * x + branch_scale * gate * v
        n = r * inv_pre * gamma_pre             (pre_norm; from the unrounded r)

    x and y are float32, float16 or bfloat16 of one shape; gate has their dtype and is None,
    [hidden], x.shape[:k] + (1, ..., 1, hidden) (one row per sample, say) or x's own shape; gammas
    are float32 [hidden] or None (ones).  Returns (r, n, inv_post, inv_pre), the last two float32
    [rows]; what a switched-off norm would give is None."""
    what = "residual_norm"
    xv, rows, cols, rs_x = _rows_view(x, what)
    _same_device(what, x, y, gamma_post, gate, gamma_pre)
    _like(what, "y", y, x)
    if gamma_post is not None and not post_norm or gamma_pre is not None and not pre_norm:
        raise ValueError(f"{what}: a gamma of a norm that is switched off")
    yv, _, _, rs_y = _rows_view(y, what)
    gamma_post, gamma_pre = _gamma("gamma_post", gamma_post, cols), _gamma("gamma_pre", gamma_pre, cols)
    gv, rs_g, per = _gate_rows(what, gate, x, rows)
    r = _dense_like(x)
    n = _dense_like(x) if pre_norm else None
    inv_post = _floats(x, rows) if post_norm else None
    inv_pre = _floats(x, rows) if pre_norm else None
    if rows and cols:
        check(lib().vbt_b200_residual_norm(
            _ptr(r), _ptr(n), _ptr(inv_post), _ptr(inv_pre), _ptr(xv), _ptr(yv), _ptr(gamma_post), _ptr(gv),
            _ptr(gamma_pre), dtype_code(x.dtype), rows, cols, rs_x, rs_y, rs_g, per, float(residual_scale),
            float(branch_scale), float(eps), int(post_norm) | 2 * int(pre_norm), stream_ptr(x)))
    return r, n, inv_post, inv_pre


def residual_norm_backward(grad_r: Optional[torch.Tensor], grad_n: Optional[torch.Tensor], y: Optional[torch.Tensor],
                           r: Optional[torch.Tensor], inv_post: Optional[torch.Tensor],
                           inv_pre: Optional[torch.Tensor], gamma_post: Optional[torch.Tensor] = None,
                           gate: Optional[torch.Tensor] = None, gamma_pre: Optional[torch.Tensor] = None, *,
                           residual_scale: float = 1.0, branch_scale: float = 1.0):
    """Backward of ``residual_norm``: from the gradients that arrive at r (None: none) and n, the
    branch's output y, and r and the reciprocal norms the forward pass returned (None where its norm
    was off), returns (grad_x, grad_y, grad_gamma_post, grad_gate, grad_gamma_pre).  Gradients of
    what was None are None; grad_gamma_* are float32 and sums over rows are reproducible run to run.
    y is only needed with post_norm or a gate, r only with pre_norm."""
    what = "residual_norm_backward"
    first = grad_n if grad_n is not None else grad_r
    if first is None:
        raise ValueError(f"{what}: no gradient given")
    post, pre = inv_post is not None, inv_pre is not None
    if pre and (grad_n is None or r is None):
        raise ValueError(f"{what}: inv_pre given without grad_n and r")
    if not pre and grad_n is not None:
        raise ValueError(f"{what}: grad_n given without inv_pre")
    if (post or gate is not None) and y is None:
        raise ValueError(f"{what}: y is needed with post_norm or a gate")
    if gamma_post is not None and not post or gamma_pre is not None and not pre:
        raise ValueError(f"{what}: a gamma of a norm that is switched off")
    xv, rows, cols, _ = _rows_view(first, what)
    _same_device(what, first, grad_r, grad_n, y, r, inv_post, inv_pre, gamma_post, gate, gamma_pre)
    views = []
    for name, t in (("grad_r", grad_r), ("grad_n", grad_n), ("y", y), ("r", r if pre else None)):
        if t is None:
            views.append((None, 0))
            continue
        _like(what, name, t, first)
        v, _, _, rs = _rows_view(t, what)
        views.append((v, rs))
    inv_post, inv_pre = _row_scalars("inv_post", inv_post, rows), _row_scalars("inv_pre", inv_pre, rows)
    gamma_post, gamma_pre = _gamma("gamma_post", gamma_post, cols), _gamma("gamma_pre", gamma_pre, cols)
    gv, rs_g, per = _gate_rows(what, gate, first, rows)
    dx = _dense_like(first)
    dy = _dense_like(first)
    dg1 = _floats(first, cols) if gamma_post is not None else None
    dg2 = _floats(first, cols) if gamma_pre is not None else None
    dgate = None
    if gate is not None:  # a gate row that no row of x uses has a gradient of zero
        dgate = _dense_like(gate) if rows else torch.zeros_like(gate, memory_format=torch.contiguous_format)
    if cols == 0:
        return dx, dy, dg1, dgate, dg2
    ws, ws_bytes = None, 0
    if rows and (dg1 is not None or dg2 is not None or dgate is not None):
        ws_bytes = _scratch_bytes("vbt_b200_residual_norm_backward_workspace_bytes", rows, cols, dtype_code(first.dtype),
                                  per, first.get_device())
        ws = first.new_empty(ws_bytes, dtype=torch.uint8)
    (drv, rs_dr), (dnv, rs_dn), (yv, rs_y), (rv, rs_r) = views
    check(lib().vbt_b200_residual_norm_backward(
        _ptr(dx), _ptr(dy), _ptr(dg1), _ptr(dgate), _ptr(dg2), _ptr(drv), _ptr(dnv), _ptr(yv), _ptr(rv),
        _ptr(inv_post), _ptr(inv_pre), _ptr(gamma_post), _ptr(gv), _ptr(gamma_pre), dtype_code(first.dtype), rows, cols,
        rs_dr, rs_dn, rs_y, rs_r, rs_g, per, float(residual_scale), float(branch_scale), int(post) | 2 * int(pre),
        _ptr(ws), ws_bytes, stream_ptr(first)))
    return dx, dy, dg1, dgate, dg2


class Checkpoint8:
    """An activation kept in 8 bits: ``q`` (int8 or float8_e4m3fn, the activation's shape) and
    ``scale`` (float32 [rows, ceil(hidden / 128)]), one scale per 128 neighbouring values of a row.
    ``dtype`` is the activation's own, what ``checkpoint8_restore`` gives back."""

    __slots__ = ("q", "scale", "fmt", "dtype")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor, fmt: str, dtype: torch.dtype):
        self.q, self.scale, self.fmt, self.dtype = q, scale, fmt, dtype

    @property
    def shape(self):
        return self.q.shape

    @property
    def device(self):
        return self.q.device

    def nbytes(self) -> int:
        return self.q.numel() + 4 * self.scale.numel()


def _q8_format(what: str, fmt: str):
    try:
        return _Q8_FORMATS[fmt]
    except (KeyError, TypeError):
        raise ValueError(f"{what}: fmt must be one of {sorted(_Q8_FORMATS)}") from None


def _new_checkpoint(x: torch.Tensor, rows: int, cols: int, fmt: str, store: torch.dtype) -> Checkpoint8:
    return Checkpoint8(torch.empty_like(x, dtype=store, memory_format=torch.contiguous_format),
                       x.new_empty(rows, -(-cols // Q8_GROUP), dtype=_F32), fmt, x.dtype)


def _held_rows(what: str, c: Checkpoint8):
    """(rows, cols, format code) of a checkpoint, its parts checked."""
    code, store = _q8_format(what, c.fmt)
    cols = c.q.shape[-1] if c.q.dim() else 1
    rows = c.q.numel() // cols if cols else 0
    if not c.q.is_cuda or not c.scale.is_cuda:
        raise RuntimeError(f"{what} requires CUDA tensors")
    if c.q.dtype != store or c.scale.dtype != torch.float32 or c.dtype not in _FLOATS:
        raise TypeError(f"{what}: not a checkpoint of format {c.fmt}")
    if c.scale.device != c.q.device or c.scale.numel() != rows * -(-cols // Q8_GROUP) or \
            not c.q.is_contiguous() or not c.scale.is_contiguous():
        raise ValueError(f"{what}: the checkpoint's values and scales do not match")
    return rows, cols, code


def checkpoint8(x: torch.Tensor, fmt: str = "int8") -> Checkpoint8:
    """Keeps x (float32, float16 or bfloat16) in 8 bits, ``fmt`` "int8" or "e4m3": with amax the
    largest magnitude of 128 neighbours, scale = amax / top and q = round(x * (top / amax)), top 127 or 448.
    A group whose amax is below 2^-119 is kept as zeros; one that holds a NaN or an infinity reads
    back as NaN throughout."""
    what = "checkpoint8"
    code, store = _q8_format(what, fmt)
    xv, rows, cols, rs = _rows_view(x, what)
    c = _new_checkpoint(x, rows, cols, fmt, store)
    if rows and cols:
        check(lib().vbt_b200_checkpoint8(_ptr(c.q), _ptr(c.scale), _ptr(xv), dtype_code(x.dtype), code, rows, cols, rs,
                                         stream_ptr(x)))
    return c


def checkpoint8_restore(c: Checkpoint8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The activation a checkpoint stands for, q * scale, in its own dtype or the given one."""
    what = "checkpoint8_restore"
    rows, cols, code = _held_rows(what, c)
    dt = c.dtype if dtype is None else dtype
    if dt not in _FLOATS:
        raise TypeError(f"{what} gives float32, float16 or bfloat16")
    out = torch.empty_like(c.q, dtype=dt)
    if rows and cols:
        check(lib().vbt_b200_checkpoint8_restore(_ptr(out), _ptr(c.q), _ptr(c.scale), dtype_code(dt), code, rows, cols,
                                                 stream_ptr(out)))
    return out


def rmsnorm_checkpoint8(x: torch.Tensor, gamma: Optional[torch.Tensor] = None, eps: float = 1e-6, fmt: str = "int8"):
    """``rmsnorm`` that also keeps its input in 8 bits, from one read of x: returns (out, inv_rms,
    checkpoint).  The checkpoint takes x's place in ``rmsnorm_backward``."""
    what = "rmsnorm_checkpoint8"
    code, store = _q8_format(what, fmt)
    xv, rows, cols, rs = _rows_view(x, what)
    _same_device(what, x, gamma)
    gamma = _gamma("gamma", gamma, cols)
    out = _dense_like(x)
    inv = _floats(x, rows)
    c = _new_checkpoint(x, rows, cols, fmt, store)
    if rows and cols:
        check(lib().vbt_b200_rmsnorm_checkpoint8(_ptr(out), _ptr(inv), _ptr(c.q), _ptr(c.scale), _ptr(xv), _ptr(gamma),
                                                 dtype_code(x.dtype), code, rows, cols, rs, float(eps), stream_ptr(x)))
    return out, inv, c


def _rmsnorm_backward8(grad_output: torch.Tensor, c: Checkpoint8, inv_rms: torch.Tensor,
                       gamma: Optional[torch.Tensor]):
    what = "rmsnorm_backward"
    rows, cols, code = _held_rows(what, c)
    if grad_output.shape != c.shape:
        raise ValueError(f"{what}: grad_output and x must have the same shape")
    if grad_output.dtype != c.dtype:
        raise TypeError(f"{what}: grad_output and x must have the same dtype")
    gv, _, _, rs = _rows_view(grad_output, what)
    _same_device(what, grad_output, c.q, inv_rms, gamma)
    inv_rms = _row_scalars("inv_rms", inv_rms, rows)
    gamma = _gamma("gamma", gamma, cols)
    dx = torch.empty_like(c.q, dtype=c.dtype)
    dgamma = _floats(c.q, cols) if gamma is not None else None
    if cols == 0:
        return dx, dgamma
    ws, ws_bytes = None, 0
    if rows and dgamma is not None:
        ws_bytes = _scratch_bytes("vbt_b200_rmsnorm_backward8_workspace_bytes", rows, cols, dtype_code(c.dtype),
                                  c.q.get_device())
        ws = c.q.new_empty(ws_bytes, dtype=torch.uint8)
    check(lib().vbt_b200_rmsnorm_backward8(_ptr(dx), _ptr(dgamma), _ptr(gv), _ptr(c.q), _ptr(c.scale), _ptr(inv_rms),
                                           _ptr(gamma), dtype_code(c.dtype), code, rows, cols, rs, _ptr(ws), ws_bytes,
                                           stream_ptr(grad_output)))
    return dx, dgamma


def _silu_mul(gate: torch.Tensor, up: torch.Tensor, fmt: Optional[str], what: str):
    gv, rows, cols, rs_g = _rows_view(gate, what)
    _same_device(what, gate, up)
    _like(what, "up", up, gate)
    uv, _, _, rs_u = _rows_view(up, what)
    out = _dense_like(gate)
    cg = cu = None
    code = 0
    if fmt is not None:
        code, store = _q8_format(what, fmt)
        cg, cu = _new_checkpoint(gate, rows, cols, fmt, store), _new_checkpoint(up, rows, cols, fmt, store)
    if rows and cols:
        check(lib().vbt_b200_silu_mul(_ptr(out), cg and _ptr(cg.q), cg and _ptr(cg.scale), cu and _ptr(cu.q),
                                      cu and _ptr(cu.scale), _ptr(gv), _ptr(uv), dtype_code(gate.dtype), code, rows, cols,
                                      rs_g, rs_u, stream_ptr(gate)))
    return out, cg, cu


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """The gated activation silu(gate) * up; gate and up of one shape and dtype, rows of any stride
    (the two halves of one projection, say)."""
    return _silu_mul(gate, up, None, "silu_mul")[0]


def silu_mul_checkpoint8(gate: torch.Tensor, up: torch.Tensor, fmt: str = "int8"):
    """``silu_mul`` that also keeps both factors in 8 bits, from one read of them: returns (out,
    gate's checkpoint, up's checkpoint) for ``silu_mul_backward``."""
    if fmt is None:
        raise ValueError("silu_mul_checkpoint8: fmt must be given")
    return _silu_mul(gate, up, fmt, "silu_mul_checkpoint8")


def silu_mul_backward(grad_output: torch.Tensor, gate, up):
    """(grad_gate, grad_up) of ``silu_mul``; gate and up are both tensors or both checkpoints."""
    what = "silu_mul_backward"
    kept = isinstance(gate, Checkpoint8)
    if kept != isinstance(up, Checkpoint8):
        raise TypeError(f"{what}: gate and up must both be tensors or both checkpoints")
    dv, rows, cols, rs_d = _rows_view(grad_output, what)
    for name, t in (("gate", gate), ("up", up)):
        _like(what, name, t, grad_output)
    if kept:
        if gate.fmt != up.fmt:
            raise ValueError(f"{what}: checkpoints of two formats")
        code = _held_rows(what, gate)[2]
        _held_rows(what, up)
        _same_device(what, grad_output, gate.q, up.q)
        a, b, sa, sb, rs_g, rs_u = gate.q, up.q, gate.scale, up.scale, cols, cols
    else:
        _same_device(what, grad_output, gate, up)
        a, _, _, rs_g = _rows_view(gate, what)
        b, _, _, rs_u = _rows_view(up, what)
        code, sa, sb = 0, None, None
    dgate = _dense_like(grad_output)
    dup = _dense_like(grad_output)
    if rows and cols:
        check(lib().vbt_b200_silu_mul_backward(_ptr(dgate), _ptr(dup), _ptr(dv), _ptr(a), _ptr(sa), _ptr(b), _ptr(sb),
                                               dtype_code(grad_output.dtype), code, rows, cols, rs_d, rs_g, rs_u,
                                               stream_ptr(grad_output)))
    return dgate, dup


_I64x15 = ctypes.c_int64 * 15
_SECTIONS = [ctypes.c_int64 * n for n in range(5)]


def _values_apart(t: torch.Tensor) -> bool:
    """Whether each value of t has memory of its own: every stride steps over all that the smaller
    strides reach."""
    reach = 0
    for st, n in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n > 1):
        if st <= reach:
            return False
        reach += (n - 1) * st
    return True


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the views may share a value: their heads lie between one another in one memory, as
    the parts of a fused projection do without sharing any."""
    if a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr() or not a.numel() or not b.numel():
        return False

    def span(t):
        end = builtins.sum((n - 1) * st for n, st in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (end + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    if a1 <= b0 or b1 <= a0:
        return False
    # parts of one projection: equal steps from token to token, and within a token apart from each other
    if a.dim() == b.dim() and a.dtype == b.dtype and a.stride()[:-2] == b.stride()[:-2] and a.shape[:-2] == b.shape[:-2]:
        step = min((st for n, st in zip(a.shape[:-2], a.stride()[:-2]) if n > 1), default=0) * a.element_size()

        def inner(t):
            return ((t.shape[-2] - 1) * t.stride(-2) + t.shape[-1]) * t.element_size()
        first, second = (a, b) if a0 <= b0 else (b, a)
        gap = second.data_ptr() - first.data_ptr()
        if inner(first) <= gap and (step == 0 or gap + inner(second) <= step):
            return False
    return True


def _head_strides(t: torch.Tensor):
    """{batch, token, head} strides of [batch, tokens, heads, dim] or [tokens, heads, dim]."""
    st = t.stride()
    return (0, st[0], st[1]) if len(st) == 3 else st[:3]


def _rotary(q, k, positions, inv_freq, sections, interleaved, inverse, out, what):
    if not q.is_cuda:
        raise RuntimeError(f"{what} requires CUDA tensors")
    if q.dtype not in _FLOATS:
        raise TypeError(f"{what} requires float32, float16 or bfloat16")
    shape = q.shape
    if len(shape) not in (3, 4):
        raise ValueError(f"{what}: q must be [tokens, heads, dim] or [batch, tokens, heads, dim]")
    _same_device(what, q, k, positions, inv_freq)
    if k is not None:
        if k.dtype != q.dtype:
            raise TypeError(f"{what}: k is {k.dtype}, expected {q.dtype}")
        if k.dim() != len(shape) or k.shape[:-2] != shape[:-2] or k.shape[-1] != shape[-1]:
            raise ValueError(f"{what}: k of shape {tuple(k.shape)} does not go with q of shape {tuple(shape)}")
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1:
        raise TypeError(f"{what}: inv_freq must be float32 of shape [pairs]")
    if positions.dtype not in (torch.int64, torch.int32, torch.float32):
        raise TypeError(f"{what}: positions must be int64, int32 or float32")
    half, dim = inv_freq.shape[0], shape[-1]
    if 2 * half > dim:
        raise ValueError(f"{what}: {half} pairs do not fit a head of {dim} values")
    lead = tuple(shape[:-2])
    pos = positions
    if sections is None:
        sections = (half,)
        pos = pos.unsqueeze(0)
    sections = [int(s) for s in sections]
    axes = len(sections)
    if not 1 <= axes <= 4 or builtins.sum(sections) != half or min(sections) < 0:
        raise ValueError(f"{what}: 1 to 4 sections that sum to the {half} pairs are needed")
    if pos.dim() != 1 + len(lead) or pos.shape[0] != axes:
        raise ValueError(f"{what}: positions of shape {tuple(positions.shape)}; expected one of "
                         f"{lead} per section")
    if pos.shape != (axes, *lead):
        try:
            pos = pos.expand((axes, *lead))
        except RuntimeError:
            raise ValueError(f"{what}: positions of shape {tuple(positions.shape)} do not broadcast to {lead}") from None
    inv_freq = inv_freq.contiguous()
    batch, tokens = (1, lead[0]) if len(lead) == 1 else lead
    ps = pos.stride()
    if len(lead) == 1:
        ps = (ps[0], 0, ps[1])
    if out is not None:
        if len(out) != 2 or (k is None) != (out[1] is None):
            raise ValueError(f"{what}: out must be a pair like (q, k)")
        for name, o, x in (("out[0]", out[0], q), ("out[1]", out[1], k)):
            if o is None:
                continue
            _same_device(what, q, o)
            _like(what, name, o, x)
            if o.stride(-1) != 1 and dim > 1:
                raise ValueError(f"{what}: {name} must have a last stride of 1")
            if not _values_apart(o):
                raise ValueError(f"{what}: {name} has values that share memory")
            # it may replace the operand of its own place; the other one, the same tensor or not, is read meanwhile
            replaces = o.data_ptr() == x.data_ptr() and o.stride() == x.stride()
            for t in (None if replaces else x, k if name == "out[0]" else q, positions, inv_freq):
                if t is not None and _overlap(o, t):
                    raise ValueError(f"{what}: {name} overlaps an input that it does not replace")
        if out[1] is not None and _overlap(*out):
            raise ValueError(f"{what}: the two outputs overlap")
    qv = q if q.stride(-1) == 1 or dim <= 1 else _ops.contiguous(q)
    qo = out[0] if out is not None else _dense_like(qv)
    strides = (*_head_strides(qo), *_head_strides(qv))
    if k is None:
        ko, kargs = None, (None, None, 0)
        strides += (0,) * 6
    else:
        kv = k if k.stride(-1) == 1 or dim <= 1 else _ops.contiguous(k)
        ko = out[1] if out is not None else _dense_like(kv)
        kargs = (ko.data_ptr(), kv.data_ptr(), kv.shape[-2])
        strides += (*_head_strides(ko), *_head_strides(kv))
    check(lib().vbt_b200_rotary(qo.data_ptr(), qv.data_ptr(), shape[-2], *kargs, _I64x15(*strides, *ps),
                                dtype_code(q.dtype), batch, tokens, dim, pos.data_ptr(), dtype_code(pos.dtype),
                                inv_freq.data_ptr(), half, _SECTIONS[axes](*sections), axes, int(interleaved),
                                int(inverse), stream_ptr(q)))
    return qo, ko


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor,
           sections=None, interleaved: bool = False, out=None):
    """Rotary positions on queries and keys, with one or several axes (time, height, width).

    q [..., tokens, heads, dim] and k [..., tokens, kv_heads, dim] (or None), with or without a
    leading batch dim and with any strides.  Pair i of a head turns by positions * inv_freq[i]
    (inv_freq: float32 [pairs], 2 * pairs <= dim; values behind the pairs are copied).  With
    ``sections`` -- how many pairs belong to each of up to four axes, in order -- positions is
    [axes, ..., tokens], without it [..., tokens]; int64, int32 or float32, dims of size 1
    broadcast.  A pair is (i, pairs + i), or (2i, 2i + 1) with ``interleaved``.  The angle is formed
    in 64 bits: far positions keep it exact.  Returns (q, k) turned, dense, or written to the pair
    ``out``, each of which may be its own operand (not the other one)."""
    return _rotary(q, k, positions, inv_freq, sections, interleaved, False, out, "rotary")


def rotary_backward(grad_q: torch.Tensor, grad_k: Optional[torch.Tensor], positions: torch.Tensor,
                    inv_freq: torch.Tensor, sections=None, interleaved: bool = False, out=None):
    """Gradients of ``rotary``'s q and k: its outputs' gradients turned back by the same angles."""
    return _rotary(grad_q, grad_k, positions, inv_freq, sections, interleaved, True, out, "rotary_backward")

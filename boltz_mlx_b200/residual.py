"""The residual path between pair layers: LayerNorm, dropout, residual add, and the three in one pass,
with gradients, over libtriattn.so (triattn_layer_norm*, triattn_dropout_add*).

    h    = layer_norm(x, weight, bias, out_dtype=torch.bfloat16)     # the LayerNorm that feeds a layer (`xn=`)
    z    = dropout_add(z, y, 0.25, seed, share=(2, 3))               # z + dropout(update), one draw per row
    z, h = dropout_add_layer_norm(z, y, weight, bias, 0.25, seed, share=(2, 3), out_dtype=torch.bfloat16)

Mirrors boltz_mlx/layers/norm.py:8-17 (LayerNorm, `.f16()`) and the add-and-norm hand-over
(boltz_mlx/kernels.py:1448-1480) of jackryan225/boltz-mlx, and adds what training needs beside them.

Dropout.  Whether a value is kept is a function of (seed, offset, position) alone, and no mask is stored:
position e of the mask tensor (the tensor's shape with size 1 along the axes in `share`) takes word e % 4
of Philox4x32-10 with key = seed and counter = (e // 4, offset) and is dropped if it is below
round(p * 2**32).  The same (seed, offset) gives the same mask, whatever the type, the strides or the
direction; a layer that must differ from another takes another offset.  Kept values are scaled by
1 / (1 - p) held in 32 bits; what is dropped contributes nothing, even where it is not finite.  `seed` may
be a CUDA int64 tensor (seed, offset), read when the kernel runs: a captured graph then draws anew on
each replay if the program changes that tensor between replays (between a forward and its backward pass it
must not change; outside a captured graph autograd checks that).

Types: an fp32 stream with an fp32 or 16-bit result, or one 16-bit type throughout; statistics and sums are
fp32.  Tensors may have any strides along the leading axes (a transposed pair tensor is read and written in
place); the last axis is read densely, else copied.  There is no CPU path.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple, Optional, Sequence, Union

import torch
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib

MAX_DIM = 8192
_CODES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_I3 = ctypes.c_int64 * 3
Seed = Union[int, torch.Tensor]


class PairDropout(NamedTuple):
    """Dropout of a pair layer's update, as the layers' `dropout=` takes it.  share: the axes of
    [B, N, N, C] that share one draw; None: the layer's own (one draw per row, per column for the
    ending node)."""

    p: float
    seed: Seed
    offset: int = 0
    share: Optional[Sequence[int]] = None


# ---- arguments ----------------------------------------------------------------------------------------
def _unsupported(msg: str):
    return _lib.TriAttnUnsupported(_lib.EUNSUPPORTED, msg)


def _code(t: torch.Tensor, name: str) -> int:
    try:
        return _CODES[t.dtype]
    except KeyError:
        raise _unsupported(f"{name}: {t.dtype} (fp32, fp16 and bf16 are supported)") from None


def _on_gpu(what: str, x: torch.Tensor, *others) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"{what} (B200) needs CUDA tensors; there is no CPU path")
    for t in others:
        if t is not None and t.device != x.device:
            raise ValueError(f"{what}: tensors on {x.device} and {t.device}")


@lru_cache(maxsize=1024)
def _shape3(shape: tuple):
    """HOST array of the three leading sizes, the rows and dim of a tensor of `shape` (at most 4 axes)."""
    lead = (1,) * (4 - len(shape)) + shape[:-1]
    return _I3(*lead), lead[0] * lead[1] * lead[2], shape[-1]


def _four(t: torch.Tensor) -> torch.Tensor:
    """t with at most four axes: the leading ones joined (a view where the strides allow it)."""
    return t if t.dim() <= 4 else t.reshape(-1, *t.shape[-3:])


def _rows(t: torch.Tensor):
    """(tensor with a dense last axis, HOST array of its leading strides or None if it is dense)."""
    if t.is_contiguous():
        return t, None
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        return t.contiguous(), None
    st = t.stride()
    return t, _I3(*((0,) * (4 - len(st)) + st[:-1]))


@lru_cache(maxsize=256)
def _share_bits(share: tuple, ndim: int) -> int:
    axes = set()
    for a in share:
        if not isinstance(a, int) or not -ndim <= a < ndim:
            raise ValueError(f"share={share}: axes of a tensor of {ndim} axes")
        axes.add(a % ndim)
    if ndim > 4:
        lead = {a for a in axes if a < ndim - 3}
        if lead and len(lead) != ndim - 3:
            raise _unsupported(f"share={share}: of {ndim} axes the first {ndim - 3} are shared together or not at all")
        axes = {a - (ndim - 4) for a in axes if a >= ndim - 3} | ({0} if lead else set())
        ndim = 4
    return sum(1 << (a + 4 - ndim) for a in axes)


def _share(share, ndim: int) -> int:
    return _share_bits(share if type(share) is tuple else tuple(share), ndim) if share else 0


def _draw(what: str, p: float, seed: Seed, offset: int, device, training: bool):
    """(p, seed, offset, DEVICE address or None, the tensor behind it)."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: p={p} must lie in [0, 1]")
    if not training:
        p = 0.0
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 2 or not seed.is_contiguous() or seed.device != device:
            raise ValueError(f"{what}: a seed tensor holds (seed, offset) as int64 on {device}")
        if offset:
            raise ValueError(f"{what}: a seed tensor brings its own offset")
        return p, 0, 0, seed.data_ptr(), seed
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        raise ValueError(f"{what}: seed and offset are numbers of 64 bits")
    return p, seed, offset, None, None


def _params(what: str, weight, bias, dim: int):
    """(weight, bias, dtype code), dense."""
    if weight is None and bias is None:
        return None, None, _lib.F32
    for t in (weight, bias):
        if t is not None and tuple(t.shape) != (dim,):
            raise ValueError(f"{what}: weight and bias must be [{dim}], got {tuple(t.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"{what}: weight is {weight.dtype}, bias {bias.dtype}")
    code = _code(weight if weight is not None else bias, "weight / bias")
    return (weight.contiguous() if weight is not None else None, bias.contiguous() if bias is not None else None, code)


def _check_dim(what: str, x: torch.Tensor) -> None:
    if x.dim() < 1:
        raise ValueError(f"{what}: a tensor without axes")
    if x.shape[-1] < 1:
        raise ValueError(f"{what}: no channels")
    if x.shape[-1] > MAX_DIM:
        raise _unsupported(f"{what}: {x.shape[-1]} channels (at most {MAX_DIM})")


def _first(t: torch.Tensor) -> int:
    return t.data_ptr()


def _last(t: torch.Tensor) -> int:
    return t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) - 1


class _on:
    """The device of a call, made current only where it is not."""

    __slots__ = ("guard",)

    def __init__(self, device: torch.device):
        self.guard = torch.cuda.device(device) if device.index != torch.cuda.current_device() else None

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *e):
        if self.guard is not None:
            self.guard.__exit__(*e)


# ---- launches -----------------------------------------------------------------------------------------
def _launch_norm(x, weight, bias, eps, out_dtype, stats: bool):
    """(h, [2, rows] mean and rstd or None)"""
    x4, xs = _rows(_four(x))
    shape, rows, dim = _shape3(x4.shape)
    w, b, pc = _params("layer_norm", weight, bias, dim)
    out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    st = torch.empty(2, rows, dtype=torch.float32, device=x.device) if stats else None
    mean = st.data_ptr() if stats else None
    with _on(x.device):
        _lib.check(_lib.lib().triattn_layer_norm(
            x4.data_ptr(), _CODES[x.dtype], xs, shape, dim, _lib.ptr(w), _lib.ptr(b), pc, eps, out.data_ptr(),
            _CODES[out_dtype], None, mean, mean + 4 * rows if stats else None, _lib.stream_handle(x.device)))
    return out, st


def _launch_norm_backward(dout, x, weight, bias, st, dsum, draw, share, want, y_dtype):
    """(dx, dy, dweight, dbias), each None unless wanted.  dout and dsum: of x's shape."""
    x4, xs = _rows(_four(x))
    g4, gs = _rows(_four(dout))
    s4, ss = _rows(_four(dsum)) if dsum is not None else (None, None)
    shape, rows, dim = _shape3(x4.shape)
    p, seed, offset, state, _ = draw
    w, _, pc = _params("layer_norm", weight, bias, dim)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if want[0] else None
    dy = torch.empty(x.shape, dtype=y_dtype, device=x.device) if want[1] else None
    dw = torch.empty(dim, dtype=weight.dtype, device=x.device) if want[2] else None
    db = torch.empty(dim, dtype=bias.dtype, device=x.device) if want[3] else None
    ws, nbytes = None, 0
    with _on(x.device):
        if dw is not None or db is not None:
            nbytes = _lib.lib().triattn_layer_norm_backward_workspace_bytes(rows, dim)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        _lib.check(_lib.lib().triattn_layer_norm_backward(
            g4.data_ptr(), _CODES[dout.dtype], gs, x4.data_ptr(), _CODES[x.dtype], xs, shape, dim, _lib.ptr(w), pc,
            st.data_ptr(), st.data_ptr() + 4 * rows, _lib.ptr(s4), ss, share, p, seed, offset, state, _lib.ptr(dx),
            _lib.ptr(dy), _CODES[y_dtype], _lib.ptr(dw), _lib.ptr(db), _lib.ptr(ws), nbytes,
            _lib.stream_handle(x.device)))
    return dx, dy, dw, db


def _launch_dropout_add(z, y, draw, share, out, out_dtype):
    """z + dropout(y) (dropout(y) with z None) in `out` or a new tensor."""
    y4, ys = _rows(_four(y))
    z4, zs = _rows(_four(z)) if z is not None else (None, None)
    shape, _, dim = _shape3(y4.shape)
    p, seed, offset, state, _ = draw
    os_ = zs if out is not None else None
    if out is None:
        out = torch.empty(y.shape, dtype=out_dtype, device=y.device)
    with _on(y.device):
        _lib.check(_lib.lib().triattn_dropout_add(
            _lib.ptr(z4), _CODES[out_dtype], zs, y4.data_ptr(), _CODES[y.dtype], ys, shape, dim, share, p, seed, offset,
            state, out.data_ptr(), _CODES[out_dtype], os_, _lib.stream_handle(y.device)))
    return out


def _launch_fused(z, y, weight, bias, eps, draw, share, out_dtype, trans_out, stats: bool):
    """(s, h, stats)"""
    z4, zs = _rows(_four(z))
    y4, ys = _rows(_four(y))
    shape, rows, dim = _shape3(z4.shape)
    w, b, pc = _params("dropout_add_layer_norm", weight, bias, dim)
    p, seed, offset, state, _ = draw
    s = torch.empty(z.shape, dtype=z.dtype, device=z.device)
    h, hs = _trans_buffer(z.shape, out_dtype, z.device, trans_out)
    st = torch.empty(2, rows, dtype=torch.float32, device=z.device) if stats else None
    mean = st.data_ptr() if stats else None
    with _on(z.device):
        _lib.check(_lib.lib().triattn_dropout_add_layer_norm(
            z4.data_ptr(), _CODES[z.dtype], zs, y4.data_ptr(), _CODES[y.dtype], ys, shape, dim, share, p, seed, offset,
            state, _lib.ptr(w), _lib.ptr(b), pc, eps, s.data_ptr(), None, h.data_ptr(), _CODES[out_dtype], hs, mean,
            mean + 4 * rows if stats else None, _lib.stream_handle(z.device)))
    return s, h, st


def _trans_buffer(shape, dtype, device, trans: bool):
    """A dense tensor of `shape`, with axes 1 and 2 swapped if `trans`, and its strides in shape's order."""
    if not trans:
        return torch.empty(shape, dtype=dtype, device=device), None
    B, I, J, C = shape
    return torch.empty(B, J, I, C, dtype=dtype, device=device), _I3(I * J * C, C, I * C)


# ---- gradients ----------------------------------------------------------------------------------------
_KEEP_ALL = (0.0, 0, 0, None, None)


class _LayerNorm(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        out, st = _launch_norm(x, weight, bias, eps, out_dtype, True)
        ctx.save_for_backward(x, weight, bias, st)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, weight, bias, st = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, _, dw, db = _launch_norm_backward(dout, x, weight, bias, st, None, _KEEP_ALL, 0,
                                              (need[0], False, need[1], need[2]), x.dtype)
        return dx, dw, db, None, None


class _DropoutAdd(Function):
    @staticmethod
    def forward(ctx, z, y, state, draw, share):
        ctx.save_for_backward(state)  # a seed tensor that changes before the backward pass is found out
        ctx.draw, ctx.share, ctx.y_dtype = draw[:4], share, y.dtype
        return _launch_dropout_add(z, y, draw, share, None, z.dtype if z is not None else y.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        state, = ctx.saved_tensors
        dy = None
        if ctx.needs_input_grad[1]:
            dy = _launch_dropout_add(None, dout, (*ctx.draw, state), ctx.share, None, ctx.y_dtype)
        return (dout if ctx.needs_input_grad[0] else None), dy, None, None, None


class _DropoutAddLayerNorm(Function):
    @staticmethod
    def forward(ctx, z, y, weight, bias, state, eps, draw, share, out_dtype, trans_out):
        s, h, st = _launch_fused(z, y, weight, bias, eps, draw, share, out_dtype, trans_out, True)
        ctx.save_for_backward(s, weight, bias, st, state)
        ctx.draw, ctx.share, ctx.y_dtype, ctx.trans = draw[:4], share, y.dtype, trans_out
        ctx.set_materialize_grads(False)
        return s, h

    @staticmethod
    @once_differentiable
    def backward(ctx, ds, dh):
        s, weight, bias, st, state = ctx.saved_tensors
        need, draw = ctx.needs_input_grad, (*ctx.draw, state)
        if dh is None:  # the norm's output is not used
            dw = torch.zeros_like(weight) if need[2] else None
            db = torch.zeros_like(bias) if need[3] else None
            if ds is None:
                return (None, None, dw, db) + (None,) * 6
            dy = _launch_dropout_add(None, ds, draw, ctx.share, None, ctx.y_dtype) if need[1] else None
            return (ds if need[0] else None, dy, dw, db) + (None,) * 6
        if ctx.trans:
            dh = dh.transpose(1, 2)
        dz, dy, dw, db = _launch_norm_backward(dh, s, weight, bias, st, ds, draw, ctx.share, need[:4], ctx.y_dtype)
        return (dz, dy, dw, db) + (None,) * 6


def _records(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- calls --------------------------------------------------------------------------------------------
def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """(x - mean) * rsqrt(var + eps) * weight + bias over the last axis (1 to 8192 channels), in
    `out_dtype` (None: x's type).  Statistics are fp32, in two passes over registers.  Differentiable once
    in x, weight and bias.  `layer_norm(z.transpose(1, 2), ...)` reads z where it lies and gives the ending
    node's `xn`."""
    _on_gpu("layer_norm", x, weight, bias)
    _check_dim("layer_norm", x)
    _code(x, "x")
    out_dtype = out_dtype or x.dtype
    if out_dtype not in _CODES:
        raise _unsupported(f"out_dtype {out_dtype}")
    if x.dtype != torch.float32 and out_dtype != x.dtype:
        x = x.float()  # exact
    if _records(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps, out_dtype)
    return _launch_norm(x, weight, bias, eps, out_dtype, False)[0]


def dropout(x: torch.Tensor, p: float, seed: Seed, offset: int = 0, *, share: Sequence[int] = (),
            training: bool = True) -> torch.Tensor:
    """x with dropped values zero and kept ones scaled by 1 / (1 - p); differentiable once."""
    _on_gpu("dropout", x)
    _code(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("dropout: no channels")
    draw, bits = _draw("dropout", p, seed, offset, x.device, training), _share(share, x.dim())
    if _records(x):
        return _DropoutAdd.apply(None, x, draw[4], draw, bits)
    return _launch_dropout_add(None, x, draw, bits, None, x.dtype)


def _check_pair(what: str, z: torch.Tensor, y: torch.Tensor) -> None:
    if z.shape != y.shape:
        raise ValueError(f"{what}: z is {tuple(z.shape)}, y {tuple(y.shape)}")
    if z.dim() < 1 or z.shape[-1] < 1:
        raise ValueError(f"{what}: no channels")
    _code(z, "z")
    _code(y, "y")
    if z.dtype != torch.float32 and y.dtype != z.dtype:
        raise _unsupported(f"{what}: y is {y.dtype} on a {z.dtype} stream")


def dropout_add(z: torch.Tensor, y: torch.Tensor, p: float, seed: Seed, offset: int = 0, *, share: Sequence[int] = (),
                training: bool = True, inplace: bool = False) -> torch.Tensor:
    """z + dropout(y) in z's type, one rounding from fp32; differentiable once in z and y.  share: the axes
    that share one draw, e.g. (2, 3) of [B, N, N, C] for one draw per row.  inplace: write into z (no
    gradients); what a shared draw drops is then neither read nor written."""
    _on_gpu("dropout_add", z, y)
    _check_pair("dropout_add", z, y)
    draw, bits = _draw("dropout_add", p, seed, offset, z.device, training), _share(share, z.dim())
    if _records(z, y):
        if inplace:
            raise RuntimeError("dropout_add: inplace=True keeps no gradients (use torch.no_grad or detach)")
        return _DropoutAdd.apply(z, y, draw[4], draw, bits)
    if not inplace:
        return _launch_dropout_add(z, y, draw, bits, None, z.dtype)
    if z.numel() and (_four(z).data_ptr() != z.data_ptr() or (z.stride(-1) != 1 and z.shape[-1] != 1)):
        raise ValueError("dropout_add: inplace=True needs a z with a dense last axis whose leading axes join into three")
    if (z.numel() and (y.data_ptr() != z.data_ptr() or y.stride() != z.stride() or y.dtype != z.dtype)
            and _first(y) <= _last(z) and _first(z) <= _last(y)):
        raise ValueError("dropout_add: inplace=True, and y overlaps z")
    _launch_dropout_add(z, y, draw, bits, z, z.dtype)
    torch.autograd.graph.increment_version(z)
    return z


def dropout_add_layer_norm(z: torch.Tensor, y: torch.Tensor, weight: Optional[torch.Tensor],
                           bias: Optional[torch.Tensor], p: float, seed: Seed, offset: int = 0, *,
                           share: Sequence[int] = (), eps: float = 1e-5, out_dtype: Optional[torch.dtype] = None,
                           trans_out: bool = False, training: bool = True):
    """(s, h): s = dropout_add(z, y, ...) and h = layer_norm(s, ...) of s as it is held, in one pass, with the
    bits of the two calls; differentiable once in z, y, weight and bias (both gradients of s, the given
    one and the norm's, are joined in one backward pass).  trans_out: h with axes 1 and 2 swapped (dense)."""
    what = "dropout_add_layer_norm"
    _on_gpu(what, z, y, weight, bias)
    _check_pair(what, z, y)
    _check_dim(what, z)
    out_dtype = out_dtype or z.dtype
    if out_dtype not in _CODES or (z.dtype != torch.float32 and out_dtype != z.dtype):
        raise _unsupported(f"{what}: out_dtype {out_dtype} of a {z.dtype} stream")
    if trans_out and z.dim() != 4:
        raise ValueError(f"{what}: trans_out needs [B, I, J, C], got {tuple(z.shape)}")
    if y.dtype != z.dtype and y.dtype != out_dtype:
        y = y.float()  # exact
    draw, bits = _draw(what, p, seed, offset, z.device, training), _share(share, z.dim())
    if _records(z, y, weight, bias):
        return _DropoutAddLayerNorm.apply(z, y, weight, bias, draw[4], eps, draw, bits, out_dtype, trans_out)
    s, h, _ = _launch_fused(z, y, weight, bias, eps, draw, bits, out_dtype, trans_out, False)
    return s, h


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last axis through `layer_norm` (boltz_mlx/layers/norm.py:8-17): same parameters and
    names.  `f16` gives the 16-bit output that the next layer takes as `xn`."""

    def __init__(self, dim: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None,
                 dtype=None) -> None:
        super().__init__(dim, eps=eps, elementwise_affine=elementwise_affine, bias=bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise _unsupported(f"LayerNorm over {len(self.normalized_shape)} axes (one is supported)")

    def _check(self, x):
        if x.shape[-1:] != torch.Size(self.normalized_shape):
            raise ValueError(f"LayerNorm: last axis {tuple(x.shape[-1:])}, expected {tuple(self.normalized_shape)}")

    def forward(self, x: torch.Tensor, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        self._check(x)
        return layer_norm(x, self.weight, self.bias, self.eps, out_dtype)

    def f16(self, x: torch.Tensor, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        return self.forward(x, out_dtype=dtype)

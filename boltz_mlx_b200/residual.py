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

Gradients are those of reverse mode.  An input with a forward-mode tangent is refused, and so is a call under a tracer
(torch.jit.trace, make_fx, torch.export) or with fake tensors; torch.compile breaks its graph around a call.
"""

from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional, Sequence, Union

import torch
from torch import nn

from . import _lib

Seed = Union[int, torch.Tensor]


class PairDropout(NamedTuple):
    """Dropout of a pair layer's update, as the layers' `dropout=` takes it.  share: the axes of
    [B, N, N, C] that share one draw; None: the layer's own (one draw per row, per column for the
    ending node)."""

    p: float
    seed: Seed
    offset: int = 0
    share: Optional[Sequence[int]] = None


def forward_only(what: str, z: torch.Tensor) -> None:
    """The layers have no gradients: a result that would lose those of z without a word is refused."""
    if torch.is_grad_enabled() and z.requires_grad:
        raise RuntimeError(f"{what}: forward only, z's gradients would be lost (use torch.no_grad or detach)")


# ---- numbers --------------------------------------------------------------------------------------------
@lru_cache(maxsize=256)
def _share_bits(share: tuple, ndim: int) -> int:
    """The library's set of shared axes of a tensor of ndim axes: bit k = axis k of [n0, n1, n2, channels]."""
    axes = set()
    for a in share:
        if not isinstance(a, int) or not -ndim <= a < ndim:
            raise ValueError(f"share={share}: axes of a tensor of {ndim} axes")
        axes.add(a % ndim)
    if ndim > 4:
        lead = {a for a in axes if a < ndim - 3}
        if lead and len(lead) != ndim - 3:
            raise _lib.TriAttnUnsupported(
                _lib.EUNSUPPORTED,
                f"share={share}: of {ndim} axes the first {ndim - 3} are shared together or not at all")
        axes = {a - (ndim - 4) for a in axes if a >= ndim - 3} | ({0} if lead else set())
        ndim = 4
    return sum(1 << (a + 4 - ndim) for a in axes)


def _share(share, ndim: int) -> int:
    return _share_bits(share if type(share) is tuple else tuple(share), ndim) if share is not None else 0


def _draw(what: str, p: float, seed: Seed, offset: int, training: bool):
    """(p, seed, offset, seed tensor or None)"""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: p={p} must lie in [0, 1]")
    if isinstance(seed, torch.Tensor):
        if offset:
            raise ValueError(f"{what}: a seed tensor brings its own offset")
        return p if training else 0.0, 0, 0, seed
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        raise ValueError(f"{what}: seed and offset are numbers of 64 bits")
    return p if training else 0.0, seed, offset, None


# ---- calls --------------------------------------------------------------------------------------------
def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """(x - mean) * rsqrt(var + eps) * weight + bias over the last axis (1 to 8192 channels), in
    `out_dtype` (None: x's type).  Statistics are fp32, in two passes over registers.  Differentiable once
    in x, weight and bias.  `layer_norm(z.transpose(1, 2), ...)` reads z where it lies and gives the ending
    node's `xn`."""
    return _lib.residual().layer_norm(x, weight, bias, eps, out_dtype)


def dropout(x: torch.Tensor, p: float, seed: Seed, offset: int = 0, *, share: Sequence[int] = (),
            training: bool = True) -> torch.Tensor:
    """x with dropped values zero and kept ones scaled by 1 / (1 - p); differentiable once."""
    return _lib.residual().dropout(x, *_draw("dropout", p, seed, offset, training), _share(share, x.dim()))


def dropout_add(z: torch.Tensor, y: torch.Tensor, p: float, seed: Seed, offset: int = 0, *, share: Sequence[int] = (),
                training: bool = True, inplace: bool = False) -> torch.Tensor:
    """z + dropout(y) in z's type, one rounding from fp32; differentiable once in z and y.  share: the axes
    that share one draw, e.g. (2, 3) of [B, N, N, C] for one draw per row.  inplace: write into z (no
    gradients); what a shared draw drops is then neither read nor written."""
    return _lib.residual().dropout_add(z, y, *_draw("dropout_add", p, seed, offset, training), _share(share, z.dim()),
                                       inplace)


def dropout_add_layer_norm(z: torch.Tensor, y: torch.Tensor, weight: Optional[torch.Tensor],
                           bias: Optional[torch.Tensor], p: float, seed: Seed, offset: int = 0, *,
                           share: Sequence[int] = (), eps: float = 1e-5, out_dtype: Optional[torch.dtype] = None,
                           trans_out: bool = False, training: bool = True):
    """(s, h): s = dropout_add(z, y, ...) and h = layer_norm(s, ...) of s as it is held, in one pass, with the
    bits of the two calls; differentiable once in z, y, weight and bias (both gradients of s, the given
    one and the norm's, are joined in one backward pass).  trans_out: h with axes 1 and 2 swapped (dense)."""
    return _lib.residual().dropout_add_layer_norm(
        z, y, weight, bias, *_draw("dropout_add_layer_norm", p, seed, offset, training), _share(share, z.dim()), eps,
        out_dtype, trans_out)


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last axis through `layer_norm` (boltz_mlx/layers/norm.py:8-17): same parameters and
    names.  `f16` gives the 16-bit output that the next layer takes as `xn`."""

    def __init__(self, dim: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None,
                 dtype=None) -> None:
        super().__init__(dim, eps=eps, elementwise_affine=elementwise_affine, bias=bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise _lib.TriAttnUnsupported(_lib.EUNSUPPORTED,
                                          f"LayerNorm over {len(self.normalized_shape)} axes (one is supported)")

    def _check(self, x):
        if x.shape[-1:] != torch.Size(self.normalized_shape):
            raise ValueError(f"LayerNorm: last axis {tuple(x.shape[-1:])}, expected {tuple(self.normalized_shape)}")

    def forward(self, x: torch.Tensor, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        self._check(x)
        return layer_norm(x, self.weight, self.bias, self.eps, out_dtype)

    def f16(self, x: torch.Tensor, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        return self.forward(x, out_dtype=dtype)

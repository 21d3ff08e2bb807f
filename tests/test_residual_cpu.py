"""CPU: the residual path's generator and oracle against published vectors and differences, and every
refusal of the Python calls and of the C entry points (nothing is launched here)."""

import ctypes
import random

import numpy as np
import pytest
import torch

import boltz_mlx_b200 as b200
from boltz_mlx_b200 import _lib, residual
from boltz_mlx_b200.build import build
from oracle.residual_ref import (dropout_add_ref, keep_mask, layer_norm_grad_ref, layer_norm_ref, philox4x32, scale_of,
                                 words)

I3 = ctypes.c_int64 * 3


@pytest.fixture(scope="module")
def L():
    build()
    return _lib.lib()


# ---- generator ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("ctr,key,out", [  # the authors' known answers for philox4x32, 10 rounds
    ([0] * 4, [0] * 2, [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
    ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
    ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
     [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]),
])
def test_generator_known_answers(ctr, key, out):
    assert philox4x32(ctr, key) == out


def test_words_are_blocks_in_order():
    seed, offset = 0x123456789ABCDEF0, (7 << 32) | 3
    w = words(11, seed, offset)
    for e in range(11):
        block = philox4x32([e // 4, 0, offset & 0xFFFFFFFF, offset >> 32], [seed & 0xFFFFFFFF, seed >> 32])
        assert w[e] == block[e % 4]


def test_keep_mask_shares_axes_and_counts():
    m = keep_mask((2, 3, 4, 5), 0.3, 9, 1, share=(2, -1))
    assert m.shape == (2, 3, 1, 1)
    assert keep_mask((64,), 0.0, 1).all() and not keep_mask((64,), 1.0, 1).any()
    n = 1 << 16
    for p in (0.1, 0.25, 0.5):  # binomial: 6 standard deviations
        assert abs(keep_mask((n,), p, 5).mean() - (1 - p)) < 6 * (p * (1 - p) / n) ** 0.5


def test_oracle_gradient_against_differences():
    g = np.random.default_rng(3)
    x, w, b, dh = g.normal(size=(3, 7)) + 1.0, g.normal(size=7), g.normal(size=7), g.normal(size=(3, 7))
    _, xh, rstd = layer_norm_ref(x, w, b)
    dx, dw, db = layer_norm_grad_ref(dh, xh, rstd, w)
    h = 1e-5  # central differences: h^2 truncation (third derivatives of order 10) and 1e-16 / h rounding, both ~ 1e-9
    for t, d in ((x, dx), (w, dw), (b, db)):
        for i in np.ndindex(t.shape):
            keep = t[i]
            t[i] = keep + h
            up = (layer_norm_ref(x, w, b)[0] * dh).sum()
            t[i] = keep - h
            down = (layer_norm_ref(x, w, b)[0] * dh).sum()
            t[i] = keep
            assert abs((up - down) / (2 * h) - d[i]) < 1e-7


def test_dropout_ref_ignores_what_it_drops():
    y = np.full(256, np.nan)
    keep = keep_mask((256,), 0.5, 4)
    out = dropout_add_ref(np.ones(256), y, 0.5, 4)
    assert (out[~keep] == 1).all() and np.isnan(out[keep]).all()
    assert scale_of(1.0) == 0.0 and scale_of(0.75) == 4.0


def test_division_by_invariant():
    """The kernels' FastDiv, in Python integers: exact for every dividend below 2^31."""
    r = random.Random(1)

    def fast(n, d):
        l = 0
        while l < 31 and (1 << l) < d:
            l += 1
        m = ((((1 << l) - d) << 32) // d + 1) & 0xFFFFFFFF
        hi = (m * n) >> 32
        assert hi + n < 1 << 32
        return (hi + n) >> l

    for d in [1, 2, 3, 5, 7, 128, 333, 1024, 65537, (1 << 30) - 1, 1 << 30, (1 << 31) - 1] + [r.randrange(1, 1 << 31) for _ in range(300)]:
        for n in [0, 1, d - 1, d, min(2 * d - 1, (1 << 31) - 1), (1 << 31) - 1] + [r.randrange(1 << 31) for _ in range(50)]:
            assert fast(n, d) == n // d, (n, d)


# ---- shared axes ----------------------------------------------------------------------------------------
def test_share_of_fewer_and_more_axes():
    assert residual._share((2, 3), 4) == 0b1100 and residual._share([-1], 2) == 0b1000 and residual._share((), 4) == 0
    assert residual._share((0,), 2) == 0b0100
    assert residual._share((0, 1), 5) == 0b0001 and residual._share((2, 4), 5) == 0b1010
    with pytest.raises(_lib.TriAttnUnsupported):
        residual._share((0,), 5)
    with pytest.raises(ValueError):
        residual._share((4,), 4)


# ---- refusals: what can be refused anywhere comes before "needs CUDA tensors" ---------------------------
def _calls(z, y, p=0.1, seed=1, offset=0, **kw):
    """dropout_add and dropout_add_layer_norm on the same arguments"""
    yield lambda: b200.dropout_add(z, y, p, seed, offset, **kw)
    yield lambda: b200.dropout_add_layer_norm(z, y, None, None, p, seed, offset, **kw)


def test_calls_refuse_cpu_tensors(L):
    x = torch.zeros(2, 8)
    for f in (lambda: b200.layer_norm(x), lambda: b200.dropout(x, 0.1, 1), *_calls(x, x), lambda: b200.LayerNorm(8)(x),
              lambda: b200.dropout_add(x, x, 0.1, 1, inplace=True), lambda: b200.layer_norm(x, torch.ones(8), torch.ones(8))):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()


def test_numbers_are_refused(L):
    x = torch.zeros(2, 8)
    for kw in ({"p": -0.1}, {"p": 1.5}, {"p": float("nan")}, {"seed": -1}, {"seed": 1 << 64}, {"offset": -1},
               {"offset": 1 << 64}, {"share": (2,)}, {"share": (-3,)}, {"seed": torch.zeros(3, dtype=torch.int64)},
               {"seed": torch.zeros(2)}, {"seed": torch.zeros(4, dtype=torch.int64)[::2]},
               {"seed": torch.zeros(2, dtype=torch.int64), "offset": 5}):
        for f in _calls(x, x, **kw):
            with pytest.raises(ValueError):
                f()
        if "share" not in kw:
            kw = {"p": 0.1, "seed": 1, **kw}
            with pytest.raises(ValueError):
                b200.dropout(x, **kw)
    assert residual._draw("f", 0.4, 1, 2, False)[0] == 0.0


def test_tensors_are_refused(L):
    z = torch.zeros(2, 8)
    for a, b in ((z, z[:1]), (z, torch.zeros(8)), (torch.zeros(()), torch.zeros(())), (z[:, :0], z[:, :0])):
        for f in _calls(a, b):
            with pytest.raises(ValueError):
                f()
    for a, b in ((z.half(), z), (z.half(), z.bfloat16()), (z.double(), z.double()), (z, z.long())):
        for f in _calls(a, b):
            with pytest.raises(NotImplementedError):
                f()
    bad = [(z, torch.zeros(7), None), (z, None, torch.zeros(7)), (z, torch.zeros(1, 8), None),
           (z, torch.zeros(8), torch.zeros(8).half()), (torch.zeros(()), None, None), (z[:, :0], None, None)]
    for x, w, b in bad:
        with pytest.raises(ValueError):
            b200.layer_norm(x, w, b)
    with pytest.raises(ValueError):
        b200.dropout_add_layer_norm(z, z, torch.zeros(7), None, 0.1, 1)
    with pytest.raises(ValueError):
        b200.dropout_add_layer_norm(z, z, None, None, 0.1, 1, trans_out=True)
    for f in (lambda: b200.layer_norm(z, torch.zeros(8).double()), lambda: b200.layer_norm(torch.zeros(1, 8193)),
              lambda: b200.dropout_add_layer_norm(torch.zeros(1, 8193), torch.zeros(1, 8193), None, None, 0.1, 1),
              lambda: b200.layer_norm(z.long()), lambda: b200.layer_norm(z, out_dtype=torch.float64),
              lambda: b200.dropout_add_layer_norm(z.half(), z.half(), None, None, 0.1, 1, out_dtype=torch.bfloat16),
              lambda: b200.LayerNorm((4, 8)),
              lambda: b200.TriangleAttention(precision="fp32").norm_input(torch.zeros(1, 4, 4, 128))):
        with pytest.raises(NotImplementedError):
            f()
    with pytest.raises(ValueError):
        b200.LayerNorm(8)(torch.zeros(2, 9))


def test_in_place_is_refused(L):
    sq = torch.zeros(3, 3, 8)
    with pytest.raises(ValueError, match="overlaps"):
        b200.dropout_add(sq, sq.transpose(0, 1), 0.1, 1, inplace=True)
    with pytest.raises(ValueError, match="dense last axis"):
        b200.dropout_add(torch.zeros(8, 4).t(), torch.zeros(4, 8), 0.1, 1, inplace=True)
    with pytest.raises(RuntimeError, match="gradients"):
        b200.dropout_add(sq.clone().requires_grad_(), sq, 0.1, 1, inplace=True)


A = 4096  # an address that validation may look at but nothing may touch


def _ln(L, x=A, xd=0, xs=None, shape=(1, 2, 3), dim=8, w=A, b=A, pd=0, eps=1e-5, out=2 * A, od=0, os_=None):
    return L.triattn_layer_norm(x, xd, xs, I3(*shape) if shape else None, dim, w, b, pd, eps, out, od, os_, None, None, None)


def test_layer_norm_entry_refuses(L):
    assert _ln(L, shape=None) == _lib.EINVAL
    assert _ln(L, dim=0) == _lib.EINVAL
    assert _ln(L, dim=8193) == _lib.EUNSUPPORTED
    assert _ln(L, shape=(1, -1, 3)) == _lib.EINVAL
    assert _ln(L, shape=(1 << 20, 1 << 20, 1)) == _lib.EUNSUPPORTED
    assert _ln(L, shape=(1 << 31, 1, 1)) == _lib.EUNSUPPORTED
    assert _ln(L, x=None) == _lib.EINVAL and _ln(L, out=None) == _lib.EINVAL
    assert _ln(L, x=A + 2) == _lib.EINVAL and _ln(L, out=A + 1) == _lib.EINVAL and _ln(L, w=A + 2) == _lib.EINVAL
    assert _ln(L, xd=7) == _lib.EUNSUPPORTED and _ln(L, pd=3) == _lib.EUNSUPPORTED
    assert _ln(L, xd=1, od=2) == _lib.EUNSUPPORTED and _ln(L, xd=2, od=0) == _lib.EUNSUPPORTED
    assert _ln(L, eps=-1.0) == _lib.EINVAL and _ln(L, eps=float("nan")) == _lib.EINVAL and _ln(L, eps=float("inf")) == _lib.EINVAL
    assert _ln(L, xs=I3(0, -8, 8)) == _lib.EINVAL and _ln(L, out=A) == _lib.EINVAL
    # an output whose rows overlap: a stride below dim, zero, or two axes that meet
    assert _ln(L, os_=I3(0, 8, 4)) == _lib.EINVAL and _ln(L, os_=I3(0, 0, 8)) == _lib.EINVAL
    assert _ln(L, os_=I3(0, 16, 8)) == _lib.EINVAL
    # an empty call is nothing, wherever the empty axis stands
    assert _ln(L, shape=(0, 2, 3), x=None, out=None) == _lib.OK
    assert _ln(L, shape=(1 << 20, 1 << 20, 0), x=None, out=None) == _lib.OK
    assert "layer_norm" in L.triattn_last_error_string().decode()


def _da(L, z=A, zd=0, y=A, yd=0, shape=(1, 2, 3), dim=8, share=0, p=0.1, state=None, out=2 * A, od=0, zs=None):
    return L.triattn_dropout_add(z, zd, zs, y, yd, None, I3(*shape), dim, share, p, 1, 0, state, out, od, None, None)


def test_dropout_add_entry_refuses(L):
    assert _da(L, p=-0.5) == _lib.EINVAL and _da(L, p=1.01) == _lib.EINVAL and _da(L, p=float("nan")) == _lib.EINVAL
    assert _da(L, share=16) == _lib.EINVAL and _da(L, share=-1) == _lib.EINVAL
    assert _da(L, state=A + 4) == _lib.EINVAL
    assert _da(L, y=None) == _lib.EINVAL and _da(L, out=None) == _lib.EINVAL
    assert _da(L, zd=1, od=0) == _lib.EUNSUPPORTED and _da(L, zd=1, od=1, yd=0) == _lib.EUNSUPPORTED
    assert _da(L, z=None, yd=1, od=2) == _lib.EUNSUPPORTED and _da(L, yd=9) == _lib.EUNSUPPORTED
    assert _da(L, dim=(1 << 30) + 1) == _lib.EUNSUPPORTED
    assert _da(L, zs=I3(-1, 8, 8)) == _lib.EINVAL
    assert _da(L, out=A, zs=I3(64, 32, 16)) == _lib.EINVAL  # in place through other strides
    assert _da(L, shape=(3, 0, 2), y=None, out=None) == _lib.OK


def test_fused_entry_refuses(L):
    def f(zd=0, yd=0, od=0, s=2 * A, y=A, out=3 * A, p=0.1, share=0, dim=8, ss=None):
        return L.triattn_dropout_add_layer_norm(A, zd, None, y, yd, None, I3(1, 2, 3), dim, share, p, 1, 0, None, A, A, 0,
                                                1e-5, s, ss, out, od, None, None, None, None)

    assert f(s=A, ss=I3(64, 32, 16)) == _lib.EINVAL and f(out=A) == _lib.EINVAL and f(s=3 * A) == _lib.EINVAL

    assert f(s=None) == _lib.EINVAL and f(y=None) == _lib.EINVAL and f(out=None) == _lib.EINVAL
    assert f(p=2.0) == _lib.EINVAL and f(share=99) == _lib.EINVAL and f(dim=9000) == _lib.EUNSUPPORTED
    assert f(zd=1, yd=1, od=0) == _lib.EUNSUPPORTED and f(zd=0, yd=1, od=2) == _lib.EUNSUPPORTED
    assert f(zd=2, yd=0, od=2) == _lib.EUNSUPPORTED


def test_backward_entry_refuses(L):
    def f(dout=A, x=A, mean=A, rstd=A, dx=A, dw=A, ws=A, nbytes=1 << 30, xd=0, gd=0, shape=(1, 2, 3), dim=8):
        return L.triattn_layer_norm_backward(dout, gd, None, x, xd, None, I3(*shape), dim, A, 0, mean, rstd, None, None, 0,
                                             0.0, 0, 0, None, dx, None, 0, dw, None, ws, nbytes, None)

    assert f(dout=None) == _lib.EINVAL and f(x=None) == _lib.EINVAL
    assert f(mean=None) == _lib.EINVAL and f(rstd=None) == _lib.EINVAL and f(mean=A + 2) == _lib.EINVAL
    assert f(ws=None) == _lib.EINVAL and f(ws=A + 8) == _lib.EINVAL and f(nbytes=16) == _lib.ENOSPACE
    assert f(xd=1, gd=0) == _lib.EUNSUPPORTED and f(dim=0) == _lib.EINVAL and f(dx=A + 1) == _lib.EINVAL
    assert f(dx=None, dw=None) == _lib.OK  # nothing wanted
    assert L.triattn_layer_norm_backward_workspace_bytes(0, 8) == 0
    assert L.triattn_layer_norm_backward_workspace_bytes(4, 9000) == 0
    assert L.triattn_layer_norm_backward_workspace_bytes(1, 8) == 64

"""GPU: the residual path (LayerNorm, dropout, residual add, their fused form and gradients) against the
64-bit oracle (oracle/residual_ref.py).

Tolerances, element by element, from the kernels' arithmetic.  u = 2^-24 is the half step of fp32, U that of
the output's type.  A row sum has at most K = 16 + 9 + 2 additions on any value's way (16 in a lane, 9 levels
over 512 lanes) and a multiplication by fp32(1 / dim) (2 u), so with A = max |x| of the row
  |d mean| <= (K + 3) u A          (one more for the backward pass, which multiplies mean by rstd first)
  |d xh|   <= rstd (|d mean| + u (|x - mean| + A u)) + |xh| e_r,   e_r = relative error of rstd
  e_r      <= ((K + 6) u + 2 |d mean| rstd) / 2 + 4 u       (squares, sum, scaling, eps; rsqrt within 2 ulp = 4 u)
  |d h|    <= |w| |d xh| + 2 u (|w xh| + |b|) + U |h|
and for the backward pass, with g = dh w, c1 = mean(g), c2 = mean(g xh),
  |d c1|   <= (K + 3) u mean|g|,   |d c2| <= (K + 5) u mean|g xh| + mean(|g| |d xh|)
  |d dx|   <= rstd (u |g| + |d c1| + |xh| |d c2| + |c2| |d xh| + 4 u (|g| + |c1| + |xh c2|)) + |dx| (e_r + u) [+ u |ds|] + U |dx|
  |d dw|   <= sum(|dh| |d xh|) + Q u sum |dh xh|,   |d db| <= Q u sum |dh|  (+ U of the parameter's type)
where Q = 100 covers the longest way of a value in a column sum of up to 8192 rows (4 rows of a lane, 8 warps, at
most 592 / 16 partial rows a warp, 16 warps, and the butterflies).  Second-order terms: a factor 1.05.
The stream s is one fused multiply-add in fp32 and one rounding, which 64 bits followed by the two roundings
reproduce, so s, and dy of a plain dropout, are compared bit for bit.
"""

import numpy as np
import pytest
import torch

import boltz_mlx_b200 as b200
from boltz_mlx_b200 import PairDropout, _lib, dropout, dropout_add, dropout_add_layer_norm, layer_norm
from oracle.residual_ref import (dropout_add_ref, keep_mask, layer_norm_grad_ref, layer_norm_ref, scale_of, words)
from oracle.triattn_ref import make_params
from tests._util import module

pytestmark = pytest.mark.gpu

F, H, B = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F, F), (F, H), (F, B), (H, H), (B, B)]
u32 = 2.0 ** -24
K, Q = 27, 100


@pytest.fixture(autouse=True)
def _status_clean():
    _lib.device_status(clear=True)
    yield
    assert _lib.device_status(clear=True) == 0


def half(t):
    return torch.finfo(t).eps / 2


def f64(t):
    return t.detach().double().cpu().numpy()


def rounded(a, t):
    """a float64 array rounded to fp32 and from there to type t, as a tensor on the GPU."""
    return torch.from_numpy(a.astype(np.float32)).to(t).cuda()


def normal(shape, t, seed, mean=0.0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std + mean).to(t).cuda()


class Row:
    """What the bounds need of one LayerNorm, in float64."""

    def __init__(self, x, w, b, eps=1e-5):
        self.x = f64(x)
        self.w = f64(w) if w is not None else np.ones(self.x.shape[-1])
        self.b = f64(b) if b is not None else np.zeros(self.x.shape[-1])
        self.h, self.xh, self.rstd = layer_norm_ref(self.x, self.w, self.b, eps)
        A = np.abs(self.x).max(-1, keepdims=True)
        dmean = (K + 3) * u32 * A
        self.er = ((K + 6) * u32 + 2 * dmean * self.rstd) / 2 + 4 * u32
        self.dxh = self.rstd * (dmean + u32 * (np.abs(self.xh) / self.rstd + A * u32)) + np.abs(self.xh) * self.er

    def tol_h(self, t):
        tiny = torch.finfo(t).smallest_normal * half(t)  # half a step of the subnormal numbers
        return 1.05 * (np.abs(self.w) * self.dxh + 2 * u32 * (np.abs(self.w * self.xh) + np.abs(self.b))
                       + half(t) * np.abs(self.h)) + tiny

    def grads(self, dh, ds=None):
        """((dx, dw, db), (tolerance of the fp32 dx, of dw, of db) without the last rounding)"""
        dh = f64(dh)
        dx, dw, db = layer_norm_grad_ref(dh, self.xh, self.rstd, self.w)
        g = np.abs(dh * self.w)
        c1, c2 = (dh * self.w).mean(-1, keepdims=True), (dh * self.w * self.xh).mean(-1, keepdims=True)
        dc1 = (K + 3) * u32 * g.mean(-1, keepdims=True)
        dc2 = (K + 5) * u32 * (g * np.abs(self.xh)).mean(-1, keepdims=True) + (g * self.dxh).mean(-1, keepdims=True)
        a = np.abs(self.xh)
        tdx = self.rstd * (u32 * g + dc1 + a * dc2 + np.abs(c2) * self.dxh + 4 * u32 * (g + np.abs(c1) + a * np.abs(c2)))
        tdx = tdx + np.abs(dx) * (self.er + u32)
        if ds is not None:
            dx = dx + f64(ds)
            tdx = tdx + u32 * (np.abs(f64(ds)) + np.abs(dx))
        lead = tuple(range(dh.ndim - 1))
        tdw = (np.abs(dh) * self.dxh).sum(lead) + Q * u32 * np.abs(dh * self.xh).sum(lead)
        tdb = Q * u32 * np.abs(dh).sum(lead)
        return (dx, dw, db), (1.05 * tdx, 1.05 * tdw, 1.05 * tdb)


def close(got, ref, tol, t, what):
    """|got - ref| <= tol + the rounding to t (tol: without it)."""
    tol = tol + 1.01 * half(t) * np.abs(ref) + torch.finfo(t).smallest_normal * half(t)
    inside(got, ref, tol, what)


def inside(got, ref, tol, what):
    d = np.abs(f64(got) - ref)
    assert got.shape == ref.shape, what
    bad = ~(d <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} outside, worst {np.nanmax(d / tol):.3g} of its tolerance"


DIMS = [1, 2, 3, 7, 8, 16, 31, 32, 33, 64, 72, 96, 100, 127, 128, 129, 130, 256, 260, 333, 384, 510, 512, 520, 768, 1000,
        1024, 1032, 2047, 2048, 4096, 4100, 8191, 8192]


# ---- LayerNorm -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("tx,to", TYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_layer_norm_and_gradients(tx, to, dim):
    for rows in ((1,), (5, 7)) if dim > 512 else ((1,), (2, 3, 11), (67,)):
        x = normal((*rows, dim), tx, dim, 0.5, 2.0).requires_grad_()
        w = normal((dim,), F, dim + 1, 1.0, 0.2).requires_grad_()
        b = normal((dim,), F, dim + 2, 0.0, 0.2).requires_grad_()
        dh = normal((*rows, dim), to, dim + 3)
        r = Row(x, w, b)
        h = layer_norm(x, w, b, out_dtype=to)
        assert h.dtype == to
        inside(h, r.h, r.tol_h(to), f"h {rows} {dim}")
        with torch.no_grad():
            assert torch.equal(layer_norm(x, w, b, out_dtype=to), h)
        dx, dw, db = torch.autograd.grad(h, (x, w, b), dh)
        (rx, rw, rb), (tx_, tw, tb) = r.grads(dh)
        assert dx.dtype == tx and dw.dtype == F
        close(dx, rx, tx_, tx, f"dx {rows} {dim}")
        close(dw, rw, tw, F, f"dw {rows} {dim}")
        close(db, rb, tb, F, f"db {rows} {dim}")


@pytest.mark.parametrize("tx,to", [(F, B), (H, H)])
def test_layer_norm_every_width(tx, to):
    """A row's lanes and pieces change with the width: all widths up to 140, and every 13th to 2100."""
    for dim in [*range(1, 140), *range(140, 2100, 13), *range(248, 2100, 248), 3000, 5000, 6000, 7777]:
        x, w = normal((3, dim), tx, dim).requires_grad_(), normal((dim,), F, dim + 1, 1.0, 0.2).requires_grad_()
        dh = normal((3, dim), to, dim + 3)
        r = Row(x, w, None)
        h = layer_norm(x, w, out_dtype=to)
        inside(h, r.h, r.tol_h(to), f"h {dim}")
        (rx, rw, _), (tx_, tw, _) = r.grads(dh)
        dx, dw = torch.autograd.grad(h, (x, w), dh)
        close(dx, rx, tx_, tx, f"dx {dim}")
        close(dw, rw, tw, F, f"dw {dim}")


@pytest.mark.parametrize("tz,ty", [(F, F), (F, B), (H, H)])
def test_dropout_every_width(tz, ty):
    for dim in [*range(1, 70), *range(70, 600, 11), *range(96, 1100, 96)]:
        z, y = normal((5, dim), tz, 1), normal((5, dim), ty, 2)
        for share in ((), (0,), (1,)):
            ref = rounded(dropout_add_ref(f64(z), f64(y), 0.4, 3, 1, share), tz)
            assert torch.equal(dropout_add(z, y, 0.4, 3, 1, share=share), ref), (dim, share)
            s, _ = dropout_add_layer_norm(z, y, None, None, 0.4, 3, 1, share=share)
            assert torch.equal(s, ref), (dim, share)


@pytest.mark.parametrize("dim", [128, 131, 1024])
def test_layer_norm_many_rows(dim):
    """More rows than one sweep of the grid, not a multiple of anything; the same bits on every run."""
    x, dh = normal((8191, dim), B, 1, 0.3).requires_grad_(), normal((8191, dim), B, 2)
    w, b = normal((dim,), F, 3, 1.0, 0.2).requires_grad_(), normal((dim,), F, 4).requires_grad_()
    r = Row(x, w, b)
    (rx, rw, rb), (tx, tw, tb) = r.grads(dh)
    first = None
    for _ in range(3):
        h = layer_norm(x, w, b)
        got = (h, *torch.autograd.grad(h, (x, w, b), dh))
        if first is None:
            first = got
            inside(h, r.h, r.tol_h(B), "h")
            close(got[1], rx, tx, B, "dx")
            close(got[2], rw, tw, F, "dw")
            close(got[3], rb, tb, F, "db")
        assert all(torch.equal(p, q) for p, q in zip(first, got))


@pytest.mark.parametrize("dim,rows", [(8, 1700001), (32, 1700001), (64, 900000), (128, 700001), (136, 300001)])
def test_layer_norm_column_sums_of_many_rows(dim, rows):
    """Every CTA's partial row has its place: the column sums of so many rows that the work is shared out twice.  A
    lane adds up at most 4 rows of 32 batches before the joins: Q = 300."""
    x, dh = normal((rows, dim), B, 1, 0.3), normal((rows, dim), B, 2)
    w, b = normal((dim,), F, 3, 1.0, 0.2).requires_grad_(), torch.zeros(dim, device="cuda").requires_grad_()
    dw, db = torch.autograd.grad(layer_norm(x, w, b), (w, b), dh)
    xd, d = x.double(), dh.double()
    c = xd - xd.mean(-1, keepdim=True)
    rstd = (c.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    xh = c * rstd
    dxh = 1.05 * ((K + 3) * u32 * xd.abs().amax(-1, keepdim=True) * rstd * (1 + xh.abs()) + (K + 14) * u32 * xh.abs())
    tw = (d.abs() * dxh).sum(0) + 300 * u32 * (d * xh).abs().sum(0)
    assert ((dw.double() - (d * xh).sum(0)).abs() <= tw).all()
    assert ((db.double() - d.sum(0)).abs() <= 300 * u32 * d.abs().sum(0)).all()


@pytest.mark.parametrize("tp", [H, B])
def test_layer_norm_16_bit_parameters_over_many_ctas(tp):
    x, dh = normal((3001, 96), F, 1), normal((3001, 96), F, 2)
    w, b = normal((96,), tp, 3, 1.0, 0.2).requires_grad_(), normal((96,), tp, 4).requires_grad_()
    (_, rw, rb), (_, tw, tb) = Row(x, w, b).grads(dh)
    dw, db = torch.autograd.grad(layer_norm(x, w, b), (w, b), dh)
    close(dw, rw, tw, tp, "dw")
    close(db, rb, tb, tp, "db")


@pytest.mark.parametrize("tp", [F, H, B])
def test_layer_norm_parameters(tp):
    """Parameters of another type, one of them, none; only the gradients that are asked for."""
    x, dh = normal((9, 96), F, 1), normal((9, 96), F, 2)
    w, b = normal((96,), tp, 3, 1.0, 0.2), normal((96,), tp, 4)
    for ww, bb in ((w, b), (w, None), (None, b), (None, None)):
        r = Row(x, ww, bb)
        inside(layer_norm(x, ww, bb), r.h, r.tol_h(F), "h")
        leaves = [t.clone().requires_grad_() if t is not None else None for t in (x, ww, bb)]
        refs, tols = r.grads(dh)
        types = (F, tp, tp)
        for k in range(3):  # each alone
            if leaves[k] is None:
                continue
            ins = [t if i == k or t is None else t.detach() for i, t in enumerate(leaves)]
            d, = torch.autograd.grad(layer_norm(*ins), ins[k], dh)
            assert d.dtype == types[k]
            close(d, refs[k], tols[k], types[k], f"gradient {k}")


def test_layer_norm_far_from_zero_and_constant_rows():
    x = normal((17, 128), F, 1, 1000.0, 0.5)
    x[3] = 7.0
    x[4] = 0.0
    w, b = normal((128,), F, 2), normal((128,), F, 3)
    r = Row(x, w, b)
    inside(layer_norm(x, w, b), r.h, r.tol_h(F), "h")
    assert torch.equal(layer_norm(x, w, b)[4], b)
    big = torch.full((1, 128), 60000.0, dtype=H, device="cuda")
    big[0, ::2] = -60000.0
    out = layer_norm(big)
    assert torch.isfinite(out).all() and float((out.abs() - 1).abs().max()) <= 2 * half(H)


def test_layer_norm_bad_values_stay_in_their_row():
    x = normal((40, 128), F, 1).requires_grad_()
    with torch.no_grad():
        x[3, 5], x[11, 0], x[20, 127] = float("nan"), float("inf"), -float("inf")
    h = layer_norm(x, out_dtype=B)
    dx, = torch.autograd.grad(h, x, torch.ones_like(h))
    rows = torch.ones(40, dtype=torch.bool, device="cuda")
    rows[[3, 11, 20]] = False
    assert torch.isfinite(h[rows]).all() and torch.isfinite(dx[rows]).all()
    assert torch.isnan(h[~rows]).all()


@pytest.mark.parametrize("tx,to", [(F, B), (B, B), (F, F)])
@pytest.mark.parametrize("dim", [8, 128, 130, 1000])
def test_layer_norm_strides(tx, to, dim):
    base = normal((3, 9, 13, dim + 8), tx, 5, 0.2)
    w, b = normal((dim,), F, 6, 1.0, 0.1), normal((dim,), F, 7)
    views = {
        "transposed": base[..., :dim].transpose(1, 2), "gap": base[:, 1:, ::2, 8:], "odd start": base[..., 1:dim + 1],
        "expanded": base[:, :1, :, :dim].expand(3, 9, 13, dim), "matrix": base[0, 0, :, :dim], "vector": base[0, 0, 0, :dim],
        "five axes": base[..., :dim].unflatten(1, (3, 3)), "last axis strided": base[0, :, :, 8:].permute(2, 0, 1)[:, :, :],
    }
    for name, v in views.items():
        ww, bb = (w, b) if v.shape[-1] == dim else (None, None)
        plain = v.contiguous()
        h = layer_norm(v, ww, bb, out_dtype=to)
        inside(h, Row(plain, ww, bb).h, Row(plain, ww, bb).tol_h(to), name)
        leaf, g = v.detach().requires_grad_(), normal(tuple(v.shape), to, 8)
        flat = plain.clone().requires_grad_()
        d1, = torch.autograd.grad(layer_norm(leaf, ww, bb, out_dtype=to), leaf, g)
        (rx, _, _), (tx_, _, _) = Row(plain, ww, bb).grads(g)
        close(d1, rx, tx_, tx, name)
        if v.dim() >= 2:  # a gradient with strides of its own, and one that is expanded
            gt = g.transpose(0, 1).contiguous().transpose(0, 1)
            d2, = torch.autograd.grad(layer_norm(flat, ww, bb, out_dtype=to), flat, gt)
            close(d2, rx, tx_, tx, name + ": strided gradient")
    x = base[0, :, :, :dim].detach().requires_grad_()
    ww = w.clone().requires_grad_()
    layer_norm(x, ww, b, out_dtype=F if tx == F else tx).float().sum().backward()
    r = Row(x, ww, b)
    (rx, rw, _), (tx_, tw, _) = r.grads(torch.ones(x.shape))
    close(x.grad, rx, tx_, tx, "sum")
    close(ww.grad, rw, tw, F, "sum")


def test_layer_norm_empty_and_wider_results():
    w = torch.ones(16, device="cuda").requires_grad_()
    b = torch.ones(16, device="cuda").requires_grad_()
    for shape in ((0, 16), (3, 0, 16), (0, 5, 2, 16)):
        x = torch.zeros(shape, device="cuda").requires_grad_()
        h = layer_norm(x, w, b, out_dtype=B)
        assert h.shape == x.shape and h.dtype == B
        dx, dw, db = torch.autograd.grad(h, (x, w, b), torch.zeros_like(h))
        assert dx.shape == x.shape and not dw.any() and not db.any()
    x = normal((5, 64), B, 1).requires_grad_()  # a 16-bit stream with another result: through an exact fp32 copy
    h = layer_norm(x, out_dtype=F)
    r = Row(x, None, None)
    inside(h, r.h, r.tol_h(F), "bf16 -> fp32")
    g = normal((5, 64), F, 2)
    (rx, _, _), (tx, _, _) = r.grads(g)
    close(torch.autograd.grad(h, x, g)[0], rx, tx + half(B) * np.abs(rx), B, "dx")


def test_layer_norm_gradient_against_differences():
    """<dx, v> against (L(x + e v) - L(x - e v)) / 2 e with L = sum(h dh) summed in 64 bits from the kernel's h.
    Truncation e^2 / 6 |L'''| with e = 2^-6 and third derivatives of order |v|^3 rstd^3 |dh| ~ 1e1 per row: below
    1e-3 * 40 rows; rounding 2 u sum|h dh| / e ~ 1e-7 * 4e3 * 64 = 0.03."""
    x, v, dh = normal((40, 128), F, 1, 0, 2.0), normal((40, 128), F, 2, 0, 0.2), normal((40, 128), F, 3)
    w = normal((128,), F, 4, 1.0, 0.2)
    e = 2.0 ** -6
    up = (layer_norm(x + e * v, w).double() * dh.double()).sum()
    down = (layer_norm(x - e * v, w).double() * dh.double()).sum()
    leaf = x.clone().requires_grad_()
    dx, = torch.autograd.grad(layer_norm(leaf, w), leaf, dh)
    assert abs(float((up - down) / (2 * e)) - float((dx.double() * v.double()).sum())) < 0.07


# ---- dropout ---------------------------------------------------------------------------------------------
SHARES = [(), (2, 3), (1, 3), (1,), (0, 1, 2), (3,), (0, 1, 2, 3), (0,)]


@pytest.mark.parametrize("tz,ty", [(F, F), (F, H), (F, B), (H, H), (B, B)])
@pytest.mark.parametrize("share", SHARES)
@pytest.mark.parametrize("dim", [1, 3, 8, 33, 128, 129, 200, 264, 300, 333, 400, 510, 512, 1000])
def test_dropout_add(tz, ty, share, dim):
    shape, p, seed, offset = (2, 5, 7, dim), 0.3, 0xDEADBEEF12345678, (1 << 40) + 5
    z, y, g = normal(shape, tz, 1), normal(shape, ty, 2), normal(shape, tz, 3)
    ref = rounded(dropout_add_ref(f64(z), f64(y), p, seed, offset, share), tz)
    z1, y1 = z.clone().requires_grad_(), y.clone().requires_grad_()
    s = dropout_add(z1, y1, p, seed, offset, share=share)
    assert torch.equal(s, ref)
    dz, dy = torch.autograd.grad(s, (z1, y1), g)
    assert torch.equal(dz, g) and dy.dtype == ty
    assert torch.equal(dy, rounded(dropout_add_ref(None, f64(g), p, seed, offset, share), ty))
    assert torch.equal(dropout_add(z, y, p, seed, offset, share=share), ref)
    # alone
    y1 = y.clone().requires_grad_()
    d = dropout(y1, p, seed, offset, share=share)
    assert torch.equal(d, rounded(dropout_add_ref(None, f64(y), p, seed, offset, share), ty))
    dd, = torch.autograd.grad(d, y1, g.to(ty))
    assert torch.equal(dd, rounded(dropout_add_ref(None, f64(g.to(ty)), p, seed, offset, share), ty))
    if tz == ty:
        zz = z.clone()
        assert dropout_add(zz, y, p, seed, offset, share=share, inplace=True) is zz and torch.equal(zz, ref)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 4095, 4096, 4097, 70001])
def test_dropout_of_vectors(n):
    for t in (F, B):
        x = normal((n,), t, n)
        assert torch.equal(dropout(x, 0.5, 11, 3), rounded(dropout_add_ref(None, f64(x), 0.5, 11, 3), t))
        big = normal((n + 1,), t, n)  # an address that is not a multiple of 16
        assert torch.equal(dropout(big[1:], 0.5, 11, 3), rounded(dropout_add_ref(None, f64(big[1:]), 0.5, 11, 3), t))


@pytest.mark.parametrize("dim", [128, 36, 33])
@pytest.mark.parametrize("share", [(), (2, 3), (1, 3), (1,)])
def test_dropout_strides(dim, share):
    base, other = normal((2, 6, 9, dim + 4), F, 1), normal((2, 9, 6, dim), F, 2)
    for z in (base[..., :dim], base[..., 4:], base[..., 1:dim + 1], base[:, :, :1, :dim].expand(2, 6, 9, dim)):
        for y in (other.transpose(1, 2), other.transpose(1, 2).contiguous()):
            ref = rounded(dropout_add_ref(f64(z), f64(y), 0.4, 77, 1, share), F)
            assert torch.equal(dropout_add(z, y, 0.4, 77, 1, share=share), ref)
    z = base.clone()[..., :dim].transpose(1, 2)  # in place, through strides; what lies between the rows stays
    whole = z.transpose(1, 2)._base
    before = whole.clone()
    y = other
    ref = rounded(dropout_add_ref(f64(z), f64(y), 0.4, 77, 1, share), F)
    dropout_add(z, y, 0.4, 77, 1, share=share, inplace=True)
    assert torch.equal(z, ref) and torch.equal(whole[..., dim:], before[..., dim:])


def test_dropout_five_axes_and_empty():
    x = normal((2, 3, 2, 5, 8), F, 1)
    assert torch.equal(dropout(x, 0.5, 3), rounded(dropout_add_ref(None, f64(x), 0.5, 3), F))
    assert torch.equal(dropout(x, 0.5, 3, share=(2, 4)), rounded(dropout_add_ref(None, f64(x), 0.5, 3, 0, (2, 4)), F))
    assert torch.equal(dropout(x, 0.5, 3, share=(0, 1)), rounded(dropout_add_ref(None, f64(x), 0.5, 3, 0, (0, 1)), F))
    assert dropout(torch.zeros(0, 8, device="cuda"), 0.5, 1).shape == (0, 8)
    e = torch.zeros(3, 0, 8, device="cuda")
    assert dropout_add(e, e.clone(), 0.5, 1).shape == e.shape
    s, h = dropout_add_layer_norm(e, e.clone(), None, None, 0.5, 1)
    assert s.shape == h.shape == e.shape


def test_dropout_ends_of_the_range_and_bad_values():
    z, y = normal((6, 128), F, 1), normal((6, 128), F, 2)
    assert torch.equal(dropout_add(z, y, 0.0, 5), z + y)
    assert torch.equal(dropout_add(z, y, 0.9, 5, training=False), z + y)
    assert torch.equal(dropout_add(z, y, 1.0, 5), z)
    assert torch.equal(dropout_add(z, y, 2.0 ** -34, 5), z + y)
    y1 = y.clone().requires_grad_()
    dy, = torch.autograd.grad(dropout_add(z, y1, 1.0, 5), y1, z)
    assert not dy.any()
    for bad in (float("nan"), float("inf")):  # what is dropped contributes nothing
        for share in ((), (1,), (0,)):
            keep = torch.from_numpy(np.broadcast_to(keep_mask((6, 128), 0.5, 9, 0, share), (6, 128)).copy()).cuda()
            yb = torch.full_like(y, bad)
            s = dropout_add(z, yb, 0.5, 9, share=share)
            assert torch.equal(s[~keep], z[~keep]) and not torch.isfinite(s[keep]).any()
            s, h = dropout_add_layer_norm(z, yb, None, None, 0.5, 9, share=share)
            assert torch.equal(s[~keep], z[~keep])
    with pytest.raises(ValueError):
        dropout_add(z, y, 1.5, 5)
    with pytest.raises(ValueError):
        dropout_add(z, y, 0.5, -1)


def test_dropout_positions_beyond_32_bits():
    """More than 2^32 positions: the last rows take the generator's words there."""
    dim, rows = 4096, (1 << 20) + 5
    x = torch.ones(1, dim, dtype=B, device="cuda").expand(rows, dim)
    out = dropout(x, 0.5, 21, 2)
    for row in (0, 1 << 20, rows - 1):
        first = row * dim
        block = words_at(first, dim, 21, 2)
        assert torch.equal(out[row] != 0, torch.from_numpy(block >= 1 << 31).cuda())
    h = layer_norm(normal((1, dim), B, 1).expand(rows, dim))
    assert torch.equal(h[0], h[-1]) and torch.equal(h[0], h[1 << 20])


def words_at(first, count, seed, offset):
    """words(first + count) without its beginning (first: a multiple of 4)."""
    from oracle.residual_ref import philox4x32
    out = []
    for e in range(first // 4, (first + count + 3) // 4):
        out += philox4x32([e & 0xFFFFFFFF, e >> 32, offset, 0], [seed, 0])
    return np.array(out[:count], np.uint64)


def test_in_place_refusals():
    z = normal((2, 3, 8), F, 1)
    with pytest.raises(RuntimeError, match="gradients"):
        dropout_add(z.clone().requires_grad_(), z, 0.1, 1, inplace=True)
    with pytest.raises(_lib.TriAttnInvalid, match="overlap"):
        e = normal((1, 3, 8), F, 1).expand(2, 3, 8)
        dropout_add(e, z, 0.1, 1, inplace=True)
    sq = normal((3, 3, 8), F, 1)
    with pytest.raises(ValueError, match="overlaps"):
        dropout_add(sq, sq.transpose(0, 1), 0.1, 1, inplace=True)
    with pytest.raises(ValueError):
        dropout_add(normal((8, 4), F, 1).t(), normal((4, 8), F, 2), 0.1, 1, inplace=True)
    twice = sq.clone()
    dropout_add(twice, twice, 0.0, 1, inplace=True)
    assert torch.equal(twice, sq + sq)
    a = normal((4, 8), F, 3).requires_grad_()
    b = a * 1.0
    c = (b * b).sum()  # keeps b for its backward pass
    with torch.no_grad():
        dropout_add(b, sq.reshape(-1, 8)[:4], 0.5, 1, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        c.backward()


# ---- fused ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tz,ty,to", [(F, F, F), (F, F, H), (F, F, B), (F, H, H), (F, B, B), (H, H, H), (B, B, B)])
@pytest.mark.parametrize("share", [(), (2, 3), (1, 3), (1,)])
@pytest.mark.parametrize("dim", [8, 33, 64, 128, 200, 512, 1000, 2056])
def test_fused_is_the_two_calls_and_its_gradients(tz, ty, to, share, dim):
    shape, p, seed, offset = (2, 3, 5, dim), 0.25, 987654321, 4
    z, y = normal(shape, tz, 1, 0.5), normal(shape, ty, 2)
    w, b = normal((dim,), F, 3, 1.0, 0.2), normal((dim,), F, 4, 0.0, 0.2)
    ds, dh = normal(shape, tz, 5), normal(shape, to, 6)
    leaves = [t.clone().requires_grad_() for t in (z, y, w, b)]
    s, h = dropout_add_layer_norm(*leaves, p, seed, offset, share=share, out_dtype=to)
    assert torch.equal(s, rounded(dropout_add_ref(f64(z), f64(y), p, seed, offset, share), tz))
    assert torch.equal(s, dropout_add(z, y, p, seed, offset, share=share))
    assert torch.equal(h, layer_norm(s.detach(), w, b, out_dtype=to))
    s0, h0 = dropout_add_layer_norm(z, y, w, b, p, seed, offset, share=share, out_dtype=to)
    assert torch.equal(s0, s) and torch.equal(h0, h)
    r = Row(s, w, b)
    inside(h, r.h, r.tol_h(to), "h")
    dz, dy, dw, db = torch.autograd.grad((s, h), leaves, (ds, dh), retain_graph=True)
    (rz, rw, rb), (tz_, tw, tb) = r.grads(dh, ds)
    close(dz, rz, tz_, tz, "dz")
    close(dw, rw, tw, F, "dw")
    close(db, rb, tb, F, "db")
    keep, scale = keep_mask(shape, p, seed, offset, share), scale_of(p)
    ry = np.where(keep, rz * scale, 0.0)
    assert dy.dtype == ty and not dy[torch.from_numpy(np.broadcast_to(~keep, shape).copy()).cuda()].any()
    close(dy, ry, scale * tz_ + u32 * np.abs(ry), ty, "dy")
    # one of the two results alone
    dz, dy, dw = torch.autograd.grad(s, leaves[:3], ds, retain_graph=True, allow_unused=True)
    assert torch.equal(dz, ds) and not dw.any()
    assert torch.equal(dy, rounded(dropout_add_ref(None, f64(ds), p, seed, offset, share), ty))
    dz, dw = torch.autograd.grad(h, (leaves[0], leaves[2]), dh, retain_graph=True)
    (rz, _, _), (tz_, _, _) = r.grads(dh)
    close(dz, rz, tz_, tz, "dz of h alone")
    close(dw, rw, tw, F, "dw of h alone")
    dy, = torch.autograd.grad(h, leaves[1], dh)
    close(dy, np.where(keep, rz * scale, 0.0), scale * tz_ + u32 * np.abs(rz * scale), ty, "dy of h alone")


@pytest.mark.parametrize("tz,to", [(F, B), (F, F), (B, B)])
def test_fused_transposed_result_and_strides(tz, to):
    base = normal((2, 9, 6, 136), tz, 1)
    z, y = base[..., :128].transpose(1, 2), normal((2, 6, 9, 128), to, 2)
    w, b = normal((128,), F, 3, 1.0, 0.2), normal((128,), F, 4)
    s, h = dropout_add_layer_norm(z, y, w, b, 0.3, 5, share=(1, 3), out_dtype=to)
    zl, wl = z.detach().requires_grad_(), w.clone().requires_grad_()
    s1, ht = dropout_add_layer_norm(zl, y, wl, b, 0.3, 5, share=(1, 3), out_dtype=to, trans_out=True)
    assert ht.is_contiguous() and torch.equal(ht, h.transpose(1, 2)) and torch.equal(s1, s)
    g = normal((2, 9, 6, 128), to, 5)
    dz, dw = torch.autograd.grad(ht, (zl, wl), g)
    z2, w2 = z.contiguous().requires_grad_(), w.clone().requires_grad_()
    _, h2 = dropout_add_layer_norm(z2, y, w2, b, 0.3, 5, share=(1, 3), out_dtype=to)
    dz2, dw2 = torch.autograd.grad(h2, (z2, w2), g.transpose(1, 2))
    assert torch.equal(dz, dz2) and torch.equal(dw, dw2)
    with pytest.raises(ValueError):
        dropout_add_layer_norm(z[0], y[0], w, b, 0.3, 5, trans_out=True)


def test_fused_refusals():
    z, y = normal((4, 8), F, 1), normal((4, 8), F, 2)
    with pytest.raises(ValueError):
        dropout_add_layer_norm(z, y[:2], None, None, 0.1, 1)
    with pytest.raises(NotImplementedError):
        dropout_add_layer_norm(z.half(), y, None, None, 0.1, 1)
    with pytest.raises(NotImplementedError):
        dropout_add_layer_norm(z.half(), y.half(), None, None, 0.1, 1, out_dtype=B)
    with pytest.raises(ValueError):
        dropout_add_layer_norm(z, y, torch.ones(7, device="cuda"), None, 0.1, 1)
    with pytest.raises(ValueError):
        dropout_add_layer_norm(z, y, torch.ones(8), None, 0.1, 1)
    with pytest.raises(NotImplementedError):
        layer_norm(z.double())
    with pytest.raises(NotImplementedError):
        layer_norm(z, out_dtype=torch.float64)


# ---- autograd, graphs, streams -----------------------------------------------------------------------------
def test_gradients_of_broadcast_inputs():
    """A stream or an update that is broadcast takes the sum of its places' gradients: fp32 sums of 30 values, off by at
    most 30 u of their absolute sum."""
    z0, y = normal((1, 1, 1, 40), F, 1).requires_grad_(), normal((2, 3, 5, 40), F, 2).requires_grad_()
    ds, dh, w = normal((2, 3, 5, 40), F, 3), normal((2, 3, 5, 40), F, 4), normal((40,), F, 5, 1.0, 0.2)
    for a, b in ((z0.expand(2, 3, 5, 40), y), (y, z0.expand(2, 3, 5, 40))):
        s, h = dropout_add_layer_norm(a, b, w, None, 0.3, 11, share=(1,))
        d0, dy = torch.autograd.grad((s, h), (z0, y), (ds, dh))
        full_a, full_b = a.detach().clone().requires_grad_(), b.detach().clone().requires_grad_()
        s2, h2 = dropout_add_layer_norm(full_a, full_b, w, None, 0.3, 11, share=(1,))
        assert torch.equal(s, s2) and torch.equal(h, h2)
        da, db = torch.autograd.grad((s2, h2), (full_a, full_b), (ds, dh))
        wide, other = (da, db) if a is not y else (db, da)
        assert torch.equal(dy, other)
        ref, tol = wide.double().sum((0, 1, 2), keepdim=True), 30 * u32 * wide.double().abs().sum((0, 1, 2), keepdim=True)
        assert ((d0.double() - ref).abs() <= tol).all()


def test_checkpointed_step_draws_the_same_mask():
    from torch.utils.checkpoint import checkpoint

    z, y = normal((4, 6, 96), F, 1).requires_grad_(), normal((4, 6, 96), F, 2).requires_grad_()
    w, g = normal((96,), F, 3, 1.0, 0.1).requires_grad_(), normal((4, 6, 96), F, 4)

    def step(z, y, w):
        s, h = dropout_add_layer_norm(z, y * y, w, None, 0.4, 5, 9)
        return dropout_add(s, h, 0.4, 5, 10, share=(0,))

    plain = torch.autograd.grad(step(z, y, w), (z, y, w), g)
    again = torch.autograd.grad(checkpoint(step, z, y, w, use_reentrant=False), (z, y, w), g)
    assert all(torch.equal(a, b) for a, b in zip(plain, again))


def test_backward_twice():
    x, w = normal((4, 8), F, 1).requires_grad_(), normal((8,), F, 2).requires_grad_()
    h = layer_norm(x, w)
    first = torch.autograd.grad(h.sum(), (x, w), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(h.sum(), (x, w))))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(h.sum(), x)


def test_two_threads_at_once():
    import threading

    x, w, g = normal((300, 256), B, 1), normal((256,), F, 2), normal((300, 256), B, 3)
    errors = []

    def work(k):
        try:
            st = torch.cuda.Stream()
            st.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(st):
                for _ in range(30):
                    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
                    s, h = dropout_add_layer_norm(xs, g, ws, None, 0.5, k, 2)
                    d = torch.autograd.grad(h, (xs, ws), g)
                    ref = torch.autograd.grad(layer_norm(s.detach().requires_grad_(), ws), ws, g)
                    st.synchronize()
                    if not torch.equal(d[1], ref[0]):
                        errors.append(k)
        except Exception as e:  # noqa: BLE001 - reported by the main thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors


def test_backward_beyond_32_bits():
    """More than 2^32 elements: the last rows' gradients are those of the first, which have the same values."""
    dim, rows = 4096, (1 << 20) + 3
    x1, g1 = normal((1, dim), B, 1), normal((1, dim), B, 2)
    x, g = x1.expand(rows, dim).requires_grad_(), g1.expand(rows, dim)
    dx, = torch.autograd.grad(layer_norm(x), x, g)
    (rx, _, _), (tx, _, _) = Row(x1, None, None).grads(g1)
    close(dx[:1], rx, tx, B, "dx")
    for row in (1 << 19, 1 << 20, rows - 1):
        assert torch.equal(dx[row], dx[0])
    del dx
    s, h = dropout_add_layer_norm(x.detach(), g, None, None, 0.5, 3, share=(1,))
    keep = torch.from_numpy(keep_mask((rows, 1), 0.5, 3, 0)).cuda()[:, 0]
    for row in (0, 1, 2, rows - 3, rows - 2, rows - 1):
        assert torch.equal(s[row], (x1.float() + 2.0 * g1.float()).to(B)[0] if keep[row] else x1[0])
    assert torch.equal(h[rows - 1], layer_norm(s[rows - 1]))


def test_inference_mode():
    z, y, w = normal((4, 8), F, 1), normal((4, 8), F, 2), normal((8,), F, 3).requires_grad_()
    want = dropout_add(z, y, 0.5, 1)
    with torch.inference_mode():
        h = layer_norm(z, w)
        zi = z + 0.0
        assert dropout_add(zi, y, 0.5, 1, inplace=True) is zi and torch.equal(zi, want)
        s, _ = dropout_add_layer_norm(z, y, w, None, 0.5, 1)
        assert torch.equal(s, want)
    assert torch.equal(h, layer_norm(z, w).detach())


def test_second_derivatives_are_refused():
    x = normal((4, 8), F, 1).requires_grad_()
    d, = torch.autograd.grad(layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


def test_a_seed_tensor_gives_the_mask_of_its_numbers_and_may_not_change():
    z, y = normal((6, 40), F, 1), normal((6, 40), F, 2).requires_grad_()
    state = torch.tensor([123456789012345, 77], dtype=torch.int64, device="cuda")
    s = dropout_add(z, y, 0.5, state)
    assert torch.equal(s, dropout_add(z, y, 0.5, 123456789012345, 77))
    w = torch.ones(40, device="cuda")
    s2, h2 = dropout_add_layer_norm(z, y, w, None, 0.5, state)
    assert torch.equal(s2, s)
    dy, = torch.autograd.grad(s, y, z, retain_graph=True)
    assert torch.equal(dy, dropout(z, 0.5, 123456789012345, 77))
    state += 1
    for out in (s, h2):
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.grad(out.sum(), y)


def test_captured_step_draws_anew_on_each_replay():
    shape = (1, 12, 12, 128)
    z, y = normal(shape, F, 1).requires_grad_(), normal(shape, F, 2).requires_grad_()
    w, b = torch.ones(128, device="cuda").requires_grad_(), torch.zeros(128, device="cuda").requires_grad_()
    ds, dh = normal(shape, F, 3), normal(shape, B, 4)
    state = torch.tensor([5, 0], dtype=torch.int64, device="cuda")

    def step(seed, offset=0):
        s, h = dropout_add_layer_norm(z, y, w, b, 0.25, seed, offset, share=(2, 3), out_dtype=B)
        return (s, h, *torch.autograd.grad((s, h), (z, y, w, b), (ds, dh)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(state)
    masks = set()
    for offset in (3, 4, 3):
        state.copy_(torch.tensor([5, offset]))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step(5, offset)):
            assert torch.equal(got, want)
        masks.add(float(out[0].double().sum()))
    assert len(masks) == 2


def test_two_streams_at_once():
    xs = [normal((700, 384), F, k).requires_grad_() for k in range(2)]
    w = normal((384,), F, 9).requires_grad_()
    g = normal((700, 384), F, 10)
    want = [torch.autograd.grad(layer_norm(x, w), (x, w), g) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(torch.autograd.grad(layer_norm(xs[k], w), (xs[k], w), g))
    torch.cuda.synchronize()
    for k in range(2):
        for d in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(d, want[k]))


# ---- the operators as the framework uses them ----------------------------------------------------------------
def test_layer_norm_module():
    ln = b200.LayerNorm(128).cuda()
    with torch.no_grad():
        ln.weight.copy_(normal((128,), F, 1, 1.0, 0.1))
        ln.bias.copy_(normal((128,), F, 2))
    assert isinstance(ln, torch.nn.LayerNorm) and sorted(ln.state_dict()) == ["bias", "weight"]
    x = normal((3, 5, 128), F, 3)
    r = Row(x, ln.weight, ln.bias)
    inside(ln(x), r.h, r.tol_h(F), "module")
    assert ln.f16(x).dtype == H and ln.f16(x, B).dtype == B
    with pytest.raises(ValueError):
        ln(x[..., :64])
    ln(x).sum().backward()
    close(ln.bias.grad, np.full(128, 15.0), np.zeros(128), F, "bias gradient")  # fifteen ones: exact
    for plain in (b200.LayerNorm(128, elementwise_affine=False).cuda(), b200.LayerNorm(128, bias=False).cuda()):
        assert torch.equal(plain(x), layer_norm(x))
    half = b200.LayerNorm(128).cuda().bfloat16()
    assert half(x.bfloat16()).dtype == B and half(x).dtype == F


@pytest.mark.parametrize("precision", ["bf16", "fp16"])
@pytest.mark.parametrize("starting", [True, False])
def test_norm_input_feeds_the_layer(precision, starting):
    """xn from norm_input gives the layer's own result within one more rounding of xn to 16 bits (the layer
    rounds the same LayerNorm to the same type, by other sums: a last-bit difference of xn at most)."""
    mod = module(make_params(5), starting, precision)
    z, m = normal((1, 40, 40, 128), F, 1), torch.ones(1, 40, 40, device="cuda")
    xn = mod.norm_input(z)
    zt = z if starting else z.transpose(1, 2)
    r = Row(zt, mod.layer_norm.weight, mod.layer_norm.bias)
    inside(xn, r.h, r.tol_h(xn.dtype), "xn")
    y, y0 = mod(z, m, xn=xn), mod(z, m)
    assert float((y - y0).abs().max()) <= 2e-2 and float((y - y0).abs().mean()) <= 5e-3


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
def test_layers_with_dropout(precision):
    """forward_residual and f16_addln with dropout are the operators on the layer's own update."""
    z, m = normal((1, 33, 33, 128), F, 1), torch.ones(1, 33, 33, device="cuda")
    m[:, 30:] = 0
    start, end = module(make_params(1), True, precision), module(make_params(2), False, precision)
    mul = b200.TriangleMultiplicationOutgoing(128, precision=precision).cuda()
    ln = torch.nn.LayerNorm(128).cuda()
    for layer, share in ((start, (2, 3)), (end, (1, 3)), (mul, (2, 3))):
        y = layer(z, m)
        for d in (PairDropout(0.25, 7, 3), PairDropout(0.25, 7, 3, (1,))):
            ax = share if d.share is None else d.share
            want = dropout_add(z, y, 0.25, 7, 3, share=ax)
            assert torch.equal(layer.forward_residual(z, m, dropout=d), want)
            zi = z.clone()
            assert layer.forward_residual(zi, m, dropout=d, inplace=True) is zi and torch.equal(zi, want)
        if precision == "fp32":
            continue
        args = (None,) if layer is mul else (layer.norm_input(z),)
        if layer is not mul:
            y = layer(z, m, xn=args[0])
        s, h = layer.f16_addln(z, m, *args, ln, dropout=PairDropout(0.25, 7, 3))
        want = dropout_add_layer_norm(z, y, ln.weight.detach(), ln.bias.detach(), 0.25, 7, 3, share=share, out_dtype=B)
        assert torch.equal(s, want[0]) and torch.equal(h, want[1])
        with pytest.raises(NotImplementedError):
            layer.f16_addln(z, m, *args, ln, w_tb=start.tb_weight16(), dropout=PairDropout(0.25, 7))
    if precision == "bf16":
        s, ht = start.f16_addln(z, m, start.norm_input(z), ln, trans_out=True, dropout=PairDropout(0.25, 7, 3))
        assert torch.equal(ht.transpose(1, 2), start.f16_addln(z, m, start.norm_input(z), ln, dropout=PairDropout(0.25, 7, 3))[1])


def test_a_chain_of_the_operators_and_its_gradients():
    """Two residual steps behind one another, as a pair block in training runs them, with elementwise updates:
    gradients of the chain against the same chain in 64 bits.  Each backward stage adds a relative error of at
    most a few hundred u to gradients of the size of their row's largest: 2e-4 of the largest is far above
    that and far below any wrong factor."""
    shape, p = (1, 9, 11, 128), 0.25
    z, c1, c2 = normal(shape, F, 1), normal(shape, F, 2), normal(shape, F, 3)
    w = [normal((128,), F, 4 + k, 1.0, 0.2) for k in range(3)]
    b = [normal((128,), F, 8 + k, 0.0, 0.2) for k in range(3)]
    g = normal(shape, F, 12)

    def chain(z, w, b, norm, fused):
        h = norm(z, w[0], b[0])
        s, h = fused(z, h * c1.to(h.dtype), w[1], b[1], 0, (2, 3))
        s, h = fused(s, h * c2.to(h.dtype), w[2], b[2], 1, (1, 3))
        return s + h

    leaves = [t.clone().requires_grad_() for t in (z, *w, *b)]
    out = chain(leaves[0], leaves[1:4], leaves[4:], layer_norm,
                lambda z, y, w, b, o, share: dropout_add_layer_norm(z, y, w, b, p, 31, o, share=share))
    got = torch.autograd.grad(out, leaves, g)

    wide = [t.double().requires_grad_() for t in (z, *w, *b)]

    def norm64(x, w, b):
        c = x - x.mean(-1, keepdim=True)
        return c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * w + b

    def fused64(z, y, w, b, o, share):
        keep = torch.from_numpy(keep_mask(shape, p, 31, o, share)).cuda()
        s = z + torch.where(keep, y * scale_of(p), 0.0)
        return s, norm64(s, w, b)

    ref = chain(wide[0], wide[1:4], wide[4:], norm64, fused64)
    for a, r in zip(got, torch.autograd.grad(ref, wide, g.double())):
        assert float((a.double() - r).abs().max()) <= 2e-4 * float(r.abs().max())


@pytest.mark.parametrize("dim,rows", [(1, 1700003), (4, 1700003), (7, 1700003), (13, 1700003), (20, 900001), (31, 900001), (63, 900001),
                                      (81, 500001), (100, 400001), (420, 100001)])
def test_narrow_odd_rows_column_sums(dim, rows):
    """Several rows to a warp, over more rows than one share of the work: the column sums with the bound of the other widths
    (a lane adds up at most 4 rows of 32 batches before the joins: 300 roundings)."""
    test_layer_norm_column_sums_of_many_rows(dim, rows)


@pytest.mark.parametrize("tz,to", [(F, B), (H, H)])
@pytest.mark.parametrize("dim", [1, 6, 8, 13, 16, 17, 31, 47, 63, 65])
def test_narrow_rows_to_the_last(dim, tz, to):
    """Warps and CTAs that the rows do not fill: every row's result and gradients, and nothing behind the last row."""
    for rows in (1, 3, 31, 32, 33, 1023, 4099):
        both = normal((2, rows + 2, dim), tz, rows)
        y, ds, dh = normal((rows, dim), tz, 5), normal((rows, dim), tz, 6), normal((rows, dim), to, 7)
        z = both[0, :rows].clone().requires_grad_()
        w = normal((dim,), F, 3, 1.0, 0.2).requires_grad_()
        y.requires_grad_()
        s, h = dropout_add_layer_norm(z, y, w, None, 0.4, 3, 1, out_dtype=to)
        ref = rounded(dropout_add_ref(f64(z), f64(y), 0.4, 3, 1, ()), tz)
        assert torch.equal(s, ref)
        r = Row(s, w, None)
        inside(h, r.h, r.tol_h(to), "h")
        (rz, _, _), (tz_, _, _) = r.grads(dh, ds)
        dz, dy, dw = torch.autograd.grad((s, h), (z, y, w), (ds, dh))
        close(dz, rz, tz_, tz, "dz")
        keep = dropout_add_ref(None, np.ones((rows, dim)), 0.4, 3, 1, ()) != 0
        assert (dy.double().cpu().numpy()[~keep] == 0).all()
        out = both[1].clone()
        before = out.clone()
        dropout_add(out[:rows], y.detach(), 0.4, 3, 1, share=(0,), inplace=True)
        assert torch.equal(out[:rows], rounded(dropout_add_ref(f64(before[:rows]), f64(y), 0.4, 3, 1, (0,)), tz))
        assert torch.equal(out[rows:], before[rows:])


@pytest.mark.parametrize("tz,ty", [(F, F), (F, B), (H, H)])
@pytest.mark.parametrize("share", [(0,), (1, 2), (1,)])
@pytest.mark.parametrize("dim", [513, 514, 516, 520, 777, 1028, 1996, 2050, 2560, 4100, 4877, 6144, 8184, 8191, 8192, 8193, 8200])
def test_dropout_wide_rows(tz, ty, share, dim):
    z, y = normal((2, 5, dim), tz, 1), normal((5, 2, dim), ty, 2).transpose(0, 1)
    ref = rounded(dropout_add_ref(f64(z), f64(y), 0.4, 3, 1, share), tz)
    assert torch.equal(dropout_add(z, y, 0.4, 3, 1, share=share), ref)
    assert torch.equal(dropout_add(z, y.contiguous(), 0.4, 3, 1, share=share), ref)
    if tz == ty:
        dropout_add(z, y, 0.4, 3, 1, share=share, inplace=True)
        assert torch.equal(z, ref)

"""GPU: calls of the residual path at the edges of what PyTorch and the C ABI allow."""

import ctypes

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

from boltz_mlx_b200 import _lib, dropout, dropout_add, dropout_add_layer_norm, layer_norm
from oracle.residual_ref import dropout_add_ref, keep_mask, scale_of
from tests.test_gpu_residual import B, F, H, Row, close, f64, half, inside, normal, rounded, u32

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status_clean():
    _lib.device_status(clear=True)
    yield
    assert _lib.device_status(clear=True) == 0


def test_forward_mode_is_refused():
    """Forward over the calls and forward over their backward passes: a tangent is refused, never dropped."""
    x, y, w = normal((3, 40), F, 1), normal((3, 40), F, 2), normal((40,), F, 3)
    leaf = x.clone().requires_grad_()
    ends = [layer_norm(leaf, w), dropout(leaf, 0.25, 1), dropout_add(y, leaf, 0.25, 1),
            dropout_add_layer_norm(leaf, y, w, None, 0.25, 1)[1], *dropout_add_layer_norm(y, leaf, w, None, 0.25, 1)]
    through = [dropout_add(leaf, y, 0.25, 1), dropout_add_layer_norm(leaf, y, w, None, 0.25, 1)[0]]
    with fwAD.dual_level():
        for t in (x, leaf):
            d = fwAD.make_dual(t, torch.ones_like(t))
            for f in (lambda: layer_norm(d, w), lambda: layer_norm(x, d[0]), lambda: dropout(d, 0.25, 1),
                      lambda: dropout_add(d, y, 0.25, 1), lambda: dropout_add(y, d, 0.25, 1),
                      lambda: dropout_add_layer_norm(d, y, w, None, 0.25, 1),
                      lambda: dropout_add_layer_norm(y, d, w, None, 0.25, 1)):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    f()
        g = fwAD.make_dual(y, torch.ones_like(y))
        for e in ends:
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(e, leaf, g, retain_graph=True)
        for e in through:  # the stream's gradient is the given one, and so is its tangent
            d = fwAD.unpack_dual(torch.autograd.grad(e, leaf, g, retain_graph=True)[0])
            assert torch.equal(d.primal, y) and torch.equal(d.tangent, torch.ones_like(y))
    for e in ends + through:  # the graphs are still good
        assert torch.isfinite(torch.autograd.grad(e, leaf, y, retain_graph=True)[0]).all()


def test_tracing_is_refused():
    """A traced call, a traced backward pass, and an in-place call on real tensors among fake ones: none is recorded as
    its uninitialised result, none changes anything."""
    x, y = normal((3, 40), F, 1), normal((3, 40), F, 2)
    leaf = x.clone().requires_grad_()
    calls = [lambda t: layer_norm(t), lambda t: dropout(t, 0.25, 1), lambda t: dropout_add(t, y, 0.25, 1),
             lambda t: dropout_add_layer_norm(t, y, None, None, 0.25, 1)[1]]
    for f in calls:
        h = f(leaf)
        g, = torch.autograd.grad(h, leaf, y, retain_graph=True)
        for trace in (lambda f: torch.jit.trace(f, (x,), check_trace=False), lambda f: make_fx(f)(x),
                      lambda f: make_fx(f, pre_dispatch=True)(x)):
            with pytest.raises(NotImplementedError, match="tracing"):
                trace(f)
        if f is not calls[2]:  # the stream's gradient of dropout_add is the given one
            with pytest.raises(RuntimeError, match="tracing"):
                make_fx(lambda g: torch.autograd.grad(h, leaf, g, retain_graph=True)[0])(y)
        with FlopCounterMode(display=False):
            assert torch.equal(f(x), h) and torch.equal(torch.autograd.grad(h, leaf, y)[0], g)
    z = x.clone()
    with FakeTensorMode():
        with pytest.raises(NotImplementedError, match="fake"):
            dropout_add(z, y, 0.25, 1, inplace=True)
    assert torch.equal(z, x)
    compiled = torch.compile(lambda t: layer_norm(t * 1.0) + 1.0, backend="eager")
    assert torch.equal(compiled(x), layer_norm(x) + 1.0)


@pytest.mark.parametrize("tx,to", [(F, F), (F, B), (H, H)])
@pytest.mark.parametrize("dim", [8, 13, 128, 333, 1000])
@pytest.mark.parametrize("rows", [1, 3, 351])
def test_gradients_of_rows_that_start_anywhere(tx, to, dim, rows):
    """x and both gradients as views from an odd element on, in rows that fill neither the warps nor the CTAs: what stands
    for the rows behind the last is zero, and copied from an address that a copy may have."""
    def at_one(t):
        r = torch.full((rows * dim + 9,), float("nan"), dtype=t.dtype, device="cuda")
        r[1:1 + rows * dim] = t.reshape(-1)
        return r[1:1 + rows * dim].view(rows, dim)

    x, y, w = at_one(normal((rows, dim), tx, 1, 0.5)), at_one(normal((rows, dim), tx, 2)), normal((dim,), F, 3, 1.0, 0.2)
    ds, dh = at_one(normal((rows, dim), tx, 5)), at_one(normal((rows, dim), to, 6))
    assert x.data_ptr() % 16 == x.element_size()
    x.requires_grad_(), w.requires_grad_()
    h = layer_norm(x, w, out_dtype=to)
    r = Row(x, w, None)
    inside(h, r.h, r.tol_h(to), "h")
    (rx, rw, _), (tx_, tw, _) = r.grads(dh)
    dx, dw = torch.autograd.grad(h, (x, w), dh)
    close(dx, rx, tx_, tx, "dx")
    close(dw, rw, tw, F, "dw")
    s, h = dropout_add_layer_norm(x, y, w, None, 0.25, 7, out_dtype=to)
    r = Row(s, w, None)
    (rx, rw, _), (tx_, tw, _) = r.grads(dh, ds)
    dx, dw = torch.autograd.grad((s, h), (x, w), (ds, dh))
    close(dx, rx, tx_, tx, "dz")
    close(dw, rw, tw, F, "dw of the fused call")


C_TYPES = {F: _lib.F32, H: _lib.F16, B: _lib.BF16}


def c_backward(x, dh, w, stats, dw, ws):
    """triattn_layer_norm_backward for dw alone, on the current stream, into a workspace of the caller's."""
    rows, dim = x.shape
    _lib.check(_lib.lib().triattn_layer_norm_backward(
        dh.data_ptr(), C_TYPES[dh.dtype], None, x.data_ptr(), C_TYPES[x.dtype], None, (ctypes.c_int64 * 3)(1, 1, rows), dim,
        w.data_ptr(), C_TYPES[w.dtype], stats.data_ptr(), stats.data_ptr() + 4 * rows, None, None, 0, 0.0, 0, 0, None, None, None,
        C_TYPES[x.dtype], dw.data_ptr(), None, ws.data_ptr(), ws.numel(), _lib.stream_handle(x.device)))


@pytest.mark.parametrize("rows,dim,t,tp", [(200001, 128, F, F), (200001, 128, B, B), (3001, 64, F, H), (8192, 4096, B, F),
                                           (777, 1000, H, F)])
def test_a_workspace_used_by_one_call_behind_another(rows, dim, t, tp):
    """The kernel that joins the partial sums is there before they are written.  Two calls in turn through one workspace, with
    nothing between them, give the bits that each gives through one of its own."""
    w = normal((dim,), tp, 1, 1.0, 0.2)
    size = _lib.lib().triattn_layer_norm_backward_workspace_bytes(rows, dim)
    sides = []
    for seed in (2, 3):
        x, dh = normal((rows, dim), t, seed, 0.5), normal((rows, dim), t, seed + 10)
        x64 = x.double()
        stats = torch.stack([x64.mean(-1), (x64.var(-1, unbiased=False) + 1e-5).rsqrt()]).float().contiguous()
        own = torch.empty_like(w)
        c_backward(x, dh, w, stats, own, torch.empty(size, dtype=torch.uint8, device="cuda"))
        xh = (x64 - stats[0].double()[:, None]) * stats[1].double()[:, None]
        ref = (dh.double() * xh).sum(0)
        # as many roundings as the longest way of a value through 200,001 rows of sums has, and those of xh
        tol = 400 * u32 * (dh.double() * xh).abs().sum(0) + 4 * u32 * (dh.double().abs() * (1 + xh.abs())).sum(0)
        assert ((own.double() - ref).abs() <= tol + 1.01 * half(tp) * ref.abs()).all()
        sides.append((x, dh, stats, own))
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    got = [torch.empty((20, dim), dtype=tp, device="cuda") for _ in sides]
    for k in range(20):
        for (x, dh, stats, _), out in zip(sides, got):
            c_backward(x, dh, w, stats, out[k], ws)
    for (*_, own), out in zip(sides, got):
        assert torch.equal(out, own.expand(20, dim))


def test_outputs_that_are_inputs():
    """What the C entries allow: an output at the place of the tensor that it is computed from, and tensors side by side in
    the rows of one buffer, equal the calls with memory of their own bit for bit."""
    L, shape, dim, p = _lib.lib(), (2, 5, 7), 136, 0.25
    i3 = (ctypes.c_int64 * 3)(*shape)
    stream = _lib.stream_handle(torch.device("cuda"))
    for t in (F, H):
        c = C_TYPES[t]
        z, y, ds, dh = (normal((*shape, dim), t, k, 0.5) for k in range(4))
        w = normal((dim,), F, 5, 1.0, 0.2)

        def add(z, zs, y, ys, out, os_, share):
            _lib.check(L.triattn_dropout_add(z, c, zs, y, c, ys, i3, dim, share, p, 5, 0, None, out, c, os_, stream))

        for share in (0, 8, 12, 4):
            want = torch.empty_like(z)
            add(z.data_ptr(), None, y.data_ptr(), None, want.data_ptr(), None, share)
            got = y.clone()  # out is y
            add(z.data_ptr(), None, got.data_ptr(), None, got.data_ptr(), None, share)
            assert torch.equal(got, want)
            side = torch.stack([z, torch.zeros_like(z), y], -2)  # z, out and y side by side
            q, s = side.data_ptr(), (ctypes.c_int64 * 3)(5 * 7 * 3 * dim, 7 * 3 * dim, 3 * dim)
            step = dim * z.element_size()
            add(q, s, q + 2 * step, s, q + step, s, share)
            assert torch.equal(side[..., 1, :], want) and torch.equal(side[..., 0, :], z) and torch.equal(side[..., 2, :], y)

        def fused(z, y, s, out):
            st = torch.empty((2, 70), device="cuda")
            _lib.check(L.triattn_dropout_add_layer_norm(
                z.data_ptr(), c, None, y.data_ptr(), c, None, i3, dim, 0, p, 5, 0, None, w.data_ptr(), None, _lib.F32, 1e-5,
                s.data_ptr(), None, out.data_ptr(), c, None, st.data_ptr(), st.data_ptr() + 280, stream))
            return s, out, st

        s, h, st = fused(z, y, torch.empty_like(z), torch.empty_like(z))
        for into in ("z", "y"):
            zc, yc = z.clone(), y.clone()
            got = fused(zc, yc, zc if into == "z" else yc, torch.empty_like(z))
            assert all(torch.equal(a, b) for a, b in zip(got, (s, h, st)))
        zc, yc = z.clone(), y.clone()
        assert all(torch.equal(a, b) for a, b in zip(fused(zc, yc, zc, yc), (s, h, st)))

        def back(dh, x, ds, dx, dy):
            ws = torch.empty(L.triattn_layer_norm_backward_workspace_bytes(70, dim), dtype=torch.uint8, device="cuda")
            dw = torch.empty_like(w)
            _lib.check(L.triattn_layer_norm_backward(
                dh.data_ptr(), c, None, x.data_ptr(), c, None, i3, dim, w.data_ptr(), _lib.F32, st.data_ptr(), st.data_ptr() + 280,
                ds.data_ptr(), None, 0, p, 5, 0, None, dx.data_ptr(), dy.data_ptr(), c, dw.data_ptr(), None, ws.data_ptr(),
                ws.numel(), stream))
            return dx, dy, dw

        want = back(dh, s, ds, torch.empty_like(z), torch.empty_like(z))
        for a, b in ((0, 1), (1, 2), (2, 0)):
            given = [dh.clone(), s.clone(), ds.clone()]
            assert all(torch.equal(u, v) for u, v in zip(back(*given, given[a], given[b]), want))


@pytest.mark.parametrize("start", [0, 1])
@pytest.mark.parametrize("rows", [1, 8])
@pytest.mark.parametrize("dim", [64, 128, 1024])
@pytest.mark.parametrize("t,far", [(F, 12345), (H, 1021)])
def test_gradients_of_rows_far_from_zero(t, far, dim, rows, start):
    """Whole numbers around a distant one: sums below 2^24, the mean and x - mean are exact in fp32, so that xh has the error of
    rstd and one rounding, however far the row is from zero (with |d mean| = 0 in the bounds of these gradients)."""
    g = torch.Generator().manual_seed(dim)
    e = torch.randint(1, 4, (rows, dim // 2), generator=g)
    whole = (torch.stack([e, -e], -1) + far).to(t).reshape(-1)
    x = torch.cat([whole[:start], whole]).cuda()[start:].view(rows, dim).requires_grad_()
    w, dh = normal((dim,), F, 3, 1.0, 0.2).requires_grad_(), normal((rows, dim), t, 4)
    h = layer_norm(x, w)
    r = Row(x, w, None)
    r.er = (27 + 6) * u32 / 2 + 4 * u32
    r.dxh = abs(r.xh) * (r.er + u32)
    inside(h, r.h, r.tol_h(t), "h")
    (rx, rw, _), (tx, tw, _) = r.grads(dh)
    dx, dw = torch.autograd.grad(h, (x, w), dh)
    close(dw, rw, tw, F, "dw")
    close(dx, rx, tx, t, "dx")


# ---- every kernel of the fused backward pass -------------------------------------------------------------------
def check_fused(z, y, w, b, ds, dh, share, p=0.25, seed=77, offset=5, trans=False):
    """dropout_add_layer_norm of leaves with these values and strides: results, and all gradients, against 64 bits."""
    leaves = [t.detach().requires_grad_() for t in (z, y, w, b)]
    s, h = dropout_add_layer_norm(*leaves, p, seed, offset, share=share, out_dtype=dh.dtype, trans_out=trans)
    assert torch.equal(s, rounded(dropout_add_ref(f64(z), f64(y), p, seed, offset, share), z.dtype))
    given = dh.transpose(1, 2) if trans else dh
    r = Row(s, w, b)
    inside(h.transpose(1, 2) if trans else h, r.h, r.tol_h(dh.dtype), "h")
    dz, dy, dw, db = torch.autograd.grad((s, h), leaves, (ds, given))
    (rz, rw, rb), (tz, tw, tb) = r.grads(dh, ds)
    close(dz, rz, tz, z.dtype, "dz")
    keep = keep_mask(z.shape, p, seed, offset, share)
    ry = np.where(keep, rz * scale_of(p), 0.0)
    close(dy, ry, np.where(keep, scale_of(p) * tz + u32 * np.abs(ry), 0.0), y.dtype, "dy")
    close(dw, rw, tw, w.dtype, "dw")
    close(db, rb, tb, b.dtype, "db")


FUSED_TYPES = [(F, F, F), (F, F, H), (F, F, B), (F, H, H), (F, B, B), (H, H, H), (B, B, B)]


@pytest.mark.parametrize("tz,ty,to", FUSED_TYPES)
@pytest.mark.parametrize("dim", [4, 13, 36, 65, 100, 101, 129, 260, 333, 388, 421, 500, 510, 700, 777, 1004, 2049, 2060, 4100, 4877,
                                 6145, 8184, 8191, 8192])
def test_fused_gradients_of_every_layout(tz, ty, to, dim):
    """Rows of whole pieces of eight, of four and of one channel, on some lanes of a warp, a warp and several, with one to all
    of their pieces there; dense, and with every tensor strided in its own way; draws per element, row, column and channel."""
    for shape in ((2, 3, 5), (3, 41, 17)) if dim < 400 else ((2, 3, 5),):
        b, i, j = shape
        z, y, ds, dh = (normal((*shape, dim), t, k, m) for t, k, m in ((tz, 1, 0.5), (ty, 2, 0.0), (tz, 3, 0.0), (to, 4, 0.0)))
        w, c = normal((dim,), F, 5, 1.0, 0.2), normal((dim,), F, 6, 0.0, 0.2)
        for share in ((), (2, 3), (1, 3), (1,)):
            check_fused(z, y, w, c, ds, dh, share)
        wide = torch.zeros((b, i, j, dim + 8), dtype=tz, device="cuda")
        wide[..., 8:] = z
        turned = torch.empty((b, j, i, dim), dtype=ty, device="cuda").copy_(y.transpose(1, 2)).transpose(1, 2)
        pad = 4 if dim % 8 else 8
        padded = torch.zeros((b, i, j + 1, dim + pad), dtype=tz, device="cuda")[:, :, :j, pad:]
        padded.copy_(ds)
        last = torch.empty((j, i, b, dim), dtype=to, device="cuda").copy_(dh.permute(2, 1, 0, 3)).permute(2, 1, 0, 3)
        for share in ((), (1, 3)):
            check_fused(wide[..., 8:], turned, w, c, padded, last, share)
            check_fused(z, y, w, c, padded, dh, share)  # the gradient of s alone is strided


@pytest.mark.parametrize("tz,ty,to", [(F, F, B), (F, B, B), (H, H, H)])
@pytest.mark.parametrize("dim", [8, 36, 100, 333, 520, 1000, 2052])
def test_fused_transposed_result_of_other_widths(tz, ty, to, dim):
    z, y, ds, dh = (normal((2, 7, 9, dim), t, k) for t, k in ((tz, 1), (ty, 2), (tz, 3), (to, 4)))
    w, b = normal((dim,), F, 5, 1.0, 0.2), normal((dim,), F, 6, 0.0, 0.2)
    for share in ((), (1, 3)):
        check_fused(z, y, w, b, ds, dh, share, trans=True)


@pytest.mark.parametrize("tz,ty,to", [(F, F, B), (H, H, H), (F, F, F)])
@pytest.mark.parametrize("dim", [1, 6, 8, 13, 16, 17, 31, 47, 63, 65])
def test_fused_gradients_of_narrow_rows_to_the_last(tz, ty, to, dim):
    """Warps and CTAs that the rows do not fill: the values of dy, and the column sums."""
    for rows in (1, 3, 31, 32, 33, 1023, 4099):
        z, y, ds, dh = (normal((rows, dim), t, k) for t, k in ((tz, rows), (ty, 5), (tz, 6), (to, 7)))
        w, b = normal((dim,), F, 8, 1.0, 0.2), normal((dim,), F, 9, 0.0, 0.2)
        for share in ((), (0,), (1,)):
            check_fused(z, y, w, b, ds, dh, share, p=0.4)


@pytest.mark.parametrize("tp", [H, B])
@pytest.mark.parametrize("dim", [13, 128, 1004])
def test_fused_parameters_in_16_bits(tp, dim):
    z, y, ds, dh = (normal((3, 7, 11, dim), F, k) for k in range(4))
    check_fused(z, y, normal((dim,), tp, 5, 1.0, 0.2), normal((dim,), tp, 6), ds, dh.to(B), (2, 3))

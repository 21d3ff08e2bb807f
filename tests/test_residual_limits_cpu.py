"""CPU: what the residual path refuses because its results would be wrong without a word, and what its build keeps in step."""

import ctypes
import itertools
import sys

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

import boltz_mlx_b200 as b200
from boltz_mlx_b200 import _lib, build


@pytest.fixture(scope="module", autouse=True)
def _built():
    build.build()


def _calls(x, y, w, b):
    """Every call on the same tensors."""
    return [lambda: b200.layer_norm(x, w, b), lambda: b200.layer_norm(x, w, b, out_dtype=torch.bfloat16),
            lambda: b200.dropout(x, 0.1, 1), lambda: b200.dropout(x, 0.1, 1, training=False),
            lambda: b200.dropout_add(x, y, 0.1, 1), lambda: b200.dropout_add(y, x, 0.1, 1),
            lambda: b200.dropout_add(x, y, 0.1, 1, inplace=True),
            lambda: b200.dropout_add_layer_norm(x, y, w, b, 0.1, 1), lambda: b200.dropout_add_layer_norm(y, x, w, b, 0.1, 1)]


def test_forward_mode_is_refused():
    """A tangent would be lost, and count as zero."""
    x, y, w, b = torch.zeros(2, 8), torch.zeros(2, 8), torch.ones(8), torch.zeros(8)
    with fwAD.dual_level():
        for f in _calls(fwAD.make_dual(x, torch.ones(2, 8)), y, w, b):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()
        dual = fwAD.make_dual(w, torch.ones(8))
        for f in (lambda: b200.layer_norm(x, dual, b), lambda: b200.layer_norm(x, w, dual),
                  lambda: b200.dropout_add_layer_norm(x, y, dual, b, 0.1, 1),
                  lambda: b200.dropout_add_layer_norm(x, y, w, dual, 0.1, 1)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()
        for f in _calls(x, y, w, b):  # none of these has a tangent
            with pytest.raises(RuntimeError, match="CUDA"):
                f()


def test_a_number_is_no_set_of_axes():
    """share=0 once counted as no shared axis, and dropped each element by itself."""
    x = torch.zeros(2, 8)
    for share in (0, 1):
        for f in (lambda: b200.dropout(x, 0.1, 1, share=share), lambda: b200.dropout_add(x, x, 0.1, 1, share=share),
                  lambda: b200.dropout_add_layer_norm(x, x, None, None, 0.1, 1, share=share)):
            with pytest.raises(TypeError):
                f()
    for share in ((), [], None, (0,), [0, 1]):
        with pytest.raises(RuntimeError, match="CUDA"):
            b200.dropout(x, 0.1, 1, share=share)


TRACERS = {
    "jit": lambda f, x: torch.jit.trace(f, (x,), check_trace=False),
    "fx": lambda f, x: make_fx(f)(x),
    "fx before dispatch": lambda f, x: make_fx(f, pre_dispatch=True)(x),
    "fx of fake tensors": lambda f, x: make_fx(f, tracing_mode="fake")(x),
    "export": lambda f, x: torch.export.export(Calls(f), (x,), strict=False),
}


class Calls(torch.nn.Module):
    def __init__(self, f):
        super().__init__()
        self.f = f

    def forward(self, x):
        return self.f(x)


@pytest.mark.parametrize("tracer", list(TRACERS))
def test_tracing_is_refused(tracer):
    """A tracer sees the allocation of the results alone, and would record that."""
    y, w, b = torch.zeros(2, 8), torch.ones(8), torch.zeros(8)
    for k in range(len(_calls(y, y, w, b))):
        with pytest.raises(NotImplementedError, match="tracing"):
            TRACERS[tracer](lambda x: _calls(x, x, w, b)[k](), torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="CUDA"):  # and nothing of it stays behind
        b200.layer_norm(y)


@torch.library.custom_op("residual_limits::norm", mutates_args=())
def _registered(x: torch.Tensor) -> torch.Tensor:
    return b200.layer_norm(x)


@_registered.register_fake
def _(x):
    return torch.empty_like(x)


@pytest.mark.parametrize("tracer", list(TRACERS))
def test_a_registered_operator_is_no_hindrance(tracer):
    """A program may register a call as an operator of its own: a tracer records that, and the call inside is not traced."""
    trace = lambda: TRACERS[tracer](lambda x: torch.ops.residual_limits.norm(x), torch.zeros(2, 8))  # noqa: E731
    if tracer in ("fx of fake tensors", "export"):
        graph = trace()
        assert "residual_limits.norm" in str(getattr(graph, "graph_module", graph).graph)
    else:  # these run what they record
        with pytest.raises(RuntimeError, match="CUDA"):
            trace()


def test_fake_tensors_are_refused():
    real, w, b = torch.zeros(2, 8), torch.ones(8), torch.zeros(8)
    with FakeTensorMode():
        for x in (torch.zeros(2, 8), torch.zeros(2, 8, device="cuda"), real):
            for f in _calls(x, x, w, b):
                with pytest.raises(NotImplementedError, match="fake"):
                    f()


def test_modes_that_record_nothing_are_no_hindrance():
    """Counting flops, or choosing what a checkpoint keeps: the calls get as far as without."""
    with FlopCounterMode(display=False):
        for f in _calls(*(torch.zeros(2, 8),) * 2, torch.ones(8), torch.zeros(8)):
            with pytest.raises(RuntimeError, match="CUDA"):
                f()


# ---- the layers ----------------------------------------------------------------------------------------------
def test_layers_refuse_to_lose_gradients():
    """forward_residual and f16_addln with dropout, and norm_input, are forward only: a z with gradients is refused, and one
    whose gradients nobody asks for gets as far as without."""
    d, ln = b200.PairDropout(0.25, 1), torch.nn.LayerNorm(128)
    calls = []
    for layer in (b200.TriangleAttention(precision="bf16"), b200.TriangleAttention(starting=False, precision="bf16"),
                  b200.TriangleMultiplicationOutgoing(128, precision="bf16")):
        calls += [lambda z, m=layer: m.forward_residual(z, dropout=d), lambda z, m=layer: m.f16_addln(z, None, None, ln, dropout=d),
                  lambda z, m=layer: m.forward_residual(z, dropout=d, inplace=True)]
        if hasattr(layer, "norm_input"):
            calls.append(layer.norm_input)
    z = torch.zeros(1, 4, 4, 128, requires_grad=True)
    for f in calls:
        with pytest.raises(RuntimeError, match="forward only"):
            f(z)
        with pytest.raises(RuntimeError, match="CUDA"):
            f(z.detach())
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            f(z)


# ---- tensors that overlap, at the C entries --------------------------------------------------------------
A = 1 << 20  # addresses that validation may look at but nothing may touch: every call here is refused


def _strides(s):
    return None if s is None else (ctypes.c_int64 * 3)(*s)


def _add(shape, dim, z, y, out, dtypes=(0, 0)):
    """triattn_dropout_add of (address, strides); what it says of them."""
    L = _lib.lib()
    rc = L.triattn_dropout_add(z[0], dtypes[0], _strides(z[1]), y[0], dtypes[1], _strides(y[1]), _strides(shape), dim, 0, 0.1, 1, 0,
                               None, out[0], dtypes[0], _strides(out[1]), None)
    assert rc == _lib.EINVAL
    return L.triattn_last_error_string().decode()


def _bytes(shape, dim, at, strides, es):
    strides = strides or (shape[1] * shape[2] * dim, shape[2] * dim, dim)
    return {at + es * sum(i * s for i, s in zip(row, strides)) + k
            for row in itertools.product(*map(range, shape)) for k in range(dim * es)}


def test_overlaps_are_refused_and_nothing_else():
    """out against z, byte by byte: y always overlaps out, so that the call is refused, for z where z does."""
    shape, dim = (2, 3, 2), 4
    layouts = [None, (48, 16, 8), (100, 30, 10), (8, 16, 4), (24, 4, 12), (8, 16, 48), (64, 16, 8)]
    n = 0
    for sz in layouts:
        for so in layouts:
            for step in (0, 8, 16, 32, 40, 64, 96, 100, 104, 192, 400, 800, 1200):
                for at in (A + step, A - step):
                    said = _add(shape, dim, (at, sz), (A + 4, (0, 0, 0)), (A, so))
                    apart = not _bytes(shape, dim, at, sz, 4) & _bytes(shape, dim, A, so, 4)
                    one = step == 0 and sz == so
                    if apart and said.count("overlaps z"):  # only where the strides differ
                        assert sz != so, (sz, so, at - A, said)
                        continue
                    assert ("out overlaps z" in said) != (apart or one), (sz, so, at - A, said)
                    assert ("out overlaps y" in said) == (apart or one), (sz, so, at - A, said)
                    n += apart
    assert n > 100


def test_column_slices_of_one_buffer_do_not_overlap():
    """z and out side by side in the rows of one buffer, out with the leading axes swapped."""
    said = _add((3, 5, 7), 8, (A, (560, 112, 16)), (A + 4, (0, 0, 0)), (A + 32, (112, 336, 1680)))
    assert "out overlaps y" in said
    said = _add((3, 5, 7), 8, (A, (560, 112, 16)), (A + 4, (0, 0, 0)), (A + 28, (112, 336, 1680)))
    assert "out overlaps z" in said


def test_other_entries_refuse_overlaps():
    L, i3 = _lib.lib(), _strides((1, 2, 3))  # 6 rows of 8: 192 bytes in fp32

    def norm(x, out, od=0, os_=None):
        return L.triattn_layer_norm(x, 0, None, i3, 8, None, None, 0, 1e-5, out, od, _strides(os_), None, None, None)

    for out in (A, A + 4, A + 188, A - 188):
        assert norm(A, out) == _lib.EINVAL, out
    assert norm(A, A - 92, od=1) == _lib.EINVAL and norm(A, A, os_=(48, 8, 16)) == _lib.EINVAL

    def fused(z=A, y=2 * A, s=3 * A, out=4 * A, ss=None, os_=None, ys=None):
        return L.triattn_dropout_add_layer_norm(z, 0, None, y, 0, _strides(ys), i3, 8, 0, 0.1, 1, 0, None, None, None, 0, 1e-5, s,
                                                _strides(ss), out, 0, _strides(os_), None, None, None)

    for kw, name in (({"s": A + 32}, "sum overlaps z"), ({"s": 2 * A, "ss": (48, 8, 16)}, "sum overlaps y"),
                     ({"s": 2 * A - 32}, "sum overlaps y"), ({"out": A}, "out overlaps z"), ({"out": A + 96}, "out overlaps z"),
                     ({"out": 2 * A + 32}, "out overlaps y"), ({"out": 2 * A, "os_": (48, 8, 16)}, "out overlaps y"),
                     ({"out": 3 * A}, "out overlaps sum"), ({"out": 3 * A + 64}, "out overlaps sum"),
                     ({"s": 2 * A, "ys": (0, 0, 0)}, "sum overlaps y")):
        assert fused(**kw) == _lib.EINVAL and name in L.triattn_last_error_string().decode(), kw

    def back(dout=A, x=2 * A, ds=3 * A, dx=4 * A, dy=5 * A, xs=None):
        return L.triattn_layer_norm_backward(dout, 0, None, x, 0, _strides(xs), i3, 8, None, 0, A, A, ds, None, 0, 0.0, 0, 0, None,
                                             dx, dy, 0, None, None, None, 0, None)

    for kw, name in (({"dx": A + 32}, "dx overlaps dout"), ({"dx": 2 * A, "xs": (48, 8, 16)}, "dx overlaps x"),
                     ({"dx": 3 * A - 32}, "dx overlaps dsum"), ({"dy": A + 32}, "dy overlaps dout"),
                     ({"dy": 2 * A + 64}, "dy overlaps x"), ({"dx": 5 * A}, "dx overlaps dy"), ({"dx": 5 * A + 32}, "dx overlaps dy")):
        assert back(**kw) == _lib.EINVAL and name in L.triattn_last_error_string().decode(), kw


def test_mean_without_rstd_is_refused():
    """The kernels write both or neither."""
    L, i3 = _lib.lib(), _strides((1, 2, 3))
    for mean, rstd in ((A, None), (None, A)):
        assert L.triattn_layer_norm(A, 0, None, i3, 8, None, None, 0, 1e-5, 2 * A, 0, None, mean, rstd, None) == _lib.EINVAL
        assert L.triattn_dropout_add_layer_norm(A, 0, None, 2 * A, 0, None, i3, 8, 0, 0.1, 1, 0, None, None, None, 0, 1e-5, 3 * A, None,
                                                4 * A, 0, None, mean, rstd, None) == _lib.EINVAL
        assert L.triattn_layer_norm_backward(A, 0, None, 2 * A, 0, None, i3, 8, None, 0, mean, rstd, None, None, 0, 0.0, 0, 0, None,
                                             3 * A, None, 0, None, None, None, 0, None) == _lib.EINVAL


# ---- the build -------------------------------------------------------------------------------------------------
def test_the_binding_is_rebuilt_for_another_pytorch(monkeypatch, tmp_path):
    ran = []
    monkeypatch.setattr(build, "_run", lambda cmd, verbose: ran.append(cmd[-1]))
    build.build()
    assert not ran and _lib.residual().built_for == build.built_for(torch)
    other = tmp_path / "_residual.so"
    other.write_bytes(build.RESIDUAL.read_bytes().replace(torch.__version__.encode(), b"0" * len(torch.__version__)))
    monkeypatch.setattr(build, "RESIDUAL", other)
    build.build()
    assert len(ran) == 1


def test_the_c_library_builds_without_pytorch(monkeypatch, capsys):
    ran = []
    monkeypatch.setattr(build, "_run", lambda cmd, verbose: ran.append(str(build.LIB) in cmd))
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build(force=True) == build.LIB and ran == [True]
    assert "left out" in capsys.readouterr().out

"""CPU: what the residual path refuses because its results would be wrong without a word, and what its build keeps in step."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

import boltz_mlx_b200 as b200
from boltz_mlx_b200 import _lib


@pytest.fixture(scope="module", autouse=True)
def _built():
    if not (_lib.LIB_PATH.exists() and _lib.RESIDUAL_PATH.exists()):
        pytest.skip("the library is not built (python -m boltz_mlx_b200.build)")


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

"""GPU: calls of the residual path at the edges of what PyTorch and the C ABI allow."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from boltz_mlx_b200 import _lib, dropout, dropout_add, dropout_add_layer_norm, layer_norm
from tests.test_gpu_residual import F, normal

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

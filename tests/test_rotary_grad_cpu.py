"""rotary() in torch's graph of gradients, without a GPU: launches are stood in for."""
import types

import pytest

torch = pytest.importorskip("torch")

import triton_ext_amd as tx  # noqa: E402
from triton_ext_amd import cache as C  # noqa: E402
from triton_ext_amd import capi  # noqa: E402


@pytest.fixture
def launches(monkeypatch):
    """The `inverse` of every launch's plan, in order; the result is a copy of x."""
    seen, native = [], capi.calls()

    def call(f, plan, x, positions, inv_freq, out, stream):
        seen.append(capi.RotaryPlan.from_address(plan).desc.inverse)
        out.copy_(x)
        return 0
    monkeypatch.setattr(C, "_native", types.SimpleNamespace(form=native.form, call=call))
    monkeypatch.setattr(C, "_current_stream", lambda device: 0)
    return seen


@pytest.mark.parametrize("inverse", [False, True])
def test_the_gradient_is_the_transposed_map(launches, inverse):
    x = torch.randn(5, 2, 64, requires_grad=True)
    y = tx.rotary(x, torch.arange(5), torch.zeros(32), inverse=inverse)
    assert y.requires_grad
    dy = torch.randn(5, 2, 64)
    y.backward(dy)
    assert launches == [inverse, not inverse] and torch.equal(x.grad, dy)


def test_second_gradients(launches):
    x = torch.randn(3, 1, 8, requires_grad=True)
    dy = torch.randn(3, 1, 8, requires_grad=True)
    y = tx.rotary(x, torch.arange(3), torch.zeros(4))
    dx, = torch.autograd.grad(y, x, dy, create_graph=True)
    ddy, = torch.autograd.grad(dx, dy, torch.ones(3, 1, 8))
    assert launches == [0, 1, 0] and torch.equal(ddy, torch.ones(3, 1, 8))


def test_what_takes_no_gradient(launches):
    x = torch.randn(5, 2, 64, requires_grad=True)
    pos, f = torch.arange(5), torch.zeros(32)
    with pytest.raises(ValueError):  # a result in a given tensor would be cut off from x
        tx.rotary(x, pos, f, out=torch.empty(5, 2, 64))
    assert not launches
    with torch.no_grad():
        out = torch.empty(5, 2, 64)
        assert tx.rotary(x, pos, f, out=out) is out and not out.requires_grad
        assert not tx.rotary(x, pos, f).requires_grad
    assert not tx.rotary(x.detach(), pos, f).requires_grad

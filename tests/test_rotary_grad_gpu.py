"""Gradients through rotary() by torch's own backward pass, against the formula's in 64 bits."""
import pytest

torch = pytest.importorskip("torch")

import triton_ext_amd as tx  # noqa: E402
from cachecase import check, gen, randn, rotate64, rotate_bound  # noqa: E402
from dotcase import say  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape,rot", [((9, 3, 64), 32), ((2, 3, 17, 80), 80), ((1, 1, 2), 2)])
@pytest.mark.parametrize("interleaved,inverse", [(False, False), (True, True)])
def test_backward(gpu, dtype, shape, rot, interleaved, inverse):
    say("rotary backward", shape, rot, dtype, interleaved, inverse)
    g = gen(sum(shape))
    x, dy = randn(g, *shape, dtype=dtype), randn(g, *shape, dtype=dtype)
    N = shape[0] if len(shape) == 3 else shape[2]
    pos, f = torch.randint(0, 9000, (N,), generator=g), tx.rotary_frequencies(rot)[0]
    xd = x.to(gpu).requires_grad_()
    y = tx.rotary(xd, pos.to(gpu), f.to(gpu), interleaved=interleaved, scale=1.25, inverse=inverse)
    for given in (dy, dy.flip(-1)):  # (a second pass adds to the first)
        y.backward(given.to(gpu), retain_graph=True)
    t = (lambda a: a) if len(shape) == 3 else (lambda a: a.transpose(1, 2))
    p = pos if len(shape) == 3 else pos.expand(shape[0], N)
    want = mag = parts = 0
    for given in (dy, dy.flip(-1)):
        w, m = rotate64(t(given), p, f, interleaved, 1.25, not inverse)
        want, mag, parts = want + w, mag + m, parts + rotate_bound(w, m, dtype)
    # each pass's bound, and one rounding of their sum
    bound = parts + rotate_bound(want, mag, dtype)
    check(xd.grad, t(want), t(bound), "dx")


def test_backward_of_views(gpu):
    """A broadcast x, a slice of a projection, and a sum's gradient, whose strides are all 0."""
    g = gen(3)
    pos, f = torch.arange(6, device=gpu), tx.rotary_frequencies(64)[0].to(gpu)
    one = randn(g, 6, 1, 64).to(gpu).requires_grad_()
    tx.rotary(one.expand(6, 4, 64), pos, f).sum().backward()
    ref = randn(gen(3), 6, 1, 64).double().requires_grad_()
    y, _ = rotate64(ref.expand(6, 4, 64), pos.cpu(), f.cpu(), False, 1.0)
    y.sum().backward()
    _, mag = rotate64(torch.ones(6, 1, 64), pos.cpu(), f.cpu(), False, 1.0)
    # four equal gradients, each within its bound, and three sums
    bound = 4 * rotate_bound(ref.grad / 4, mag, torch.float32) + 3 * 2.0 ** -24 * 4 * mag
    check(one.grad, ref.grad, bound, "broadcast")
    qkv = randn(g, 6, 8, 64).to(gpu).requires_grad_()
    tx.rotary(qkv[:, 2:5], pos, f).square().sum().backward()
    got = qkv.grad.cpu()
    assert not got[:, :2].any() and not got[:, 5:].any()
    # |y| = |x|: the gradient of the sum of squares is 2 x, with two maps' roundings
    x = qkv.detach().cpu()[:, 2:5].double()
    _, mag = rotate64(x, pos.cpu(), f.cpu(), False, 1.0)
    twice = rotate64(mag, 0 * pos.cpu(), f.cpu(), False, 1.0)[1]
    check(got[:, 2:5], 2 * x, 2 * 2 * rotate_bound(twice, twice, torch.float32), "slice")


def test_backward_on_a_named_stream(gpu):
    g = gen(4)
    pos, f = torch.arange(6, device=gpu), tx.rotary_frequencies(64)[0].to(gpu)
    x = randn(g, 6, 3, 64).to(gpu)
    want = tx.rotary(torch.ones_like(x), pos, f, inverse=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    x.requires_grad_()
    y = tx.rotary(x, pos, f, stream=side.cuda_stream)
    side.synchronize()
    y.sum().backward()
    torch.cuda.synchronize()
    assert torch.equal(x.grad, want)

"""Counter-based dropout against its 64-bit restatement (tests/_fp8_ref.py).

The mask is exact.  A kept value is one float32 product (2^-24 of it), with a
residual one float32 sum more, then one rounding to the type: half a step."""
import numpy as np
import pytest
import torch

import _fp8_ref as ref

pytestmark = pytest.mark.gpu

B, F = torch.bfloat16, torch.float32
KEY = dict(seed=0xFEDCBA9876543, site=3, step=17)


def close(got, x, f, residual=None):
    want = x.double() * f + (0.0 if residual is None else residual.double())
    mag = (x.double() * f).abs() + (0.0 if residual is None else residual.double().abs())
    slack = torch.finfo(got.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -23 * mag
    assert got.shape == x.shape and got.dtype == x.dtype
    assert bool(((got.double() - want).abs() <= slack).all())


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("p", [0.0, 1e-5, 0.1, 0.5, 0.999, 1.0])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (2049,), (16, 768), (33, 501), (3, 5, 77)])
def test_dropout_and_gradients(shape, p, dtype):
    import advanced_optimizers_b200 as A
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(shape, generator=g, device="cuda").to(dtype).requires_grad_()
    r = torch.randn(shape, generator=g, device="cuda").to(dtype).requires_grad_()
    dy = torch.randn(shape, generator=g, device="cuda").to(dtype)
    f = ref.keep_factor(shape, p, **KEY)
    y = A.philox_dropout(x, p, **KEY)
    close(y.detach(), x.detach(), f)
    assert torch.equal(y.detach() != 0, (f > 0) & (x.detach() != 0))
    close(torch.autograd.grad(y, x, dy)[0], dy, f)
    y = A.philox_dropout(x, p, residual=r, **KEY)
    close(y.detach(), x.detach(), f, r.detach())
    gx, gr = torch.autograd.grad(y, (x, r), dy)
    close(gx, dy, f)
    assert torch.equal(gr, dy)


@pytest.mark.parametrize("dtype", [B, F])
def test_dropped_infinities_and_nan_are_zero(dtype):
    import advanced_optimizers_b200 as A
    n = 4096
    f = ref.keep_factor((n,), 0.5, **KEY)
    x = torch.where(f > 0, torch.ones(n, device="cuda").double(), torch.full((n,), float("nan"), device="cuda").double()).to(dtype)
    x[(f == 0).nonzero()[::2, 0]] = float("inf")
    y = A.philox_dropout(x, 0.5, **KEY)
    assert torch.equal(y, (2.0 * (f > 0)).to(dtype))
    assert torch.equal(A.philox_dropout(x, 0.5, residual=torch.ones_like(x), **KEY), (1 + 2.0 * (f > 0)).to(dtype))


@pytest.mark.parametrize("dtype", [B, F])
def test_strides_and_unaligned_views(dtype):
    import advanced_optimizers_b200 as A
    wide = torch.randn(40, 130, device="cuda").to(dtype)
    flat = torch.randn(1003, device="cuda").to(dtype)
    for t in (wide.t(), wide[:, 1:50], wide[::2], flat[1:], flat[3:900], wide[:1].expand(40, 130)):
        close(A.philox_dropout(t, 0.3, **KEY), t, ref.keep_factor(tuple(t.shape), 0.3, **KEY))
        got = A.philox_dropout(t, 0.3, residual=t, **KEY)
        close(got, t, ref.keep_factor(tuple(t.shape), 0.3, **KEY), t)
    leaf = wide.clone().requires_grad_()
    g, = torch.autograd.grad(A.philox_dropout(leaf, 0.3, **KEY).sum(), leaf)   # an expanded dy
    close(g, torch.ones_like(wide), ref.keep_factor((40, 130), 0.3, **KEY))


def test_seed_site_and_step_each_matter():
    import advanced_optimizers_b200 as A
    x = torch.ones(4096, device="cuda")
    seen = [A.philox_dropout(x, 0.5, **{**KEY, **c}) for c in ({}, dict(seed=1), dict(seed=1 << 40), dict(site=4), dict(step=18))]
    for i in range(len(seen)):
        for j in range(i):
            assert 0.4 < float((seen[i] != seen[j]).float().mean()) < 0.6
    assert torch.equal(A.philox_dropout(x, 0.5, **KEY), seen[0])


def test_rate_and_mean():
    """Over 2^22 elements the kept share is within 5 sigma of the realised probability, and the mean of ones stays one."""
    import advanced_optimizers_b200 as A
    n = 1 << 22
    for p in (0.1, 0.5, 0.9):
        y = A.philox_dropout(torch.ones(n, device="cuda"), p, **KEY)
        q = 1 - round(p * 65536) / 65536
        kept = float((y != 0).double().mean())
        assert abs(kept - q) <= 5 * np.sqrt(q * (1 - q) / n)
        assert abs(float(y.double().mean()) - 1) <= 5 * np.sqrt((1 - q) / (q * n)) + 2.0 ** -23


def test_step_on_the_device_and_captured():
    import advanced_optimizers_b200 as A
    x = torch.randn(1000, device="cuda", requires_grad=True)
    dy = torch.randn(1000, device="cuda")
    step = torch.tensor(17, device="cuda")
    kw = dict(seed=KEY["seed"], site=3)

    def run(at):
        y = A.philox_dropout(x, 0.4, step=at, **kw)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        warm = run(step)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(warm, run(17)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(step)
    for at in (3, 2 ** 32 - 1):
        step.fill_(at)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, run(at)))
    y = A.philox_dropout(x, 0.4, step=step, **kw)
    step.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, dy)


def test_past_32_bits():
    import advanced_optimizers_b200 as A
    n = (1 << 32) + 12345
    x = torch.ones(n, dtype=B, device="cuda")
    y = A.philox_dropout(x, 0.25, **KEY)
    first = n - 5000
    T = round(0.25 * 65536)
    keep = ref.random16(5000, KEY["seed"], KEY["site"], KEY["step"], first) >= T
    assert torch.equal((y[first:] != 0).cpu(), keep)
    keep = ref.random16(5000, KEY["seed"], KEY["site"], KEY["step"]) >= T
    assert torch.equal((y[:5000] != 0).cpu(), keep)


def test_empty():
    import advanced_optimizers_b200 as A
    x = torch.zeros(0, 5, device="cuda", requires_grad=True)
    y = A.philox_dropout(x, 0.5)
    assert tuple(y.shape) == (0, 5) and tuple(torch.autograd.grad(y.sum(), x)[0].shape) == (0, 5)


def test_gradient_of_the_gradient():
    import advanced_optimizers_b200 as A
    x = torch.randn(300, device="cuda", requires_grad=True)
    dy = torch.randn(300, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(A.philox_dropout(x, 0.5, **KEY), x, dy, create_graph=True)
    gg, = torch.autograd.grad(g, dy, torch.ones_like(g))
    assert torch.equal(gg, (2.0 * (ref.keep_factor((300,), 0.5, **KEY) > 0)).float())

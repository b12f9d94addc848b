"""Layer norm and its gradients against their 64-bit formulas (tests/_rows_ref.py)."""
import pytest
import torch

import _rows_ref as ref

pytestmark = pytest.mark.gpu

B, F = torch.bfloat16, torch.float32


def make(R, C, dtype, wdtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + R + C)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = (n(R, C) * (1 + 9 * (torch.rand(C, generator=g, device="cuda") < 0.02)) + n(R, 1)).to(dtype)
    return x, (1 + 0.2 * n(C)).to(wdtype), (0.2 * n(C)).to(wdtype), n(R, C).to(dtype)


def check(x, w, b, dy, eps=1e-5):
    import advanced_optimizers_b200 as A
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = A.layer_norm(*leaves, eps)
    C = x.shape[-1]
    o = ref.LayerNorm(x.reshape(-1, C), w, b, eps)
    want, slack = o.forward()
    ref.close(y.reshape(-1, C), want, slack, x.dtype)
    grads = iter(torch.autograd.grad(y, [t for t in leaves if t is not None], dy))
    for t, (want, slack) in zip(leaves, o.backward(dy.reshape(-1, C))):
        if t is not None:
            ref.close(next(grads).reshape(want.shape), want, slack, t.dtype)


@pytest.mark.parametrize("dtype,wdtype", [(B, B), (B, F), (F, F), (F, B)])
@pytest.mark.parametrize("R,C", [(1, 1), (3, 2), (1, 7), (9, 8), (70, 129), (33, 256), (64, 257), (17, 512), (40, 768), (2500, 768), (5, 1000), (11, 1024),
                                 (9, 1025), (700, 2048), (31, 2049), (1200, 4096), (300, 5003), (7, 8192), (9, 8200), (5, 12001), (3, 16384), (6, 16392),
                                 (2, 40003)])
def test_layer_norm_and_gradients(R, C, dtype, wdtype):
    check(*make(R, C, dtype, wdtype))


@pytest.mark.parametrize("C", [100, 2048, 5003, 20000])
def test_optional_weight_and_bias(C):
    x, w, b, dy = make(50, C, B, B)
    for ww, bb in ((None, None), (w, None), (None, b)):
        check(x, ww, bb, dy)


@pytest.mark.parametrize("need", ["x", "w", "b", "xw", "wb", "xb"])
@pytest.mark.parametrize("C", [300, 2050, 9000])
def test_gradients_that_are_asked_for(C, need):
    import advanced_optimizers_b200 as A
    x, w, b, dy = make(77, C, F, F)
    leaves = dict(x=x, w=w, b=b)
    for k in need:
        leaves[k].requires_grad_()
    got = torch.autograd.grad(A.layer_norm(x, w, b), [leaves[k] for k in need], dy)
    all3 = dict(zip("xwb", ref.LayerNorm(x.detach(), w.detach(), b.detach(), 1e-5).backward(dy)))
    for k, g in zip(need, got):
        ref.close(g, *all3[k], F)


@pytest.mark.parametrize("dtype", [B, F])
def test_shapes_and_strides(dtype):
    g = torch.Generator(device="cuda").manual_seed(5)
    wide = torch.randn(40, 2100, generator=g, device="cuda").to(dtype)
    _, w, b, _ = make(1, 2051, dtype, F)
    for x in (wide[:, 1:2052], wide[:, 8:2059], wide[::3, :2051], wide.t()[:2051].t(), wide[:1].expand(9, 2100)[:, :2051],
              wide[:, :2051].reshape(4, 10, 2051)[:, 1:], wide[0, :2051]):
        dy = torch.randn(x.shape, generator=g, device="cuda").to(dtype)
        check(x, w, b, dy)
        check(x, w[::1], b.flip(0), dy[..., :1].expand_as(dy))
    wd = torch.randn(40, 2100, generator=g, device="cuda").to(dtype)
    check(wide[:, :2048], w[1:2049], b[3:2051], wd[:, 1:2049])
    check(wide[:, :1000], w[1:1001], b[3:1003], wd[:, 2:1002])


def test_hard_rows():
    """Rows of one value, a mean far from 0, tiny and huge values: the variance is that of the differences from the mean."""
    import advanced_optimizers_b200 as A
    C = 3000
    g = torch.Generator(device="cuda").manual_seed(1)
    n = torch.randn(8, C, generator=g, device="cuda")
    x = torch.stack([torch.full((C,), 5.0, device="cuda"), 1000 + n[1], 1e4 + 0.1 * n[2], 1e-15 * n[3], 1e15 * n[4], torch.zeros(C, device="cuda"),
                     n[6], n[7]])
    x[6, 17] = 1e4
    w, b, dy = torch.ones(C, device="cuda"), torch.zeros(C, device="cuda"), torch.randn(8, C, generator=g, device="cuda")
    check(x, w, b, dy)
    check(x, w, b, dy, eps=1e-12)
    y = A.layer_norm(x, w, b)
    assert bool((y[0] == 0).all()) and bool((y[5] == 0).all())
    bad = x.clone()
    bad[2, 3], bad[4, 5] = float("nan"), float("inf")
    y = A.layer_norm(bad, w, b)
    assert bool(y[[2, 4]].isnan().all()) and torch.equal(y[[0, 1, 3, 5, 6, 7]], A.layer_norm(x, w, b)[[0, 1, 3, 5, 6, 7]])


def test_empty_calls():
    import advanced_optimizers_b200 as A
    w, b = (torch.ones(24, device="cuda", requires_grad=True) for _ in range(2))
    x = torch.empty(0, 3, 24, device="cuda", requires_grad=True)
    y = A.layer_norm(x, w, b)
    assert y.shape == x.shape
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert dx.shape == x.shape and bool((dw == 0).all()) and bool((db == 0).all())


@pytest.mark.parametrize("R,C", [(3000, 768), (1500, 2048), (700, 10000)])
def test_repeats_bit_for_bit_on_other_streams_and_in_graphs(R, C):
    import advanced_optimizers_b200 as A
    x, w, b, dy = make(R, C, B, F)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    run = lambda: torch.autograd.grad(A.layer_norm(*leaves), leaves, dy)  # noqa: E731
    want = run()
    same = lambda got: all(torch.equal(g, t) for g, t in zip(got, want))  # noqa: E731
    assert same(run()) and same(run())
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            got += [run() for _ in range(4)]
    torch.cuda.synchronize()
    assert all(map(same, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    with torch.no_grad():
        x.mul_(0.5).add_(0.25)
        dy.mul_(-2)
    graph.replay()
    for g, (want, slack), t in zip(out, ref.LayerNorm(x.detach(), w.detach(), b.detach(), 1e-5).backward(dy), leaves):
        ref.close(g, want, slack, t.dtype)


@pytest.mark.parametrize("C", [600, 3001])
def test_gradient_against_differences(C):
    """The kernel's own difference quotient along a direction, within its rounding and the 64-bit quotient's truncation."""
    import advanced_optimizers_b200 as A
    x, w, b, dy = make(20, C, F, F)
    v = torch.randn_like(x)
    step = 2.0 ** -6
    leaf = x.clone().requires_grad_()
    slope = float((torch.autograd.grad(A.layer_norm(leaf, w, b), leaf, dy)[0].double() * v.double()).sum())
    hi, lo = x + step * v, x - step * v
    f = lambda t: float((A.layer_norm(t, w, b).double() * dy.double()).sum())  # noqa: E731
    o = [ref.LayerNorm(t, w, b, 1e-5).forward() for t in (hi, lo)]
    exact = float(((o[0][0] - o[1][0]) * dy.double()).sum()) / (2 * step)
    (dx, ox), _, _ = ref.LayerNorm(x, w, b, 1e-5).backward(dy)
    moved = float(((hi - x).double() - step * v.double()).abs().mul(dx.abs()).sum()) * 4 / step   # the steps' own rounding
    rounding = float(sum(((s + ref.U * y.abs()) * dy.double().abs()).sum() for y, s in o)) / (2 * step) + float((ox * v.double().abs()).sum())
    truncation = abs(exact - float((dx * v.double()).sum()))
    assert abs((f(hi) - f(lo)) / (2 * step) - slope) <= truncation + rounding + moved


def test_more_than_2_to_32_elements():
    import advanced_optimizers_b200 as A
    R, C = (1 << 21) + 5, 2056
    x = torch.zeros(R, C, dtype=B, device="cuda")
    x[-3:, ::2] = 1.0
    x.requires_grad_()
    y = A.layer_norm(x)
    want = ref.LayerNorm(x[-3:].detach(), None, None, 1e-5)
    ref.close(y[-3:], *want.forward(), B)
    assert bool((y[: R - 3 : 1000] == 0).all())
    dy = torch.zeros_like(y)
    dy[-1] = torch.arange(C, device="cuda") % 7
    dx, = torch.autograd.grad(y, x, dy)
    ref.close(dx[-3:], *want.backward(dy[-3:])[0], B)
    assert bool((dx[: R - 3 : 1000] == 0).all())


def test_hooks_on_saved_tensors_and_other_derivatives():
    import advanced_optimizers_b200 as A
    x, w, b, dy = make(60, 300, F, F)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(A.layer_norm(*leaves), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = A.layer_norm(*leaves)
    assert all(torch.equal(g, t) for g, t in zip(torch.autograd.grad(y, leaves, dy), want))
    y = A.layer_norm(*leaves)
    with torch.no_grad():
        x.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaves, dy)
    g, = torch.autograd.grad(A.layer_norm(*leaves), w, dy.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    from torch.autograd import forward_ad
    x, w, b = (t.detach() for t in leaves)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args in ((dual(x), w, b), (x, dual(w), b), (x, w, dual(b))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                A.layer_norm(*args)


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("R", [1, 5, 7, 8, 9, 15, 17, 40, 600])
@pytest.mark.parametrize("C", [1, 5, 331, 1001, 1003, 5003, 6007])
def test_rows_between_boundaries(C, R, dtype):
    """Rows that begin anywhere between two 16-byte boundaries: alike in x, y, dy and dx, or each in their own way."""
    x, w, b, dy = make(R, C, dtype, dtype)

    def placed(t, pitch, offset):
        flat = torch.full((R * pitch + offset + 8,), float("nan"), dtype=dtype, device="cuda")   # outside the rows
        v = flat.as_strided((R, C), (pitch, 1), offset)
        v.copy_(t)
        return v

    for px, ox, pd, od in ((C, 0, C, 0), (C + 8, 0, C + 16, 8), (C, 0, C + 1, 0), (C, 3, C, 1), (C + 2, 1, C + 2, 1)):
        check(placed(x, px, ox), w, b, placed(dy, pd, od))


@pytest.mark.parametrize("dtype,wdtype", [(B, B), (F, F), (F, B)])
@pytest.mark.parametrize("R,C", [(1, 8193), (200, 12288), (190, 12001), (700, 16384), (7, 16385), (40, 20011), (100, 33000), (20, 50000), (17, 65536), (9, 65537),
                                 (6, 70001), (40, 131072)])
def test_wide_rows(R, C, dtype, wdtype):
    """Rows that take two, four and eight CTAs, and wider ones."""
    check(*make(R, C, dtype, wdtype))


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("R", [1, 7, 9, 33])
@pytest.mark.parametrize("C", [8195, 12001, 30011, 61000, 61447, 66666])
def test_wide_rows_between_boundaries(C, R, dtype):
    x, w, b, dy = make(R, C, dtype, dtype)
    for px, ox, pd, od in ((C, 0, C + 16, 8), (C + 1, 1, C, 2)):
        xs, dys = (torch.full((R * p + o + 8,), float("nan"), dtype=dtype, device="cuda").as_strided((R, C), (p, 1), o) for p, o in ((px, ox), (pd, od)))
        xs.copy_(x)
        dys.copy_(dy)
        check(xs, w, b, dys)


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("R", [296, 297, 400])
def test_many_wide_rows(R, dtype):
    check(*make(R, 17408, dtype, dtype))


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("C", [1, 8, 100, 500, 768, 1000, 1024, 1030, 4096, 5003, 8192, 10000, 16384, 20000, 32768, 40001, 65536, 70000])
def test_rows_of_one_value(C, dtype):
    """Their sum is exact (values of eight bits or fewer), so their mean and every difference from it are: y is the bias and dweight 0."""
    import advanced_optimizers_b200 as A
    values = torch.tensor([3.296875, 100.0, -1000.0, 5.0, 0.001953125 * 211, -77.0, 1.0, 2.0 ** 20], dtype=dtype, device="cuda")
    x = values[:, None].repeat(1, C).requires_grad_()
    _, w, b, dy = make(8, C, dtype, dtype)
    w.requires_grad_()
    for eps in (1e-5, 1e-12):
        y = A.layer_norm(x, w, b, eps)
        assert torch.equal(y, b.expand_as(y))
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        ref.close(dx, *ref.LayerNorm(torch.zeros_like(x), w.detach(), b, eps).backward(dy)[0], dtype)
        assert bool((dw == 0).all())


@pytest.mark.parametrize("C", [256, 1000, 1024, 1031, 4096, 5000, 5003, 8192, 12288, 16384])
def test_a_mean_far_from_zero(C):
    """Rows of integers around their mean, whose sums are below 2^24: mean and differences are exact, and the results within the bounds of
    the rows without the mean."""
    g = torch.Generator(device="cuda").manual_seed(C)
    half = torch.randint(-2, 3, (16, C // 2), generator=g, device="cuda").float()
    d = torch.cat([half, -half, torch.zeros(16, C % 2, device="cuda")], 1)
    mean = 1000.0 + torch.arange(16, device="cuda")[:, None]
    _, w, b, dy = make(16, C, F, F)
    import advanced_optimizers_b200 as A
    leaves = [t.requires_grad_() for t in (d + mean, w, b)]
    o = ref.LayerNorm(d, w.detach(), b.detach(), 1e-5)
    y = A.layer_norm(*leaves)
    ref.close(y, *o.forward(), F)
    for got, want in zip(torch.autograd.grad(y, leaves, dy), o.backward(dy)):
        ref.close(got, *want, F)


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("C", [40, 701, 4096, 5003, 9000])
def test_tiny_rows_without_eps(C, dtype):
    """Rows of a spread of 2^-66: 1 / var is beyond float32, rstd, its square root, and the gradient are not.  Half of a row is one value
    and half another, so that its sums are exact."""
    import advanced_optimizers_b200 as A
    x = torch.zeros(9, C, dtype=dtype, device="cuda")
    x[:, : C // 2], x[:, C // 2 : C // 2 * 2] = 2.0 ** -66, -(2.0 ** -66)
    _, w, b, dy = make(9, C, dtype, dtype)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    o = ref.LayerNorm(x.detach(), w.detach(), b.detach(), 0.0)
    # the squares, 2^-132, are denormal numbers of 17 bits: the sum of the squares is exact, its mean off by 2^-18 of it
    rel = 2.0 ** -18
    y = A.layer_norm(*leaves, 0.0)
    want, slack = o.forward()
    ref.close(y, want, slack + rel * (o.h * o.w).abs(), dtype)
    (dx, ox), (dw, ow), (db, ob) = o.backward(dy)
    g = torch.autograd.grad(y, leaves, dy)
    size = o.rstd * (dy.double() * o.w).abs().amax(1, keepdim=True) * 3   # of dx's terms: |h| is about 1
    ref.close(g[0], dx, ox + 3 * rel * size, dtype)
    ref.close(g[1], dw, ow + rel * (dy.double() * o.h).abs().sum(0), dtype)
    ref.close(g[2], db, ob, dtype)


@pytest.mark.parametrize("dtype,wdtype", [(B, B), (B, F), (F, F)])
@pytest.mark.parametrize("R,C", [(256, 1024), (1000, 776), (4097, 1024), (515, 1001), (600, 713), (300, 1023)])
def test_rows_of_up_to_1024_columns_that_a_cta_takes(R, C, dtype, wdtype):
    check(*make(R, C, dtype, wdtype))
    x, w, b, dy = make(R, C + 1, dtype, wdtype)
    check(x[:, 1:], w[1:], b[1:], dy[:, :-1])

"""The block quantiser, the block-scaled fp8 product and the fp8 linear layer
against 64-bit restatements (tests/_fp8_ref.py).

Tolerances.  Codes and scales: equal (scaling by a power of two is exact, so a
code carries the one rounding that the restatement carries too).  Products:
one rounding to the output type (half a step, eps / 2 of the value) plus the
float32 accumulation.  A tensor-core instruction adds 32 exact products to the
accumulator after aligning all 33 to the largest, so each loses less than 2^-23
of it (truncation to 24 bits): at most 33 * 2^-23 * S per instruction and
(K / 32) * 33 * 2^-23 * S over K, S the sum of the products' magnitudes; with
the few float32 additions of a split K that is within (K + 64) * 2^-22 * S."""
import pytest
import torch

import _fp8_ref as ref

pytestmark = pytest.mark.gpu

E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
B, F = torch.bfloat16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close_product(got, a, b, what="", extra=None, after=lambda t: t):
    """got against after(a @ b^T), a and b float64 values."""
    want = after(a @ b.t())
    mag = a.abs() @ b.abs().t()
    slack = (a.shape[1] + 64) * 2.0 ** -22 * mag * (1.0 if extra is None else extra)
    # two float32 roundings of the epilogue (bias, dropout) and one of the residual, on values up to |want| + slack's mag
    slack = slack + half_step(got.dtype) * want.abs() * (1 + 2.0 ** -10)
    diff = (got.double() - want).abs()
    assert got.shape == want.shape
    bad = ~(diff <= slack + 1e-300)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, first {torch.nonzero(bad)[0].tolist()}, " \
                                f"worst {float((diff / (slack + 1e-300)).max()):.3g} of the tolerance"


def check_blocks(b, x, block, dtype):
    q, e = ref.quantize(x, block, dtype)
    assert b.codes.dtype == dtype and tuple(b.codes.shape) == tuple(x.shape)
    got = b.codes.to(torch.float64)
    same = (got == q) | (torch.isnan(got) & torch.isnan(q))
    assert bool(same.all()), f"{int((~same).sum())} codes differ, first {torch.nonzero(~same)[0].tolist()}"
    assert torch.equal(b.scales.view(torch.uint8).to(torch.int64) - 127, e)
    assert b.block == ((128, 128) if block == 128 and x.shape[0] > 1 else (1, 128)) or x.shape[0] <= 1


def data(rows, cols, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + rows * 31 + cols)
    x = torch.randn(rows, cols, generator=g, device="cuda")
    return (x * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g, device="cuda").float())).to(dtype)


@pytest.mark.parametrize("layout", ["rows", "cols", "both"])
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("code", [E4, E5])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (7, 130), (128, 128), (129, 257), (257, 387), (300, 1000), (2, 4096), (1000, 64)])
def test_quantize(rows, cols, code, dtype, block, layout):
    import advanced_optimizers_b200 as A
    x = data(rows, cols, dtype)
    q = A.quantize_fp8(x, (block, 128), code, layout)
    r, c = (q if layout == "both" else (q, None) if layout == "rows" else (None, q))
    if r is not None:
        check_blocks(r, x, block, code)
    if c is not None:
        check_blocks(c, x.t(), block, code)


@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("code", [E4, E5])
@pytest.mark.parametrize("dtype", [B, F])
def test_quantize_special_values(dtype, code, block):
    """Zeros of both signs, infinities and NaN, values at and around the type's
    largest, ties between codes, and the smallest and largest numbers."""
    import advanced_optimizers_b200 as A
    big = ref.LARGEST[code]
    x = data(260, 390, F, 5)
    x[0:128, 0:128] = 0.0
    x[1, 5] = -0.0
    x[130, 128:256] = 0.0
    x[131, 130], x[132, 131], x[133, 132] = float("inf"), float("-inf"), float("nan")
    x[134, 256:384] = float("nan")
    x[135, 128:256] = torch.linspace(-big, big, 128, device="cuda")          # the largest value itself, and ties
    x[136, 128:256] = torch.linspace(-1.01 * big, 1.01 * big, 128, device="cuda")
    x[137, 128:256] = torch.arange(128, device="cuda") * 2.0 ** -10 * big    # ties and small codes
    x[138, 128:256] = 3.0e38
    x[139, 128:256] = torch.linspace(-1, 1, 128, device="cuda") * 2.0 ** -126
    x[140, 128:256] = 2.0 ** -140
    x[256:260, :] = torch.linspace(-1, 1, 390, device="cuda") * 1.0e-37
    x = x.to(dtype)
    r, c = A.quantize_fp8(x, (block, 128), code, "both")
    check_blocks(r, x, block, code)
    check_blocks(c, x.t(), block, code)
    check_blocks(A.quantize_fp8(x, (block, 128), code, "rows"), x, block, code)


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("first,cols", [(0, 200), (3, 200), (8, 256), (1, 1), (2, 300), (5, 261), (7, 384)])
def test_quantize_strided_rows(first, cols, dtype):
    """A slice of columns, aligned or not, and a transposed matrix; nothing outside is touched."""
    import advanced_optimizers_b200 as A
    wide = data(300, 521, dtype)
    x = wide[:, first:first + cols]
    for t in (x, x.t(), x[::2], x[:, ::2]):
        r, c = A.quantize_fp8(t, layout="both")
        check_blocks(r, t, 1, E4)
        check_blocks(c, t.t(), 1, E4)
        check_blocks(A.quantize_fp8(t), t, 1, E4)


def test_quantize_empty():
    import advanced_optimizers_b200 as A
    for shape in ((0, 64), (64, 0), (0, 0)):
        r, c = A.quantize_fp8(torch.empty(shape, device="cuda"), layout="both")
        assert tuple(r.codes.shape) == shape and tuple(c.codes.shape) == shape[::-1]


def test_quantize_past_32_bits():
    """More than 2^32 elements: the last rows are those of a small matrix."""
    import advanced_optimizers_b200 as A
    cols, rows = 16400, 262200
    x = torch.zeros(rows, cols, dtype=B, device="cuda")
    tail = data(300, cols, B)
    x[-300:] = tail
    q = A.quantize_fp8(x)
    small = A.quantize_fp8(tail)
    assert torch.equal(q.codes[-300:].view(torch.uint8), small.codes.view(torch.uint8))
    assert torch.equal(q.scales[-300:].view(torch.uint8), small.scales.view(torch.uint8))
    assert int(q.codes[:1000].view(torch.uint8).max()) == 0
    del q
    rows -= rows % 128                      # the same slabs for the columns' blocks
    c = A.quantize_fp8(x[-rows:], layout="cols")
    small = A.quantize_fp8(tail[-256:], layout="cols")
    assert torch.equal(c.codes[:, -256:].view(torch.uint8), small.codes.view(torch.uint8))


def operands(m, n, k, ta, tb, square, seed=0):
    import advanced_optimizers_b200 as A
    a = A.quantize_fp8(data(m, k, F, seed), (1, 128), ta)
    b = A.quantize_fp8(data(n, k, F, seed + 1) * 0.02, (128 if square else 1, 128), tb)
    return a, b


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 200, 4096), (3, 257, 129), (16, 1024, 512), (33, 384, 1000), (64, 100, 640),
          (65, 130, 2048), (128, 128, 128), (128, 256, 96), (129, 256, 640), (130, 1000, 385), (257, 129, 1024),
          (333, 2041, 1000), (512, 512, 4096), (1000, 33, 700), (777, 1, 300), (1024, 768, 14336)]


@pytest.mark.parametrize("out", [B, F])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul(m, n, k, out):
    import advanced_optimizers_b200 as A
    for ta, tb, square in ((E4, E4, True), (E5, E4, False), (E4, E5, True), (E5, E5, False)):
        a, b = operands(m, n, k, ta, tb, square)
        d = A.fp8_matmul(a, b, out)
        assert d.dtype == out
        close_product(d, ref.values(a), ref.values(b), f"{ta} {tb} {square}")
    A.check_fp8_errors()


VARIANTS = [256, 224, 192, 128] + [swap + 1000 * split + bn for swap in (0, 100000) for split in (1, 2, 4, 8)
                                   for bn in (32, 64, 128, 256)]


@pytest.mark.parametrize("out", [B, F])
@pytest.mark.parametrize("variant", VARIANTS)
def test_matmul_every_variant(variant, out):
    """Each kernel the rule can pick, over whole and ragged tiles, short and long K, with every part of the epilogue."""
    from advanced_optimizers_b200 import check_fp8_errors, fp8
    from advanced_optimizers_b200.dropout import drop_fields
    split = variant % 100000 // 1000
    for m, n, k in ((300, 520, 4224), (97, 261, 640), (513, 1000, 2100), (1, 7, 5000), (700, 900, 17000), (2500, 3100, 130)):
        if split > -(-(-(-k // 128)) // 4):
            continue
        a, b = operands(m, n, k, E4, E5, n % 2 == 0)
        av, bv = ref.values(a), ref.values(b)
        close_product(fp8._gemm(a, b, torch.empty(m, n, dtype=out, device="cuda"), variant=variant), av, bv, f"{m} {n} {k}")
        if m < 1000:
            bias, res = data(1, n, out, 7)[0], data(m, n, out, 8)
            key = (77, 3, 5)
            drop = drop_fields(0.25, *key, None)
            d = fp8._gemm(a, b, torch.empty(m, n, dtype=out, device="cuda"), bias, res, drop, variant)
            f = ref.keep_factor((m, n), 0.25, *key)
            want = (av @ bv.t() + bias.double()) * f + res.double()
            mag = (av.abs() @ bv.abs().t() + bias.double().abs()) * f + res.double().abs()
            slack = ((k + 64) * 2.0 ** -22 + 3 * 2.0 ** -23) * mag + half_step(out) * want.abs() * (1 + 2.0 ** -10)
            assert bool(((d.double() - want).abs() <= slack).all()), (m, n, k)
    check_fp8_errors()


@pytest.mark.parametrize("m,n,k", [(4096, 4096, 8192), (300, 14336, 4096), (8, 4096, 14336), (2048, 2048, 2048)])
def test_matmul_large_float32(m, n, k):
    """float32 results: the error of the whole matrix stays near float32's."""
    import advanced_optimizers_b200 as A
    a, b = operands(m, n, k, E4, E4, False)
    d = A.fp8_matmul(a, b, F).double()
    want = ref.values(a) @ ref.values(b).t()
    rel = float((d - want).norm() / want.norm())
    print("relative error", m, n, k, rel)
    # each of the K / 32 instructions loses less than 2^-23 of the accumulator on each of its lanes' sums; their sum is a
    # random walk at worst as long as the bound of one step times K / 32
    assert rel <= (k / 32) * 2.0 ** -23, rel


@pytest.mark.parametrize("m,n,k", [(5, 300, 512), (200, 300, 512), (300, 700, 384)])
def test_matmul_nan_stays_in_its_row(m, n, k):
    import advanced_optimizers_b200 as A
    x, w = data(m, k, F), data(n, k, F, 3)
    x[m // 2, 130] = float("nan")
    w[n - 1, 5] = float("inf")
    d = A.fp8_matmul(A.quantize_fp8(x), A.quantize_fp8(w), F)
    bad = torch.isnan(d)
    want = torch.zeros_like(bad)
    want[m // 2, :] = True
    want[:, n - 1] = True
    assert torch.equal(bad, want)


def test_matmul_given_blocks():
    """Codes and scales made elsewhere: any pitch, any alignment, views of larger tensors."""
    import advanced_optimizers_b200 as A
    g = torch.Generator(device="cuda").manual_seed(1)
    for m, k in ((1, 1000), (5, 100), (130, 513), (64, 640)):
        nb = -(-k // 128)
        codes = torch.randn(m, k + 7, generator=g, device="cuda").to(E4)[:, 3:3 + k]
        scales = torch.randint(120, 134, (m, nb + 3), generator=g, device="cuda", dtype=torch.uint8)[:, 1:1 + nb]
        a = A.Fp8Blocks(codes, scales.view(torch.float8_e8m0fnu))
        want = codes.double() * ref.blocked(ref.pow2(scales.long() - 127), m, k, 1)
        assert torch.equal(ref.values(a), want)
        close_product(A.fp8_matmul(a, a, F), want, want)


def test_matmul_scale_range():
    """Scales far apart between blocks and operands."""
    import advanced_optimizers_b200 as A
    a, b = operands(200, 260, 1024, E4, E4, False)
    sa = a.scales.view(torch.uint8)
    sb = b.scales.view(torch.uint8)
    sa.copy_(torch.randint(60, 190, sa.shape, device="cuda", dtype=torch.uint8))
    sb.copy_(torch.randint(100, 150, sb.shape, device="cuda", dtype=torch.uint8))
    close_product(A.fp8_matmul(a, b, F), ref.values(a), ref.values(b))


def test_matmul_empty():
    import advanced_optimizers_b200 as A
    z = lambda r, k: A.quantize_fp8(torch.zeros(r, k, device="cuda"))  # noqa: E731
    assert tuple(A.fp8_matmul(z(0, 64), z(5, 64)).shape) == (0, 5)
    assert tuple(A.fp8_matmul(z(5, 64), z(0, 64)).shape) == (5, 0)
    assert torch.equal(A.fp8_matmul(z(5, 0), z(3, 0)), torch.zeros(5, 3, dtype=B, device="cuda"))


def test_matmul_repeats_bit_for_bit():
    import advanced_optimizers_b200 as A
    for m, n, k in ((1, 4096, 4096), (40, 1000, 2048), (512, 512, 4096), (2048, 4096, 1024)):
        a, b = operands(m, n, k, E4, E4, True)
        first = A.fp8_matmul(a, b, F)
        for _ in range(3):
            assert torch.equal(first, A.fp8_matmul(a, b, F))


def linear_reference(x, w, bias, residual, dy, p, key, out_dtype):
    T, N = x.shape[0], w.shape[0]
    f = ref.keep_factor((T, N), p, *key)
    T16 = round(p * 65536)
    f32 = float(torch.tensor(65536 / (65536 - T16) if T16 < 65536 else 0.0, dtype=F))
    xq, wq = ref.quantized(x, 1), ref.quantized(w, 128)
    g32 = (dy.float() * f32) * (f > 0)                    # float32, as it is quantised
    g, gt = ref.quantized(g32, 1), ref.quantized(g32.t(), 1)
    xt = ref.quantized(x.t(), 1)
    return f, xq, wq, g32.double(), g, gt, xt


@pytest.mark.parametrize("xd,wd", [(B, B), (F, F), (B, F), (F, B)])
@pytest.mark.parametrize("T,N,K,p,bias,residual", [
    (1, 128, 64, 0.0, False, False), (1, 300, 500, 0.25, True, True), (9, 257, 130, 0.5, True, False),
    (128, 128, 128, 0.1, False, True), (200, 385, 513, 0.1, True, True), (300, 96, 1000, 0.0, True, True),
    (513, 1000, 384, 0.3, True, True), (129, 130, 131, 1.0, True, True)])
def test_linear_and_gradients(T, N, K, p, bias, residual, xd, wd):
    import advanced_optimizers_b200 as A
    g = torch.Generator(device="cuda").manual_seed(T + N + K)
    x = torch.randn(T, K, generator=g, device="cuda").to(xd).requires_grad_()
    w = (torch.randn(N, K, generator=g, device="cuda") * 0.05).to(wd).requires_grad_()
    b = torch.randn(N, generator=g, device="cuda").to(xd).requires_grad_() if bias else None
    r = torch.randn(T, N, generator=g, device="cuda").to(xd).requires_grad_() if residual else None
    dy = torch.randn(T, N, generator=g, device="cuda").to(xd)
    key = (0x123456789AB, 7, 11)
    y = A.fp8_linear(x, w, b, residual=r, dropout_p=p, seed=key[0], site=key[1], step=key[2])
    leaves = [t for t in (x, w, b, r) if t is not None]
    grads = dict(zip([n for n, t in (("x", x), ("w", w), ("b", b), ("r", r)) if t is not None],
                     torch.autograd.grad(y, leaves, dy)))
    f, xq, wq, g32, gq, gt, xt = linear_reference(x.detach(), w.detach(), b, r, dy, p, key, xd)
    bd = b.detach().double() if bias else torch.zeros(N, dtype=torch.float64, device="cuda")
    rd = r.detach().double() if residual else 0.0
    # the epilogue rounds in float32 after the bias, the dropout and the residual: 3 * 2^-24 of the largest of the values
    want = (xq @ wq.t() + bd) * f + rd
    mag = (xq.abs() @ wq.abs().t() + bd.abs()) * f + (r.detach().double().abs() if residual else 0.0)
    slack = ((K + 64) * 2.0 ** -22 + 3 * 2.0 ** -23) * mag + half_step(xd) * want.abs() * (1 + 2.0 ** -10)
    assert bool(((y.detach().double() - want).abs() <= slack + 1e-300).all())
    assert y.dtype == xd and grads["x"].dtype == xd and grads["w"].dtype == wd
    close_product(grads["x"], gq, wq.t(), "dx")
    close_product(grads["w"], gt, xt, "dw")
    if bias:
        slack = (T + 2) * 2.0 ** -23 * g32.abs().sum(0) + half_step(xd) * g32.sum(0).abs() * (1 + 2.0 ** -10)
        assert bool(((grads["b"].double() - g32.sum(0)).abs() <= slack + 1e-300).all())
    if residual:
        assert torch.equal(grads["r"], dy)
    A.check_fp8_errors()


def test_linear_some_gradients():
    """Only the wanted gradients are computed, and each is what the full set gives."""
    import advanced_optimizers_b200 as A
    x, w, b, r, dy = data(200, 300, B), data(260, 300, B, 1) * 0.1, data(1, 260, B, 2)[0], data(200, 260, B, 3), data(200, 260, B, 4)
    kw = dict(dropout_p=0.2, seed=5, site=1, step=2)

    def run(want):
        leaves = [t.detach().clone().requires_grad_(n in want) for n, t in zip("xwbr", (x, w, b, r))]
        y = A.fp8_linear(leaves[0], leaves[1], leaves[2], residual=leaves[3], **kw)
        return y, dict(zip([n for n in "xwbr" if n in want],
                           torch.autograd.grad(y, [t for n, t in zip("xwbr", leaves) if n in want], dy)))

    y0, full = run("xwbr")
    for want in ("x", "w", "b", "r", "xw", "wb", "xr", "bx"):
        y, got = run(want)
        assert torch.equal(y, y0)
        for n in got:
            assert torch.equal(got[n], full[n]), (want, n)
    with torch.no_grad():
        assert torch.equal(A.fp8_linear(x, w, b, residual=r, **kw), y0)


def test_linear_shapes_strides_and_kept_weights():
    import advanced_optimizers_b200 as A
    w = (data(96, 160, F, 1) * 0.1).requires_grad_()
    blocks = A.quantize_fp8(w, (128, 128), layout="both")
    wide = data(12 * 5, 400, F).view(12, 5, 400)
    x = wide[:, :, 40:200].detach().requires_grad_()
    y = A.fp8_linear(x, w, weight_blocks=blocks)
    assert tuple(y.shape) == (12, 5, 96)
    flat = A.fp8_linear(x.detach().reshape(60, 160), w.detach())
    assert torch.equal(y.detach().view(60, 96), flat)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))     # an expanded dy
    ones = torch.ones(60, 96, device="cuda")
    x2, w2 = x.detach().reshape(60, 160).requires_grad_(), w.detach().clone().requires_grad_()
    hx, hw = torch.autograd.grad(A.fp8_linear(x2, w2), (x2, w2), ones)
    assert torch.equal(gx.reshape(60, 160), hx) and torch.equal(gw, hw)
    one = A.fp8_linear(x.detach()[0, 0], w)
    assert tuple(one.shape) == (96,)
    none = torch.zeros(0, 160, device="cuda", requires_grad=True)
    y = A.fp8_linear(none, w, torch.zeros(96, device="cuda"))
    gx, gw = torch.autograd.grad(y.sum(), (none, w))
    assert tuple(y.shape) == (0, 96) and tuple(gx.shape) == (0, 160) and float(gw.abs().max()) == 0.0


def test_linear_gradients_against_differences():
    """d(sum(y dy)) along a direction in x: the layer is linear in the numbers
    its quantised operands stand for, so with x, dy and weights that are their
    own quantised values (small integers) the difference quotient is exact up
    to the float32 sums."""
    import advanced_optimizers_b200 as A
    g = torch.Generator(device="cuda").manual_seed(2)
    ints = lambda *s: torch.randint(-7, 8, s, generator=g, device="cuda").float()  # noqa: E731
    x, w, dy, step = ints(130, 140), ints(70, 140), ints(130, 70), ints(130, 140)
    x, w = x.requires_grad_(), w.requires_grad_()
    f = lambda a, b: (A.fp8_linear(a, b, dropout_p=0.5, seed=3) * dy).double().sum()  # noqa: E731
    gx, gw = torch.autograd.grad(f(x, w), (x, w))
    with torch.no_grad():
        along = (f(x + step, w) - f(x - step, w)) / 2
        wstep = ints(70, 140)
        wlong = (f(x, w + wstep) - f(x, w - wstep)) / 2
    # integers below 15 are exact in e4m3 (4 significant bits), products and sums of them exact in float32
    assert float((gx.double() * step).sum()) == float(along)
    assert float((gw.double() * wstep).sum()) == float(wlong)


def test_linear_on_another_stream_and_captured():
    """A captured forward and backward pass, replayed with the step advanced on the device, draws the masks of those steps."""
    import advanced_optimizers_b200 as A
    x, w = data(150, 256, B).requires_grad_(), (data(200, 256, B, 1) * 0.1).requires_grad_()
    dy = data(150, 200, B, 2)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")

    def run():
        y = A.fp8_linear(x, w, dropout_p=0.3, seed=9, site=4, step=step)
        return (y.detach(),) + torch.autograd.grad(y, (x, w), dy)

    def eager(at):
        y = A.fp8_linear(x, w, dropout_p=0.3, seed=9, site=4, step=at)
        return (y.detach(),) + torch.autograd.grad(y, (x, w), dy)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        warm = run()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(warm, eager(0)):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for at in (5, 6):
        step.fill_(at)
        graph.replay()
        for a, b in zip(outs, eager(at)):
            assert torch.equal(a, b)
    # a step written between the passes is refused
    y = A.fp8_linear(x, w, dropout_p=0.3, step=step)
    step.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, (x, w), dy)


def test_training_run_with_an_optimizer():
    """fp8_linear, philox_dropout and an optimizer step together: two steps run, gradients reach every parameter."""
    import advanced_optimizers_b200 as A
    g = torch.Generator(device="cuda").manual_seed(0)
    w1 = torch.nn.Parameter((torch.randn(256, 128, generator=g, device="cuda") * 0.05).bfloat16())
    w2 = torch.nn.Parameter((torch.randn(128, 256, generator=g, device="cuda") * 0.05).bfloat16())
    b2 = torch.nn.Parameter(torch.zeros(128, device="cuda", dtype=B))
    opt = A.AdamW_adv([w1, w2, b2], lr=1e-3, state_precision="int8_sr")
    x = torch.randn(70, 128, generator=g, device="cuda").bfloat16()
    for step in range(2):
        before = [p.detach().clone() for p in (w1, w2, b2)]
        h = A.philox_dropout(torch.relu(A.fp8_linear(x, w1)), 0.1, site=0, step=step)
        y = A.fp8_linear(h, w2, b2, residual=x, dropout_p=0.1, site=1, step=step)
        y.float().square().mean().backward()
        for p in (w1, w2, b2):
            assert p.grad is not None and bool(torch.isfinite(p.grad).all()) and float(p.grad.abs().max()) > 0
        opt.step()
        opt.zero_grad()
        for p, q in zip((w1, w2, b2), before):
            assert not torch.equal(p.detach(), q)
    A.check_fp8_errors()


def test_products_on_two_streams_at_once():
    import advanced_optimizers_b200 as A
    cases = [operands(m, n, k, E4, E4, True, i) for i, (m, n, k) in enumerate(((8, 4096, 4096), (700, 2048, 2048), (33, 500, 8192)))]
    want = [A.fp8_matmul(a, b, F) for a, b in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] += [A.fp8_matmul(a, b, F) for a, b in cases]
    torch.cuda.synchronize()
    for results in got:
        for i, d in enumerate(results):
            assert torch.equal(d, want[i % 3])
    A.check_fp8_errors()


def test_products_captured_and_replayed_on_new_data():
    """A captured chain quantise -> product -> product, as the first call that would need the error word, and replays on other data."""
    import advanced_optimizers_b200 as A
    from advanced_optimizers_b200 import fp8
    x = data(40, 512, B)
    w1, w2 = (A.quantize_fp8(data(n, k, F, n) * 0.05, (128, 128)) for n, k in ((768, 512), (300, 768)))

    def chain():
        return A.fp8_matmul(A.quantize_fp8(A.fp8_matmul(A.quantize_fp8(x), w1)), w2, F)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        chain()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    word, fp8._ERR.word = fp8._ERR.word, None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain()
    fp8._ERR.word = word
    for seed in (5, 6, 7):
        x.copy_(data(40, 512, B, seed))
        graph.replay()
        assert torch.equal(out, chain())


def test_a_matrix_times_itself():
    import advanced_optimizers_b200 as A
    x = data(260, 384, F).requires_grad_()
    y = A.fp8_linear(x, x)
    dy = data(260, 260, F, 1)
    g, = torch.autograd.grad(y, x, dy)
    a, b = x.detach().clone().requires_grad_(), x.detach().clone().requires_grad_()
    ga, gb = torch.autograd.grad(A.fp8_linear(a, b), (a, b), dy)
    assert torch.equal(g, ga + gb)


def test_refusals_on_the_device():
    import advanced_optimizers_b200 as A
    x = torch.zeros(4, 256, device="cuda")
    q = A.quantize_fp8(x)
    with pytest.raises(NotImplementedError):
        A.quantize_fp8(x.half())
    with pytest.raises(NotImplementedError):
        A.fp8_matmul(q, q, torch.float16)
    with pytest.raises(ValueError, match="quantised along"):
        A.fp8_matmul(q, A.quantize_fp8(x[:, :128]))
    with pytest.raises(ValueError, match="need scales"):
        A.Fp8Blocks(q.codes, q.scales[:, :1])
    with pytest.raises(ValueError, match="weight_blocks"):
        A.fp8_linear(x, torch.zeros(8, 256, device="cuda"), weight_blocks=A.quantize_fp8(x, (128, 128), layout="both"))
    with pytest.raises(ValueError, match="bias"):
        A.fp8_linear(x, torch.zeros(8, 256, device="cuda"), torch.zeros(7, device="cuda"))
    with pytest.raises(ValueError, match="residual"):
        A.fp8_linear(x, torch.zeros(8, 256, device="cuda"), residual=torch.zeros(4, 9, device="cuda"))
    with pytest.raises(NotImplementedError):
        A.fp8_linear(x.half(), torch.zeros(8, 256, device="cuda"))


def test_second_derivatives_are_refused():
    import advanced_optimizers_b200 as A
    x, w = data(40, 128, F).requires_grad_(), data(50, 128, F, 1).requires_grad_()
    dy = data(40, 50, F, 2).requires_grad_()
    y = A.fp8_linear(x, w)
    want = torch.autograd.grad(A.fp8_linear(x, w), (x, w), dy.detach())
    got = torch.autograd.grad(y, (x, w), dy, create_graph=True)
    assert all(torch.equal(a.detach(), b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(got[0].sum(), dy)


def test_kept_blocks_are_saved_tensors():
    """They go with the graph's other saved tensors: through hooks that move them, and released by the backward pass."""
    import advanced_optimizers_b200 as A
    x, w, dy = data(40, 256, B).requires_grad_(), data(130, 256, B, 1).requires_grad_(), data(40, 130, B, 2)
    want = torch.autograd.grad(A.fp8_linear(x, w), (x, w), dy)
    with torch.autograd.graph.save_on_cpu():
        y = A.fp8_linear(x, w)
    filler = torch.randint(0, 255, (1 << 20,), device="cuda", dtype=torch.uint8)   # over what was moved away
    got = torch.autograd.grad(y, (x, w), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and filler.numel()
    y = A.fp8_linear(x, w)
    torch.autograd.grad(y, (x, w), dy)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, (x, w), dy)
    y = A.fp8_linear(x, w)
    torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, w), dy), want))


@pytest.mark.parametrize("variant", [0, 1256, 101256])
def test_matmul_past_32_bits(variant):
    """A result of more than 2^32 elements: its last rows are those of a small product."""
    from advanced_optimizers_b200 import check_fp8_errors, fp8
    m, n, k = 66000, 66048, 160
    a, b = operands(m, n, k, E4, E4, False)
    d = fp8._gemm(a, b, torch.empty(m, n, dtype=B, device="cuda"), variant=variant)
    check_fp8_errors()
    tail = fp8.Fp8Blocks(a.codes[-300:], a.scales[-300:])
    want = fp8._gemm(tail, b, torch.empty(300, n, dtype=B, device="cuda"), variant=variant)
    assert torch.equal(d[-300:], want)
    close_product(want[-200:, -200:], ref.values(tail)[-200:], ref.values(b)[-200:])
    close_product(d[:200, :200], ref.values(a)[:200], ref.values(b)[:200])


def test_a_wait_that_gave_up_is_reported_once():
    """The word a kernel's bounded wait would set (here set by the host): the next call and check_fp8_errors raise, then calls work again."""
    import advanced_optimizers_b200 as A
    from advanced_optimizers_b200 import _lib, fp8
    a, b = operands(8, 128, 256, E4, E4, True)
    want = A.fp8_matmul(a, b)
    fp8._ERR.view[0] = 1
    with pytest.raises(_lib.AdvOptError, match="bounded wait"):
        A.fp8_matmul(a, b)
    fp8._ERR.view[0] = 1
    with pytest.raises(_lib.AdvOptError, match="bounded wait"):
        A.check_fp8_errors()
    A.check_fp8_errors()
    assert torch.equal(A.fp8_matmul(a, b), want)


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("T,N", [(256, 384), (150, 261)])
def test_linear_infinities_in_dropped_places(T, N, dtype):
    """What is dropped does not reach a gradient, whatever stands there; a kept infinity reaches its row of dx and of dweight alone."""
    import advanced_optimizers_b200 as A
    x, w = data(T, 256, dtype).requires_grad_(), (data(N, 256, dtype, 1) * 0.1).requires_grad_()
    b = torch.zeros(N, device="cuda", dtype=dtype, requires_grad=True)
    key = (123, 4, 5)
    f = ref.keep_factor((T, N), 0.5, *key)
    dy = torch.where(f > 0, data(T, N, dtype, 2).float(), torch.zeros((), device="cuda")).to(dtype)
    run = lambda g: torch.autograd.grad(A.fp8_linear(x, w, b, dropout_p=0.5, seed=key[0], site=key[1], step=key[2]), (x, w, b), g)  # noqa: E731
    want = run(dy)
    bad = dy.clone()
    at = (f == 0).nonzero()
    bad[at[::3, 0], at[::3, 1]] = float("inf")
    bad[at[1::3, 0], at[1::3, 1]] = float("nan")
    for got, w0 in zip(run(bad), want):
        assert bool(torch.isfinite(got).all()) and torch.equal(got, w0)
    i, j = (f > 0).nonzero()[1000].tolist()
    bad[i, j] = float("-inf")
    dx, dw, db = run(bad)
    rows = torch.zeros(T, dtype=torch.bool, device="cuda")
    rows[i] = True
    assert torch.equal(torch.isnan(dx).all(1), rows) and torch.equal(torch.isnan(dx).any(1), rows)
    cols = torch.zeros(N, dtype=torch.bool, device="cuda")
    cols[j] = True
    assert torch.equal(torch.isnan(dw).all(1), cols) and torch.equal(torch.isnan(dw).any(1), cols)
    assert torch.equal(~torch.isfinite(db), cols)

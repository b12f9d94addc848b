"""Sums of the fp8 product at long K, compared for equality.

Small integers: with operands that are whole numbers of magnitude at most 16
every product and every sum of up to 2^15 of them is below 2^24, so float32
holds them exactly in any order, and a bfloat16 result is the exact sum's one
rounding.  A block, tail or chunk that is lost, doubled or misplaced shows.

Cuts: a float32 result of long K is the float32 sum, in order, of the products
of chunks of at most 64 blocks: those of a CTA's accumulators, then those of
the cluster that K is split over, then those of the launches.  So it equals the
chunks' products, each made by a call of its own and added here."""
import functools

import pytest
import torch

import _fp8_ref as ref

pytestmark = pytest.mark.gpu

E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
B, F = torch.bfloat16, torch.float32
PAIRS = [256, 224, 192, 128]
SINGLES = [swap + 1000 * split + bn for swap in (0, 100000) for split in (1, 2, 4, 8) for bn in (32, 64, 128, 256)]


def whole(rows, k, code, square, seed):
    """Fp8Blocks of whole numbers up to 16 in magnitude, a power of two apart between blocks, and those numbers."""
    import advanced_optimizers_b200 as A
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(-4, 5, (rows, k), generator=g, device="cuda").double()
    block = 128 if square else 1
    f = torch.randint(0, 3, (-(-rows // block), -(-k // 128)), generator=g, device="cuda")
    x = x * ref.blocked(ref.pow2(f), rows, k, block)
    b = A.quantize_fp8(x.float(), (block, 128), code)
    assert torch.equal(ref.values(b), x)
    return b, x


def splits(variant, k):
    return variant % 100000 // 1000 <= -(-k // 512)


@pytest.mark.parametrize("out", [B, F])
@pytest.mark.parametrize("variant", [0] + PAIRS + SINGLES)
def test_whole_numbers_are_summed_exactly(variant, out):
    from advanced_optimizers_b200 import check_fp8_errors, fp8
    for m, n, k in ((700, 900, 17000), (130, 261, 32700), (1, 7, 5000)):
        if splits(variant, k):
            (a, av), (b, bv) = whole(m, k, E4, False, m), whole(n, k, E5, n % 2 == 0, n)
            d = fp8._gemm(a, b, torch.full((m, n), float("nan"), dtype=out, device="cuda"), variant=variant)
            assert torch.equal(d, (av @ bv.t()).to(out)), (m, n, k)
    check_fp8_errors()


MANY = [(2500, 3100, 130, B), (2500, 3100, 130, F), (1300, 4000, 8320, B), (1300, 4000, 8320, F), (2500, 3099, 130, F), (70, 50, 140000, F), (70, 50, 300100, F)]


@pytest.mark.parametrize("variant,m,n,k,out", [(v, *c) for v in [0] + PAIRS + [1256, 101064, 2128, 108032] for c in MANY if splits(v, c[2])])
def test_bias_dropout_and_residual_of_many_tiles(variant, m, n, k, out):
    """More tiles than pairs of CTAs, and chunked sums: the extras are applied once, to the whole sum.  All steps are
    exact: the factor of the kept ones is 2, bias and residual are whole numbers."""
    from advanced_optimizers_b200 import check_fp8_errors, fp8
    from advanced_optimizers_b200.dropout import drop_fields
    (a, av), (b, bv) = whole(m, k, E4, False, 1), whole(n, k, E4, True, 2)
    if k > 1 << 15:      # keep the sums below 2^24
        keep = torch.arange(k, device="cuda") % 5 == 0
        av = av * keep
        a.codes.view(torch.uint8).mul_(keep.to(torch.uint8))
        assert torch.equal(ref.values(a), av)
    g = torch.Generator(device="cuda").manual_seed(3)
    bias = torch.randint(-100, 101, (n,), generator=g, device="cuda").to(out)
    res = torch.randint(-100, 101, (m, n), generator=g, device="cuda").to(out)
    key = (77, 3, 5)
    f = ref.keep_factor((m, n), 0.5, *key)
    d = fp8._gemm(a, b, torch.full((m, n), float("nan"), dtype=out, device="cuda"), bias, res, drop_fields(0.5, *key, None), variant)
    want = (av @ bv.t() + bias.double()) * f + res.double()
    assert float(want.abs().max()) < 2 ** 24
    assert torch.equal(d, want.to(out))
    check_fp8_errors()


def starts(total, parts):
    """total things in parts, as even as they come: where each starts, and the end."""
    return [total * i // parts for i in range(parts + 1)]


def chunks(first, last, parts):
    """Blocks first .. last - 1 in equal parts of whole scale words (four blocks)."""
    size = -(-(-(-(last - first) // parts)) // 4) * 4
    return [(i, min(i + size, last)) for i in range(first, last, size)]


def plan(variant, k):
    """[launches or chunks of D's sum][CTAs of a cluster][accumulators] of (first block, last block)."""
    nb = -(-k // 128)
    if variant < 1000:
        return [[[c]] for c in chunks(0, nb, -(-nb // 64))]
    split, bn, groups = variant % 100000 // 1000, variant % 1000, -(-nb // 4)
    accs = {32: 7, 64: 7, 128: 3, 256: 1}[bn]
    at, out = starts(groups, -(-groups // (16 * split * accs))), []
    for g0, g1 in zip(at, at[1:]):
        ranks = [(4 * (g0 + r0), min(4 * (g0 + r1), nb)) for r0, r1 in zip(starts(g1 - g0, split), starts(g1 - g0, split)[1:])]
        out.append([chunks(i, j, -(-(j - i) // 64)) for i, j in ranks])
    return out


def sum_of_chunks(a, b, variant):
    """The plan's products, each by a call that sums at most 64 blocks in one accumulator of the same tile, added up here."""
    from advanced_optimizers_b200 import fp8
    one = variant if variant < 1000 else variant - variant % 100000 + 1000 + variant % 1000   # split 1

    def product(i, j):
        part = [fp8.Fp8Blocks(q.codes[:, 128 * i:min(128 * j, q.k)], q.scales[:, i:j]) for q in (a, b)]
        return fp8._gemm(*part, torch.empty(a.rows, b.rows, dtype=F, device="cuda"), variant=one)

    add = lambda terms: functools.reduce(torch.add, terms)  # noqa: E731
    p = plan(variant, a.k)
    assert all(j - i <= 64 for d in p for r in d for i, j in r)
    return add(add(add(product(*c) for c in r) for r in d) for d in p), sum(len(r) for d in p for r in d)


def operands(m, n, k):
    import advanced_optimizers_b200 as A
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    return [A.quantize_fp8(torch.randn(r, k, generator=g, device="cuda")) for r in (m, n)]


@pytest.mark.parametrize("variant", PAIRS + SINGLES)
def test_float32_results_are_sums_of_chunks(variant):
    from advanced_optimizers_b200 import check_fp8_errors, fp8
    for m, n, k in ((300, 520, 17000), (33, 100, 70000), (130, 70, 300100)):
        a, b = operands(m, n, k)
        want, parts = sum_of_chunks(a, b, variant)
        d = fp8._gemm(a, b, torch.full((m, n), float("nan"), dtype=F, device="cuda"), variant=variant)
        assert torch.equal(d, want), (m, n, k, parts)
    assert parts > 8      # a CTA's sum was cut
    check_fp8_errors()


@pytest.mark.parametrize("m,n,k", [(256, 256, 131072), (64, 128, 300000), (1024, 1024, 131072), (5, 4096, 70016), (17, 33, 1000000)])
def test_float32_results_of_the_rule_s_choice_are_sums_of_chunks(m, n, k):
    """Weight gradients over many tokens: whichever variant the rule picks cuts its sums."""
    import advanced_optimizers_b200 as A
    a, b = operands(m, n, k)
    d = A.fp8_matmul(a, b, F)
    assert any(torch.equal(d, sum_of_chunks(a, b, v)[0]) for v in PAIRS + SINGLES)
    A.check_fp8_errors()


def test_a_captured_long_sum_with_extras():
    """Its launches follow one another in a graph, on other data at each replay."""
    import advanced_optimizers_b200 as A
    from advanced_optimizers_b200 import fp8
    x, w = (torch.randn(r, 140000, device="cuda") for r in (70, 50))
    bias, res = torch.randn(50, device="cuda"), torch.randn(70, 50, device="cuda")
    out = torch.empty(70, 50, device="cuda")

    def run(d):
        return fp8._gemm(A.quantize_fp8(x), A.quantize_fp8(w), d, bias, res, variant=2128)

    run(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(out)
    for _ in range(2):
        x.normal_()
        graph.replay()
        assert torch.equal(out, run(torch.empty_like(out)))

"""Token embedding and its gradient against 64-bit sums (tests/_rows_ref.py)."""
import pytest
import torch

import _rows_ref as ref

pytestmark = pytest.mark.gpu

B, F = torch.bfloat16, torch.float32


def make(T, V, C, dtype, ids="zipf", seed=0, id_dtype=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed + T + V + C)
    if ids == "zipf":
        t = (torch.rand(T, generator=g, device="cuda", dtype=torch.float64) * torch.log(torch.tensor(float(V)))).exp().long().sub(1).clamp(0, V - 1)
    elif ids == "same":
        t = torch.full((T,), V // 2, device="cuda")
    elif ids == "each":
        t = torch.randperm(max(T, V), generator=g, device="cuda")[:T] % V
    else:
        t = torch.randint(V, (T,), generator=g, device="cuda").sort().values
    w = torch.randn(V, C, generator=g, device="cuda").to(dtype)
    dy = torch.randn(T, C, generator=g, device="cuda").to(dtype)
    return t.to(id_dtype), w, dy


def check(ids, w, dy, scale=1.0, padding=None):
    import advanced_optimizers_b200 as A
    w = w.detach().requires_grad_()
    y = A.embedding(ids, w, scale=scale, padding_idx=padding)
    want = w.detach()[ids.long()].double() * scale
    ref.close(y, want, ref.U * want.abs() if scale != 1.0 else torch.zeros_like(want), w.dtype)
    if scale == 1.0:
        assert torch.equal(y.detach(), w.detach()[ids.long()])
    dw, = torch.autograd.grad(y, w, dy)
    ref.close(dw, *ref.embedding_grad(ids, dy, w.shape[0], scale, padding), w.dtype)
    return dw


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("T,V,C", [(1, 1, 1), (1, 7, 8), (31, 5, 3), (32, 33, 264), (33, 512, 256), (100, 511, 129), (1000, 513, 20), (2049, 300, 64), (256, 20000, 5), (256, 70, 520),
                                   (4096, 50304, 72), (9001, 1000, 136), (70000, 262145, 8), (257, 100, 5003)])
def test_embedding_and_gradient(T, V, C, dtype):
    ids, w, dy = make(T, V, C, dtype)
    check(ids, w, dy)


@pytest.mark.parametrize("how", ["same", "each", "sorted"])
@pytest.mark.parametrize("T,V,C", [(1, 3, 40), (64, 64, 8), (1025, 40, 300), (33000, 70, 24)])
def test_orders_of_ids(T, V, C, how):
    ids, w, dy = make(T, V, C, F, how)
    check(ids, w, dy, scale=0.37)
    check(ids.int(), w, dy, padding=V // 2)


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("padding", [0, 3, -1])
def test_scale_and_padding(dtype, padding):
    ids, w, dy = make(3000, 50, 136, dtype, id_dtype=torch.int32)
    dw = check(ids, w, dy, scale=8.5, padding=padding)
    assert bool((dw[padding] == 0).all())


def test_shapes_strides_and_empty_calls():
    import advanced_optimizers_b200 as A
    ids, w, _ = make(24, 50, 48, F)
    wide = torch.randn(50, 61, device="cuda")
    for table in (w, wide[:, :48], wide[:, 1:49], wide[:, 3:52], wide.t()[:48].t(), w[::2], wide[:1].expand(50, 61)):
        for t in (ids % table.shape[0], (ids % table.shape[0]).view(4, 6), (ids % table.shape[0]).view(4, 6).t(), (ids % table.shape[0])[::3]):
            assert torch.equal(A.embedding(t, table), table[t])
            leaf = table.detach().clone().requires_grad_()
            y = A.embedding(t, leaf)
            dy = torch.randn(y.shape, device="cuda")
            for g in (dy, dy.transpose(0, 1).contiguous().transpose(0, 1), dy[..., :1].expand_as(dy)):
                dw, = torch.autograd.grad(y, leaf, g, retain_graph=True)
                ref.close(dw, *ref.embedding_grad(t, g.reshape(*t.shape, -1), leaf.shape[0], 1.0, None), F)
    leaf = w.clone().requires_grad_()
    y = A.embedding(ids[:0], leaf)
    assert y.shape == (0, 48)
    assert torch.equal(torch.autograd.grad(y.sum(), leaf)[0], torch.zeros_like(w))
    assert A.embedding(ids, w[:, :0]).shape == (24, 0)
    assert A.embedding(ids[0], w).shape == (48,)


def test_ids_outside_the_table():
    import advanced_optimizers_b200 as A
    A.check_index_errors()
    ids, w, dy = make(300, 50, 24, B)
    bad = ids.clone()
    bad[7], bad[100], bad[299], bad[32] = -1, 50, 1 << 40, -(1 << 50)
    leaf = w.clone().requires_grad_()
    y = A.embedding(bad, leaf)
    wrong = (bad < 0) | (bad >= 50)
    assert bool(y[wrong].isnan().all()) and torch.equal(y[~wrong].detach(), w[bad[~wrong]])
    dw, = torch.autograd.grad(y, leaf, dy)
    ref.close(dw, *ref.embedding_grad(bad, dy, 50, 1.0, None), B)
    with pytest.raises(A.embeddings.L.AdvOptError, match="outside its table"):
        A.check_index_errors()
    A.embedding(bad, w)
    torch.cuda.synchronize()
    with pytest.raises(A.embeddings.L.AdvOptError, match="outside its table"):
        A.embedding(ids, w)
    assert torch.equal(A.embedding(ids, w), w[ids])
    A.check_index_errors()


def test_infinities_stay_in_their_rows():
    import advanced_optimizers_b200 as A
    ids, w, dy = make(500, 60, 40, F)
    dy[3, 5], dy[77, 0] = float("inf"), float("nan")
    leaf = w.requires_grad_()
    dw, = torch.autograd.grad(A.embedding(ids, leaf), leaf, dy)
    touched = torch.zeros_like(dw, dtype=torch.bool)
    touched[ids[3], 5] = touched[ids[77], 0] = True
    assert torch.equal(~dw.isfinite(), touched)


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("T", [200, 20000])
def test_repeats_bit_for_bit_on_other_streams_and_in_graphs(T, dtype):
    import advanced_optimizers_b200 as A
    ids, w, dy = make(T, 400, 264, dtype)
    leaf = w.requires_grad_()
    run = lambda: torch.autograd.grad(A.embedding(ids, leaf, padding_idx=3), leaf, dy)[0]  # noqa: E731
    want = run()
    for _ in range(3):
        assert torch.equal(run(), want)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            got.append([run() for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for gs in got for g in gs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    new = torch.randint_like(ids, 400)
    ids.copy_(new)
    dy.mul_(2)
    graph.replay()
    ref.close(out, *ref.embedding_grad(ids, dy, 400, 1.0, 3), dtype)


@pytest.mark.parametrize("repeat", [1, 100])
def test_more_than_2_to_32_elements(repeat):
    import advanced_optimizers_b200 as A
    V, C = 70000, 65536
    w = torch.zeros(V, C, dtype=B, device="cuda")
    ids = torch.tensor([0, V - 1, 65537, V - 1], device="cuda").repeat(repeat)
    w[V - 1], w[65537] = 3.0, 5.0
    leaf = w.requires_grad_()
    y = A.embedding(ids, leaf)
    assert y.float().mean(1).tolist() == [0.0, 3.0, 5.0, 3.0] * repeat
    dw, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert [float(dw[i].float().mean()) for i in (0, 1, 65537, V - 2, V - 1)] == [n * repeat for n in (1.0, 0.0, 1.0, 0.0, 2.0)]
    total = sum(float(part.float().sum()) for part in dw.split(10000))
    assert total == 4.0 * C * repeat


def test_hooks_on_saved_tensors_and_other_derivatives():
    import advanced_optimizers_b200 as A
    ids, w, dy = make(200, 40, 16, F)
    leaf = w.requires_grad_()
    want, = torch.autograd.grad(A.embedding(ids, leaf), leaf, dy)
    with torch.autograd.graph.save_on_cpu():
        y = A.embedding(ids, leaf)
    assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], want)
    y = A.embedding(ids, leaf)
    ids.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaf, dy)
    y = A.embedding(ids, leaf)
    g, = torch.autograd.grad(y, leaf, dy.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    from torch.autograd import forward_ad
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        A.embedding(ids, forward_ad.make_dual(w.detach(), w.detach()))

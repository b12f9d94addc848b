"""Autograd rules of the dropout and fp8 operators on the device: saved-tensor
hooks, checkpointing and forward-mode derivatives.  Results are compared for
equality with those of the same call without them."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu

B, F = torch.bfloat16, torch.float32


def inputs(T=70, N=200, K=256, dtype=B):
    g = torch.Generator(device="cuda").manual_seed(T + N + K)
    x = torch.randn(T, K, generator=g, device="cuda").to(dtype).requires_grad_()
    w = (torch.randn(N, K, generator=g, device="cuda") * 0.05).to(dtype).requires_grad_()
    b = torch.randn(N, generator=g, device="cuda").to(dtype).requires_grad_()
    dy = torch.randn(T, N, generator=g, device="cuda").to(dtype)
    return x, w, b, dy


def linear(x, w, b, step):
    import advanced_optimizers_b200 as A
    return A.fp8_linear(x, w, b, dropout_p=0.4, seed=9, site=4, step=step)


def dropout(x, step):
    import advanced_optimizers_b200 as A
    return A.philox_dropout(x, 0.4, seed=9, site=4, step=step)


@pytest.mark.parametrize("how", ["advanced", "freed"])
def test_device_step_on_saved_tensors_kept_elsewhere(how):
    """The backward pass draws the forward pass's mask from the kept copy of the step, though the caller's was advanced or freed."""
    x, w, b, dy = inputs()
    want_l = torch.autograd.grad(linear(x, w, b, 7), (x, w, b), dy)
    want_d, = torch.autograd.grad(dropout(w, 7), w, w.detach())
    with torch.autograd.graph.save_on_cpu():
        step = torch.full((1,), 7, dtype=torch.int64, device="cuda")
        y, d = linear(x, w, b, step), dropout(w, step)
    step.fill_(8)                     # freed memory is anyone's
    if how == "freed":
        del step
        others = [torch.full((1,), 8, dtype=torch.int64, device="cuda") for _ in range(64)]
        assert len(others) == 64
    for got, want in zip(torch.autograd.grad(y, (x, w, b), dy), want_l):
        assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(d, w, w.detach())[0], want_d)


def test_device_step_under_checkpointing():
    x, w, b, dy = inputs()
    want_l = torch.autograd.grad(linear(x, w, b, 7), (x, w, b), dy)
    want_d, = torch.autograd.grad(dropout(w, 7), w, w.detach())
    step = torch.full((1,), 7, dtype=torch.int64, device="cuda")
    for got, want in zip(torch.autograd.grad(checkpoint(linear, x, w, b, step, use_reentrant=False), (x, w, b), dy), want_l):
        assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(checkpoint(dropout, w, step, use_reentrant=False), w, w.detach())[0], want_d)
    y, d = checkpoint(linear, x, w, b, step, use_reentrant=False), checkpoint(dropout, w, step, use_reentrant=False)
    step.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, (x, w, b), dy)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(d, w, w.detach())


@pytest.mark.parametrize("p", [0.0, 1e-6, 1.0])
def test_a_step_that_no_mask_depends_on_may_be_advanced(p):
    import advanced_optimizers_b200 as A
    x, w, b, dy = inputs()
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    lin = lambda s: A.fp8_linear(x, w, b, dropout_p=p, step=s)  # noqa: E731
    drop = lambda s: A.philox_dropout(w, p, step=s)  # noqa: E731
    y, d = lin(step), drop(step)
    step.add_(1)
    for got, want in zip(torch.autograd.grad(y, (x, w, b), dy), torch.autograd.grad(lin(0), (x, w, b), dy)):
        assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(d, w, w.detach())[0], torch.autograd.grad(drop(0), w, w.detach())[0])


def test_forward_mode_is_refused():
    """It was lost without a word where the call does not go through an autograd function."""
    import advanced_optimizers_b200 as A
    from torch.autograd import forward_ad
    x, w, b, _ = (t.detach() for t in inputs())
    r = torch.zeros(70, 200, device="cuda", dtype=B)
    for guard in (torch.enable_grad, torch.no_grad):
        with guard(), forward_ad.dual_level():
            dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
            for call in (lambda: A.philox_dropout(dual(x), 0.3), lambda: A.philox_dropout(x, 0.3, residual=dual(x)),
                         lambda: A.fp8_linear(dual(x), w, b, residual=r), lambda: A.fp8_linear(x, dual(w), b, residual=r),
                         lambda: A.fp8_linear(x, w, dual(b), residual=r), lambda: A.fp8_linear(x, w, b, residual=dual(r))):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
            assert tuple(A.philox_dropout(x, 0.3).shape) == tuple(x.shape)
            assert tuple(A.fp8_linear(x, w, b, residual=r).shape) == (70, 200)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: A.philox_dropout(t, 0.3), (x,), (x,))


@pytest.mark.parametrize("N,K", [(1, 300), (200, 1), (1, 1), (200, 300)])
def test_weight_blocks_made_from_their_tensors(N, K):
    """Also of a single row or column, whose scales do not tell the two block shapes apart."""
    import advanced_optimizers_b200 as A
    x, w, b, dy = inputs(70, N, K)
    blocks = A.quantize_fp8(w, (128, 128), layout="both")
    again = [A.Fp8Blocks(q.codes, q.scales) for q in blocks]
    y, want = A.fp8_linear(x, w, b, weight_blocks=blocks), A.fp8_linear(x, w, b)
    z = A.fp8_linear(x, w, b, weight_blocks=again)
    assert torch.equal(y, want) and torch.equal(z, want)
    grads = [torch.autograd.grad(t, (x, w, b), dy) for t in (want, y, z)]
    for got in grads[1:]:
        assert all(torch.equal(g, h) for g, h in zip(got, grads[0]))
    rows = A.quantize_fp8(w, (1, 128), layout="both")
    if N > 1 and K > 1:
        with pytest.raises(ValueError, match="weight_blocks"):
            A.fp8_linear(x, w, b, weight_blocks=rows)


def test_a_residual_s_gradient_does_not_read_the_step():
    import advanced_optimizers_b200 as A
    x, w, b, dy = (t.detach() for t in inputs())
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    r, q = (torch.zeros(s, device="cuda", dtype=B, requires_grad=True) for s in ((70, 200), (70, 256)))
    y = A.fp8_linear(x, w, b, residual=r, dropout_p=0.4, step=step)
    d = A.philox_dropout(x, 0.4, residual=q, step=step)
    step.add_(1)
    assert torch.equal(torch.autograd.grad(y, r, dy)[0], dy)
    assert torch.equal(torch.autograd.grad(d, q, x)[0], x)

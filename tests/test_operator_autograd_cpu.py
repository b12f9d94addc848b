"""Autograd rules of the dropout and fp8 operators that need no GPU: the kernel
launches are replaced by readers of the addresses that they are given."""
import ctypes
import gc
import types

import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks
from torch.utils.checkpoint import checkpoint


@pytest.fixture
def steps_read(monkeypatch):
    """`_Dropout` on CPU tensors: a launch multiplies by the step at the address of its fields, and notes it."""
    from advanced_optimizers_b200 import dropout
    seen = []

    def launch(x, residual, fields):
        step = ctypes.c_int64.from_address(fields[1]).value if fields[1] else fields[3]
        seen.append(step)
        return x * step if residual is None else residual + x * step

    monkeypatch.setattr(dropout, "_launch", launch)
    return seen


def apply(x, step):
    from advanced_optimizers_b200.dropout import _Dropout, drop_fields
    return _Dropout.apply(x, None, step, drop_fields(0.5, 1, 0, step, x.device))


copying = lambda: saved_tensors_hooks(lambda t: t.clone(), lambda t: t)  # noqa: E731


def test_step_of_a_copied_saved_tensor_is_the_forward_pass_s(steps_read):
    """A hook that keeps a copy keeps the step's value too, whatever the caller does to the tensor in between."""
    x, step = torch.ones(4, requires_grad=True), torch.tensor([7])
    with copying():
        y = apply(x, step)
    step.add_(1)
    g, = torch.autograd.grad(y.sum(), x)
    assert steps_read == [7, 7] and torch.equal(g, torch.full((4,), 7.0))


def test_step_of_a_copied_saved_tensor_outlives_the_caller_s(steps_read):
    x, step = torch.ones(4, requires_grad=True), torch.tensor([7])
    kept = step                       # the test's own reference, so that the overwritten memory stays the test's
    with copying():
        y = apply(x, step)
    del step
    gc.collect()
    kept.data.fill_(99)               # what the address holds once it is someone else's
    torch.autograd.grad(y.sum(), x)
    assert steps_read == [7, 7]


def test_step_of_the_second_derivative_is_the_saved_one(steps_read):
    x, dy, step = torch.ones(4, requires_grad=True), torch.ones(4, requires_grad=True), torch.tensor([7])
    with copying():
        y = apply(x, step)
        step.add_(1)
        g, = torch.autograd.grad(y, x, dy, create_graph=True)
    torch.autograd.grad(g.sum(), dy)
    assert steps_read == [7, 7, 7]


def test_step_written_between_the_passes_is_refused(steps_read):
    x, step = torch.ones(4, requires_grad=True), torch.tensor([7])
    y = apply(x, step)
    step.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)
    step = torch.tensor([7])
    y = checkpoint(apply, x, step, use_reentrant=False)
    step.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)
    assert 8 not in steps_read


def test_step_under_checkpointing(steps_read):
    x, step = torch.ones(4, requires_grad=True), torch.tensor([7])
    g, = torch.autograd.grad(checkpoint(apply, x, step, use_reentrant=False).sum(), x)
    assert torch.equal(g, torch.full((4,), 7.0)) and set(steps_read) == {7}


@pytest.mark.parametrize("unpacked", [torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int64),
                                      torch.zeros(1, dtype=torch.int64, device="meta")])
def test_a_hook_that_gives_another_kind_of_step_is_refused(steps_read, unpacked):
    x, step = torch.ones(4, requires_grad=True), torch.tensor([7])
    with saved_tensors_hooks(lambda t: t, lambda t: unpacked):
        y = apply(x, step)
    with pytest.raises(RuntimeError, match="for the step"):
        torch.autograd.grad(y.sum(), x)
    assert steps_read == [7]


@pytest.mark.parametrize("kept", [dict(size=-1), dict(size=1), dict(dtype=torch.int8), dict(device="meta"), dict(stride=2)])
def test_a_hook_that_gives_other_kept_blocks_is_refused(kept):
    """Before any launch: the kernels would read what is not there."""
    from advanced_optimizers_b200 import fp8
    T, N, K = 5, 40, 256
    size = fp8._kept_at(0, T, N, K, True, True, True)[2] + kept.get("size", 0)
    t = torch.zeros(size * kept.get("stride", 1), dtype=kept.get("dtype", torch.uint8),
                    device=kept.get("device", "cpu"))[::kept.get("stride", 1)]
    ctx = types.SimpleNamespace(saved_tensors=(t,), needs_input_grad=(True, True, False, False), K=K, blocks=None, keeps=True,
                                stepped=False, drop=fp8.NO_DROP, w_dtype=torch.float32)
    with pytest.raises(RuntimeError, match="for the kept blocks"):
        fp8._linear_backward(ctx, torch.zeros(T, N))


@pytest.mark.parametrize("p,reads", [(0.0, False), (1e-6, False), (0.5, True), (1.0, False)])
def test_a_mask_that_is_the_same_at_every_step_reads_none(p, reads):
    from advanced_optimizers_b200.dropout import drop_fields
    step = torch.tensor([7])
    assert drop_fields(p, 1, 0, step, step.device)[1] == (step.data_ptr() if reads else 0)
    with pytest.raises(ValueError, match="step tensor"):
        drop_fields(p, 1, 0, torch.zeros(2, dtype=torch.int64), step.device)


def test_tangents_are_found():
    """At the level they belong to, with gradients off, and through the functional transform."""
    from torch.autograd import forward_ad
    from advanced_optimizers_b200._device import refuse_tangents
    x = torch.ones(3)
    refuse_tangents("op", x, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        refuse_tangents("op", x, None)
        for guard in (torch.enable_grad, torch.no_grad):
            with guard(), pytest.raises(NotImplementedError, match="op: forward-mode"):
                refuse_tangents("op", None, x, dual)

    def seen(t):
        with pytest.raises(NotImplementedError, match="forward-mode"):
            refuse_tangents("op", t)
        return t

    torch.func.jvp(seen, (x,), (x,))


def test_a_residual_s_gradient_does_not_read_the_step(steps_read):
    from advanced_optimizers_b200.dropout import _Dropout, drop_fields
    x, r, step = torch.ones(4), torch.zeros(4, requires_grad=True), torch.tensor([7])
    y = _Dropout.apply(x, r, step, drop_fields(0.5, 1, 0, step, x.device))
    step.add_(1)
    g, = torch.autograd.grad(y.sum(), r)
    assert torch.equal(g, torch.ones(4)) and steps_read == [7]

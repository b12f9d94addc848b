"""Log-probabilities of tokens and the losses over them against their 64-bit
formulas (tests/_rows_ref.py)."""
import pytest
import torch

import _rows_ref as ref

pytestmark = pytest.mark.gpu

B, F = torch.bfloat16, torch.float32
IGNORE = -100
INF, NAN = float("inf"), float("nan")


def rand(*shape, seed=0, dtype=F):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def check_logprobs(logits, tokens, dlp, temperature=1.0, ignore=IGNORE):
    import advanced_optimizers_b200 as A
    leaf = logits.detach().requires_grad_()
    lp = A.token_logprobs(leaf, tokens, temperature=temperature, ignore_index=ignore)
    want, slack, _, _ = ref.logprobs(logits.detach(), tokens, temperature, ignore)
    ref.close(lp, want, slack, F)
    dx, = torch.autograd.grad(lp, leaf, dlp)
    want, slack = ref.logprobs_grad(logits.detach(), tokens, temperature, ignore, dlp)
    ref.close(dx, want, slack, logits.dtype)
    with torch.no_grad():
        assert torch.equal(A.token_logprobs(leaf, tokens, temperature=temperature, ignore_index=ignore).nan_to_num(7.0), lp.nan_to_num(7.0))


def case(R, V, dtype, seed=0):
    x = rand(R, V, seed=seed, dtype=dtype) * 3
    t = torch.randint(V, (R,), generator=torch.Generator(device="cuda").manual_seed(R + V), device="cuda")
    return x, t, rand(R, seed=seed + 1)


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("R,V", [(1, 1), (5, 2), (3, 7), (40, 33), (300, 50), (17, 1001), (9, 2048), (1300, 2049), (33, 4096), (50, 4104), (7, 5003),
                                 (1, 16384), (1, 32769), (2, 50257), (200, 50257), (300, 32777), (620, 16400), (1, 128256), (40, 128256), (149, 70001),
                                 (3, 262145)])
def test_logprobs_and_gradient(R, V, dtype):
    x, t, g = case(R, V, dtype)
    check_logprobs(x, t, g)


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("temperature", [0.05, 0.7, 30.0])
def test_temperatures(dtype, temperature):
    for R, V in ((50, 1000), (20, 9001)):
        x, t, g = case(R, V, dtype)
        check_logprobs(x, t.int(), g, temperature)


@pytest.mark.parametrize("R,V", [(60, 513), (60, 30001), (300, 30001), (300, 100)])
def test_ignored_tokens_and_rows_without_a_gradient(R, V):
    """Neither are read: what they hold does not matter."""
    import advanced_optimizers_b200 as A
    x, t, g = case(R, V, F)
    t[::3] = IGNORE
    g[1::3] = 0
    check_logprobs(x, t, g)
    check_logprobs(x, torch.where(t == IGNORE, 5, t), g, ignore=5)
    x[::3] = NAN
    x[1::3, 7] = INF
    leaf = x.requires_grad_()
    lp = A.token_logprobs(leaf, t)
    dx, = torch.autograd.grad(lp, leaf, g)
    assert bool((lp[::3] == 0).all()) and bool(lp[1::3].isnan().all()) and bool(lp[2::3].isfinite().all())
    assert bool((dx[::3] == 0).all()) and bool((dx[1::3] == 0).all()) and bool(dx[2::3].isfinite().all())


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("V,times", [(40, 1), (700, 1), (20011, 1), (20011, 15)])
def test_infinities_nan_and_lowest_values(V, times, dtype):
    low = torch.finfo(dtype).min
    x, t, g = case(12, V, dtype)
    t[:] = torch.arange(12, device="cuda") + 20
    x[0, :20] = -INF                  # part of the vocabulary masked
    x[1] = -INF                       # all of it: NaN
    x[2] = -INF
    x[2, 22] = 1.5                    # one token left: probability 1
    x[3, 23] = -INF                   # the token itself masked
    x[4, 3] = INF
    x[5, 3] = NAN
    x[6] = low                        # a mask of the type's lowest value in every place
    x[7] = low
    x[7, 27] = 0.0
    x[8, :-1] = -INF                  # only the last one
    x[9, 1:] = -INF                   # only the first one
    x[10] = -torch.finfo(dtype).min   # the largest finite value everywhere
    x[11] = 0.0
    check_logprobs(x.repeat(times, 1), t.repeat(times), g.repeat(times))


@pytest.mark.parametrize("dtype", [B, F])
def test_growing_and_falling_rows(dtype):
    """Every block of a row raises the running maximum, or none after the first does."""
    V = 60001
    x = torch.stack([torch.linspace(-50, 50, V, device="cuda"), torch.linspace(50, -50, V, device="cuda"), torch.linspace(0, 1, V, device="cuda") * 1e4])
    check_logprobs(x.to(dtype), torch.tensor([V - 1, 5, V - 1], device="cuda"), torch.ones(3, device="cuda"))


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("V,S,T", [(61, 4, 9), (1027, 4, 9), (8200, 4, 9), (20003, 4, 9), (9001, 6, 60)])
def test_strides_and_shapes_of_logits(V, S, T, dtype):
    x = rand(S, T, V + 5, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    views = [x[:, :-1, :V], x[:, 1:, 1 : V + 1], x[:, ::2, 3 : V + 3], x[::2, :, :V], x[0, :, :V], x[0, 0, :V], x.transpose(0, 1)[:, :, :V],
             x[:, :, :V].reshape(2, S // 2, T, V), rand(V, 30, dtype=dtype).t(), x[:1, :1, :V].expand(3, 5, V), x[:, :1, :V].expand(S, 3, V)]
    for v in views:
        t = torch.randint(V, v.shape[:-1], generator=g, device="cuda")
        check_logprobs(v, t, torch.randn(t.shape, generator=g, device="cuda"))
        if t.dim() == 2:
            check_logprobs(v, t.t().contiguous().t(), torch.randn(1, device="cuda").expand(t.shape))


def test_tokens_outside_the_vocabulary():
    import advanced_optimizers_b200 as A
    A.check_index_errors()
    for V in (50, 20000):
        x, t, g = case(8, V, F)
        t[1], t[3], t[5], t[6] = -1, V, 1 << 33, IGNORE
        leaf = x.requires_grad_()
        lp = A.token_logprobs(leaf, t)
        assert lp.isnan().tolist() == [False, True, False, True, False, True, False, False]
        dx, = torch.autograd.grad(lp, leaf, g)
        assert dx.isnan().all(1).tolist() == [False, True, False, True, False, True, False, False]
        assert dx.isnan().any(1).tolist() == dx.isnan().all(1).tolist()
        with pytest.raises(A.embeddings.L.AdvOptError, match="outside its table"):
            A.check_index_errors()


def test_logprobs_more_than_2_to_32_elements():
    import advanced_optimizers_b200 as A
    R, V = 33000, 131072
    x = torch.zeros(R, V, dtype=B, device="cuda")
    t = torch.arange(R, device="cuda")
    x[-1, R - 1] = 5.0
    leaf = x.requires_grad_()
    lp = A.token_logprobs(leaf, t)
    want, slack, _, _ = ref.logprobs(x[-2:].detach(), t[-2:], 1.0, IGNORE)
    ref.close(lp[-2:], want, slack, F)
    ref.close(lp[:2], *ref.logprobs(x[:2].detach(), t[:2], 1.0, IGNORE)[:2], F)
    dx, = torch.autograd.grad(lp.sum(), leaf)
    for rows in (slice(0, 2), slice(R - 2, R)):
        ref.close(dx[rows], *ref.logprobs_grad(x[rows].detach(), t[rows], 1.0, IGNORE, torch.ones(2, device="cuda")), B)


def answers(R, C, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + R + C)
    mask = torch.rand(R, C, generator=g, device="cuda") < 0.7
    if R > 2:
        mask[R // 2] = False
    return mask


def policy_case(R, C, dtype, seed=0):
    old = -rand(R, C, seed=seed).abs()
    lp, refp = old + 0.2 * rand(R, C, seed=seed + 1), old + 0.3 * rand(R, C, seed=seed + 2)
    return [t.to(dtype) for t in (lp, old, refp)]


def check_policy(lp, old, adv, mask, refp, clip=(0.2, 0.2), kl_weight=0.0, average="tokens", dloss=1.0):
    import advanced_optimizers_b200 as A
    leaf = lp.detach().requires_grad_()
    r = A.policy_loss(leaf, old, adv, mask, ref_logprobs=refp, clip=clip, kl_weight=kl_weight, average=average)
    want = ref.policy(lp.detach(), old, adv, mask, refp, clip, kl_weight, average)
    for k in ("loss", "kl", "clip_fraction"):
        ref.close(getattr(r, k), *want[k], F)
    g, = torch.autograd.grad(r.loss, leaf, torch.tensor(dloss, device="cuda"))
    ref.close(g, want["grad"][0] * dloss, want["grad"][1] * abs(dloss), lp.dtype)
    with torch.no_grad():
        again = A.policy_loss(leaf, old, adv, mask, ref_logprobs=refp, clip=clip, kl_weight=kl_weight, average=average)
    assert all(torch.equal(a, b) for a, b in zip(again, r))


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("R,C", [(1, 1), (1, 2), (3, 31), (8, 501), (64, 1024), (65, 1024), (33, 1025), (7, 9001), (200, 2051), (1025, 40), (3000, 3)])
def test_policy_loss_and_gradient(R, C, dtype):
    lp, old, refp = policy_case(R, C, dtype)
    adv = rand(R, C, seed=9, dtype=dtype)
    mask = answers(R, C)
    check_policy(lp, old, adv, mask, refp, kl_weight=0.05)
    check_policy(lp, old, adv[:, 0], mask, refp, kl_weight=0.05, average="sequences", dloss=-2.5)
    check_policy(lp, old, adv, None, None, clip=(0.1, 0.3), average="sequences")
    check_policy(lp, old, adv[:, 0], None, None)


def test_policy_clipping_at_its_borders():
    old = torch.full((2, 8), -1.0, device="cuda")
    d = torch.tensor([0.0, 0.1823, 0.1824, 1.0, -0.2231, -0.2232, -5.0, 80.0], device="cuda")
    adv = torch.tensor([[1.0] * 8, [-1.0] * 8], device="cuda")
    for clip in ((0.2, 0.2), (0.0, 0.0), (1.0, 0.5)):
        check_policy(old + d, old, adv, None, None, clip=clip)
    check_policy(old + d, old, adv * 0, None, None)


def test_policy_kl_near_zero():
    """e^q - q - 1 where it cancels: within a few roundings of it, not of its terms."""
    import advanced_optimizers_b200 as A
    q = torch.tensor([[2.0 ** -k * s for k in range(0, 20) for s in (1, -1)]], device="cuda")
    zero = torch.zeros_like(q)
    r = A.policy_loss(zero, zero, zero, None, ref_logprobs=q, kl_weight=1.0)
    each = [A.policy_loss(zero[:, :1], zero[:, :1], zero[:, :1], ref_logprobs=q[:, i : i + 1], kl_weight=1.0).kl for i in range(q.shape[1])]
    want = ref.policy(zero, zero, zero, None, q, (0.2, 0.2), 1.0, "tokens")
    ref.close(r.kl, *want["kl"], F)
    for i, k in enumerate(each):
        w = ref.policy(zero[:, :1], zero[:, :1], zero[:, :1], None, q[:, i : i + 1], (0.2, 0.2), 1.0, "tokens")["kl"][0]
        assert abs(float(k) - float(w)) <= 16 * ref.U * float(w)


@pytest.mark.parametrize("dtype", [B, F])
def test_masked_places_are_not_looked_at(dtype):
    import advanced_optimizers_b200 as A
    for R, C in ((6, 700), (90, 1500)):
        lp, old, refp = policy_case(R, C, dtype)
        adv, mask = rand(R, C, seed=4, dtype=dtype), answers(R, C)
        spoilt = []
        for t, bad in ((lp, NAN), (old, -INF), (refp, torch.finfo(dtype).min), (adv, INF)):
            t = t.clone()
            t[~mask] = bad
            spoilt.append(t)
        check_policy(spoilt[0], spoilt[1], spoilt[3], mask, spoilt[2], kl_weight=0.1)
        leaf = spoilt[0].requires_grad_()
        r = A.policy_loss(leaf, spoilt[1], spoilt[3], mask, ref_logprobs=spoilt[2], kl_weight=0.1)
        g, = torch.autograd.grad(r.loss, leaf, torch.tensor(INF, device="cuda"))
        assert bool((g[~mask] == 0).all())
        even = R // 2 * 2
        spoilt = [t.detach()[:even] for t in spoilt]
        check_preference(spoilt[0], spoilt[2], mask[:even])
        leaf = spoilt[0].requires_grad_()
        g, = torch.autograd.grad(A.preference_loss(leaf, spoilt[2], mask[:even]).loss, leaf, torch.tensor(INF, device="cuda"))
        assert bool((g[~mask[:even]] == 0).all())


@pytest.mark.parametrize("R,C", [(1, 5), (4, 300), (80, 2000)])
def test_nothing_in_the_mask(R, C):
    import advanced_optimizers_b200 as A
    lp, old, refp = policy_case(2 * R, C, F)
    mask = torch.zeros(2 * R, C, dtype=torch.bool, device="cuda")
    leaf = lp.requires_grad_()
    for average in ("tokens", "sequences"):
        r = A.policy_loss(leaf, old, rand(2 * R), mask, ref_logprobs=refp, kl_weight=0.1, average=average)
        assert [float(t) for t in r] == [0.0, 0.0, 0.0]
        assert bool((torch.autograd.grad(r.loss, leaf)[0] == 0).all())
    for average in (False, True):
        r = A.preference_loss(leaf, refp, mask, average=average)
        assert bool((r.chosen_rewards == 0).all()) and abs(float(r.loss) - 0.6931471805599453) <= 2 * ref.U
        assert bool((torch.autograd.grad(r.loss, leaf)[0] == 0).all())


def test_empty_batches():
    import advanced_optimizers_b200 as A
    for shape in ((0, 5), (5, 0), (0, 0)):
        e = torch.empty(shape, device="cuda", requires_grad=True)
        r = A.policy_loss(e, e.detach(), e.detach()[:, 0] if shape[1] else e.new_empty(shape[0]), e.detach() > 0)
        assert [float(t) for t in r] == [0.0, 0.0, 0.0]
        assert torch.autograd.grad(r.loss, e)[0].shape == shape
    e = torch.empty(4, 0, device="cuda", requires_grad=True)
    r = A.preference_loss(e)
    assert abs(float(r.loss) - 0.6931471805599453) <= 2 * ref.U and r.chosen_rewards.tolist() == [0.0, 0.0]
    assert torch.autograd.grad(r.loss, e)[0].shape == (4, 0)


def check_preference(lp, refp, mask, beta=0.1, e=0.0, average=False, dloss=1.0):
    import advanced_optimizers_b200 as A
    leaf = lp.detach().requires_grad_()
    r = A.preference_loss(leaf, refp, mask, beta=beta, label_smoothing=e, average=average)
    want = ref.preference(lp.detach(), refp, mask, beta, e, average)
    for k in ("loss", "chosen_rewards", "rejected_rewards"):
        ref.close(getattr(r, k), *want[k], F)
    g, = torch.autograd.grad(r.loss, leaf, torch.tensor(dloss, device="cuda"))
    ref.close(g, want["grad"][0] * dloss, want["grad"][1] * abs(dloss), lp.dtype)
    with torch.no_grad():
        again = A.preference_loss(leaf, refp, mask, beta=beta, label_smoothing=e, average=average)
    assert all(torch.equal(a, b) for a, b in zip(again, r))


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("P,C", [(1, 1), (1, 33), (4, 333), (32, 1024), (33, 1024), (17, 3001), (3, 10000), (1500, 7), (130, 4095)])
def test_preference_loss_and_gradient(P, C, dtype):
    refp = -rand(2 * P, C).abs()
    lp = (refp + 0.2 * rand(2 * P, C, seed=1)).to(dtype)
    refp, mask = refp.to(dtype), answers(2 * P, C)
    check_preference(lp, refp, mask)
    check_preference(lp, refp, mask, beta=0.5, e=0.2, average=True, dloss=-3.0)
    check_preference(lp, None, None, beta=0.01)
    check_preference(lp, None, mask, beta=2.0, average=True)


def test_preference_of_far_apart_pairs():
    lp = torch.tensor([[-1.0], [-1e4], [-1.0], [-3e38], [-1e4], [-1.0], [-1.0], [-1.0]], device="cuda")
    for e in (0.0, 0.1, 1.0):
        check_preference(lp, None, None, beta=1.0, e=e)


@pytest.mark.parametrize("dtype", [B, F])
def test_strides_of_losses(dtype):
    wide = -rand(40, 1100, dtype=dtype).abs()
    old = -rand(40, 1207, seed=3, dtype=dtype).abs()
    mask = answers(41, 1300)
    adv = rand(40, 1111, seed=5, dtype=dtype)
    for C in (1000, 1037):
        check_policy(wide[:, 3 : C + 3], old[:, 1 : C + 1], adv[:, :C], mask[1:, 5 : C + 5], old[:, 9 : C + 9], kl_weight=0.1)
        check_policy(wide[::2, :C], old[::2, :C], adv[::2, 4], mask[:40:2, :C], None, average="sequences")
        check_policy(wide[:1, :C].expand(5, C), old.t()[:C, :5].t(), adv[:1, :C].expand(5, C), mask[:1, :C].expand(5, C), None)
        check_preference(wide[:, 3 : C + 3], old[:, 1 : C + 1], mask[1:, 5 : C + 5])
        check_preference(wide[:2, :C].t().contiguous().t(), old[:1, :C].expand(2, C), mask[:1, :C].expand(2, C))


@pytest.mark.parametrize("R,C", [(8, 501), (300, 3000)])
def test_losses_repeat_on_other_streams_and_in_graphs(R, C):
    import advanced_optimizers_b200 as A
    lp, old, refp = policy_case(R, C, F)
    adv, mask = rand(R), answers(R, C)
    x, t, _ = case(R, 3001, B)
    leaf, xl = lp.requires_grad_(), x.requires_grad_()

    def run():
        a = A.policy_loss(leaf, old, adv, mask, ref_logprobs=refp, kl_weight=0.1)
        b = A.preference_loss(leaf, refp, mask)
        c = A.token_logprobs(xl, t)
        return [*a, *b, c, *torch.autograd.grad(a.loss, leaf), *torch.autograd.grad(b.loss, leaf), *torch.autograd.grad(c.sum(), xl)]

    same = lambda a, b: all(torch.equal(p, q) for p, q in zip(a, b))  # noqa: E731
    want = [w.detach() for w in run()]   # no eager graph of the leaves may live during a capture
    assert same(run(), want)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            got += [[g.detach() for g in run()] for _ in range(3)]
    torch.cuda.synchronize()
    assert all(same(g, want) for g in got)
    del got
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append([o.detach() for o in run()])
    with torch.no_grad():
        lp.mul_(1.01)
        x.add_(0.5)
        mask.logical_not_()
    for graph in graphs:
        graph.replay()
    want = run()
    assert all(same(o, want) for o in outs)


@pytest.mark.parametrize("R,V", [(5, 50257), (300, 9001), (200, 70001), (400, 40), (200, 900)])
def test_logprobs_of_every_variant_in_a_graph(R, V):
    """Two graphs of the same call in turn, each with its own buffers, on inputs that changed since their capture."""
    import advanced_optimizers_b200 as A
    x, t, g = case(R, V, B)
    leaf = x.requires_grad_()

    def run():
        lp = A.token_logprobs(leaf, t, temperature=0.9)
        return [lp.detach(), *torch.autograd.grad(lp, leaf, g)]

    run()
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run())
    with torch.no_grad():
        x.mul_(1.25)
        t.copy_(t.flip(0))
    t[::7] = IGNORE
    for graph in graphs * 2:
        graph.replay()
    want = run()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


def test_gradients_against_differences():
    """The kernels' own difference quotients along a direction, within their rounding and the 64-bit quotients' truncation."""
    import advanced_optimizers_b200 as A
    R, C = 6, 800
    lp, old, refp = policy_case(R, C, F)
    adv, mask, v = rand(R, C, seed=3), answers(R, C), rand(R, C, seed=8)
    step = 2.0 ** -7
    # no direction at tokens whose ratio is near a border of the clipping: the loss has corners there
    r = (lp.double() - old.double()).exp()
    v = torch.where(((r - 0.8).abs() < 0.1) | ((r - 1.2).abs() < 0.1), 0.0, v)
    for kernel, oracle in (
            (lambda t: A.policy_loss(t, old, adv, mask, ref_logprobs=refp, kl_weight=0.1).loss, lambda t: ref.policy(t, old, adv, mask, refp, (0.2, 0.2), 0.1, "tokens")),
            (lambda t: A.preference_loss(t, refp, mask, beta=0.3).loss, lambda t: ref.preference(t, refp, mask, 0.3, 0.0, False))):
        leaf = lp.clone().requires_grad_()
        slope = float((torch.autograd.grad(kernel(leaf), leaf)[0].double() * v.double()).sum())
        hi, lo = lp + step * v, lp - step * v
        quotient = (float(kernel(hi)) - float(kernel(lo))) / (2 * step)
        o = [oracle(hi)["loss"], oracle(lo)["loss"]]
        g = oracle(lp)["grad"]
        exact = float(o[0][0] - o[1][0]) / (2 * step)
        rounding = sum(float(s + 2 * ref.U * abs(y)) for y, s in o) / (2 * step) + float((g[1] * v.double().abs()).sum()) + 4 * ref.U * abs(slope)
        truncation = abs(exact - float((g[0] * v.double()).sum()))
        assert abs(quotient - slope) <= truncation + rounding


def test_hooks_on_saved_tensors_and_other_derivatives():
    import advanced_optimizers_b200 as A
    lp, old, refp = policy_case(6, 70, F)
    mask = answers(6, 70)
    x, t, dlp = case(30, 500, B)
    leaf, xl = lp.requires_grad_(), x.requires_grad_()
    calls = [(lambda: A.policy_loss(leaf, old, rand(6), mask).loss, leaf, None), (lambda: A.preference_loss(leaf, refp, mask).loss, leaf, None),
             (lambda: A.token_logprobs(xl, t), xl, dlp)]
    for call, to, d in calls:
        want, = torch.autograd.grad(call(), to, d)
        with torch.autograd.graph.save_on_cpu():
            y = call()
        assert torch.equal(torch.autograd.grad(y, to, d, retain_graph=True)[0], want)
        assert torch.equal(torch.autograd.grad(y, to, d)[0], want)
        y = call()
        d = torch.ones_like(y).requires_grad_()
        g, = torch.autograd.grad(y, to, d, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()
    r = A.policy_loss(leaf, old, rand(6), mask)
    (r.loss * 2).backward()
    assert not r.kl.requires_grad and not r.clip_fraction.requires_grad
    assert not A.preference_loss(leaf, refp, mask).chosen_rewards.requires_grad
    for const in (dict(old_logprobs=leaf), dict(advantages=leaf), dict(ref_logprobs=leaf)):
        kw = {**dict(old_logprobs=old, advantages=refp, ref_logprobs=refp), **const}
        with pytest.raises(ValueError, match="constant"):
            A.policy_loss(leaf, kw["old_logprobs"], kw["advantages"], mask, ref_logprobs=kw["ref_logprobs"])
    with pytest.raises(ValueError, match="constant"):
        A.preference_loss(leaf, leaf)
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t.detach(), torch.ones_like(t))  # noqa: E731
        for call in (lambda: A.policy_loss(dual(lp), old, old), lambda: A.policy_loss(lp.detach(), dual(old), old),
                     lambda: A.preference_loss(dual(lp)), lambda: A.token_logprobs(dual(x), t)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


@pytest.mark.parametrize("dtype", [B, F])
@pytest.mark.parametrize("R,C", [(3, 40), (3, 41), (70, 3000)])
def test_a_reference_without_weight_changes_nothing(R, C, dtype):
    """kl_weight = 0: the KL term is only reported, and where it is beyond float32 neither the loss nor a gradient sees it."""
    import advanced_optimizers_b200 as A
    lp, old, refp = policy_case(R, C, dtype)
    refp[0, 3], refp[1, 0], lp[2, 5] = 100.0, 3e4, -INF
    adv, mask = rand(R, C, seed=9, dtype=dtype), answers(R, C)
    mask[0, 3] = mask[1, 0] = mask[2, 5] = True
    leaf = lp.requires_grad_()
    for average in ("tokens", "sequences"):
        plain, seen = A.policy_loss(leaf, old, adv, mask, average=average), A.policy_loss(leaf, old, adv, mask, ref_logprobs=refp, average=average)
        assert bool(plain.loss.isfinite()) and torch.equal(seen.loss, plain.loss) and torch.equal(seen.clip_fraction, plain.clip_fraction)
        a, b = (torch.autograd.grad(r.loss, leaf)[0] for r in (plain, seen))
        assert bool(a.isfinite().all()) and torch.equal(a, b)
        assert not bool(seen.kl.isfinite())


def test_ratios_beyond_float32():
    """e^d A is 0 where the advantage is, and a number of its own where e^d alone has left float32."""
    d = torch.tensor([[87.0, 88.5, 89.0, 95.0, 100.0, 150.0, 176.0, 250.0, 700.0], [88.0, 88.8, 90.0, 100.0, 120.0, 0.1, -3.0, -300.0, 0.0]], device="cuda")
    old = torch.full_like(d, -1.0)
    old[0, -2:], old[1, 7] = -800.0, 0.0
    adv = torch.zeros_like(d)
    check_policy(old + d, old, adv, None, None)
    check_policy(old + d, old, adv[:, 0], None, None, average="sequences")
    adv[1] = torch.tensor([-1.0, -1e-3, -1e-4, -1e-8, -1e-20, -1.0, -1.0, -1.0, -1.0], device="cuda")
    check_policy(old + d, old, adv, None, None)
    check_policy(old + d, old, adv, None, old + d, kl_weight=0.1)


def test_preference_of_impossible_sequences():
    """A term without weight is left out: a rejected sequence of probability 0 costs nothing, a chosen one is infinite."""
    import advanced_optimizers_b200 as A
    lp = torch.full((4, 40), -1.0, device="cuda")
    lp[2, 7] = -INF   # rejected
    for e, want in ((0.0, 0.6931471805599453 / 2), (0.1, INF), (1.0, INF)):
        leaf = lp.clone().requires_grad_()
        r = A.preference_loss(leaf, label_smoothing=e)
        assert float(r.loss) == want if want == INF else abs(float(r.loss) - want) <= 2 * ref.U
        g, = torch.autograd.grad(r.loss, leaf)
        assert bool(g.isfinite().all()) and (e > 0 or bool((g[[0, 2]] == 0).all()))
        chosen = torch.cat([lp[2:], lp[:2]]).requires_grad_()   # the other way round
        r = A.preference_loss(chosen, label_smoothing=1 - e)
        assert float(r.loss) == want if want == INF else abs(float(r.loss) - want) <= 2 * ref.U
        g, = torch.autograd.grad(r.loss, chosen)
        assert bool(g.isfinite().all()) and (e > 0 or bool((g[[0, 2]] == 0).all()))

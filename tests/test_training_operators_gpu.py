"""The operators together, as a trainer uses them: embedding, layer norm, fp8 or
plain products, dropout, log-probabilities and both losses, with gradients and
optimizer steps."""
import pytest
import torch

import _rows_ref as ref

pytestmark = pytest.mark.gpu

B, F, D = torch.bfloat16, torch.float32, torch.float64
IGNORE = -100


def weights(V, C, H, seed=0, dtype=F, spread=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    return dict(emb=n(V, C) * spread, w1=1 + 0.1 * n(C), b1=0.1 * n(C), up=n(H, C) * C ** -0.5, down=n(C, H) * H ** -0.5, w2=1 + 0.1 * n(C), b2=0.1 * n(C))


def batch(S, T, V, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(V, (S, T), generator=g, device="cuda")
    mask = torch.rand(S, T, generator=g, device="cuda") < 0.6
    mask[0] = False
    old = -torch.rand(S, T, generator=g, device="cuda") * 3
    adv = torch.randn(S, generator=g, device="cuda")
    return ids, mask, old, adv


def model(p, ids):
    """A two-layer model with a tied head: logits of the next tokens."""
    import advanced_optimizers_b200 as A
    x = A.embedding(ids, p["emb"], scale=1.5)
    h = A.layer_norm(x, p["w1"], p["b1"])
    h = torch.nn.functional.linear(torch.tanh(torch.nn.functional.linear(h, p["up"])), p["down"])
    x = A.layer_norm(x + h, p["w2"], p["b2"])
    return torch.nn.functional.linear(x, p["emb"])


def plain_model(p, ids):
    """The same in elementary operations, float64."""
    def norm(x, w, b):
        x = x - x.mean(-1, keepdim=True)
        return x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b
    x = p["emb"][ids] * 1.5
    h = norm(x, p["w1"], p["b1"])
    h = torch.tanh(h @ p["up"].t()) @ p["down"].t()
    return norm(x + h, p["w2"], p["b2"]) @ p["emb"].t()


def loss_of(logits, ids, mask, old, adv, kind):
    import advanced_optimizers_b200 as A
    # a row's logits are of the token behind it: strided logits, shifted ids; masked tokens are ignored and not read
    tokens = torch.where(mask[:, 1:], ids[:, 1:], IGNORE)
    lp = A.token_logprobs(logits[:, :-1], tokens)
    if kind == "policy":
        return A.policy_loss(lp, old[:, 1:], adv, mask[:, 1:], ref_logprobs=old[:, 1:], kl_weight=0.05, average="sequences").loss
    return A.preference_loss(lp, old[:, 1:], mask[:, 1:], beta=0.1).loss


def plain_loss(logits, ids, mask, old, adv, kind):
    lp = torch.log_softmax(logits[:, :-1], -1).gather(-1, ids[:, 1:, None])[..., 0]
    mask, old = mask[:, 1:], old[:, 1:].double()
    if kind == "policy":
        r, q = (lp - old).exp(), old - lp
        a = adv.double()[:, None]
        each = 0.05 * (q.exp() - q - 1) - torch.minimum(r * a, r.clamp(0.8, 1.2) * a)
        n = mask.sum(1)
        return ((each * mask).sum(1) / n.clamp(min=1)).sum() / (n > 0).sum()
    s = ((lp - old) * mask).sum(1)
    h = 0.1 * (s[: len(s) // 2] - s[len(s) // 2 :])
    return -torch.nn.functional.logsigmoid(h).mean()


@pytest.mark.parametrize("kind", ["policy", "preference"])
@pytest.mark.parametrize("S,T,V,C,H,spread", [(4, 17, 61, 48, 96, 0.5), (6, 130, 1003, 200, 256, 0.5), (4, 17, 61, 48, 96, 0.05),
                                              (6, 130, 1003, 200, 256, 0.05)])
def test_a_model_s_gradients(S, T, V, C, H, spread, kind):
    """The gradient of every parameter through the whole run, against float64.  float32 arithmetic with products of up to 1003 terms keeps
    1e-4 of a gradient's norm: each of some ten operations is off by at most sqrt(1003) 2^-24 = 2e-6 of its result's norm, and the layer
    norms (whose rows have a spread of about 1) and the softmax grow that by less than ten."""
    p = {k: v.requires_grad_() for k, v in weights(V, C, H, spread=spread).items()}
    q = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    ids, mask, old, adv = batch(S, T, V)
    loss = loss_of(model(p, ids), ids, mask, old, adv, kind)
    want = plain_loss(plain_model(q, ids), ids, mask, old, adv, kind)
    if float(want) > torch.finfo(F).max:   # the KL term of far-off log-probabilities: beyond float32
        assert float(loss) == float("inf")
        return
    assert abs(float(loss) - float(want)) <= 1e-4 * abs(float(want))
    for k, g, w in zip(p, torch.autograd.grad(loss, list(p.values())), torch.autograd.grad(want, list(q.values()))):
        assert float((g.double() - w).norm()) <= 1e-4 * float(w.norm()), k


@pytest.mark.parametrize("spread", [0.5, 0.05])
@pytest.mark.parametrize("opt", ["AdamW_adv", "Muon_adv"])
def test_training_steps_with_the_package_s_layers_and_optimizers(opt, spread):
    """bf16 weights, fp8 products, dropout: every step's gradients are finite, reach every parameter and move it."""
    import advanced_optimizers_b200 as A
    S, T, V, C, H = 4, 33, 512, 256, 512
    p = {k: torch.nn.Parameter(v) for k, v in weights(V, C, H, dtype=B, spread=spread).items()}
    if opt == "Muon_adv":
        o = A.Muon_adv([dict(params=[p["up"], p["down"]], optim_type="muon"), dict(params=[v for k, v in p.items() if k not in ("up", "down")],
                                                                                   optim_type="adam")], lr=1e-2)
    else:
        o = A.AdamW_adv(list(p.values()), lr=1e-2)
    ids, mask, old, adv = batch(S, T, V)
    for step in range(3):
        x = A.embedding(ids, p["emb"], scale=1.5)
        h = A.fp8_linear(A.layer_norm(x, p["w1"], p["b1"]), p["up"])
        x = A.fp8_linear(torch.tanh(h), p["down"], residual=x, dropout_p=0.1, site=1, step=step)
        logits = A.layer_norm(x, p["w2"], p["b2"]) @ p["emb"].t()
        loss = loss_of(logits, ids, mask, old, adv, ("policy", "preference")[step % 2]) if step < 2 else -A.token_logprobs(logits, ids).mean()
        if not loss.isfinite():   # the KL term of far-off log-probabilities: beyond float32
            assert step == 0 and spread == 0.5 and float(plain_loss(logits.double(), ids, mask, old, adv, "policy")) > torch.finfo(F).max
            continue
        before = {k: v.detach().clone() for k, v in p.items()}
        loss.backward()
        for k, v in p.items():
            assert v.grad.isfinite().all() and float(v.grad.float().norm()) > 0, k
        o.step()
        o.zero_grad()
        for k, v in p.items():
            assert v.isfinite().all() and not torch.equal(v, before[k]), k
    A.check_fp8_errors()
    A.check_index_errors()


def test_a_captured_step_replays_with_new_inputs():
    """Forward and backward of the whole run in one graph, replayed on other inputs, is what an eager run gives."""
    S, T, V, C, H = 4, 40, 300, 128, 192
    p = {k: v.requires_grad_() for k, v in weights(V, C, H).items()}
    ids, mask, old, adv = batch(S, T, V)

    def run():
        loss = loss_of(model(p, ids), ids, mask, old, adv, "policy")
        return [loss.detach(), *torch.autograd.grad(loss, list(p.values()))]

    run()   # the libraries' own set-up
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in (5, 6):
        for t, new in zip((ids, mask, old, adv), batch(S, T, V, seed)):
            t.copy_(new)
        graph.replay()
        got = [t.clone() for t in out]
        for g, w in zip(got, run()):
            # the library's products may take other kernels on other streams: within float32's rounding
            assert float((g - w).norm()) <= 1e-5 * float(w.norm())


def test_calls_on_a_stream_that_is_not_the_current_one_s_default():
    """Results used on the calling stream alone: no call waits for, or lets run ahead of, another stream."""
    import advanced_optimizers_b200 as A
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    ids = torch.arange(600, device="cuda") % 50
    w = torch.randn(50, 264, device="cuda")
    torch.cuda.synchronize()
    outs = []
    for s in (a, b) * 4:
        with torch.cuda.stream(s):
            leaf = w.clone().requires_grad_()
            y = A.layer_norm(A.embedding(ids, leaf, scale=2.0))
            outs.append(torch.autograd.grad(A.token_logprobs(y, ids % 264).sum(), leaf)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_threads_call_at_once():
    import threading

    import advanced_optimizers_b200 as A
    ids = torch.randint(400, (3000,), device="cuda")
    w = torch.randn(400, 72, device="cuda")
    lp, old, mask = -torch.rand(16, 700, device="cuda"), -torch.rand(16, 700, device="cuda"), torch.rand(16, 700, device="cuda") < 0.5
    adv = torch.randn(16, device="cuda")
    torch.cuda.synchronize()

    def run():
        leaf, l2 = w.clone().requires_grad_(), lp.clone().requires_grad_()
        y = A.layer_norm(A.embedding(ids, leaf))
        r = A.policy_loss(l2, old, adv, mask)
        return [*torch.autograd.grad(y.square().sum(), leaf), r.loss.detach(), *torch.autograd.grad(r.loss, l2),
                *torch.autograd.grad(A.preference_loss(l2, old, mask).loss, l2)]

    want, got = run(), []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got.append(run())
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 20 and all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_index_error_of_a_captured_call_is_reported():
    import advanced_optimizers_b200 as A
    A.check_index_errors()
    ids, w = torch.arange(8, device="cuda"), torch.randn(8, 16, device="cuda")
    A.embedding(ids, w)   # an eager call: the word is there
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = A.embedding(ids, w)
    graph.replay()
    assert torch.equal(y, w)
    A.check_index_errors()
    ids[3] = 8
    graph.replay()
    with pytest.raises(A.embeddings.L.AdvOptError, match="outside its table"):
        A.check_index_errors()
    assert bool(y[3].isnan().all())


@pytest.mark.parametrize("S,T,V,C,H", [(4, 17, 61, 48, 96), (6, 130, 1003, 200, 256)])
def test_a_model_s_policy_gradients_near_its_reference(S, T, V, C, H):
    """As above, with old log-probabilities near the model's own, as a trainer has them, so that every term is a number; none of the ratios is
    within 0.08 of a border of the clipping (log 1.2 and log 0.8)."""
    p = {k: v.requires_grad_() for k, v in weights(V, C, H).items()}
    q = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    ids, mask, _, adv = batch(S, T, V)
    logits = plain_model(q, ids)
    lp = torch.log_softmax(logits.detach()[:, :-1], -1).gather(-1, ids[:, 1:, None])[..., 0]
    apart = torch.tensor([-0.5, -0.1, 0.0, 0.1, 0.3], dtype=D, device="cuda")[torch.arange(S * (T - 1), device="cuda") % 5].view(S, T - 1)
    old = torch.cat([torch.zeros(S, 1, dtype=D, device="cuda"), lp - apart], 1).float()
    want = plain_loss(logits, ids, mask, old, adv, "policy")
    loss = loss_of(model(p, ids), ids, mask, old, adv, "policy")
    for k, g, w in zip(p, torch.autograd.grad(loss, list(p.values())), torch.autograd.grad(want, list(q.values()))):
        assert float(w.norm()) > 0 and float((g.double() - w).norm()) <= 1e-4 * float(w.norm()), k


@pytest.mark.parametrize("S,T,V", [(4, 17, 61), (3, 9, 1003), (40, 30, 5003)])
def test_shifted_tokens_of_whole_logits(S, T, V):
    """The last place ignored: the same log-probabilities and gradients as of the logits without it, and zeros there."""
    import advanced_optimizers_b200 as A
    ids, mask, _, _ = batch(S, T, V)
    g = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randn(S, T, V, generator=g, device="cuda", dtype=B).requires_grad_()
    tokens = torch.full_like(ids, IGNORE)
    tokens[:, :-1] = torch.where(mask[:, 1:], ids[:, 1:], IGNORE)
    d = torch.randn(S, T, generator=g, device="cuda")
    lp, cut = A.token_logprobs(logits, tokens), A.token_logprobs(logits[:, :-1], tokens[:, :-1])
    assert torch.equal(lp[:, :-1], cut) and bool((lp[:, -1] == 0).all())
    assert torch.equal(torch.autograd.grad(lp, logits, d)[0], torch.autograd.grad(cut, logits, d[:, :-1].contiguous())[0])

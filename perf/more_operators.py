"""What is measured of the token embedding, the layer norm, the tokens'
log-probabilities and the policy and preference losses.

`run` computes one pass in plain torch operations (`own` false) or through
the package's entry points (`own` true).  Sizes are GPT-2 small's (768,
vocabulary 50257), the 1.3B GPT's (2048, 50304), Llama-3-8B's (4096, 128256)
and odd ones between.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}
IGNORED = -100
BETA = 0.1


def listed():
    return [
        # the last tokens of a few sequences: latency
        dict(name="embedding 16 of 50304x2048 bf16 fwd", op="embedding", tokens=16, vocab=50304, width=2048, dtype="bf16", scaled=False, padded=0.0, backward=False),
        # a ragged training batch of GPT-2 small with padding, fp32 weights, scaled embeddings
        dict(name="embedding 16381 of 50257x768 f32 both", op="embedding", tokens=16381, vocab=50257, width=768, dtype="f32", scaled=True, padded=0.1, backward=True),
        # a training batch of Llama-3-8B: the dense gradient of a large table
        dict(name="embedding 8192 of 128256x4096 bf16 both", op="embedding", tokens=8192, vocab=128256, width=4096, dtype="bf16", scaled=False, padded=0.0, backward=True),
        # an odd token count and an odd width: rows of every alignment
        dict(name="layer_norm 1000x5003 bf16 both", op="layer_norm", rows=1000, cols=5003, dtype="bf16", wdtype="bf16", affine=True, backward=True),
        # a training batch's hidden states, fp32 weights
        dict(name="layer_norm 16384x4096 bf16 both", op="layer_norm", rows=16384, cols=4096, dtype="bf16", wdtype="f32", affine=True, backward=True),
        # scoring the last tokens of a few sequences
        dict(name="logprobs 17x128256 bf16 fwd", op="logprobs", rows=17, vocab=128256, dtype="bf16", temperature=0.7, prompt=0.0, backward=False),
        # a fine-tuning batch of GPT-2 small: an odd vocabulary, prompts ignored, fp32 logits
        dict(name="logprobs 2047x50257 f32 both", op="logprobs", rows=2047, vocab=50257, dtype="f32", temperature=1.0, prompt=0.25, backward=True),
        # a training batch over Llama-3-8B's vocabulary
        dict(name="logprobs 4096x128256 bf16 both", op="logprobs", rows=4096, vocab=128256, dtype="bf16", temperature=1.0, prompt=0.0, backward=True),
        # a small group of answers, one advantage each
        dict(name="policy 8x501 f32", op="policy", seqs=8, tokens=501, dtype="f32", advantage="sequence", kl=0.04, average="sequences"),
        # a large batch with an advantage for each token
        dict(name="policy 512x8192 f32", op="policy", seqs=512, tokens=8192, dtype="f32", advantage="token", kl=0.02, average="tokens"),
        # a few pairs
        dict(name="preference 4x333 f32", op="preference", pairs=4, tokens=333, dtype="f32", reference=True, smoothing=0.0, average=False),
        # a large batch of pairs, log-probabilities kept in bf16, an odd length
        dict(name="preference 256x4095 bf16", op="preference", pairs=256, tokens=4095, dtype="bf16", reference=True, smoothing=0.1, average=True),
    ]


def _size(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n // 64 * 64 if n > 128 and rng.random() < 0.4 else n))


def draw(rng):
    op = rng.choice(["embedding", "layer_norm", "logprobs", "policy", "preference"])
    dtype = rng.choice(["bf16", "f32"])
    if op == "embedding":
        vocab, width = _size(rng, 100, 262144), _size(rng, 8, 8192)
        vocab = min(vocab, 128256 * 4096 * 2 // (width * SIZE[dtype]))
        tokens = min(_size(rng, 1, 65536), 128256 * 4096 * 2 // (width * SIZE[dtype]))
        return dict(op=op, tokens=tokens, vocab=vocab, width=width, dtype=dtype, scaled=rng.random() < 0.5, padded=rng.choice([0.0, 0.0, 0.1, 0.4]),
                    backward=rng.random() < 0.7)
    if op == "layer_norm":
        rows, cols = _size(rng, 1, 65536), _size(rng, 2, 16384)
        return dict(op=op, rows=min(rows, 16384 * 4096 * 2 // (cols * SIZE[dtype])), cols=cols, dtype=dtype, wdtype=rng.choice([dtype, "f32"]),
                    affine=rng.random() < 0.9, backward=rng.random() < 0.7)
    if op == "logprobs":
        rows, vocab = _size(rng, 1, 65536), _size(rng, 32, 262144)
        return dict(op=op, rows=max(1, min(rows, 4096 * 128256 * 2 // (vocab * SIZE[dtype]))), vocab=vocab, dtype=dtype,
                    temperature=rng.choice([0.7, 1.0, 1.0, 1.3]), prompt=rng.choice([0.0, 0.25, 0.5]), backward=rng.random() < 0.7)
    n, tokens = _size(rng, 1, 1024), _size(rng, 1, 16384)
    n = max(1, min(n, 512 * 8192 // tokens))
    if op == "policy":
        return dict(op=op, seqs=n, tokens=tokens, dtype=dtype, advantage=rng.choice(["sequence", "token"]), kl=rng.choice([0.0, 0.01, 0.04, 0.1]),
                    average=rng.choice(["sequences", "tokens"]))
    return dict(op=op, pairs=max(1, n // 2), tokens=tokens, dtype=dtype, reference=rng.random() < 0.8, smoothing=rng.choice([0.0, 0.0, 0.1]),
                average=rng.random() < 0.3)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _answers(g, rows, tokens):
    """A mask of answers: each row has a prompt ahead and padding behind, and some rows are nothing but padding."""
    at = torch.arange(tokens, device="cuda")
    first = (torch.rand(rows, 1, generator=g, device="cuda") * 0.3 * tokens).long()
    last = ((0.5 + 0.6 * torch.rand(rows, 1, generator=g, device="cuda")) * tokens).ceil().long()
    mask = (at >= first) & (at < last)
    if rows > 16:
        mask[torch.rand(rows, generator=g, device="cuda") < 0.02] = False
    return mask


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, s = case, dict(case=case)
    op, dt = c["op"], DTYPES[c["dtype"]]
    if op == "embedding":
        T, V, C = c["tokens"], c["vocab"], c["width"]
        # frequencies fall off as one over the rank; the padding token is the last one
        ids = (torch.rand(T, generator=g, device="cuda", dtype=torch.float64) * math.log(V)).exp().long().sub_(1).clamp_(0, V - 1)
        s["ids"] = torch.where(torch.rand(T, generator=g, device="cuda") < c["padded"], V - 1, ids)
        s["weight"] = (_normal(g, V, C) * 0.02).to(dt).requires_grad_(c["backward"])
        s["scale"] = math.sqrt(C) if c["scaled"] else 1.0
        s["padding"] = V - 1 if c["padded"] else None
        s["dy"] = (_normal(g, T, C) * 1e-3).to(dt) if c["backward"] else None
    elif op == "layer_norm":
        R, C, wd = c["rows"], c["cols"], DTYPES[c["wdtype"]]
        # hidden states: rows of other scales and means, some columns ten times as large
        x = _normal(g, R, C) * (1.0 + 9.0 * (torch.rand(C, generator=g, device="cuda") < 0.02))
        s["x"] = ((x + _normal(g, R, 1) * 0.5) * torch.rand(R, 1, generator=g, device="cuda").add_(0.5)).to(dt).requires_grad_(c["backward"])
        s["w"] = (1 + 0.1 * _normal(g, C)).to(wd).requires_grad_(c["backward"]) if c["affine"] else None
        s["b"] = (0.1 * _normal(g, C)).to(wd).requires_grad_(c["backward"]) if c["affine"] else None
        s["dy"] = (_normal(g, R, C) * 1e-3).to(dt) if c["backward"] else None
    elif op == "logprobs":
        R, V = c["rows"], c["vocab"]
        x = _normal(g, R, V).mul_(2.5)
        tokens = torch.randint(V, (R,), generator=g, device="cuda")
        x[torch.arange(R, device="cuda"), tokens] += 6.0   # the tokens that came are likely ones
        s["logits"] = x.to(dt).requires_grad_(c["backward"])
        tokens[: int(R * c["prompt"])] = IGNORED
        s["tokens"] = tokens
        s["dlp"] = (_normal(g, R) / R) if c["backward"] else None
    elif op == "policy":
        B, T = c["seqs"], c["tokens"]
        old = -_normal(g, B, T).square() * 1.2
        s["old"] = old.to(dt)
        s["lp"] = (old + _normal(g, B, T) * 0.15).clamp_(max=0).to(dt).requires_grad_()
        s["ref"] = (old + _normal(g, B, T) * 0.2).clamp_(max=0).to(dt) if c["kl"] else None
        s["adv"] = (_normal(g, B) if c["advantage"] == "sequence" else _normal(g, B, T)).to(dt)
        s["mask"] = _answers(g, B, T)
    else:
        R, T = 2 * c["pairs"], c["tokens"]
        ref = -_normal(g, R, T).square() * 1.2
        s["ref"] = ref.to(dt) if c["reference"] else None
        s["lp"] = (ref + _normal(g, R, T) * 0.1 + _normal(g, R, 1) * 0.02).clamp_(max=0).to(dt).requires_grad_()
        s["mask"] = _answers(g, R, T)
    return s


# ---- the plain forms ----
def _plain(s):
    c = s["case"]
    op, dt = c["op"], DTYPES[c["dtype"]]
    if op == "embedding":
        w, ids = s["weight"].detach(), s["ids"]
        y = (w[ids].float() * s["scale"]).to(dt)
        if not c["backward"]:
            return [y]
        dw = torch.zeros(w.shape, device=w.device).index_add_(0, ids, s["dy"].float())
        if s["padding"] is not None:
            dw[s["padding"]] = 0
        return [y, (dw * s["scale"]).to(dt)]
    if op == "layer_norm":
        x = s["x"].detach().float()
        w, b = (s["w"].detach().float(), s["b"].detach().float()) if c["affine"] else (1.0, 0.0)
        x = x - x.mean(1, keepdim=True)
        r = torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-5)
        h = x * r
        y = (h * w + b).to(dt)
        if not c["backward"]:
            return [y]
        dy = s["dy"].float()
        t = dy * w
        dx = r * (t - t.mean(1, keepdim=True) - h * (t * h).mean(1, keepdim=True))
        out = [y, dx.to(dt)]
        return out + [(dy * h).sum(0).to(DTYPES[c["wdtype"]]), dy.sum(0).to(DTYPES[c["wdtype"]])] if c["affine"] else out
    if op == "logprobs":
        z = s["logits"].detach().float() / c["temperature"]
        kept = s["tokens"] != IGNORED
        at = torch.where(kept, s["tokens"], 0)[:, None]
        z = z - z.amax(1, keepdim=True)
        e = z.exp()
        total = e.sum(1, keepdim=True)
        lp = torch.where(kept, (z.gather(1, at) - total.log())[:, 0], 0.0)
        if not c["backward"]:
            return [lp]
        k = torch.where(kept, s["dlp"], 0.0)[:, None] / c["temperature"]
        dx = e * (-k / total)
        dx.scatter_add_(1, at, k)
        return [lp, dx.to(dt)]
    if op == "policy":
        lo = hi = 0.2
        mask, lp = s["mask"], s["lp"].detach()
        adv = s["adv"].float()
        adv = adv[:, None] if c["advantage"] == "sequence" else adv
        d = lp.double() - s["old"].double()   # near a border of the clipping, 32 bits decide otherwise
        rho = d.exp().float()
        clipped = ((adv > 0) & (d > math.log1p(hi))) | ((adv < 0) & (d < math.log1p(-lo)))
        gain = torch.where(clipped, torch.where(adv > 0, 1 + hi, 1 - lo) * adv, rho * adv)
        slope = -torch.where(clipped, 0.0, rho * adv)
        kl = torch.zeros_like(gain)
        if c["kl"]:
            q = s["ref"].double() - lp.double()   # near 0, e^q - q - 1 cancels
            kl = (q.exp() - q - 1).float()
            slope = slope + c["kl"] * (-torch.expm1(q)).float()
        count = mask.sum().clamp(min=1).float()
        if c["average"] == "tokens":
            weight = mask / count
        else:
            n = mask.sum(1, keepdim=True)
            weight = mask / n.clamp(min=1) / (n > 0).sum().clamp(min=1)
        mean = lambda v: (torch.where(mask, v, 0.0) * weight).double().sum().float()  # noqa: E731
        return [mean(c["kl"] * kl - gain), (mask * kl).double().sum().float() / count, (mask & clipped).sum() / count,
                torch.where(mask, slope * weight, 0.0).to(dt)]
    mask, lp = s["mask"], s["lp"].detach()
    ratio = lp.float() - (s["ref"].float() if c["reference"] else 0.0)
    n = mask.sum(1).clamp(min=1).float() if c["average"] else torch.ones(mask.shape[0], device=lp.device)
    total = torch.where(mask, ratio, 0.0).double().sum(1).float() / n
    P, e = c["pairs"], c["smoothing"]
    h = BETA * (total[:P] - total[P:])
    softplus = lambda v: v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))  # noqa: E731
    loss = ((1 - e) * softplus(-h) + e * softplus(h)).mean()
    k = BETA / P * (e - 1 / (1 + h.exp()))
    k = torch.cat([k, -k]) / n
    return [loss, BETA * total[:P], BETA * total[P:], torch.where(mask, k[:, None], 0.0).to(dt)]


# ---- the package's calls ----
def _own(s):
    import advanced_optimizers_b200 as A
    c = s["case"]
    op = c["op"]
    if op == "embedding":
        y = A.embedding(s["ids"], s["weight"], scale=s["scale"], padding_idx=s["padding"])
        return [y, *torch.autograd.grad(y, s["weight"], s["dy"])] if c["backward"] else [y]
    if op == "layer_norm":
        y = A.layer_norm(s["x"], s["w"], s["b"], eps=1e-5)
        leaves = [t for t in (s["x"], s["w"], s["b"]) if t is not None]
        return [y, *torch.autograd.grad(y, leaves, s["dy"])] if c["backward"] else [y]
    if op == "logprobs":
        lp = A.token_logprobs(s["logits"], s["tokens"], temperature=c["temperature"], ignore_index=IGNORED)
        return [lp, *torch.autograd.grad(lp, s["logits"], s["dlp"])] if c["backward"] else [lp]
    if op == "policy":
        r = A.policy_loss(s["lp"], s["old"], s["adv"], s["mask"], ref_logprobs=s["ref"], clip=(0.2, 0.2), kl_weight=c["kl"], average=c["average"])
        return [r.loss, r.kl, r.clip_fraction, *torch.autograd.grad(r.loss, s["lp"])]
    r = A.preference_loss(s["lp"], s["ref"], s["mask"], beta=BETA, label_smoothing=c["smoothing"], average=c["average"])
    return [r.loss, r.chosen_rewards, r.rejected_rewards, *torch.autograd.grad(r.loss, s["lp"])]


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    c, size = case, SIZE[case["dtype"]]
    if c["op"] == "embedding":
        n = c["tokens"] * c["width"]
        fwd = 8 * c["tokens"] + size * (min(c["tokens"], c["vocab"]) * c["width"] / 2 + n)   # about half of the tokens are repeats
        return {"bytes": fwd + (size * (n + c["vocab"] * c["width"]) if c["backward"] else 0), "flops": 0}
    if c["op"] == "layer_norm":
        return {"bytes": c["rows"] * c["cols"] * size * (4 if c["backward"] else 2), "flops": 0}
    if c["op"] == "logprobs":
        n, ignored = c["rows"] * c["vocab"], int(c["rows"] * c["prompt"]) * c["vocab"]
        return {"bytes": 12 * c["rows"] + size * (n - ignored + (n if c["backward"] else 0)), "flops": 0}
    if c["op"] == "policy":
        n = c["seqs"] * c["tokens"]
        return {"bytes": n * (1 + size * (3 + (c["kl"] > 0) + (c["advantage"] == "token"))), "flops": 0}
    n = 2 * c["pairs"] * c["tokens"]
    return {"bytes": n * (1 + size * (2 + c["reference"])), "flops": 0}


# ---- the definitions in 64 bits ----
def exact(case, seed):
    s, c = prepare(case, seed), case
    op = c["op"]
    if op == "embedding":
        w = s["weight"].detach()
        y = torch.nn.functional.embedding(s["ids"], w).double() * s["scale"]
        if not c["backward"]:
            return [y]
        dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
        kept = torch.ones_like(s["ids"], dtype=torch.bool) if s["padding"] is None else s["ids"] != s["padding"]
        return [y, dw.index_put_((s["ids"][kept],), s["dy"][kept].double() * s["scale"], accumulate=True)]
    if op == "layer_norm":
        leaves = [t.detach().double().requires_grad_() for t in (s["x"], s["w"], s["b"]) if t is not None]
        var, mean = torch.var_mean(leaves[0], dim=1, correction=0, keepdim=True)
        y = (leaves[0] - mean) / (var + 1e-5).sqrt()
        y = y * leaves[1] + leaves[2] if c["affine"] else y
        return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"].double())] if c["backward"] else [y.detach()]
    if op == "logprobs":
        kept = (s["tokens"] != IGNORED).nonzero()[:, 0]
        z = s["logits"].detach().double().div_(c["temperature"])
        lse = torch.logsumexp(z, 1)
        lp = torch.zeros_like(lse)
        lp[kept] = z[kept, s["tokens"][kept]] - lse[kept]
        if not c["backward"]:
            return [lp]
        k = torch.zeros_like(lse)
        k[kept] = s["dlp"][kept].double() / c["temperature"]
        dx = z.sub_(lse[:, None]).exp_().mul_(-k[:, None])
        dx[kept, s["tokens"][kept]] += k[kept]
        return [lp, dx]
    mask = s["mask"]
    lp = s["lp"].detach().double().requires_grad_()
    if op == "policy":
        adv = s["adv"].double().view(mask.shape[0], -1)
        rho = (lp - s["old"].double()).exp()
        one, two = rho * adv, rho.clamp(0.8, 1.2) * adv
        each = -torch.minimum(one, two)
        q = s["ref"].double() - lp if c["kl"] else torch.zeros_like(rho)
        kl = torch.expm1(q) - q
        each = each + c["kl"] * kl
        n = mask.sum(1)
        rows = n > 0
        if c["average"] == "tokens":
            loss = each[mask].sum() / n.sum().clamp(min=1)
        else:
            loss = ((each * mask)[rows].sum(1) / n[rows]).sum() / rows.sum().clamp(min=1)
        count = n.sum().clamp(min=1).double()
        return [loss.detach(), kl.detach()[mask].sum() / count, (one > two)[mask].sum() / count, *torch.autograd.grad(loss, lp)]
    ratio = lp - s["ref"].double() if c["reference"] else lp
    total = (ratio * mask).sum(1)
    total = total / mask.sum(1).clamp(min=1) if c["average"] else total
    chosen, rejected = (BETA * total).chunk(2)
    h, e = chosen - rejected, c["smoothing"]
    loss = -((1 - e) * torch.nn.functional.logsigmoid(h) + e * torch.nn.functional.logsigmoid(-h)).mean()
    return [loss.detach(), chosen.detach(), rejected.detach(), *torch.autograd.grad(loss, lp)]

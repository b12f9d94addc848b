"""64-bit restatements of the embedding, layer norm, log-probability and loss
operators, and bounds of what their float32 arithmetic may be off by.

U is half a step of float32.  A float32 sum of n terms is off by at most
(depth of its tree) U times the sum of the magnitudes; a result is rounded to
its type once, by at most finfo.eps / 2 of it."""
import torch

U = 2.0 ** -24
D = torch.float64


def close(got, want, slack, dtype):
    """got (of dtype) is within its type's rounding and `slack` of want; NaN where want is NaN, equal infinities."""
    assert got.dtype == dtype and got.shape == want.shape, (got.dtype, got.shape, want.shape)
    g = got.detach().double()
    tol = torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2.0 ** -10) + slack + torch.finfo(dtype).tiny
    same = (g == want) | (g.isnan() & want.isnan())
    ok = same | ((g - want).abs() <= tol)
    if not bool(ok.all()):
        i = int((~ok).reshape(-1).nonzero()[0])
        raise AssertionError(f"element {i}: got {g.reshape(-1)[i].item()!r}, want {want.reshape(-1)[i].item()!r}; "
                             f"{int((~ok).sum())} of {ok.numel()} are off")


def embedding_grad(ids, dy, vocab, scale, padding):
    """(dweight, its slack)"""
    flat, g = ids.reshape(-1).long(), dy.reshape(-1, dy.shape[-1]).double()
    keep = (flat >= 0) & (flat < vocab)
    if padding is not None:
        keep &= flat != padding % vocab
    flat, g = flat[keep], g[keep]
    dw = torch.zeros(vocab, g.shape[1], dtype=D, device=dy.device)
    mag = dw.clone().index_add_(0, flat, g.abs())
    n = torch.zeros(vocab, dtype=D, device=dy.device).index_add_(0, flat, torch.ones_like(flat, dtype=D))
    return dw.index_add_(0, flat, g) * scale, (n[:, None] + 2) * U * mag * abs(scale)


class LayerNorm:
    """Values and slacks of a layer norm of x [R, C]."""

    def __init__(self, x, w, b, eps):
        self.x, C = x.double(), x.shape[1]
        self.w = torch.ones(C, dtype=D, device=x.device) if w is None else w.double()
        self.b = torch.zeros(C, dtype=D, device=x.device) if b is None else b.double()
        self.depth = 64 + C / 1024       # a thread's elements, a warp's five steps, 32 warps
        self.mean = self.x.mean(1, keepdim=True)
        d = self.x - self.mean
        var = (d * d).mean(1, keepdim=True) + eps
        self.rstd = var.rsqrt()
        off = (self.depth + 2) * U * self.x.abs().mean(1, keepdim=True)          # of the mean
        rel = 0.5 * ((self.depth + 6) * U + off * off / var) + 4 * U             # of rstd
        self.h = d * self.rstd
        self.h_off = self.rstd * (U * d.abs() + off) + self.h.abs() * (rel + 2 * U)
        self.rel = rel

    def forward(self):
        y = self.h * self.w + self.b
        return y, self.w.abs() * self.h_off + 2 * U * ((self.h * self.w).abs() + self.b.abs())

    def backward(self, dy):
        """((dx, slack), (dw, slack), (db, slack))"""
        dy = dy.double()
        g, h, R = dy * self.w, self.h, dy.shape[0]
        mean = lambda t: t.mean(1, keepdim=True)  # noqa: E731
        s1, s2 = mean(g), mean(g * h)
        o1 = (self.depth + 4) * U * mean(g.abs())
        o2 = (self.depth + 4) * U * mean((g * h).abs()) + mean(g.abs() * self.h_off)
        dx = self.rstd * (g - s1 - h * s2)
        ox = self.rstd * (o1 + h.abs() * o2 + s2.abs() * self.h_off + 4 * U * (g.abs() + s1.abs() + (h * s2).abs())) + dx.abs() * (self.rel + 2 * U)
        ow = (R + 64) * U * (dy * h).abs().sum(0) + (dy.abs() * self.h_off).sum(0)
        return (dx, ox), ((dy * h).sum(0), ow), (dy.sum(0), (R + 64) * U * dy.abs().sum(0))


def logprobs(logits, tokens, temperature, ignore):
    """(lp, slack, p, p's relative slack): rows of p that are ignored are whatever the formula gives."""
    V = logits.shape[-1]
    x, t = logits.double().reshape(-1, V), tokens.reshape(-1).long()
    z = x / temperature
    m = z.amax(1, keepdim=True)
    # infinite maxima: inf - inf
    e = (z - m).exp()
    s = e.sum(1, keepdim=True)
    far = torch.where(z.isinf(), 0.0, (m - z).abs())
    # A term has its exponential's error (2^-22) and three roundings of its argument.  A lane's sum is rescaled, which is an exponential and
    # roundings more, at most twice for what lies ahead of and behind the row's 16-byte boundaries, once when its lanes join, then with each
    # part of 6 KB of its row that a lane joins (two of up to 16, or one in 32 of more) and twice more.  The sums' trees are 72 deep at most:
    # 48 of a lane's pairs, their join, two, five steps, two or more parts, twice five steps.
    rel = (9 + V / 32768) * (2.0 ** -22 + 4 * U) + 72 * U + (3 * U * (far * e).sum(1, keepdim=True) / s)
    bad = (t < 0) | (t >= V)
    zt = z.gather(1, t.clamp(0, V - 1)[:, None])
    lp = zt - m - s.log()
    lp_off = rel + 4 * U * torch.where(zt.isinf() | m.isinf(), 0.0, (zt - m).abs()) + 3 * U * s.log().abs()
    lp = torch.where((t == ignore)[:, None], 0.0, torch.where(bad[:, None], float("nan"), lp))
    return (lp[:, 0].reshape(tokens.shape), lp_off[:, 0].reshape(tokens.shape), (e / s).reshape(logits.shape),
            (rel + 2.0 ** -22 + 3 * U * far + 4 * U).reshape(logits.shape))


def logprobs_grad(logits, tokens, temperature, ignore, dlp):
    """(dlogits, slack)"""
    V = logits.shape[-1]
    _, _, p, rel = logprobs(logits, tokens, temperature, ignore)
    p, rel, t = p.reshape(-1, V), rel.reshape(-1, V), tokens.reshape(-1).long()
    g = dlp.double().reshape(-1, 1) / temperature
    hit = torch.zeros_like(p)
    inside = (t >= 0) & (t < V)
    hit[inside.nonzero()[:, 0], t[inside]] = 1.0
    # an exponential below 2^-126 is flushed to 0 before the factor |g| / s <= |g| comes to it
    out, off = g * (hit - p), g.abs() * (p * rel + 3 * U * (hit + p) + 2.0 ** -126)
    out[~inside] = float("nan")
    nothing = (g[:, 0] == 0) | (t == ignore)
    out[nothing], off[nothing] = 0.0, 0.0
    return out.reshape(logits.shape), torch.nan_to_num(off, nan=0.0, posinf=0.0).reshape(logits.shape)


def policy(lp, old, adv, mask, ref, clip, kl_weight, average):
    """dict of (value, slack): loss, kl, clip_fraction, grad (for dloss = 1)."""
    R, C = lp.shape
    mask = torch.ones(R, C, dtype=torch.bool, device=lp.device) if mask is None else mask
    hide = lambda t: torch.where(mask, t.double(), 0.0)  # noqa: E731
    lp, old = hide(lp), hide(old)
    adv = hide(adv if adv.dim() == 2 else adv[:, None].expand(R, C))
    d = lp - old
    r = d.exp()
    one, two = r * adv, r.clamp(1 - clip[0], 1 + clip[1]) * adv
    clipped = (one > two) & mask
    gain = torch.minimum(one, two)
    gain_off = torch.where(clipped, 3 * U * gain.abs(), gain.abs() * (6 * U + U * d.abs()))
    slope, slope_off = torch.where(clipped, 0.0, -one), torch.where(clipped, 0.0, gain_off)
    kl = kl_off = torch.zeros_like(d)
    if ref is not None:
        q = hide(ref) - lp
        e1 = torch.expm1(q)
        kl = torch.where(q.abs() < 1e-3, q * q / 2 * (1 + q / 3 * (1 + q / 4 * (1 + q / 5))), e1 - q)
        kl_off = e1.abs() * U * q.abs() + 8 * U * (torch.where(q.abs() > 0.5, e1.abs() + q.abs(), kl))
        slope = slope - kl_weight * e1
        slope_off = slope_off + abs(kl_weight) * (3 * U * e1.abs() + q.exp() * U * q.abs())
    n = mask.sum(1, keepdim=True).double()
    N = n.sum().clamp(min=1)
    w = mask / N if average == "tokens" else mask / n.clamp(min=1) / (n > 0).sum().clamp(min=1)
    each = kl_weight * kl - gain
    each_off = abs(kl_weight) * kl_off + gain_off + 40 * U * (abs(kl_weight) * kl + gain.abs())   # a lane's 32 tokens and five steps
    grad = slope * w
    return dict(loss=((each * w).sum(), (each_off * w).sum()), kl=((kl * mask).sum() / N, ((kl_off + 40 * U * kl) * mask).sum() / N),
                clip_fraction=(clipped.sum() / N, torch.zeros((), dtype=D, device=lp.device)),
                grad=(grad, slope_off * w + 6 * U * grad.abs()))


def preference(lp, ref, mask, beta, e, average):
    """dict of (value, slack): loss, chosen, rejected, grad (for dloss = 1)."""
    R, C = lp.shape
    P = R // 2
    mask = torch.ones(R, C, dtype=torch.bool, device=lp.device) if mask is None else mask
    diff = torch.where(mask, lp.double() - (0.0 if ref is None else ref.double()), 0.0)
    n = mask.sum(1).double().clamp(min=1) if average else torch.ones(R, dtype=D, device=lp.device)
    reward = beta * diff.sum(1) / n
    off = abs(beta) * 40 * U * diff.abs().sum(1) / n      # a lane's 32 tokens, five steps, the difference itself
    h, h_off = reward[:P] - reward[P:], off[:P] + off[P:]
    soft = torch.nn.functional.softplus
    sig = torch.sigmoid
    loss = ((1 - e) * soft(-h) + e * soft(h)).mean()
    k = beta / P * (e * sig(h) - (1 - e) * sig(-h))
    k_off = abs(beta) / P * h_off
    k, k_off = torch.cat([k, -k]) / n, torch.cat([k_off, k_off]) / n
    return dict(loss=(loss, h_off.mean() + 2 * U * loss), chosen_rewards=(reward[:P], off[:P]), rejected_rewards=(reward[P:], off[P:]),
                grad=(torch.where(mask, k[:, None], 0.0), torch.where(mask, (k_off + 4 * U * k.abs())[:, None], 0.0)))

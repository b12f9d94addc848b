"""What is measured of the block-scaled 8-bit product, its quantiser, the fp8
linear layer and the counter-based dropout.

`run` computes one pass in plain torch operations (`own` false) or through
the package's entry points (`own` true).  Sizes are Llama-3-8B's (hidden 4096,
ffn 14336, kv 1024), the 1.3B GPT's (2048, 8192) and odd ones between.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
SIZE = {"bf16": 2, "f32": 4}
DROP_STREAM = 4


def listed():
    return [
        # the hidden state of a few tokens through dropout: latency
        dict(name="dropout 16x768 f32 fwd", op="dropout", rows=16, cols=768, dtype="f32", p=0.1, residual=False, backward=False),
        # an odd token count and an odd width, both directions
        dict(name="dropout 1023x5003 bf16 both", op="dropout", rows=1023, cols=5003, dtype="bf16", p=0.2, residual=True, backward=True),
        # the residual dropout of a training batch, both directions
        dict(name="dropout 16384x4096 bf16 both", op="dropout", rows=16384, cols=4096, dtype="bf16", p=0.1, residual=True, backward=True),
        # the activations of a small decode batch
        dict(name="quantize 7x4096 bf16 rows", op="quantize", rows=7, cols=4096, dtype="bf16", block=1, layout="rows", codes="e4m3"),
        # a training batch's activations, kept for both products
        dict(name="quantize 8192x4096 bf16 both", op="quantize", rows=8192, cols=4096, dtype="bf16", block=1, layout="both", codes="e4m3"),
        # fp32 master weights of an odd shape after a step, e5m2
        dict(name="quantize 5000x2049 f32 tiles", op="quantize", rows=5000, cols=2049, dtype="f32", block=128, layout="both", codes="e5m2"),
        # one token through an up projection
        dict(name="matmul 1x14336x4096 bf16", op="matmul", m=1, n=14336, k=4096, out="bf16", a="e4m3", b="e4m3", tile_b=True),
        # a ragged weight gradient: mixed types, fp32 out
        dict(name="matmul 333x2041x1000 f32", op="matmul", m=333, n=2041, k=1000, out="f32", a="e5m2", b="e4m3", tile_b=False),
        # a prompt through an up projection
        dict(name="matmul 8192x14336x4096 bf16", op="matmul", m=8192, n=14336, k=4096, out="bf16", a="e4m3", b="e4m3", tile_b=True),
        # a weight gradient over a batch's tokens, fp32 out
        dict(name="matmul 4096x4096x8192 f32", op="matmul", m=4096, n=4096, k=8192, out="f32", a="e4m3", b="e4m3", tile_b=False),
        # a training step of a GPT projection: bias, residual dropout, all gradients
        dict(name="linear 1000x2048x2048 f32", op="linear", tokens=1000, n=2048, k=2048, dtype="f32", p=0.1, bias=True, residual=True, backward=True),
        # a training step of a down projection
        dict(name="linear 8192x4096x14336 bf16", op="linear", tokens=8192, n=4096, k=14336, dtype="bf16", p=0.1, bias=False, residual=True, backward=True),
    ]


def _size(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n // 128 * 128 if n > 256 and rng.random() < 0.5 else n))


def draw(rng):
    op = rng.choice(["dropout", "quantize", "matmul", "linear"])
    if op == "dropout":
        rows, cols = _size(rng, 1, 16384), _size(rng, 1, 14336)
        rows = min(rows, (16384 * 4096) // cols)
        return dict(op=op, rows=rows, cols=cols, dtype=rng.choice(["bf16", "f32"]), p=rng.choice([0.05, 0.1, 0.2, 0.5]),
                    residual=rng.random() < 0.5, backward=rng.random() < 0.5)
    if op == "quantize":
        rows, cols = _size(rng, 1, 16384), _size(rng, 64, 14336)
        rows = min(rows, (8192 * 4096) // cols)
        return dict(op=op, rows=rows, cols=cols, dtype=rng.choice(["bf16", "f32"]), block=rng.choice([1, 128]),
                    layout=rng.choice(["rows", "cols", "both"]), codes=rng.choice(["e4m3", "e5m2"]))
    m, n, k = _size(rng, 1, 8192), _size(rng, 64, 14336), _size(rng, 64, 14336)
    m = max(1, min(m, (8192 * 4096 * 8192) // (n * k)))
    if op == "matmul":
        return dict(op=op, m=m, n=n, k=k, out=rng.choice(["bf16", "f32"]), a=rng.choice(["e4m3", "e5m2"]), b=rng.choice(["e4m3", "e5m2"]),
                    tile_b=rng.random() < 0.5)
    return dict(op=op, tokens=m, n=n, k=k, dtype=rng.choice(["bf16", "f32"]), p=rng.choice([0.0, 0.1, 0.2]), bias=rng.random() < 0.5,
                residual=rng.random() < 0.5, backward=rng.random() < 0.7)


def _activations(g, rows, cols, dtype):
    """Unit normal values with some columns ten times as large, as hidden states have."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= 1.0 + 9.0 * (torch.rand(cols, generator=g, device="cuda") < 0.02)
    return x.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case, seed=seed & 0xFFFFFFFFFFFF, site=seed % 97, step=seed % 1009)
    op = case["op"]
    if op == "dropout":
        dt = DTYPES[case["dtype"]]
        s["x"] = _activations(g, case["rows"], case["cols"], dt).requires_grad_(case["backward"])
        s["residual"] = _activations(g, case["rows"], case["cols"], dt).requires_grad_(case["backward"]) if case["residual"] else None
        s["dy"] = (torch.randn(case["rows"], case["cols"], generator=g, device="cuda") * 1e-3).to(dt) if case["backward"] else None
    elif op == "quantize":
        s["x"] = _activations(g, case["rows"], case["cols"], DTYPES[case["dtype"]])
    elif op == "matmul":
        a = _activations(g, case["m"], case["k"], torch.float32)
        b = torch.randn(case["n"], case["k"], generator=g, device="cuda") * 0.02
        s["a"] = _quantize(a, 1, case["a"])
        s["b"] = _quantize(b, 128 if case["tile_b"] else 1, case["b"])
        for q in ("a", "b"):   # a handle's codes have rows of whole 16 bytes
            codes, scales = s[q]
            wide = torch.zeros(codes.shape[0], -(-case["k"] // 16) * 16, dtype=torch.uint8, device="cuda")
            wide[:, : case["k"]] = codes.view(torch.uint8)
            s[q] = (wide.view(codes.dtype)[:, : case["k"]], scales)
    else:
        dt = DTYPES[case["dtype"]]
        T, N, K = case["tokens"], case["n"], case["k"]
        grad = case["backward"]
        s["x"] = _activations(g, T, K, dt).requires_grad_(grad)
        s["w"] = (torch.randn(N, K, generator=g, device="cuda") * 0.02).to(dt).requires_grad_(grad)
        s["bias"] = (torch.randn(N, generator=g, device="cuda") * 0.1).to(dt).requires_grad_(grad) if case["bias"] else None
        s["residual"] = _activations(g, T, N, dt).requires_grad_(grad) if case["residual"] else None
        s["dy"] = (torch.randn(T, N, generator=g, device="cuda") * 1e-3).to(dt) if grad else None
    return s


# ---- the plain forms ----
def _mul_hi_lo(a, m):
    """(high, low) words of the 32 x 32 bit products, in int64."""
    low = (a & 0xFFFF) * m
    high = (a >> 16) * m
    low = low + ((high & 0xFFFF) << 16)
    return (high >> 16) + (low >> 32), low & 0xFFFFFFFF


def _keep(n, p, s, device):
    """Which of n elements are kept, and the factor of the kept ones."""
    T = int(round(p * 65536))
    grp = torch.arange((n + 7) // 8, dtype=torch.int64, device=device)
    c0, c1 = grp & 0xFFFFFFFF, (grp >> 32) | (DROP_STREAM << 24)
    c2, c3 = torch.full_like(grp, s["site"]), torch.full_like(grp, s["step"])
    k0, k1 = s["seed"] & 0xFFFFFFFF, s["seed"] >> 32
    for _ in range(10):
        h0, l0 = _mul_hi_lo(c0, 0xD2511F53)
        h1, l1 = _mul_hi_lo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    r = torch.stack([c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16], dim=1)
    return r.reshape(-1)[:n] >= T, (65536.0 / (65536 - T) if T < 65536 else 0.0)


def _dropped(v, keep, scale):
    return torch.where(keep.view(v.shape), v.float() * scale, torch.zeros((), device=v.device))


def _blocks(x, block):
    """x padded with zeros and cut into blocks: [row blocks, block, column blocks, 128]."""
    R, C = x.shape
    x = torch.nn.functional.pad(x, (0, -C % 128, 0, -R % block))
    return x.view((R + block - 1) // block, block, (C + 127) // 128, 128)


def _pow2(e, dtype=torch.float32):
    """2^e for whole e, from its bits: exact, which pow need not be."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64).to(dtype)


def _quantize(x, block, codes):
    """(codes, scales) of x in blocks of block x 128."""
    R, C = x.shape
    x = x.float()
    x = torch.where(torch.isfinite(x), x, torch.full((), math.nan, device=x.device))
    b = _blocks(x, block)
    top = torch.nan_to_num(b, nan=0.0).abs().amax(dim=(1, 3))
    frac, ex = torch.frexp(top)
    e = ex - torch.where(frac <= 0.875, 9 if codes == "e4m3" else 16, 8 if codes == "e4m3" else 15)
    e = torch.where(top > 0, e, torch.zeros_like(e)).clamp(min=-127)
    q = (b * _pow2(-e)[:, None, :, None]).reshape(b.shape[0] * block, -1)[:R, :C]
    return q.to(DTYPES[codes]), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _values(codes, scales, dtype=torch.float32):
    """The numbers that codes and scales stand for."""
    R, C = codes.shape
    e = scales.view(torch.uint8).to(torch.int64) - 127
    block = 1 if scales.shape[0] == R else 128
    e = _pow2(e, dtype).repeat_interleave(block, 0)[:R].repeat_interleave(128, 1)[:, :C]
    return codes.to(dtype) * e


def _round_trip(x, block):
    return _values(*_quantize(x, block, "e4m3"))


def _plain(s):
    c = s["case"]
    if c["op"] == "dropout":
        x = s["x"].detach()
        keep, scale = _keep(x.numel(), c["p"], s, x.device)
        y = _dropped(x, keep, scale)
        y = (y + s["residual"].detach().float() if c["residual"] else y).to(x.dtype)
        if not c["backward"]:
            return [y]
        return [y, _dropped(s["dy"], keep, scale).to(x.dtype)] + ([s["dy"]] if c["residual"] else [])
    if c["op"] == "quantize":
        out = []
        if c["layout"] in ("rows", "both"):
            out += _quantize(s["x"], c["block"], c["codes"])
        if c["layout"] in ("cols", "both"):
            out += _quantize(s["x"].t(), c["block"], c["codes"])
        return out
    if c["op"] == "matmul":
        return [(_values(*s["a"]) @ _values(*s["b"]).t()).to(DTYPES[c["out"]])]
    x, w = s["x"].detach(), s["w"].detach()
    T, N = c["tokens"], c["n"]
    wq = _round_trip(w, 128)
    y = _round_trip(x, 1) @ wq.t()
    if c["bias"]:
        y = y + s["bias"].detach().float()
    keep, scale = _keep(T * N, c["p"], s, x.device) if c["p"] else (torch.ones(T * N, dtype=torch.bool, device=x.device), 1.0)
    y = _dropped(y, keep, scale)
    y = (y + s["residual"].detach().float() if c["residual"] else y).to(x.dtype)
    if not c["backward"]:
        return [y]
    g = _dropped(s["dy"], keep, scale)
    dx = (_round_trip(g, 1) @ wq).to(x.dtype)
    dw = (_round_trip(g.t(), 1) @ _round_trip(x.t(), 1).t()).to(x.dtype)
    out = [y, dx, dw]
    if c["bias"]:
        out.append(g.sum(0).to(x.dtype))
    if c["residual"]:
        out.append(s["dy"])
    return out


# ---- the package's calls ----
def _own(s):
    import advanced_optimizers_b200 as A
    c = s["case"]
    if c["op"] == "dropout":
        y = A.philox_dropout(s["x"], c["p"], seed=s["seed"], site=s["site"], step=s["step"], residual=s["residual"])
        if not c["backward"]:
            return [y]
        leaves = [t for t in (s["x"], s["residual"]) if t is not None]
        return [y] + list(torch.autograd.grad(y, leaves, s["dy"]))
    if c["op"] == "quantize":
        q = A.quantize_fp8(s["x"], block=(c["block"], 128), dtype=DTYPES[c["codes"]], layout=c["layout"])
        return [t for b in (q if c["layout"] == "both" else (q,)) for t in (b.codes, b.scales)]
    if c["op"] == "matmul":
        return [A.fp8_matmul(A.Fp8Blocks(*s["a"]), A.Fp8Blocks(*s["b"]), out_dtype=DTYPES[c["out"]])]
    y = A.fp8_linear(s["x"], s["w"], s["bias"], residual=s["residual"], dropout_p=c["p"], seed=s["seed"], site=s["site"], step=s["step"])
    if not c["backward"]:
        return [y]
    leaves = [t for t in (s["x"], s["w"], s["bias"], s["residual"]) if t is not None]
    return [y] + list(torch.autograd.grad(y, leaves, s["dy"]))


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    c = case
    if c["op"] == "dropout":
        n, size = c["rows"] * c["cols"], SIZE[c["dtype"]]
        return {"bytes": n * size * (2 + c["residual"] + 2 * c["backward"]), "flops": 0}
    if c["op"] == "quantize":
        n, layouts = c["rows"] * c["cols"], 2 if c["layout"] == "both" else 1
        return {"bytes": n * (SIZE[c["dtype"]] + layouts * (1 + 1 / (128 * c["block"]))), "flops": 0}
    if c["op"] == "matmul":
        m, n, k = c["m"], c["n"], c["k"]
        scales = k / 128 * (m + n / (128 if c["tile_b"] else 1))
        return {"bytes": (m + n) * k + scales + m * n * SIZE[c["out"]], "flops": 2 * m * n * k}
    t, n, k, size = c["tokens"], c["n"], c["k"], SIZE[c["dtype"]]
    fwd = t * k + n * k + t * n * (1 + c["residual"])
    bwd = t * n + t * k + n * k if c["backward"] else 0
    return {"bytes": size * (fwd + bwd), "flops": 2 * t * n * k * (3 if c["backward"] else 1)}


# ---- the definitions in 64 bits ----
def _exact_keep(n, p, s):
    T = int(round(p * 65536))
    u = np.uint64
    grp = np.arange((n + 7) // 8, dtype=u)
    low = u(0xFFFFFFFF)
    c = [grp & low, (grp >> u(32)) | u(DROP_STREAM << 24), np.full_like(grp, s["site"]), np.full_like(grp, s["step"])]
    key = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32]
    for i in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        ka, kb = u((key[0] + i * 0x9E3779B9) & 0xFFFFFFFF), u((key[1] + i * 0xBB67AE85) & 0xFFFFFFFF)
        c = [(b >> u(32)) ^ c[1] ^ ka, b & low, (a >> u(32)) ^ c[3] ^ kb, a & low]
    r = np.empty((grp.size, 8), dtype=np.uint16)
    for e in range(8):
        r[:, e] = (c[e // 2] >> u(16 * (e % 2))) & u(0xFFFF)
    keep = torch.from_numpy(r.reshape(-1)[:n].astype(np.int32) >= T).cuda()
    return keep.double() * (65536 / (65536 - T) if T < 65536 else 0.0)


def _power(e):
    """2^e for whole e in float64, without pow's last-bit errors."""
    return (e.long() + 1023).bitwise_left_shift(52).view(torch.float64)


def _exact_codes(x, block, codes):
    """(codes' values, scales) of finite x: the least power of two that brings the block's largest value into the type's range, and the nearest value of the type."""
    largest, digits, lowest = (448.0, 3, -6) if codes == "e4m3" else (57344.0, 2, -14)
    R, C = x.shape
    x = x.double()
    nb = (C + 127) // 128
    full = torch.zeros(-(-R // block) * block, nb * 128, dtype=torch.float64, device=x.device)
    full[:R, :C] = x
    top = full.abs().view(-1, block, nb, 128).amax(3).amax(1)
    e = torch.floor(torch.log2(top.clamp(min=1e-300) / largest)) - 1
    for _ in range(2):
        e = e + (top > largest * _power(e))
    e = torch.where(top > 0, e, torch.zeros_like(e)).clamp(min=-127.0)
    scale = _power(e)
    q = full / scale.repeat_interleave(block, 0).repeat_interleave(128, 1)
    at = torch.floor(torch.log2(q.abs().clamp(min=1e-30)))
    at = at + (q.abs() >= _power(at + 1)).double() - (q.abs() < _power(at)).double()
    grid = _power(at.clamp(min=lowest) - digits)
    return (torch.round(q / grid) * grid)[:R, :C], scale


def _exact_values(x, block):
    q, scale = _exact_codes(x, block, "e4m3")
    return q * scale.repeat_interleave(block, 0)[: q.shape[0]].repeat_interleave(128, 1)[:, : q.shape[1]]


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "dropout":
        f = _exact_keep(c["rows"] * c["cols"], c["p"], s).view(c["rows"], c["cols"])
        y = s["x"].detach().double() * f
        if c["residual"]:
            y = y + s["residual"].detach().double()
        return [y] + ([s["dy"].double() * f] if c["backward"] else []) + ([s["dy"].double()] if c["backward"] and c["residual"] else [])
    if c["op"] == "quantize":
        out = []
        if c["layout"] != "cols":
            out += _exact_codes(s["x"], c["block"], c["codes"])
        if c["layout"] != "rows":
            out += _exact_codes(s["x"].t(), c["block"], c["codes"])
        return out
    if c["op"] == "matmul":
        return [torch.matmul(_values(*s["a"], dtype=torch.float64), _values(*s["b"], dtype=torch.float64).mT)]
    T, N = c["tokens"], c["n"]
    x, w = s["x"].detach(), s["w"].detach()
    f = _exact_keep(T * N, c["p"], s).view(T, N)
    wv = _exact_values(w, 128)
    y = torch.matmul(_exact_values(x, 1), wv.mT)
    if c["bias"]:
        y += s["bias"].detach().double()
    y *= f
    if c["residual"]:
        y += s["residual"].detach().double()
    out = [y]
    if c["backward"]:
        dy = s["dy"].double()
        gf = (dy * f)
        out.append(torch.matmul(_exact_values(gf, 1), wv))
        out.append(torch.matmul(_exact_values(gf.mT, 1), _exact_values(x.mT, 1).mT))
        if c["bias"]:
            out.append(gf.sum(0))
        if c["residual"]:
            out.append(dy)
    return out

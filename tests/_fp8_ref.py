"""Plain 64-bit restatements of the block quantiser, the fp8 product and the
counter-based dropout, for the tests."""
import numpy as np
import torch

DROP_STREAM = 4
LARGEST = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
DIGITS = {torch.float8_e4m3fn: (3, -6), torch.float8_e5m2: (2, -14)}


def pow2(e):
    """2^e as float64 from its bits, e whole and within +-1000."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def blocked(scales, rows, cols, block):
    """A value per block, spread over the block's elements."""
    return scales.repeat_interleave(block, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def exponent(v):
    """floor(log2 v) of positive float64 values, exactly."""
    return (v.view(torch.int64) >> 52) - 1023


def quantize(x, block, dtype):
    """(values of the codes in float64, exponents of the scales) of x [R][C] in block x 128 blocks."""
    R, C = x.shape
    x = x.double()
    finite = torch.isfinite(x)
    mb, nb = -(-R // block), -(-C // 128)
    pad = torch.zeros(mb * block, nb * 128, dtype=torch.float64, device=x.device)
    pad[:R, :C] = torch.where(finite, x.abs(), torch.zeros_like(x))
    top = pad.view(mb, block, nb, 128).amax(dim=(1, 3))
    e = exponent(top.clamp(min=1e-300)) - exponent(torch.tensor([LARGEST[dtype]], dtype=torch.float64, device=x.device))
    e = torch.where(top > LARGEST[dtype] * pow2(e), e + 1, e)
    e = torch.where(top > 0, e.clamp(min=-127), torch.zeros_like(e))
    q = x / blocked(pow2(e), R, C, block)
    digits, lowest = DIGITS[dtype]
    grid = pow2(exponent(q.abs().clamp(min=1e-300).nan_to_num(posinf=1.0)).clamp(min=lowest) - digits)
    q = torch.where(finite, torch.round(q / grid) * grid, torch.full_like(q, float("nan")))
    return q, e


def quantized(x, block, dtype=torch.float8_e4m3fn):
    """The numbers that the codes and scales of x stand for."""
    q, e = quantize(x, block, dtype)
    return q * blocked(pow2(e), x.shape[0], x.shape[1], block)


def values(b):
    """The numbers that an Fp8Blocks stands for."""
    e = b.scales.view(torch.uint8).to(torch.int64) - 127
    return b.codes.to(torch.float64) * blocked(pow2(e), b.rows, b.k, b.block[0])


def random16(n, seed, site, step, first=0):
    """The generator's 16-bit values of elements first .. first + n - 1."""
    g0, g1 = first // 8, (first + n + 7) // 8
    u = np.uint64
    low = u(0xFFFFFFFF)
    grp = np.arange(g0, g1, dtype=u)
    c = [grp & low, (grp >> u(32)) | u(DROP_STREAM << 24), np.full_like(grp, site), np.full_like(grp, step)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ u(k0), b & low, (a >> u(32)) ^ c[3] ^ u(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    r = np.stack([(c[i >> 1] >> u(16 * (i & 1))) & u(0xFFFF) for i in range(8)], axis=1).reshape(-1)
    return torch.from_numpy(r[first - 8 * g0: first - 8 * g0 + n].astype(np.int64))


def keep_factor(shape, p, seed, site, step, device="cuda"):
    """0 where an element is dropped, else the factor of the kept ones (float64)."""
    n = int(np.prod(shape))
    T = round(p * 65536)
    f = (random16(n, seed, site, step) >= T).double() * (65536 / (65536 - T) if T < 65536 else 0.0)
    return f.view(shape).to(device)

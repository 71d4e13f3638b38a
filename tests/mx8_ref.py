"""FP8 by blocks of 128 from its definition, in float64 on whatever device the inputs are (the oracle of mx8's tests)."""
import numpy as np
import torch

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
HALF = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}      # a rounding is off by at most this, relative to the value


def magnitudes():
    """every finite magnitude of E4M3, in the order of its codes"""
    return [(m / 8 if e == 0 else 1 + m / 8) * 2.0 ** (max(e, 1) - 7) for e in range(16) for m in range(8)][:127]


def quantize(x):
    """(codes uint8 [M, K], scales uint8 [M, K / 128]): the smallest power of two, 2^-127 at least, with which no magnitude is above 448; the
    nearest element, of two as near the even code"""
    v = x.detach().cpu().double().reshape(x.shape[0], -1, 128).numpy()
    grid = np.array(magnitudes())
    mid = (grid[1:] + grid[:-1]) / 2
    most = np.abs(v).max(-1)
    bad = ~np.isfinite(most)
    exp = np.full(most.shape, -127)
    for s in range(-127, 128):
        exp = np.where(most > 448.0 * 2.0 ** s, s + 1, exp)
    exp = np.where(bad, 128, exp)
    a = np.abs(np.where(bad[..., None], 0.0, v)) / 2.0 ** exp[..., None].astype(np.float64)
    code = np.searchsorted(mid, a, side="left")                  # midpoints below the value
    at = np.minimum(code, len(mid) - 1)
    code = code + ((mid[at] == a) & (code < len(mid)) & (code % 2 == 1))
    sign = np.signbit(np.where(bad[..., None], 0.0, v))
    return (code + 128 * sign).astype(np.uint8).reshape(x.shape[0], -1), (exp + 127).astype(np.uint8)


def values(codes):
    """float64 of E4M3 codes"""
    grid = magnitudes() + [float("nan")]
    return torch.tensor(grid + [-g for g in grid], dtype=torch.float64, device=codes.device)[codes.long()]


def powers(scales):
    s = torch.exp2(scales.double() - 127.0)
    return torch.where(scales == 255, torch.full_like(s, float("nan")), s)


def rounded(x):
    """float64 of the quantised rows"""
    c, s = quantize(x)
    c, s = torch.from_numpy(c).to(x.device), torch.from_numpy(s).to(x.device)
    return values(c) * powers(s).repeat_interleave(128, 1)


def weight(v, s):
    """float64 of an MXFP8 tensor's bytes"""
    return values(v) * powers(s).repeat_interleave(128, 0)[:v.shape[0]].repeat_interleave(128, 1)


def gate(y, gelu=False):
    g, u = y.chunk(2, -1)
    z = 1.59576912160573071176 * g * (1 + 0.044715 * g * g) if gelu else g
    return g * torch.sigmoid(z) * u


def make_weight(seed, rows, K, spread=2):
    """bytes of a tensor of values of the order of 0.02"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = (torch.randn(rows, K, generator=g, device="cuda") * 90).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, torch.randint(115 - spread, 116 + spread, (-(-rows // 128), K // 128), generator=g, device="cuda", dtype=torch.uint8)


def make_x(seed, rows, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000)
    x = torch.randn(rows, K, generator=g, device="cuda")
    x[:, torch.randperm(K, generator=g, device="cuda")[:2]] *= 20
    return x.to(dtype)


KEPT = 2.0 ** -10, 2.0 ** -13


def check(got, x, w, glu=False, gelu=False):
    """got [M, N] against float64 products of x [M, K] and w [N, K] (the values behind the codes).  Rounding to the type costs HALF of the value.
    The matrix cores keep 14 bits of products, aligned to the largest of eight: each product is off by at most 2^-13 of that, the eight by
    2^-10, so a sum by 2^-10 of its sum of magnitudes at most; in the 2-norm the errors of a group are no more alike than its products,
    which leaves 2^-13.  fp32 sums add K * 2^-24 of the magnitudes, far below that.  A gated result has two such factors, the slope of the
    gate at most 1.13, and the hardware's exponential and reciprocal, 2^-20 together."""
    got, half = got.double(), HALF[got.dtype]
    y, mag = x @ w.T, (x.abs() @ w.abs().T) * KEPT[0]
    rel = KEPT[1] + half / 3 ** 0.5 * 1.05      # a rounding is spread evenly: a third of its square; 5 % for few values
    tol = mag
    if glu:
        (g, u), (dg, du) = y.chunk(2, -1), mag.chunk(2, -1)
        y = gate(y, gelu)
        tol = 1.13 * dg * (u.abs() + du) + gate(torch.cat((g.abs() + dg, torch.ones_like(u)), -1), gelu).abs() * du + 2.0 ** -20 * y.abs()
        rel = rel + 1.5 * KEPT[1]
    assert got.shape == y.shape
    assert torch.equal(got.isnan(), y.isnan())
    ok = ~y.isnan()
    err, want, tol = (got - y)[ok], y[ok], tol[ok]
    assert (err.abs() <= half * want.abs() + tol + 1e-30).all(), float((err.abs() - half * want.abs() - tol).max())
    if want.numel() >= 64:      # a norm of enough values
        assert err.norm() <= rel * want.norm() * (1.0 if want.numel() >= 1024 else 1.3), float(err.norm() / want.norm())

"""Plain 64-bit forms of the microscaled operators, written out from the format: element grids, block scales, sums."""
import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
E2M3 = np.array([(m / 8 if e == 0 else 1 + m / 8) * 2.0 ** (max(e, 1) - 1) for e in range(4) for m in range(8)])
GRID = {"MXFP4": E2M1, "MXFP6": E2M3}


def plain_scales(laid, M, K):
    """[M, whole groups of eight] of scales laid out [blocks of 32 rows][groups of 256 columns][32][8]"""
    return laid.reshape(-(-M // 32), -(-K // 256), 32, 8).transpose(0, 2, 1, 3).reshape(-(-M // 32) * 32, -1)[:M]


def quantize(x, dtype):
    """(codes uint8 [M, K], scale bytes [M, K / 32]) of fp64 rows"""
    grid = GRID[dtype]
    v = np.asarray(x, np.float64).reshape(len(x), -1, 32)
    finite = np.isfinite(v).all(-1)
    most = np.where(finite, np.abs(np.where(np.isfinite(v), v, 0)).max(-1), 0)
    e = np.where(most > 0, np.frexp(most)[1] - 1, -200)
    byte = np.where(finite, np.clip(e - 2, -127, 127) + 127, 255).astype(np.uint8)
    a = np.abs(np.where(finite[..., None], v, 0)) / np.exp2(np.where(finite, byte, 127).astype(np.float64) - 127)[..., None]
    mid = (grid[1:] + grid[:-1]) / 2
    code = np.searchsorted(mid, a, side="left")
    at = np.minimum(code, len(mid) - 1)
    code = code + ((mid[at] == a) & (code < len(mid)) & ((at + 1) % 2 == 0))
    sign = np.signbit(np.where(finite[..., None], v, 0))
    code = code + sign * len(grid)
    return code.reshape(len(x), -1).astype(np.uint8), byte


def pack(codes, dtype):
    """value bytes of quantised rows: whole groups of 256 columns; E2M3's 24 bytes a block as 16 of each of eight blocks, then 8 of each"""
    M, K = codes.shape
    codes = np.concatenate([codes, np.zeros((M, -K % 256), np.uint8)], 1)
    if dtype == "MXFP4":
        return codes[:, 0::2] | (codes[:, 1::2] << 4)
    bits = (codes.reshape(M, -1, 8, 32, 1) >> np.arange(6)) & 1
    blocks = np.packbits(bits.astype(np.uint8).reshape(M, -1, 8, 192), axis=-1, bitorder="little")
    return np.concatenate([blocks[..., :16].reshape(M, -1, 128), blocks[..., 16:].reshape(M, -1, 64)], -1).reshape(M, -1)


def values(codes, scales, dtype):
    """fp64 values of codes [M, K] with scales [M, >= K / 32]"""
    grid = np.concatenate([GRID[dtype], -GRID[dtype]])
    s = scales[:, : codes.shape[1] // 32].astype(np.float64)
    s = np.where(s == 255, np.nan, np.exp2(s - 127))
    return (grid[codes].reshape(len(codes), -1, 32) * s[..., None]).reshape(len(codes), -1)


def unpack(v):
    return np.stack([v & 15, v >> 4], -1).reshape(len(v), -1)


def weight(rng, rows, K, lo=118, hi=126):
    """(value bytes, scale bytes, fp64 values) of an MXFP4 tensor"""
    v = rng.integers(0, 256, (rows, K // 2), dtype=np.uint8)
    s = rng.integers(lo, hi, (rows, K // 32), dtype=np.uint8)
    return v, s, values(unpack(v), s, "MXFP4")


def sum_bound(x, w):
    """How far a product of quantised rows and weights may be off, element by element, from its sums in 64 bits.  Every product of two
    codes and their scales is exact.  The sum of a row passes through no more than K / 8 additions in the matrix cores and 24
    more where pieces of K meet, each off by at most 2^-24 of a partial sum, which the sum of magnitudes bounds."""
    return (np.abs(x) @ np.abs(w).T) * ((x.shape[1] / 8 + 24) * 2.0 ** -24)


def glu(y, gelu=False):
    g, u = np.split(y, 2, -1)
    z = 1.59576912160573071176 * g * (1 + 0.044715 * g * g) if gelu else g
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-z)) * u


def glu_bound(y, err, gelu=False):
    """act has a slope of at most 1.13 (both activations) and |act(g)| <= |g|; the sigmoid from a base-2 exponential and a reciprocal is off
    by the rounding of its argument, |z| 2^-23 relative, and four roundings"""
    g, u = np.split(y, 2, -1)
    eg, eu = np.split(err, 2, -1)
    z = np.abs(1.59576912160573071176 * g * (1 + 0.044715 * g * g) if gelu else g)
    h = np.abs(glu(y, gelu))
    return 1.13 * eg * (np.abs(u) + eu) + np.abs(g) * eu + h * (np.minimum(z, 100) + 4) * 2.0 ** -23 + 1e-30


HALF = {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def check(got, want, err, dtype, l2=None):
    """got: torch tensor on any device; NaN where and only where want has it; elsewhere within err and the rounding to dtype"""
    got = got.double().cpu().numpy().reshape(want.shape)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), f"NaN in {np.isnan(got).sum()} places, {nan.sum()} wanted"
    half = HALF[dtype]
    tiny = 2.0 ** -25 if dtype == "float16" else 0.0    # half a step of fp16's subnormals
    off = np.abs(got - want)[~nan]
    room = (err * (1 + half) + half * np.abs(want) + tiny)[~nan]
    assert (off <= room).all(), f"{(off > room).sum()} of {off.size} beyond their bound, worst {np.nanmax(off / np.maximum(room, 1e-300)):.2f} times it"
    if l2 is not None and off.size:
        rel = np.sqrt((off ** 2).sum() / max((want[~nan] ** 2).sum(), 1e-300))
        assert rel <= l2 + half, f"2-norm {rel:.2e}"

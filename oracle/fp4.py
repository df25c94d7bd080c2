"""CPU oracle of the RMS norm with an 8-bit output and of the microscaled 4-bit format, in 64 bits (numpy).

Written from the definitions in include/samq.h; shares nothing with the CUDA path.  Test-only."""
import numpy as np

BLOCK = {"mxfp4": 32, "nvfp4": 16}
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
# border between code i and i + 1; a value on it takes the even code
BORDERS = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
E4M3 = np.array([m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])


def _nearest_even(v, table):
    """Index of the entry of an ascending table nearest to v >= 0, ties to the even index, saturating."""
    hi = np.clip(np.searchsorted(table, v), 1, len(table) - 1)
    lo = hi - 1
    mid = (table[lo] + table[hi]) / 2
    return np.where((v > mid) | ((v == mid) & (lo % 2 == 1)), hi, lo)


def quantize(x, fmt, g=1.0):
    """x float64 [M, K] -> (codes uint8 [M, K], scale bytes uint8 [M, blocks], values float64 [M, K])."""
    x = np.asarray(x, np.float64)
    M, K = x.shape
    b = BLOCK[fmt]
    nb = -(-K // b)
    z = np.zeros((M, nb * b))
    z[:, :K] = x
    z = z.reshape(M, nb, b)
    finite = np.isfinite(z).all(-1)
    zf = np.where(finite[..., None], z, 0.0)
    amax = np.abs(zf).max(-1)
    if fmt == "mxfp4":
        e = np.frexp(np.where(amax > 0, amax, 1e-300))[1] - 1
        byte = np.clip(e - 2 + 127, 0, 252)
        scale = 2.0 ** (byte - 127.0)
        byte = np.where(finite, byte, 0xFF)
    else:
        byte = np.maximum(_nearest_even(np.minimum(amax / (6.0 * g), 448.0), E4M3), 1)
        scale = E4M3[byte] * g
        byte = np.where(finite, byte, 0x7F)
    v = np.abs(zf) / scale[..., None]
    code = np.zeros(v.shape, np.int64)
    for i, border in enumerate(BORDERS):
        code += (v >= border) if i % 2 else (v > border)
    value = np.where(np.signbit(zf), -1.0, 1.0) * E2M1[code] * scale[..., None]
    value[~finite] = np.nan
    code = code + 8 * np.signbit(zf)
    return (code.reshape(M, -1)[:, :K].astype(np.uint8), byte.astype(np.uint8), value.reshape(M, -1)[:, :K])


def groups(fmt, K):
    return -(-K // 256) * (64 // BLOCK[fmt])


def pack_codes(codes, pitch):
    M, K = codes.shape
    z = np.zeros((M, 2 * pitch), np.uint8)
    z[:, :K] = codes
    return z[:, 0::2] | (z[:, 1::2] << 4)


def tile_scales(byte, fmt, K):
    """[M, blocks] -> the tiles [ceil(M/128), G, 32, 4, 4], zero outside."""
    M, nb = byte.shape
    G = groups(fmt, K)
    t = np.zeros((-(-M // 128), G, 32, 4, 4), np.uint8)
    r, j = np.meshgrid(np.arange(M), np.arange(nb), indexing="ij")
    t[r // 128, j // 4, r % 32, r % 128 // 32, j % 4] = byte
    return t


def scale_value(byte, fmt, g=1.0):
    return 2.0 ** (byte.astype(np.float64) - 127) if fmt == "mxfp4" else E4M3[byte] * g


def code_value(code):
    return np.where(code & 8, -1.0, 1.0) * E2M1[code & 7]


def rms_norm(h, w, eps, qmax=127.0):
    """h, w float64 -> (y / s, s [M]) of the definition."""
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * w
    s = np.maximum(np.abs(y).max(-1, keepdims=True), 1e-5) / qmax
    return y / s, s[:, 0]


def gelu(y):
    import torch
    return 0.5 * y * (1.0 + torch.erf(torch.from_numpy(y / np.sqrt(2.0))).numpy())

"""Plain 64-bit numpy forms of the 4-bit matrices, rotary positions and dropout, written from their definitions in include/kiln_b200.h."""
import numpy as np
import torch

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MX4, NV4 = 0, 1
BLOCK = {MX4: 32, NV4: 16}


def round_e4m3(v):
    """To the nearest E4M3 number, ties to even, at most 448; v >= 0."""
    v = np.asarray(v, np.float64)
    _, e = np.frexp(np.maximum(v, 1e-300))
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.minimum(np.round(v / step) * step, 448.0)


def quantise(x, fmt, exp=0):
    """(codes 0..15 [rows, cols], scale [rows, blocks], value [rows, cols]); a block with an infinity or a NaN has a NaN scale."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    b = BLOCK[fmt]
    y = np.zeros((rows, -(-cols // b) * b))
    y[:, :cols] = x * 2.0 ** -exp
    y = y.reshape(rows, -1, b)
    bad = ~np.isfinite(y).all(2)
    y = np.where(bad[:, :, None], 0.0, y)
    top = np.abs(y).max(2)
    if fmt == MX4:
        s = np.ldexp(1.0, np.maximum(np.frexp(top)[1] - 1 - 2, -127))
        s = np.where(top == 0, 2.0 ** -127, s)
    else:
        s = np.maximum(round_e4m3(top / 6.0), 2.0 ** -9)
    v = np.minimum(np.abs(y) / s[:, :, None], 6.0)
    step = np.where(v < 2, 0.5, np.where(v < 4, 1.0, 2.0))
    v = np.round(v / step) * step
    code = np.searchsorted(E2M1, v) + 8 * np.signbit(y)
    s = np.where(bad, np.nan, s)
    val = np.where(np.signbit(y), -v, v) * s[:, :, None] * 2.0 ** exp
    return code.reshape(rows, -1)[:, :cols], s, val.reshape(rows, -1)[:, :cols]


def read4(codes, scales, rows, cols, fmt, exp=0):
    """The matrix that the two buffers (numpy bytes) stand for, by the layout's description."""
    r, c = np.arange(rows)[:, None], np.arange(cols)[None, :]
    byte = codes[r, c // 2]
    code = np.where(c % 2 == 0, byte & 15, byte >> 4).astype(np.int64)
    blk = c // BLOCK[fmt]
    pieces = -(-(-(-cols // BLOCK[fmt])) // 4)
    sb = scales[((r // 128) * pieces + blk // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + blk % 4].astype(np.int64)
    if fmt == MX4:
        s = np.where(sb == 255, np.nan, np.ldexp(1.0, sb - 127))
    else:
        s = np.where(sb == 127, np.nan, np.where(sb >= 8, (8 + sb % 8) * np.ldexp(1.0, sb // 8 - 10), sb * 2.0 ** -9))
    v = E2M1[code % 8] * s * 2.0 ** exp
    return np.where(code >= 8, -v, v)


def buffers(q):
    return q.codes.cpu().numpy(), q.scales.cpu().numpy()


def held(q):
    return read4(*buffers(q), q.rows, q.cols, q.fmt, q.exp)


def gelu64(v):
    from scipy.special import ndtr
    return v * ndtr(v)


def rope64(x, heads, dim, rot, pos, freq, axis, half, amplitude=1.0, inverse=False):
    """x [rows, heads * dim] in 64 bits; pos [rows, axes]."""
    x = np.array(x, np.float64).reshape(len(x), -1)
    y = x.copy()
    axis = np.zeros(rot // 2, int) if axis is None else axis
    n = rot // 2
    for h in range(heads):
        for i in range(n):
            # positions times frequencies turn many times: reduced by whole turns in long double
            t = np.asarray(pos[:, axis[i]], np.longdouble) * np.longdouble(freq[i])
            t = np.asarray(np.remainder(t, 2 * np.longdouble("3.14159265358979323846264338327950288")), np.float64) * (-1 if inverse else 1)
            a, b = (h * dim + i, h * dim + n + i) if half else (h * dim + 2 * i, h * dim + 2 * i + 1)
            y[:, a] = amplitude * (x[:, a] * np.cos(t) - x[:, b] * np.sin(t))
            y[:, b] = amplitude * (x[:, b] * np.cos(t) + x[:, a] * np.sin(t))
    return y


def dropout_words(rows, cols, seed, offset):
    """The 16-bit number of every element: Philox4x32 with ten rounds in Python's integers, vectorised over numpy objects of 64 bits."""
    m = 0xffffffff
    g = -(-cols // 8)
    c = [np.tile(np.arange(g, dtype=np.uint64), rows), np.repeat(np.arange(rows, dtype=np.uint64), g),
         np.full(rows * g, offset & m, np.uint64), np.full(rows * g, offset >> 32, np.uint64)]
    k0, k1 = seed & m, seed >> 32
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & np.uint64(m), (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & np.uint64(m)]
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    return np.stack(c, 1).astype("<u4").view("<u2").reshape(rows, 8 * g)[:, :cols].astype(np.int64)


TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}     # of a rounding, relative

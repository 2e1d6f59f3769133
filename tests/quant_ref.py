"""64-bit restatement of the 8-bit operators (numpy), written from their definitions, and the
tolerances their tests use.

scale = max(max|y| / 448, 2^-126) over 128 consecutive values of a row or a 128 x 128 block;
q = the e4m3 value nearest to y / scale; the pair stands for q * scale."""
import numpy as np

G = 128
TOP = 448.0
FLOOR = 2.0 ** -126


def e4m3_values():
    """Value of every e4m3 bit pattern (0x7f and 0xff are NaN; there are no infinities)."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e.astype(np.float64) - 10))
    v = np.where(b & 128, -v, v)
    v[[127, 255]] = np.nan
    return v


VALUES = e4m3_values()


def decode(bits):
    return VALUES[bits]


def half_step(t):
    """Half the distance between neighbouring e4m3 values around |t| (the smallest step is 2^-9)."""
    e = np.maximum(np.floor(np.log2(np.maximum(np.abs(t), 2.0 ** -6))), -6)
    return 2.0 ** (e - 4)


def encode(t):
    """Bit patterns of the nearest e4m3 values (for making operands: ties go either way)."""
    step = 2 * half_step(t)
    v = np.clip(np.rint(t / step) * step, -TOP, TOP)
    order = np.argsort(VALUES[:127])
    bits = order[np.searchsorted(VALUES[:127][order], np.abs(v))]
    return (bits | np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def blocks(n, b=G):
    return -(-n // b)


def spread(s, rows, cols, block_rows):
    """Scales to one per element."""
    return np.repeat(np.repeat(s, block_rows, 0)[:rows], G, 1)[:, :cols]


def scales(y, block_rows):
    rows, cols = y.shape
    s = np.zeros((blocks(rows, block_rows), blocks(cols)))
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            s[i, j] = np.max(np.abs(y[i * block_rows:(i + 1) * block_rows, j * G:(j + 1) * G]))
    return np.maximum(s / TOP, FLOOR)


def check_pair(y, bits, s, block_rows, rel, t_abs=0.0):
    """`bits`, `s` are what the device made of y.  `rel` bounds the relative error of the fp32
    arithmetic in front of the rounding: of y itself, and of the maximum.  The scale adds one
    division (2^-24) and y / scale a reciprocal and a product (2^-24 each), so the value that is
    rounded is off by at most 2 rel + 2^-22 of itself, and q by half an e4m3 step beside that.  `t_abs`
    bounds what subnormal values in front of the rounding lose, in units of q."""
    rows, cols = y.shape
    want = scales(y, block_rows)
    assert np.all(np.abs(s - want) <= want * (rel + 2.0 ** -23 + t_abs / TOP)), "scale"
    t = y / spread(np.asarray(s, np.float64), rows, cols, block_rows)
    q = decode(bits)
    off = np.abs(q - np.clip(t, -TOP, TOP)) - half_step(t) - np.abs(t) * (2 * rel + 2.0 ** -22) - t_abs
    assert np.all(off <= 0), f"q is {off.max()} beyond the nearest value"


def rmsnorm(x, gain, eps):
    x = x.astype(np.float64)
    return x / np.sqrt(np.mean(x * x, 1, keepdims=True) + eps) * gain


def silu(v):
    return v / (1 + np.exp(-v))


def swiglu(x):
    h = x.shape[1] // 2
    return silu(x[:, :h].astype(np.float64)) * x[:, h:]


def operands(rng, rows, cols, block_rows, std=1.0):
    """A quantised matrix made on the host: (q bits, fp32 scales, 64-bit values it stands for)."""
    y = rng.standard_normal((rows, cols)) * std
    s = scales(y, block_rows).astype(np.float32)
    bits = encode(y / spread(s.astype(np.float64), rows, cols, block_rows))
    return bits, s, decode(bits) * spread(s.astype(np.float64), rows, cols, block_rows)


def product_tolerance(av, bv, c, slope=1.0):
    """|device - exact| for C = A B^T of the values av [M,K], bv [N,K].  Products of two e4m3 values
    are exact; each of the K additions and each scaling may lose 2^-23 (truncation) of the sum of
    magnitudes; the output is rounded to bf16 once (2^-8 of itself).  `slope` bounds the derivative
    of the epilogue."""
    k = av.shape[1]
    size = np.abs(av) @ np.abs(bv).T
    return np.abs(c) * 2.0 ** -8 + slope * size * (k + 8) * 2.0 ** -23 + 1e-30

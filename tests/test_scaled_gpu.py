"""8-bit path: quantisation to e4m3 with a scale per 128 values (plain, behind RMSNorm and behind
SwiGLU) and the block-scaled product, against 64-bit restatements (tests/quant_ref.py)."""
import ctypes as C
import math

import numpy as np
import pytest

import habu_b200 as hb
import oracle
import quant_ref as qr
from habu_b200 import model_ir
from util import SEED

pytestmark = pytest.mark.gpu

PAT = 0xA5                  # fills e4m3 buffers around the output
F_PAT = np.float32(-7.25)   # fills scale buffers


def _up(ctx, ptr, a):
    a = np.ascontiguousarray(a)
    ctx._check(model_ir._lib.hb_upload(ctx._h, C.c_void_p(ptr), a.ctypes.data_as(C.c_void_p), a.nbytes))
    ctx.sync()


def _bf16(rng, shape, std=1.0):
    x = oracle.round_bf16((rng.standard_normal(shape) * std).astype(np.float32))
    return x, oracle.to_bf16_bits(x)


class Out:
    """A (q, scale) pair inside pattern-filled buffers: pitched rows, guard bands, and for the
    scales a row pitch or the transposed order."""

    def __init__(self, ctx, rows, cols, block_rows=1, pad=0, scale_t=False):
        self.ctx, self.rows, self.cols = ctx, rows, cols
        self.pitch = (cols + 15) // 16 * 16 + pad
        self.qbuf = ctx.upload(np.full(64 + rows * self.pitch + 64, PAT, np.uint8))
        self.q = ctx.wrap(self.qbuf.ptr + 64, (rows, cols), hb.HB_E4M3, (self.pitch, 1))
        self.sr, self.sc = qr.blocks(rows, block_rows), qr.blocks(cols)
        self.scale_t = scale_t
        self.sp = (self.sr if scale_t else self.sc) + 3
        self.sbuf = ctx.upload(np.full(16 + (self.sc if scale_t else self.sr) * self.sp + 16, F_PAT, np.float32))
        self.scale = ctx.wrap(self.sbuf.ptr + 64, (self.sr, self.sc), hb.HB_F32, (1, self.sp) if scale_t else (self.sp, 1))

    def finish(self):
        raw = self.ctx.download(self.qbuf)
        body = raw[64:-64].reshape(self.rows, self.pitch)
        assert (raw[:64] == PAT).all() and (raw[-64:] == PAT).all() and (body[:, self.cols:] == PAT).all(), "q: write outside"
        s = self.ctx.download(self.sbuf)
        n = self.sc if self.scale_t else self.sr
        sb = s[16:16 + n * self.sp].reshape(n, self.sp)
        w = self.sr if self.scale_t else self.sc
        assert (s[:16] == F_PAT).all() and (s[16 + n * self.sp:] == F_PAT).all() and (sb[:, w:] == F_PAT).all(), "scale: write outside"
        out = body[:, :self.cols].copy(), (sb[:, :w].T if self.scale_t else sb[:, :w]).copy()
        self.ctx.free(self.qbuf), self.ctx.free(self.sbuf)
        return out


SHAPES = [(1, 8), (1, 128), (3, 129), (5, 136), (128, 128), (129, 127), (200, 1000), (37, 4096), (300, 264), (2, 16384), (1000, 24)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize(ctx, rows, cols, block_rows, dtype):
    rng = np.random.default_rng(rows * 7 + cols)
    x, bits = _bf16(rng, (rows, cols), 3.0)
    if dtype == "f32":
        x = (rng.standard_normal((rows, cols)) * 3).astype(np.float32)
    dx = ctx.upload(bits if dtype == "bf16" else x)
    for pad, scale_t in ((0, False), (16, True)):
        out = Out(ctx, rows, cols, block_rows, pad, scale_t)
        ctx.quantize(dx, out.q, out.scale, block_rows)
        q, s = out.finish()
        qr.check_pair(x.astype(np.float64), q, s, block_rows, 0.0)     # the input is exact: no error in front of the rounding
    ctx.free(dx)


@pytest.mark.parametrize("shift,pitch,qshift,qpitch", [(0, 41, 0, 48), (1, 48, 0, 48), (0, 48, 3, 48), (0, 48, 0, 43), (3, 45, 5, 41)])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_odd_addresses_and_pitches(ctx, shift, pitch, qshift, qpitch, block_rows):
    rows, cols = 150, 40
    rng = np.random.default_rng(shift * 100 + pitch + qpitch)
    x, bits = _bf16(rng, (rows, cols))
    host = np.full(shift + rows * pitch, 0x7FC0, np.uint16)            # NaN in the padding: it must not be read into a maximum
    host[shift:].reshape(rows, pitch)[:, :cols] = bits
    buf = ctx.upload(host)
    qb = ctx.upload(np.full(qshift + rows * qpitch, PAT, np.uint8))
    dx = ctx.wrap(buf.ptr + 2 * shift, (rows, cols), hb.HB_BF16, (pitch, 1))
    q = ctx.wrap(qb.ptr + qshift, (rows, cols), hb.HB_E4M3, (qpitch, 1))
    _, s = ctx.quantize(dx, q, None, block_rows)
    raw = ctx.download(qb)
    body = raw[qshift:].reshape(rows, qpitch)
    assert (raw[:qshift] == PAT).all() and (body[:, cols:] == PAT).all()
    qr.check_pair(x.astype(np.float64), body[:, :cols], ctx.download(s), block_rows, 0.0)
    for t in (buf, qb, s):
        ctx.free(t)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_special_values(ctx, block_rows):
    """Zeros, the smallest and largest magnitudes, values on e4m3 steps and ties, NaN and infinity."""
    rows, cols = 130, 512
    x = np.zeros((rows, cols), np.float32)
    x[1, :128] = 2.0 ** -149
    x[2, :128] = 3.0e38
    x[3, :128] = np.linspace(-448, 448, 128)                            # scale 1: 448 itself included
    x[4, :128] = np.concatenate([qr.VALUES[:127], [448.0]])             # every positive e4m3 value, scale 1
    x[5, :127] = np.diff(qr.VALUES[:127], append=480.0) / 2 + qr.VALUES[:127]   # every tie
    x[5, 126:128] = 448.0
    x[6, 5] = np.nan
    x[6, 6:128] = 1.0
    x[7, 130] = np.inf
    x[7, 131] = 1.0
    x[8, 300] = -0.0
    x[129, 400:] = 5.0
    dx = ctx.upload(x)
    q, s = ctx.quantize(dx, block_rows=block_rows)
    bits = np.ascontiguousarray(_pitched(ctx, q))
    sc = ctx.download(s)
    assert np.isnan(qr.decode(bits[6, 5])), "a NaN stays one"
    vals = qr.decode(bits)
    finite = np.isfinite(x)
    if block_rows == 1:
        assert sc[0, 0] == np.float32(2.0 ** -126) and (bits[0] == 0).all()
        assert np.array_equal(vals[4, :128], x[4, :128].astype(np.float64)), "values on the grid are kept"
        # ties go to the even mantissa
        assert ((bits[5, :126] & 1) == 0).all()
        assert np.all(vals[6, 6:128] == 448.0) and sc[6, 0] == np.float32(1 / 448)
        assert np.isinf(sc[7, 1]) and np.isnan(vals[7, 130] * sc[7, 1]) and np.isnan(vals[7, 131] * sc[7, 1])
        clean = np.ones(rows, bool)
        clean[[6, 7]] = False
        qr.check_pair(x[clean].astype(np.float64), bits[clean], sc[clean], 1, 0.0)
    else:
        assert np.isinf(sc[0, 1]) and np.all(np.isnan((vals[:128, 128:256] * sc[0, 1])[finite[:128, 128:256]]))
        assert sc[0, 3] == np.float32(2.0 ** -126) and sc[1, 3] == np.float32(5 / 448)
        assert np.all(vals[129, 400:] == 448.0)
    for t in (dx, q, s):
        ctx.free(t)


def _pitched(ctx, q):
    """Rows of an e4m3 tensor with a row pitch, on the host."""
    rows, cols = q.shape
    flat = ctx.wrap(q.ptr, (rows, q.stride[0]), hb.HB_E4M3)
    return ctx.download(flat)[:, :cols]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 128), (5, 136), (37, 512), (2, 2048), (130, 2056), (16, 4096), (7, 8200), (3, 16384)])
def test_rmsnorm_quant(ctx, rows, cols, residual):
    rng = np.random.default_rng(rows + cols)
    x, xb = _bf16(rng, (rows, cols), 2.0)
    r, rb = _bf16(rng, (rows, cols), 2.0)
    g, gb = _bf16(rng, (cols,), 0.5)
    if rows > 2:                     # a row of zeros (the statistic is eps alone) and one of large values
        xb[1] = 0
        x[1] = r[1] = 0
        rb[1] = 0
        x[2] *= np.float32(2.0 ** 40)
        xb[2] = oracle.to_bf16_bits(x[2])
    dx, dg = ctx.upload(xb), ctx.upload(gb)
    pitch = cols + 8                 # strided residual, padding kept
    rh = np.full((rows, pitch), 0x1234, np.uint16)
    rh[:, :cols] = rb
    dr = ctx.upload(rh)
    drv = ctx.wrap(dr.ptr, (rows, cols), hb.HB_BF16, (pitch, 1))
    out = Out(ctx, rows, cols, 1, 16, rows % 2 == 0)
    ctx.rmsnorm_quant(dx, dg, out.q, out.scale, 1e-5, drv if residual else None)
    q, s = out.finish()
    base = x
    if residual:
        base = oracle.round_bf16((x.astype(np.float64) + r).astype(np.float32))   # the sum of two bf16 values is exact in 64 bits ...
        got = ctx.download(dr)
        assert np.array_equal(got[:, :cols], oracle.to_bf16_bits(base)) and (got[:, cols:] == 0x1234).all()
    # mean of squares: up to 64 additions per thread, 5 + 8 across threads (2^-24 each: 2^-17.7 on the
    # sum, half on the root), rsqrt 2 ulp, three products: below 2^-17 of y
    qr.check_pair(qr.rmsnorm(base, g.astype(np.float64), 1e-5), q, s, 1, 2.0 ** -17)
    for t in (dx, dg, dr):
        ctx.free(t)


def test_rmsnorm_quant_keeps_a_bad_row_to_itself(ctx):
    rng = np.random.default_rng(5)
    x, xb = _bf16(rng, (4, 256))
    g, gb = _bf16(rng, (256,))
    xb[1, 17] = 0x7FC0               # NaN
    xb[2, 200] = 0x7F80              # infinity: its square makes the statistic infinite
    q, s = ctx.rmsnorm_quant(ctx.upload(xb), ctx.upload(gb))
    v = qr.decode(_pitched(ctx, q)) * qr.spread(ctx.download(s).astype(np.float64), 4, 256, 1)
    assert np.isnan(v[1]).all() and np.isnan(v[2, 200]) and (v[2, :128] == 0).all()
    qr.check_pair(qr.rmsnorm(x[[0, 3]], g.astype(np.float64), 1e-5), _pitched(ctx, q)[[0, 3]], ctx.download(s)[[0, 3]], 1, 2.0 ** -17)


@pytest.mark.parametrize("rows,half", [(1, 8), (2, 128), (5, 136), (300, 264), (16, 14336), (33, 2048), (1000, 16)])
def test_swiglu_quant(ctx, rows, half):
    rng = np.random.default_rng(rows + half)
    x, xb = _bf16(rng, (rows, 2 * half), 3.0)
    if rows > 1:
        x[1, :half] = -200.0         # silu(-200) is -0 in fp32
        xb[1, :half] = oracle.to_bf16_bits(np.full(half, -200, np.float32))
    dx = ctx.upload(xb)
    out = Out(ctx, rows, half, 1, 0, rows % 2 == 0)
    ctx.swiglu_quant(dx, out.q, out.scale)
    q, s = out.finish()
    y = qr.swiglu(x)
    if rows > 1:
        assert (qr.decode(q[1]) == 0).all() and (s[1] == np.float32(2.0 ** -126)).all()
    # exp with the argument's rounding (|v| 2^-24 log2 e, |v| < 20 here) and 2 ulp, division 2 ulp, one product: below 2^-18
    keep = [i for i in range(rows) if rows == 1 or i != 1]
    qr.check_pair(y[keep], q[keep], s[keep], 1, 2.0 ** -18)
    ctx.free(dx)


# ------------------------------------------------------------------ product
def _upload_pair(ctx, bits, s, pad=0, scale_t=False):
    """Host pair -> device views with padded rows (the padding holds e4m3 NaNs)."""
    rows, cols = bits.shape
    pitch = (cols + 15) // 16 * 16 + pad
    h = np.full((rows, pitch), 0x7F, np.uint8)
    h[:, :cols] = bits
    d = ctx.upload(h)
    sp = (s.shape[0] if scale_t else s.shape[1]) + 1
    sh = np.full((s.shape[1] if scale_t else s.shape[0], sp), np.nan, np.float32)
    sh[:, :-1] = s.T if scale_t else s
    ds = ctx.upload(sh)
    return (ctx.wrap(d.ptr, (rows, cols), hb.HB_E4M3, (pitch, 1), d),
            ctx.wrap(ds.ptr, s.shape, hb.HB_F32, (1, sp) if scale_t else (sp, 1), ds))


def _free(ctx, *ts):
    for t in ts:
        ctx.free(t.owner)


class COut:
    def __init__(self, ctx, M, N, pad=0, shift=0):
        self.ctx, self.M, self.N, self.ld, self.front = ctx, M, N, N + pad, 64 + shift
        self.buf = ctx.upload(np.full(self.front + M * self.ld + 64, 0xBEEF, np.uint16))
        self.t = ctx.wrap(self.buf.ptr + 2 * self.front, (M, N), hb.HB_BF16, (self.ld, 1))

    def finish(self):
        raw = self.ctx.download(self.buf)
        body = raw[self.front:-64].reshape(self.M, self.ld)
        assert (raw[:self.front] == 0xBEEF).all() and (raw[-64:] == 0xBEEF).all() and (body[:, self.N:] == 0xBEEF).all()
        self.ctx.free(self.buf)
        return oracle.from_bf16_bits(np.ascontiguousarray(body[:, :self.N])).astype(np.float64)


# rows around the limits of the few-row kernel and of the tiles; columns around blocks of 128; k around 128 and 16
PRODUCTS = [(1, 256, 128), (1, 1, 1), (1, 6144, 512), (2, 300, 100), (16, 256, 4096), (16, 1000, 1000), (17, 384, 136), (63, 130, 300),
            (64, 512, 2048), (65, 512, 256), (64, 100, 128), (128, 128, 128), (129, 129, 129), (200, 255, 384), (256, 256, 640),
            (300, 1000, 520), (333, 72, 2056), (511, 1025, 16), (700, 520, 1160), (1000, 8, 256), (1500, 2304, 384),
            # long sums of few tiles (split over a cluster), and a wide product of one tile row (128 x 256 tiles)
            (65, 130, 7000), (128, 520, 4096), (200, 100, 6000), (100, 9500, 256), (128, 10000, 200)]


@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_matmul_scaled(ctx, M, N, K):
    rng = np.random.default_rng(M * 31 + N * 7 + K)
    ab, sa, av = qr.operands(rng, M, K, 1)
    bb, sb, bv = qr.operands(rng, N, K, 128)
    want = av @ bv.T
    tol = qr.product_tolerance(av, bv, want)
    for pad, scale_t, cpad, shift in ((0, False, 0, 0), (16, True, 8, 0), (48, False, 3, 1)):
        A, SA = _upload_pair(ctx, ab, sa, pad, scale_t)
        B, SB = _upload_pair(ctx, bb, sb, pad, scale_t)
        c = COut(ctx, M, N, cpad, shift)
        ctx.matmul_scaled(A, SA, B.T, SB.T, c.t, weights=pad == 0)
        got = c.finish()
        assert np.all(np.abs(got - want) <= tol), (pad, float(np.max(np.abs(got - want) - tol)))
        _free(ctx, A, SA, B, SB)


@pytest.mark.parametrize("epi", [hb.HB_EPI_GELU, hb.HB_EPI_SWIGLU, hb.HB_EPI_RESIDUAL])
@pytest.mark.parametrize("M,N,K", [(1, 256, 128), (16, 512, 384), (64, 264, 1000), (129, 136, 200), (300, 1000, 520), (513, 770, 256),
                                   (100, 202, 6100), (128, 9600, 200), (1300, 2310, 136)])
def test_matmul_scaled_epilogues(ctx, M, N, K, epi):
    rng = np.random.default_rng(M + N + K + epi)
    ab, sa, av = qr.operands(rng, M, K, 1)
    bb, sb, bv = qr.operands(rng, N, K, 128, K ** -0.5)
    r, rb = _bf16(rng, (M, N + 5))
    acc = av @ bv.T
    if epi == hb.HB_EPI_GELU:
        from math import erf
        want = acc * 0.5 * (1 + np.vectorize(erf)(acc / np.sqrt(2)))
        tol = qr.product_tolerance(av, bv, want, 1.13)               # |gelu'| < 1.13
        tol += np.abs(acc) * 2.0 ** -22                               # erff: 2 ulp of a value of at most 1
    elif epi == hb.HB_EPI_SWIGLU:
        g, u = acc[:, 0::2], acc[:, 1::2]
        want = qr.silu(g) * u
        t = qr.product_tolerance(av, bv, acc * 0)
        # |silu'| < 1.1, |silu(g)| <= |g|: errors of the gate times |u|, of the up value times |g|; the fp32 silu itself 2^-18
        tol = np.abs(want) * (2.0 ** -8 + 2.0 ** -18) + 1.1 * t[:, 0::2] * np.abs(u) + t[:, 1::2] * np.abs(g) + 1.1 * t[:, 0::2] * t[:, 1::2]
    else:
        want = acc + r[:, :N]
        tol = qr.product_tolerance(av, bv, want) + np.abs(want) * 2.0 ** -23
    for cpad, shift in ((0, 0), (8, 0), (3, 1)):
        A, SA = _upload_pair(ctx, ab, sa)
        B, SB = _upload_pair(ctx, bb, sb)
        R = ctx.upload(rb)
        c = COut(ctx, M, want.shape[1], cpad, shift)
        res = ctx.wrap(R.ptr, (M, N), hb.HB_BF16, (N + 5, 1)) if epi == hb.HB_EPI_RESIDUAL else None
        ctx.matmul_scaled(A, SA, B.T, SB.T, c.t, epilogue=epi, residual=res)
        got = c.finish()
        assert np.all(np.abs(got - want) <= tol), float(np.max(np.abs(got - want) - tol))
        _free(ctx, A, SA, B, SB)
        ctx.free(R)


@pytest.mark.parametrize("M,N,K", [(16, 512, 1024), (48, 256, 512), (130, 300, 640), (600, 520, 896), (100, 300, 6400), (128, 9600, 384),
                                   (1300, 2304, 384)])
def test_matmul_scaled_is_exact_on_small_integers(ctx, M, N, K):
    """Integers up to 8 and power-of-two scales: every partial sum fits fp32, so the result is the
    exact sum rounded to bf16, whatever the order.  A scale that lands on the wrong row, column or
    k-block shows at once, because every one of them differs."""
    rng = np.random.default_rng(M)
    a = rng.integers(-8, 9, (M, K)).astype(np.float64)
    b = rng.integers(-8, 9, (N, K)).astype(np.float64)
    sa = 2.0 ** rng.integers(-2, 3, (M, qr.blocks(K)))
    sb = 2.0 ** rng.integers(-2, 3, (qr.blocks(N), qr.blocks(K)))
    want = (a * qr.spread(sa, M, K, 1)) @ (b * qr.spread(sb, N, K, 128)).T
    A, SA = _upload_pair(ctx, qr.encode(a), sa.astype(np.float32))
    B, SB = _upload_pair(ctx, qr.encode(b), sb.astype(np.float32))
    got = ctx.download(ctx.matmul_scaled(A, SA, B.T, SB.T))
    assert np.array_equal(got, oracle.to_bf16_bits(want.astype(np.float32)))
    _free(ctx, A, SA, B, SB)


@pytest.mark.parametrize("M,N,K", [(5, 300, 700), (64, 512, 1024), (200, 300, 700), (520, 512, 512)])
def test_matmul_scaled_keeps_nan_to_its_row_and_column(ctx, M, N, K):
    """A NaN value or scale of A reaches its own output row only, one of B its own column (a scale:
    its block of columns)."""
    rng = np.random.default_rng(N)
    ab, sa, av = qr.operands(rng, M, K, 1)
    bb, sb, bv = qr.operands(rng, N, K, 128)
    want = av @ bv.T
    tol = qr.product_tolerance(av, bv, want)
    ab, sb, sa = ab.copy(), sb.copy(), sa.copy()
    ab[M // 2, K - 1] = 0x7F
    sa[0, 1] = np.nan
    sb[-1, 0] = np.inf
    A, SA = _upload_pair(ctx, ab, sa)
    B, SB = _upload_pair(ctx, bb, sb)
    got = oracle.from_bf16_bits(ctx.download(ctx.matmul_scaled(A, SA, B.T, SB.T))).astype(np.float64)
    n0 = (qr.blocks(N) - 1) * 128
    bad = np.zeros((M, N), bool)
    bad[[M // 2, 0]] = True
    bad[:, n0:] = True
    assert np.isnan(got[[M // 2, 0]]).all() and (~np.isfinite(got[:, n0:])).all()
    assert np.all(np.abs(got - want)[~bad] <= tol[~bad])
    _free(ctx, A, SA, B, SB)


@pytest.mark.parametrize("M", [1, 16, 40, 64, 100, 700])
def test_matmul_scaled_repeats_bit_for_bit(ctx, M):
    rng = np.random.default_rng(M)
    N, K = 2000, 2176
    ab, sa, _ = qr.operands(rng, M, K, 1)
    bb, sb, _ = qr.operands(rng, N, K, 128)
    A, SA = _upload_pair(ctx, ab, sa)
    B, SB = _upload_pair(ctx, bb, sb)
    first = ctx.download(ctx.matmul_scaled(A, SA, B.T, SB.T))
    outs = [ctx.matmul_scaled(A, SA, B.T, SB.T, weights=i % 2 == 0) for i in range(12)]     # back to back, nothing waits between
    for o in outs:
        assert np.array_equal(ctx.download(o), first)
        ctx.free(o)
    _free(ctx, A, SA, B, SB)


@pytest.mark.parametrize("rows", [1, 16, 64, 200])
def test_a_feed_forward_sublayer(ctx, rows):
    """The operators as they are used together, enqueued without a wait: norm with the residual's
    addition -> gate/up product -> SwiGLU -> down product.  Each step is checked against the 64-bit
    formula on the device's own input of that step, so every tolerance is that of one operator."""
    d, F = 512, 1024
    rng = np.random.default_rng(rows)
    x, xb = _bf16(rng, (rows, d))
    r, rb = _bf16(rng, (rows, d))
    g, gb = _bf16(rng, (d,))
    w1 = (rng.standard_normal((2 * F, d)) * d ** -0.5).astype(np.float32)
    w2 = (rng.standard_normal((d, F)) * F ** -0.5).astype(np.float32)
    dw1, dw2 = ctx.upload(w1), ctx.upload(w2)
    q1, s1 = ctx.quantize(dw1, block_rows=128)
    q2, s2 = ctx.quantize(dw2, block_rows=128)
    dx, dr, dg = ctx.upload(xb), ctx.upload(rb), ctx.upload(gb)
    h, hs = ctx.rmsnorm_quant(dx, dg, residual=dr)
    gu = ctx.matmul_scaled(h, hs, q1.T, s1.T, weights=True)
    a, as_ = ctx.swiglu_quant(gu)
    out = ctx.matmul_scaled(a, as_, q2.T, s2.T, weights=True)
    val = lambda q, s, b: qr.decode(_pitched(ctx, q)) * qr.spread(ctx.download(s).astype(np.float64), *q.shape, b)
    base = oracle.round_bf16((x.astype(np.float64) + r).astype(np.float32))
    assert np.array_equal(ctx.download(dr), oracle.to_bf16_bits(base))
    qr.check_pair(qr.rmsnorm(base, g.astype(np.float64), 1e-5), _pitched(ctx, h), ctx.download(hs), 1, 2.0 ** -17)
    hv, w1v, w2v, av = val(h, hs, 1), val(q1, s1, 128), val(q2, s2, 128), val(a, as_, 1)
    guv = oracle.from_bf16_bits(ctx.download(gu)).astype(np.float64)
    want = hv @ w1v.T
    assert np.all(np.abs(guv - want) <= qr.product_tolerance(hv, w1v, want))
    qr.check_pair(qr.swiglu(guv), _pitched(ctx, a), ctx.download(as_), 1, 2.0 ** -18)
    want = av @ w2v.T
    got = oracle.from_bf16_bits(ctx.download(out)).astype(np.float64)
    assert np.all(np.abs(got - want) <= qr.product_tolerance(av, w2v, want))
    for t in (dw1, dw2, q1, s1, q2, s2, dx, dr, dg, h, hs, gu, a, as_, out):
        ctx.free(t)


def test_offsets_beyond_32_bits(ctx):
    """Rows more than 2^31 elements apart: every row index is multiplied by its pitch in 64 bits.  The
    operators touch a few rows of a buffer that is otherwise left alone."""
    far = (1 << 31) + 64
    rows, cols, N = 3, 256, 300
    rng = np.random.default_rng(9)
    x, xb = _bf16(rng, (rows, cols))
    r, rb = _bf16(rng, (rows, cols))
    g, gb = _bf16(rng, (cols,))
    bx, bq, bc = ctx.empty((2 * far + 1024,)), ctx.empty((2 * far + 1024,), hb.HB_E4M3), ctx.empty((2 * far + 1024,))
    dx = ctx.wrap(bx.ptr, (rows, cols), hb.HB_BF16, (far, 1))
    dr = ctx.wrap(bc.ptr, (rows, cols), hb.HB_BF16, (far, 1))
    dq = ctx.wrap(bq.ptr, (rows, cols), hb.HB_E4M3, (far, 1))
    for i in range(rows):
        _up(ctx, bx.ptr + 2 * i * far, xb[i])
        _up(ctx, bc.ptr + 2 * i * far, rb[i])

    def fetch(buf, elem, dtype, width):
        return np.stack([ctx.download(ctx.wrap(buf.ptr + elem * i * far, (width,), dtype)) for i in range(rows)])
    _, s = ctx.quantize(dx, dq, None, 1)
    qr.check_pair(x.astype(np.float64), fetch(bq, 1, hb.HB_E4M3, cols), ctx.download(s), 1, 0.0)
    _, s = ctx.quantize(dx, dq, None, 128)
    qr.check_pair(x.astype(np.float64), fetch(bq, 1, hb.HB_E4M3, cols), ctx.download(s), 128, 0.0)
    _, s = ctx.swiglu_quant(dx, ctx.wrap(bq.ptr, (rows, cols // 2), hb.HB_E4M3, (far, 1)))
    qr.check_pair(qr.swiglu(x), fetch(bq, 1, hb.HB_E4M3, cols // 2), ctx.download(s), 1, 2.0 ** -18)
    _, s = ctx.rmsnorm_quant(dx, ctx.upload(gb), dq, residual=dr)
    base = oracle.round_bf16((x.astype(np.float64) + r).astype(np.float32))
    assert np.array_equal(fetch(bc, 2, hb.HB_BF16, cols), oracle.to_bf16_bits(base))
    ab = fetch(bq, 1, hb.HB_E4M3, cols)
    sa = ctx.download(s)
    qr.check_pair(qr.rmsnorm(base, g.astype(np.float64), 1e-5), ab, sa, 1, 2.0 ** -17)
    # the product: A, the residual and C with that pitch, and B for the few-row kernel
    av = qr.decode(ab) * qr.spread(sa.astype(np.float64), rows, cols, 1)
    bb, sb, bv = qr.operands(rng, N, cols, 128)
    B, SB = _upload_pair(ctx, bb, sb)
    dc = ctx.wrap(bx.ptr, (rows, N), hb.HB_BF16, (far, 1))
    for i in range(rows):
        _up(ctx, bc.ptr + 2 * i * far, oracle.to_bf16_bits(np.zeros(N, np.float32) + i))
    ctx.matmul_scaled(dq, s, B.T, SB.T, dc, epilogue=hb.HB_EPI_RESIDUAL, residual=ctx.wrap(bc.ptr, (rows, N), hb.HB_BF16, (far, 1)))
    want = av @ bv.T + np.arange(rows)[:, None]
    got = oracle.from_bf16_bits(fetch(bx, 2, hb.HB_BF16, N)).astype(np.float64)
    assert np.all(np.abs(got - want) <= qr.product_tolerance(av, bv, want) + np.abs(want) * 2.0 ** -23)
    # roles exchanged: the far-pitched matrix as B (three columns of C), 200 rows of A: the tile kernels
    ab2, sa2, av2 = qr.operands(rng, 200, cols, 1)
    A2, SA2 = _upload_pair(ctx, ab2, sa2)
    bs = ctx.upload(np.full((1, 2), 0.5, np.float32))
    c2 = ctx.matmul_scaled(A2, SA2, dq.T, bs.T)
    bv2 = qr.decode(ab) * 0.5
    want = av2 @ bv2.T
    got = oracle.from_bf16_bits(ctx.download(c2)).astype(np.float64)
    assert np.all(np.abs(got - want) <= qr.product_tolerance(av2, bv2, want))
    for t in (bx, bq, bc):
        ctx.free(t)
    _free(ctx, B, SB, A2, SA2)


@pytest.mark.parametrize("M", [3, 90, 700])
@pytest.mark.parametrize("N", [301, 302, 304])
@pytest.mark.parametrize("epi", [hb.HB_EPI_NONE, hb.HB_EPI_RESIDUAL])
def test_matmul_scaled_output_alignments(ctx, M, N, epi):
    """Outputs and residuals whose rows start on 16, 4 or 2 bytes, in every combination that a pitch and a
    start allow: 16-, 4- and 2-byte pieces, and TMA where it is possible."""
    K = 2304
    rng = np.random.default_rng(N + M)
    ab, sa, av = qr.operands(rng, M, K, 1)
    bb, sb, bv = qr.operands(rng, N, K, 128)
    acc = av @ bv.T
    A, SA = _upload_pair(ctx, ab, sa)
    B, SB = _upload_pair(ctx, bb, sb)
    for pad, shift in ((0, 0), (8 - N % 8, 0), (2 - N % 2, 0), (8 - N % 8, 2), (1 - N % 2, 1)):
        c = COut(ctx, M, N, pad, shift)
        res, want = None, acc
        if epi == hb.HB_EPI_RESIDUAL:
            r, rb = _bf16(rng, (M, N + pad))
            rbuf = ctx.upload(np.concatenate([np.full(shift, 0x7FC0, np.uint16), rb.reshape(-1)]))
            res = ctx.wrap(rbuf.ptr + 2 * shift, (M, N), hb.HB_BF16, (N + pad, 1))
            want = acc + r[:, :N]
        ctx.matmul_scaled(A, SA, B.T, SB.T, c.t, epilogue=epi, residual=res)
        got = c.finish()
        tol = qr.product_tolerance(av, bv, want) + np.abs(want) * 2.0 ** -23
        assert np.all(np.abs(got - want) <= tol), (pad, shift)
    _free(ctx, A, SA, B, SB)


def test_operators_follow_the_context_stream(ctx):
    """On a caller's stream, and back: ordered with what the caller queues there."""
    torch = pytest.importorskip("torch")
    rows, d, N = 64, 512, 640
    rng = np.random.default_rng(11)
    gb = _bf16(rng, (d,))[1]
    dg = ctx.upload(gb)
    w = ctx.quantize(ctx.upload(rng.standard_normal((N, d)).astype(np.float32)), block_rows=128)
    ctx.sync()
    st = torch.cuda.Stream()
    ctx.set_stream(st.cuda_stream)
    try:
        with torch.cuda.stream(st):
            x = torch.zeros(rows, d, device="cuda", dtype=torch.bfloat16)
            outs = []
            for i in range(6):
                x += 1 + i                                # queued on the same stream, in front of the norm
                x[:, i] = -3
                t = ctx.wrap(x.data_ptr(), (rows, d), hb.HB_BF16)
                h = ctx.rmsnorm_quant(t, dg)
                outs.append((x.clone(), ctx.matmul_scaled(*h, w[0].T, w[1].T, weights=True)))
        st.synchronize()
    finally:
        ctx.set_stream(None)
    for xi, o in outs:
        t = ctx.wrap(xi.data_ptr(), (rows, d), hb.HB_BF16)
        h = ctx.rmsnorm_quant(t, dg)
        again = ctx.matmul_scaled(*h, w[0].T, w[1].T)
        assert np.array_equal(ctx.download(o), ctx.download(again))


def test_two_contexts_at_once():
    """Nothing is shared between contexts, and the product keeps no scratch at all: two contexts on their
    own streams, working at the same time."""
    rng = np.random.default_rng(12)
    M, N, K = 16, 1024, 4096
    cs = [hb.Context(0), hb.Context(0)]
    work = []
    for c in cs:
        ab, sa, av = qr.operands(rng, M, K, 1)
        bb, sb, bv = qr.operands(rng, N, K, 128)
        A, SA = _upload_pair(c, ab, sa)
        B, SB = _upload_pair(c, bb, sb)
        work.append((c, A, SA, B, SB, av @ bv.T, qr.product_tolerance(av, bv, av @ bv.T), [c.empty((M, N)) for _ in range(20)]))
    for i in range(20):
        for c, A, SA, B, SB, _, _, outs in work:
            c.matmul_scaled(A, SA, B.T, SB.T, outs[i], weights=True)
    for c, *_, want, tol, outs in work:
        for o in outs:
            got = oracle.from_bf16_bits(c.download(o)).astype(np.float64)
            assert np.all(np.abs(got - want) <= tol)
    for c in cs:
        c.close()


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_around_the_floor(ctx, block_rows):
    """Groups whose largest value runs from far below 448 x 2^-126, where the scale meets its floor, to far
    above it: the pair stands for the values on both sides."""
    rows, cols = 256, 128
    rng = np.random.default_rng(13)
    top = 2.0 ** np.linspace(-149, -100, rows if block_rows == 1 else 2)
    y = rng.uniform(-1, 1, (rows, cols)) * np.repeat(top, rows // len(top))[:, None]
    x = y.astype(np.float32)
    q, s = ctx.quantize(ctx.upload(x), block_rows=block_rows)
    bits, sc = _pitched(ctx, q), ctx.download(s)
    assert not np.isnan(qr.decode(bits)).any()
    qr.check_pair(x.astype(np.float64), bits, sc, block_rows, 0.0)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", [(37, 256), (5, 2560), (300, 1920), (3, 10240)])
def test_rmsnorm_quant_around_the_floor(ctx, rows, cols, residual):
    """Gains that take whole groups from far below the floor of the scale to far above it, beside rows of
    zeros, of a statistic that overflows, and with a NaN or an infinity."""
    rng = np.random.default_rng(rows)
    x, xb = _bf16(rng, (rows, cols))
    g, gb = _bf16(rng, (cols,))
    g *= np.repeat(2.0 ** np.linspace(-133, -100, cols // 128).round(), 128)
    gb = oracle.to_bf16_bits(g.astype(np.float32))
    g = oracle.round_bf16(g.astype(np.float32)).astype(np.float64)
    x[0], xb[0] = 0, 0
    huge = 2.0 ** 100                # squares beyond fp32: the root's inverse is 0
    xb[1] = oracle.to_bf16_bits((x[1] * huge).astype(np.float32))
    xb[2, cols - 1] = 0x7FC0
    if rows > 3:
        xb[3, 5] = 0xFF80            # minus infinity
    dx, dr = ctx.upload(xb), ctx.upload(np.zeros((rows, cols), np.uint16))
    out = Out(ctx, rows, cols, 1, 16, False)
    ctx.rmsnorm_quant(dx, ctx.upload(gb), out.q, out.scale, 1e-5, dr if residual else None)
    q, s = out.finish()
    if residual:
        assert np.array_equal(ctx.download(dr)[[0, 1]], xb[[0, 1]])
    v = qr.decode(q)
    assert (v[0] == 0).all() and (v[1] == 0).all() and (s[:2] == np.float32(qr.FLOOR)).all()
    assert np.isnan(v[2]).all()
    if rows > 3:
        assert np.isnan(v[3, 5]) and (np.delete(v[3], 5) == 0).all()
    # x * gain is formed first: below 2^-126 it is off by 2^-150, which the root's inverse (at most 1.2 for
    # rows of unit variance) and a scale of 2^-126 or more turn into 1.2 * 2^-24 units of q
    good = [0] + list(range(4, rows))
    qr.check_pair(qr.rmsnorm(x[good], g, 1e-5), q[good], s[good], 1, 2.0 ** -17, 2.0 ** -23)


@pytest.mark.parametrize("step,K", [(64, 16), (1, 256), (100, 4096), (1300, 16)])
def test_gelu_epilogue_over_its_range(ctx, step, K):
    """Products of a single 1 with a_scale as the argument: from far below zero, where the output is a
    vanishing product, through zero to far above, infinities and NaN; every form of the product."""
    x = np.concatenate([np.linspace(-14, 14, 700), np.linspace(-6, 6, 500), [0.0, -0.0, 1e-30, -1e-30, 1e30, -1e30, 3e38, -3e38],
                        np.linspace(-0.01, 0.01, 92)]).astype(np.float32)
    if step == 1:
        x = x[::50]
    N = 24
    one = np.zeros((step, K), np.uint8)
    one[:, 3] = qr.encode(np.ones(1))[0]
    w = np.zeros((N, K), np.uint8)
    w[:, 3] = one[0, 3]
    A, B = ctx.upload(one), ctx.upload(w)
    SB = ctx.upload(np.ones((1, K // 128 if K > 128 else 1), np.float32))
    got = []
    for at in range(0, len(x), step):
        s = np.ones((step, SB.shape[1]), np.float32)
        part = x[at:at + step]
        s[:len(part), 0] = part
        c = ctx.matmul_scaled(A, ctx.upload(s), B.T, SB.T, epilogue=hb.HB_EPI_GELU)
        got.append(oracle.from_bf16_bits(ctx.download(c))[:len(part)])
    got = np.concatenate(got).astype(np.float64)
    v = x.astype(np.float64)
    tail = np.array([0.5 * abs(t) * math.erfc(abs(t) / math.sqrt(2)) for t in v])
    want = np.maximum(v, 0) - tail
    # erfc to 2^-17 of itself (|x| < 5.2), 2^-14 (up to 6), 2^-4.9; three roundings to fp32; the one to bf16.
    # The exponential gives 0 for an erfc below 2^-126: the product with |x| / 2 then loses at most
    # |x| / 2 * 2^-126 (and |x| / 2 is taken as 8 at most).
    off = np.where(np.abs(v) < 5.2, 2.0 ** -17, np.where(np.abs(v) < 6, 2.0 ** -14, 2.0 ** -4.9))
    tol = np.abs(want) * (2.0 ** -8 + 2.0 ** -21) + tail * off * (1 + 2.0 ** -8) + np.minimum(np.abs(v) / 2, 8) * 2.0 ** -126 + 2.0 ** -133
    assert np.all(np.abs(got - want[:, None]) <= tol[:, None])
    s = np.ones((step, SB.shape[1]), np.float32)
    for value in (np.inf, np.nan):
        s[0, 0] = value
        c = oracle.from_bf16_bits(ctx.download(ctx.matmul_scaled(A, ctx.upload(s), B.T, SB.T, epilogue=hb.HB_EPI_GELU)))
        assert np.isnan(c[0]).all() if np.isnan(value) else (c[0] == np.inf).all()


@pytest.mark.parametrize("M,N,K", [(4100, 1158, 144), (2050, 4614, 128), (200, 38402, 128), (600, 1414, 256)])
@pytest.mark.parametrize("epi", [hb.HB_EPI_NONE, hb.HB_EPI_SWIGLU, hb.HB_EPI_RESIDUAL])
def test_matmul_scaled_tiles_at_odd_addresses(ctx, M, N, K, epi):
    """Whole tiles whose rows start on every multiple of two bytes, from one row to the next and from one
    start to another, for every width that a warp writes; the edges beside them stay as they were."""
    rng = np.random.default_rng(N)
    ab, sa, av = qr.operands(rng, M, K, 1)
    bb, sb, bv = qr.operands(rng, N, K, 128)
    A, SA = _upload_pair(ctx, ab, sa)
    B, SB = _upload_pair(ctx, bb, sb)
    acc = av @ bv.T
    size = np.abs(av) @ np.abs(bv).T
    if epi == hb.HB_EPI_SWIGLU:
        base, slope = qr.silu(acc[:, 0::2]) * acc[:, 1::2], None
        # |silu'| < 1.1: the two factors' errors, each (K + 8) 2^-23 of its sums; silu itself 2^-20
        e = (K + 8) * 2.0 ** -23
        loose = 1.1 * np.abs(acc[:, 1::2]) * size[:, 0::2] * e + np.abs(acc[:, 0::2]) * size[:, 1::2] * e + np.abs(base) * 2.0 ** -19
    else:
        base, loose = acc, size * (K + 8) * 2.0 ** -23
    out = base.shape[1]
    for pad, shift in ((1, 0), (0, 1), (3, 2), (2, 3), (5, 7)):
        c = COut(ctx, M, out, pad, shift)
        res, want = None, base
        if epi == hb.HB_EPI_RESIDUAL:
            r, rb = _bf16(rng, (M, out + pad))
            rbuf = ctx.upload(np.concatenate([np.full(shift, 0x7FC0, np.uint16), rb.reshape(-1)]))
            res = ctx.wrap(rbuf.ptr + 2 * shift, (M, out), hb.HB_BF16, (out + pad, 1))
            want = base + r[:, :out]
        ctx.matmul_scaled(A, SA, B.T, SB.T, c.t, epilogue=epi, residual=res)
        got = c.finish()
        assert np.all(np.abs(got - want) <= np.abs(want) * (2.0 ** -8 + 2.0 ** -22) + loose + 1e-30), (pad, shift)
    _free(ctx, A, SA, B, SB)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_fp32_rounds_once(ctx, block_rows):
    """fp32 values a unit in the last place on either side of the points half-way between two e4m3 values, for
    many scales: q is the nearest value of the quotient in 64 bits wherever that is not a tie itself."""
    rng = np.random.default_rng(5)
    rows, cols = 256, 256
    x = rng.uniform(-1, 1, (rows, cols)).astype(np.float32)
    top = rng.uniform(1, 2, (rows // block_rows, 2)).astype(np.float32)
    tops = np.repeat(np.repeat(top, block_rows, 0), 128, 1).astype(np.float64)
    vals = np.sort(qr.VALUES[:127])
    half = (vals[1:] + vals[:-1]) / 2
    pick = half[rng.integers(0, len(half), (rows, cols))] * tops / 448
    x = np.nextafter(pick.astype(np.float32), np.where(rng.random((rows, cols)) < 0.5, np.float32(0), np.float32(9)), dtype=np.float32)
    x = np.where(rng.random((rows, cols)) < 0.3, pick.astype(np.float32), x) * np.where(rng.random((rows, cols)) < 0.5, 1, -1).astype(np.float32)
    for i in range(rows // block_rows):
        for j in range(2):
            x[i * block_rows, 128 * j] = top[i, j]
    q, s = ctx.quantize(ctx.upload(x), block_rows=block_rows)
    t = x.astype(np.float64) * 448 / tops                # (two roundings of 2^-53)
    lower = np.searchsorted(half, np.abs(t))
    tie = np.abs(np.abs(t) - half[np.minimum(lower, len(half) - 1)]) <= np.abs(t) * 2.0 ** -51
    tie |= np.abs(np.abs(t) - half[np.maximum(lower - 1, 0)]) <= np.abs(t) * 2.0 ** -51
    want = np.copysign(vals[lower], t)
    assert np.array_equal(qr.decode(_pitched(ctx, q))[~tie], want[~tie]) and (~tie).mean() > 0.5

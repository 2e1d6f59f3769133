"""The 8-bit operators on the executor, and the decoder graphs that use them (``e4m3=True``): the nodes
against the same calls on the context (bit for bit), capture and replay, the generation step and the
prompt against their bf16 forms on the weights that the quantised ones stand for."""
import ctypes as C

import numpy as np
import pytest

import habu_b200 as hb
import oracle
import quant_ref as qr
from habu_b200 import model_ir
from habu_b200.graph import Graph
from habu_b200.model_ir import HabuError
from habu_b200.tp import DecoderConfig, DecodeGraph, DecoderGraph, decode_layer, shard_layer
from oracle import decoder

pytestmark = pytest.mark.gpu


def _up(ctx, t, a):
    a = np.ascontiguousarray(a)
    ctx._check(model_ir._lib.hb_upload(ctx._h, C.c_void_p(t.ptr), a.ctypes.data_as(C.c_void_p), a.nbytes))
    ctx.sync()


def _bits(rng, shape, std=1.0):
    return oracle.to_bf16_bits((rng.standard_normal(shape) * std).astype(np.float32))


def test_nodes_equal_the_calls_bit_for_bit(ctx):
    rows, d, F = 70, 256, 384
    rng = np.random.default_rng(1)
    dx, dr, dg = ctx.upload(_bits(rng, (rows, d))), ctx.upload(_bits(rng, (rows, d))), ctx.upload(_bits(rng, (d,)))
    r0 = ctx.download(dr)
    w1 = ctx.quantize(ctx.upload(_bits(rng, (2 * F, d), d ** -0.5)), block_rows=128)
    w2 = ctx.quantize(ctx.upload(_bits(rng, (d, F), F ** -0.5)), block_rows=128)
    out = ctx.empty((rows, d))
    # the calls
    h = ctx.rmsnorm_quant(dx, dg, residual=dr)
    r1 = ctx.download(dr)
    act = ctx.matmul_scaled(*h, w1[0].T, w1[1].T, epilogue=hb.HB_EPI_SWIGLU)
    a = ctx.quantize(act)
    want = ctx.download(ctx.matmul_scaled(*a, w2[0].T, w2[1].T))
    gu = ctx.matmul_scaled(*h, w1[0].T, w1[1].T)
    s = ctx.swiglu_quant(gu)
    want2 = ctx.download(ctx.matmul_scaled(*s, w2[0].T, w2[1].T))
    # the same on a graph: every temporary, the scales included, is planner-owned
    g = Graph(ctx)
    x, r, gain, o = g.input(dx), g.input(dr), g.input(dg), g.input(out)
    W1, W2 = [g.input(t.T) for t in w1], [g.input(t.T) for t in w2]
    hq = g.temp_quantised(rows, d)
    g.rmsnorm_quant(x, gain, *hq, residual=r)
    ga = g.temp((rows, F))
    g.matmul_scaled(*hq, *W1, ga, epilogue=hb.HB_EPI_SWIGLU)
    gq = g.temp_quantised(rows, F)
    g.quantize(ga, *gq)
    g.matmul_scaled(*gq, *W2, o, weights=True)
    out2 = ctx.empty((rows, d))
    o2 = g.input(out2)
    ggu = g.temp((rows, 2 * F))
    g.matmul_scaled(*hq, *W1, ggu)
    gs = g.temp_quantised(rows, F)
    g.swiglu_quant(ggu, *gs)
    g.matmul_scaled(*gs, *W2, o2)
    g.plan()
    assert "e4m3" in g.describe() and "rmsnorm_quant" in g.describe()
    for run in range(3):                          # eager, eager, replayed
        _up(ctx, dr, r0)
        if run < 2:
            g.run()
        else:
            g.capture()
            g.replay()
        ctx.sync()
        assert np.array_equal(ctx.download(dr), r1)
        assert np.array_equal(ctx.download(out), want) and np.array_equal(ctx.download(out2), want2), run
    g.close()


def test_graph_refusals(ctx):
    rows, d = 8, 256
    rng = np.random.default_rng(2)
    w = ctx.quantize(ctx.upload(_bits(rng, (d, d))), block_rows=128)
    dx, dg, out = ctx.upload(_bits(rng, (rows, d))), ctx.upload(_bits(rng, (d,))), ctx.empty((rows, d))
    # scales that no node wrote are not read
    g = Graph(ctx)
    q, s = g.temp_quantised(rows, d)
    other = g.temp((rows, 2), hb.HB_F32)
    g.quantize(g.input(dx), q, s)
    g.matmul_scaled(q, other, g.input(w[0].T), g.input(w[1].T), g.input(out))
    with pytest.raises(HabuError, match="before any node writes"):
        g.plan()
    g.close()
    g = Graph(ctx)
    q, s = g.temp_quantised(rows, d)
    g.quantize(g.input(dx), q, s)
    with pytest.raises(HabuError, match="no residual input"):
        g.matmul_scaled(q, s, g.input(w[0].T), g.input(w[1].T), g.input(out), epilogue=hb.HB_EPI_RESIDUAL)
    with pytest.raises(HabuError, match="unknown tensor"):
        g.matmul_scaled(q, s, g.input(w[0].T), 99, g.input(out))
    g.close()
    g = Graph(ctx)                                 # a gain of the wrong length
    q, s = g.temp_quantised(rows, d)
    g.rmsnorm_quant(g.input(dx), g.view(g.input(dg), 0, (d // 2,), (1,)), q, s)
    g.plan()
    with pytest.raises(HabuError, match="gain"):
        g.run()
    g.close()


def _stands_for(layer):
    """The bf16 layer whose matrices are what the quantised ones stand for, rounded to bf16."""
    out = {}
    for k, v in layer.items():
        if k in ("g1", "g2"):
            out[k] = v
            continue
        y = v.astype(np.float64)
        s = qr.scales(y, 128).astype(np.float32).astype(np.float64)
        f = qr.spread(s, *y.shape, 128)
        out[k] = oracle.round_bf16((qr.decode(qr.encode(y / f)) * f).astype(np.float32))
    return out


def _bits_layer(lw):
    return {k: oracle.to_bf16_bits(v) for k, v in lw.items()}


CFG = DecoderConfig(d_model=512, n_q_heads=4, n_kv_heads=2, head_dim=128, ffn_hidden=1024, n_layers=2, batch=2, seq=40)


def _far(a, b):
    return float(np.linalg.norm(a.astype(np.float64) - b) / np.linalg.norm(b))


def test_generation_and_prompt_with_e4m3_weights(ctx):
    """Quantising an activation is off by at most 2^-4 of a value, evenly spread over the step: 2^-4 /
    sqrt(3) in the mean square at the top of a step and half that at its bottom.  A product of such
    values with exact ones has the same relative error in its norm; four products a layer add up in the
    sublayers' outputs (the residual stream itself is exact), so two layers stay below 4 x 2^-4 /
    sqrt(3) = 0.15 of the norm.  A wrong scale, block or operand is off by about its whole norm."""
    S = CFG.seq
    layers = [decoder.make_layer(CFG, i) for i in range(CFG.n_layers)]
    xs = decoder.make_input(CFG)
    e4 = DecodeGraph(ctx, CFG, [_bits_layer(decode_layer(l, CFG)) for l in layers], CFG.batch, s_max=S, e4m3=True)
    bf = DecodeGraph(ctx, CFG, [_bits_layer(_stands_for(decode_layer(l, CFG))) for l in layers], CFG.batch, s_max=S)
    x3 = xs.reshape(CFG.batch, S, -1)
    eager = []
    for t in range(S):
        xt = oracle.to_bf16_bits(np.ascontiguousarray(x3[:, t]))
        for dg in (e4, bf):
            _up(ctx, dg.x, xt)
            dg.step()
        ctx.sync()
        eager.append(ctx.download(e4.out))
        want = oracle.from_bf16_bits(ctx.download(bf.out)).astype(np.float64)
        got = oracle.from_bf16_bits(eager[-1]) - x3[:, t]           # what the layers added
        assert _far(got, want - x3[:, t]) < 0.15, t
    # half the weight bytes (the scales are 2^-12 of the elements)
    assert e4.bytes_per_step(1) < 0.52 * bf.bytes_per_step(1)
    # replayed: the same bits, token after token, with another graph of the same context in between
    rep = DecodeGraph(ctx, CFG, [_bits_layer(decode_layer(l, CFG)) for l in layers], CFG.batch, s_max=S, e4m3=True)
    _up(ctx, rep.x, oracle.to_bf16_bits(np.ascontiguousarray(x3[:, 0])))
    rep.capture()
    rep.set_pos(0)
    bf.set_pos(0)
    for t in range(S):
        _up(ctx, rep.x, oracle.to_bf16_bits(np.ascontiguousarray(x3[:, t])))
        rep.step()
        bf.step()
        ctx.sync()
        assert np.array_equal(ctx.download(rep.out), eager[t]), t
    # the prompt graph (gate and up rows interleaved, SwiGLU in the product's epilogue)
    pre = DecoderGraph(ctx, CFG, 1, 0, [_bits_layer(shard_layer(l, CFG, 1, 0)) for l in layers], e4m3=True)
    ref = DecoderGraph(ctx, CFG, 1, 0, [_bits_layer(_stands_for(shard_layer(l, CFG, 1, 0))) for l in layers])
    for dg in (pre, ref):
        dg.plan()
        _up(ctx, dg.x0, oracle.to_bf16_bits(xs))
        dg.run()
    ctx.sync()
    got = oracle.from_bf16_bits(ctx.download(pre.out))
    want = oracle.from_bf16_bits(ctx.download(ref.out)).astype(np.float64)
    assert _far(got - xs, want - xs) < 0.15
    # and the prompt's rows are the generation's tokens
    gen = np.stack([oracle.from_bf16_bits(e) for e in eager], 1).reshape(xs.shape)
    assert _far(gen - xs, (got - xs).astype(np.float64)) < 0.15


def test_decoder_graph_refuses_what_e4m3_does_not_cover(ctx):
    layers = [_bits_layer(shard_layer(decoder.make_layer(CFG, 0), CFG, 1, 0))]
    with pytest.raises(ValueError, match="one rank"):
        DecoderGraph(ctx, CFG, 2, 0, layers, e4m3=True)
    one = DecoderGraph(ctx, CFG, 1, 0, layers)
    with pytest.raises(ValueError, match="same precision"):
        DecoderGraph(ctx, CFG, 1, 0, layers, e4m3=True, share=one)


def test_other_operators_refuse_e4m3(ctx):
    """An e4m3 tensor where an operator takes bare pointers to wider elements is refused before a launch."""
    q, _ = ctx.quantize(ctx.upload(np.zeros((32, 256), np.uint16)))
    gain, ids = ctx.upload(np.zeros(256, np.uint16)), ctx.upload(np.zeros(4, np.int32))
    before = ctx.launches
    for call in (lambda: ctx.rmsnorm(q, gain), lambda: ctx.rmsnorm(gain, gain, out=q), lambda: ctx.rope(q, 32, 2, 128), lambda: ctx.embedding(q, ids),
                 lambda: ctx.swiglu(q), lambda: ctx.gelu(q), lambda: ctx.add(q, q), lambda: ctx.argmax(q), lambda: ctx.mse(q, q),
                 lambda: ctx.matmul(q, q.T)):
        with pytest.raises(hb.HabuError):
            call()
    assert ctx.launches == before

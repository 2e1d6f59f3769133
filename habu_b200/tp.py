"""Megatron-style tensor-parallel decoder block on the model-IR executor.

Sharding (rank r of n): query heads and KV heads are split by head, so grouped-query
groups stay rank-local; the QKV and gate/up projections are column-parallel, the
attention-out and FFN-down projections row-parallel, each followed by one sum-allreduce
of the [tokens, d_model] partial result.  RMSNorm, RoPE and the residual stream are
replicated.  Weights are stored the way the matmul node wants a column-major B: one
row per output feature, K contiguous.

Pure index arithmetic lives in the ``shard_*`` functions (no GPU needed); ``DecoderGraph``
builds the node list for one rank.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List

import numpy as np

from . import _capi


@dataclass(frozen=True)
class DecoderConfig:
    d_model: int = 4096
    n_q_heads: int = 32
    n_kv_heads: int = 8
    head_dim: int = 128
    ffn_hidden: int = 14336
    n_layers: int = 2
    batch: int = 4
    seq: int = 2048
    eps: float = 1e-5
    rope_base: float = 10000.0

    @property
    def tokens(self) -> int:
        return self.batch * self.seq

    def flops(self) -> float:
        """Algorithmic flop of one forward (GEMMs + causal attention by the usual count)."""
        T, d, hd = self.tokens, self.d_model, self.head_dim
        qkv = 2.0 * T * d * (self.n_q_heads + 2 * self.n_kv_heads) * hd
        attn = 4.0 * self.batch * self.n_q_heads * self.seq * self.seq * hd / 2
        out = 2.0 * T * self.n_q_heads * hd * d
        ffn = 2.0 * T * d * 2 * self.ffn_hidden + 2.0 * T * self.ffn_hidden * d
        return self.n_layers * (qkv + attn + out + ffn)


def shard_range(total: int, world: int, rank: int):
    if total % world:
        raise ValueError(f"{total} does not split over {world} ranks")
    per = total // world
    return rank * per, (rank + 1) * per


def check_shardable(cfg: DecoderConfig, world: int):
    if cfg.n_q_heads % cfg.n_kv_heads:
        raise ValueError("query heads must be a multiple of KV heads")
    for name, v in (("n_kv_heads", cfg.n_kv_heads), ("n_q_heads", cfg.n_q_heads), ("ffn_hidden", cfg.ffn_hidden)):
        if v % world:
            raise ValueError(f"{name}={v} does not split over {world} ranks")
    if (cfg.ffn_hidden // world) % 8:
        raise ValueError("local FFN width must be a multiple of 8")


def shard_layer(full: Dict[str, np.ndarray], cfg: DecoderConfig, world: int, rank: int) -> Dict[str, np.ndarray]:
    """Slice one layer's full weights ([out_features, in_features] each) for `rank`.

    full: wq [Hq*hd, d], wk/wv [Hkv*hd, d], wo [d, Hq*hd], wg/wu [F, d], wd [d, F], g1/g2 [d].
    Returns wqkv [(q+2kv)_local*hd, d], wo [d, q_local*hd], wgu [2*F_local, d] with rows
    interleaved (gate_j, up_j), wd [d, F_local], and the replicated gains.
    """
    check_shardable(cfg, world)
    hd = cfg.head_dim
    q0, q1 = shard_range(cfg.n_q_heads, world, rank)
    k0, k1 = shard_range(cfg.n_kv_heads, world, rank)
    f0, f1 = shard_range(cfg.ffn_hidden, world, rank)
    wqkv = np.concatenate([full["wq"][q0 * hd:q1 * hd], full["wk"][k0 * hd:k1 * hd], full["wv"][k0 * hd:k1 * hd]], 0)
    wgu = np.empty((2 * (f1 - f0), cfg.d_model), full["wg"].dtype)
    wgu[0::2] = full["wg"][f0:f1]
    wgu[1::2] = full["wu"][f0:f1]
    return {"wqkv": np.ascontiguousarray(wqkv), "wo": np.ascontiguousarray(full["wo"][:, q0 * hd:q1 * hd]),
            "wgu": wgu, "wd": np.ascontiguousarray(full["wd"][:, f0:f1]), "g1": full["g1"], "g2": full["g2"]}


QUANTISED = ("wqkv", "wo", "wgu", "wd")       # the weight matrices of a layer; the gains stay bf16


def upload_layer(ctx, layer: Dict[str, np.ndarray], e4m3: bool) -> Dict[str, object]:
    """Device tensors of one layer's weights (bf16 bit patterns).  With `e4m3` every matrix is
    quantised on the device in 128 x 128 blocks (a (q, scale) pair instead of a tensor) and its
    bf16 copy is freed."""
    dev = {}
    for k, v in layer.items():
        t = ctx.upload(v)
        if e4m3 and k in QUANTISED:
            dev[k] = ctx.quantize(t, block_rows=128)
            ctx.sync()
            ctx.free(t)
        else:
            dev[k] = t
    return dev


class _Products:
    """The products of a layer on an executor graph, in bf16 or with e4m3 operands: where an activation
    comes from (a norm, SwiGLU, attention) and the product that takes it."""

    def __init__(self, g, e4m3: bool, eps: float, weights: bool):
        self.g, self.e4m3, self.eps, self.weights = g, e4m3, eps, weights

    def weight(self, v):
        """Graph ids of one weight: B as [in, out], and its scales."""
        return (self.g.input(v[0].T), self.g.input(v[1].T)) if isinstance(v, tuple) else self.g.input(v.T)

    def norm(self, x, gain, rows, cols, residual=None):
        if self.e4m3:
            h = self.g.temp_quantised(rows, cols)
            self.g.rmsnorm_quant(x, gain, *h, residual=residual, eps=self.eps)
        else:
            h = self.g.temp((rows, cols))
            self.g.rmsnorm(x, gain, h, residual=residual, eps=self.eps)
        return h

    def swiglu(self, gu, rows, half):
        if self.e4m3:
            act = self.g.temp_quantised(rows, half)
            self.g.swiglu_quant(gu, *act)
        else:
            act = self.g.temp((rows, half))
            self.g.swiglu(gu, act)
        return act

    def operand(self, x, rows, cols):
        """A bf16 activation as an operand of :meth:`matmul`."""
        if not self.e4m3:
            return x
        h = self.g.temp_quantised(rows, cols)
        self.g.quantize(x, *h)
        return h

    def matmul(self, a, w, out, epilogue=_capi.HB_EPI_NONE):
        if self.e4m3:
            self.g.matmul_scaled(*a, *w, out, epilogue=epilogue, weights=self.weights)
        else:
            self.g.matmul(a, w, out, epilogue=epilogue, weights=self.weights)


class DecoderGraph:
    """Node list of the decoder forward for one rank; weights are bf16 bit patterns.

    With ``chunks > 1`` the batch is cut into that many micro-batches (whole sequences, so
    attention stays local to a chunk).  Each chunk runs the same nodes on its own rows, and
    the two allreduces of a chunk are put on the executor's side stream: while chunk c is
    being summed over NVLink, the tensor cores work on chunk c+1.
    """

    def __init__(self, ctx, cfg: DecoderConfig, world: int, rank: int, layers: List[Dict[str, np.ndarray]],
                 algo: int = _capi.HB_AR_AUTO, chunks: int = 1, fused: bool = False, gathered: bool = False,
                 fused_form: int = 0, fused_ctas: int = 0, share=None, e4m3: bool = False):
        """`e4m3`: weights and the inputs of their products in 8 bits (``Context.matmul_scaled``), one rank
        only; attention, the residual stream and the outputs of the products stay bf16.  `fused_form` / `fused_ctas`: kernel form of the fused collective for this graph's runs
        (``Context.comm_configure``).  `share`: another DecoderGraph of the same rank whose uploaded
        weights and input buffer this one reuses (schedule variants of one model)."""
        from .graph import Graph
        check_shardable(cfg, world)
        if e4m3 and world > 1:
            raise ValueError("e4m3 weights are supported on one rank")
        if share is not None and bool(e4m3) != share.e4m3:
            raise ValueError("a graph shares weights only with one of the same precision")
        self.e4m3 = bool(e4m3)
        self._out_id = None
        self.fused_form, self.fused_ctas, self._share = fused_form, fused_ctas, share
        self.schedule = {"chunks": chunks, "fused": bool(fused and world > 1), "gathered": bool(gathered and world > 1),
                         "fused_form": fused_form, "fused_ctas": fused_ctas,
                         "collective": {_capi.HB_AR_AUTO: "auto", _capi.HB_AR_NCCL: "nccl", _capi.HB_AR_P2P: "p2p",
                                        _capi.HB_AR_NVLS: "nvls"}.get(algo, str(algo))}
        if fused and world > 1:
            self._build_fused(ctx, cfg, world, rank, layers, algo, chunks, gathered)
            return
        if cfg.batch % chunks:
            raise ValueError(f"batch {cfg.batch} does not split into {chunks} chunks")
        self.ctx, self.cfg, self.world, self.rank, self.chunks = ctx, cfg, world, rank, chunks
        T, d, hd = cfg.tokens, cfg.d_model, cfg.head_dim
        ql, kl, fl = cfg.n_q_heads // world, cfg.n_kv_heads // world, cfg.ffn_hidden // world
        W = (ql + 2 * kl) * hd
        Bc = cfg.batch // chunks            # sequences per chunk
        Tc = Bc * cfg.seq                   # tokens per chunk
        side = 1 if (chunks > 1 and world > 1) else 0
        g = self.graph = Graph(ctx)
        self.x0 = share.x0 if share is not None else ctx.empty((T, d))
        self._out = ctx.empty((T, d))
        x0, out = g.input(self.x0), g.input(self._out)
        rows = lambda t, c: g.view(t, c * Tc * d, (Tc, d), (d, 1))       # chunk c of a [T, d] tensor
        self.weights = []
        ops = _Products(g, e4m3, cfg.eps, weights=False)
        x = None                                  # residual stream [T, d], planner-owned after layer 0
        pending = [None] * chunks                 # per chunk: sublayer output not yet added into the stream
        for li, lw in enumerate(layers):
            dev = share.weights[li] if share is not None else upload_layer(ctx, lw, e4m3)
            self.weights.append(dev)
            w = {k: g.input(v) if k in ("g1", "g2") else ops.weight(v) for k, v in dev.items()}
            first = x is None
            if first:
                x = g.temp((T, d))
            # ---- attention sublayer, chunk by chunk
            aos = []
            for c in range(chunks):
                if first:
                    h = ops.norm(rows(x0, c), w["g1"], Tc, d)
                else:
                    h = ops.norm(pending[c], w["g1"], Tc, d, residual=rows(x, c))
                qkv = g.temp((Tc, W))
                ops.matmul(h, w["wqkv"], qkv)
                g.rope(g.view(qkv, 0, (Tc, ql * hd), (W, 1)), cfg.seq, ql, hd, cfg.rope_base)
                g.rope(g.view(qkv, ql * hd, (Tc, kl * hd), (W, 1)), cfg.seq, kl, hd, cfg.rope_base)
                v4 = lambda off, H: g.view(qkv, off, (Bc, cfg.seq, H, hd), (cfg.seq * W, W, hd, 1))
                attn = g.temp((Tc, ql * hd))
                g.attention(v4(0, ql), v4(ql * hd, kl), v4((ql + kl) * hd, kl),
                            g.view(attn, 0, (Bc, cfg.seq, ql, hd), (cfg.seq * ql * hd, ql * hd, hd, 1)), causal=True)
                ao = g.temp((Tc, d), symmetric=True)
                ops.matmul(ops.operand(attn, Tc, ql * hd), w["wo"], ao)
                g.all_reduce(ao, algo, stream=side)
                aos.append(ao)
            # ---- FFN sublayer, chunk by chunk
            for c in range(chunks):
                if first:
                    g.add(rows(x0, c), aos[c], rows(x, c))
                    h2 = ops.norm(rows(x, c), w["g2"], Tc, d)
                else:
                    h2 = ops.norm(aos[c], w["g2"], Tc, d, residual=rows(x, c))
                act = g.temp((Tc, fl))
                ops.matmul(h2, w["wgu"], act, epilogue=_capi.HB_EPI_SWIGLU)
                fo = g.temp((Tc, d), symmetric=True)
                ops.matmul(ops.operand(act, Tc, fl), w["wd"], fo)
                g.all_reduce(fo, algo, stream=side)
                pending[c] = fo
        for c in range(chunks):
            g.add(rows(x, c), pending[c], rows(out, c))
        self.symmetric_needed = None

    def _build_fused(self, ctx, cfg, world, rank, layers, algo, chunks=1, gathered=False):
        """Sequence-parallel form: each allreduce + residual add + RMSNorm becomes one fused
        node (reduce-scatter, add and norm on this rank's rows, all-gather of the normalised
        rows); the residual stream is sharded by rows and gathered once at the end.

        With ``chunks > 1`` the token rows are cut into that many row blocks and every
        row-parallel product, its fused collective and the column-parallel product that
        consumes the gathered rows run block by block: the collective of block c goes to the
        executor's side stream and crosses NVLink while the tensor cores work on block c+1
        (and, later, on the consumer of block c).  A rank owns rows/world rows of EVERY block,
        so the sharding of the residual stream is the same in all collectives.  The values do
        not depend on ``chunks``: every output row is computed by the same arithmetic.

        With ``gathered`` (one row block only) the fused collectives go to the side stream and
        the column-parallel product that consumes their gathered rows is not ordered behind them
        by an event: it waits block by block for the "rows ready" words the collective publishes
        and starts with this rank's own rows, so the all-gather runs under the product."""
        from .graph import Graph
        if gathered and chunks != 1:
            raise ValueError("gathered products take the whole gathered tensor: chunks must be 1")
        if cfg.tokens % (world * chunks):
            raise ValueError("tokens must split evenly over the ranks and row blocks")
        self.ctx, self.cfg, self.world, self.rank, self.chunks = ctx, cfg, world, rank, chunks
        T, d, hd = cfg.tokens, cfg.d_model, cfg.head_dim
        ql, kl, fl = cfg.n_q_heads // world, cfg.n_kv_heads // world, cfg.ffn_hidden // world
        W = (ql + 2 * kl) * hd
        Tc = T // chunks
        side = 1 if (chunks > 1 or gathered) else 0
        g = self.graph = Graph(ctx)
        share = self._share
        self.x0 = share.x0 if share is not None else ctx.empty((T, d))
        x0 = g.input(self.x0)
        self.weights = share.weights if share is not None else [{k: ctx.upload(v) for k, v in lw.items()} for lw in layers]
        ws = [{k: g.input(v if k in ("g1", "g2") else v.T) for k, v in dev.items()} for dev in self.weights]
        rows = lambda t, c, n: g.view(t, c * Tc * n, (Tc, n), (n, 1)) if chunks > 1 else t   # row block c of a [T, n] tensor
        x = g.temp((T, d))                          # residual stream: only this rank's rows of each block are live
        h = g.temp((T, d))
        g.rmsnorm(x0, ws[0]["g1"], h, eps=cfg.eps)
        # The four exchange buffers are allocated once and reused by every layer: the planner
        # packs by position in the node list, and a buffer that it placed over another one still
        # being read on the side stream would make the executor serialise the two streams.
        ao, h2, fo, nxt = (g.temp((T, d), symmetric=True) for _ in range(4))
        for li, w in enumerate(ws):
            qkv = g.temp((T, W))
            attn = g.temp((T, ql * hd))
            # When a row block is a whole number of sequences, its QKV product, RoPE and attention
            # form a chain of their own: block 0's chain runs while the previous layer's last
            # collective is still gathering block 1.  Otherwise RoPE and attention take all rows.
            per_block = chunks > 1 and Tc % cfg.seq == 0
            xin = x0 if li == 0 else x

            def attention_out(c):
                g.matmul(rows(attn, c, ql * hd), w["wo"], rows(ao, c, d))
                g.all_reduce_norm(rows(ao, c, d), w["g2"], rows(xin, c, d), rows(x, c, d), rows(h2, c, d), eps=cfg.eps,
                                  algo=algo, stream=side, ready_words=gathered)
            for c in range(chunks):                 # block c starts as soon as its gathered rows have landed
                g.matmul(rows(h, c, d), w["wqkv"], rows(qkv, c, W), gathered=gathered and li > 0)
                if per_block:
                    # the whole attention sublayer of block c, so that its collective runs under the
                    # QKV product, RoPE, attention and output product of block c+1
                    r0, Bc = c * Tc, Tc // cfg.seq
                    g.rope(g.view(qkv, r0 * W, (Tc, ql * hd), (W, 1)), cfg.seq, ql, hd, cfg.rope_base)
                    g.rope(g.view(qkv, r0 * W + ql * hd, (Tc, kl * hd), (W, 1)), cfg.seq, kl, hd, cfg.rope_base)
                    v4 = lambda off, H: g.view(qkv, r0 * W + off, (Bc, cfg.seq, H, hd), (cfg.seq * W, W, hd, 1))
                    g.attention(v4(0, ql), v4(ql * hd, kl), v4((ql + kl) * hd, kl),
                                g.view(attn, r0 * ql * hd, (Bc, cfg.seq, ql, hd), (cfg.seq * ql * hd, ql * hd, hd, 1)),
                                causal=True)
                    attention_out(c)
            if not per_block:
                g.rope(g.view(qkv, 0, (T, ql * hd), (W, 1)), cfg.seq, ql, hd, cfg.rope_base)
                g.rope(g.view(qkv, ql * hd, (T, kl * hd), (W, 1)), cfg.seq, kl, hd, cfg.rope_base)
                v4 = lambda off, H: g.view(qkv, off, (cfg.batch, cfg.seq, H, hd), (cfg.seq * W, W, hd, 1))
                g.attention(v4(0, ql), v4(ql * hd, kl), v4((ql + kl) * hd, kl),
                            g.view(attn, 0, (cfg.batch, cfg.seq, ql, hd), (cfg.seq * ql * hd, ql * hd, hd, 1)), causal=True)
                for c in range(chunks):
                    attention_out(c)
            act = g.temp((T, fl))
            last = li + 1 == len(ws)
            for c in range(chunks):
                g.matmul(rows(h2, c, d), w["wgu"], rows(act, c, fl), epilogue=_capi.HB_EPI_SWIGLU, gathered=gathered)
                g.matmul(rows(act, c, fl), w["wd"], rows(fo, c, d))
                g.all_reduce_norm(rows(fo, c, d), None if last else ws[li + 1]["g1"], rows(x, c, d), rows(x, c, d),
                                  rows(nxt, c, d), eps=cfg.eps, gather_only=last, algo=algo, stream=side,
                                  ready_words=gathered and not last)
            if last:
                self._out_id = nxt
            else:
                h = nxt
        self.symmetric_needed = None

    @property
    def out(self):
        """The output tensor [tokens, d_model] (valid after plan())."""
        if self._out_id is not None:
            return self.graph.tensor(self._out_id)
        return self._out

    def plan(self):
        arena, sym = self.graph.plan()
        self.symmetric_needed = sym
        return arena, sym

    def run(self):
        if self.world > 1:
            self.ctx.comm_configure(self.fused_form, self.fused_ctas)
        self.graph.run()


# Schedules of the tensor-parallel block worth timing on a given box: how the fused collectives
# overlap the products around them.  Which one wins depends on the rank count (at 2 GPUs the
# collectives are a quarter of the step, at 8 more than half) and on the NVLink fabric.
#   - one row block, collectives on the main stream (nothing overlaps; fastest collective kernel);
#   - two row blocks: the collective of block c on the side stream under the products of block c+1
#     (warp-per-row form, few CTAs, beside the GEMM on the same SMs);
#   - one row block, gathered products: the column-parallel product after each collective waits
#     for its rows block by block and runs under the all-gather.
def candidate_schedules(world: int, gathered: bool = False):
    """`gathered` adds the gathered-product schedules (measured slower than two row blocks at 2
    GPUs: 3.73 against 3.29 ms; not measured on more)."""
    if world <= 1:
        return [dict(chunks=1, fused=False)]
    out = [dict(chunks=1, fused=True, fused_form=1),
           dict(chunks=2, fused=True, fused_form=2, fused_ctas=64),
           dict(chunks=2, fused=True, fused_form=2, fused_ctas=128),
           dict(chunks=2, fused=True, fused_form=1)]
    # (Plain peer loads and stores instead of the in-switch reduction move fewer bytes per link on
    # two ranks -- 153 against 203 us for one exchange -- but the whole step was not faster with
    # them: 3.41 against 3.35 ms; pass algo=HB_AR_P2P to DecoderGraph to use them.)
    if gathered:
        out += [dict(chunks=1, fused=True, gathered=True, fused_form=2, fused_ctas=128),
                dict(chunks=1, fused=True, gathered=True, fused_form=2, fused_ctas=64)]
    return out


def pick_schedule(graphs, measure):
    """Times every candidate graph with `measure(run) -> ms` (the caller's device timer; with
    several ranks it must return the same number on all of them, e.g. the maximum) and returns
    (index of the fastest, all timings)."""
    times = [float(measure(g.run)) for g in graphs]
    return int(np.argmin(times)), times


def decode_layer(full: Dict[str, np.ndarray], cfg: DecoderConfig) -> Dict[str, np.ndarray]:
    """One layer's weights in the form the decode graph wants (single rank): wqkv
    [(Hq+2Hkv)*hd, d], wo [d, Hq*hd], wgu [2F, d] with the F gate rows first and the F up rows
    second (the stand-alone SwiGLU kernel reads the two halves), wd [d, F], and the gains."""
    return {"wqkv": np.ascontiguousarray(np.concatenate([full["wq"], full["wk"], full["wv"]], 0)),
            "wo": np.ascontiguousarray(full["wo"]), "wgu": np.ascontiguousarray(np.concatenate([full["wg"], full["wu"]], 0)),
            "wd": np.ascontiguousarray(full["wd"]), "g1": full["g1"], "g2": full["g2"]}


class DecodeGraph:
    """One generation step of the decoder block for `batch` sequences on one GPU: the new
    token's embedding in, its output row out, key/value caches of `s_max` positions per layer.
    The projections are M = batch products (the stream-K kernel for M <= 64), attention is the
    split-KV single-query kernel, and the position is a device-side counter that the last node
    advances, so every step enqueues exactly the same launches (``advance=False`` keeps the
    position fixed: the benchmark's steady-state step)."""

    def __init__(self, ctx, cfg: DecoderConfig, layers: List[Dict[str, np.ndarray]], batch: int, s_max: int,
                 advance: bool = True, len_hint: int = 0, e4m3: bool = False):
        """`e4m3`: weights and the inputs of their products in 8 bits (``Context.matmul_scaled``), which
        halves the weight bytes of a step; the caches, attention and the residual stream stay bf16."""
        from .graph import Graph
        self.ctx, self.cfg, self.batch, self.s_max, self.e4m3 = ctx, cfg, batch, s_max, bool(e4m3)
        d, hd, Hq, Hkv, F = cfg.d_model, cfg.head_dim, cfg.n_q_heads, cfg.n_kv_heads, cfg.ffn_hidden
        W = (Hq + 2 * Hkv) * hd
        B = batch
        g = self.graph = Graph(ctx)
        self.x = ctx.empty((B, d))
        self.out = ctx.empty((B, d))
        self.pos = ctx.upload(np.zeros(1, np.int32))
        self.kv = [ctx.empty((2 * B, s_max, Hkv, hd)) for _ in layers]
        x_in, out, pos = g.input(self.x), g.input(self.out), g.input(self.pos)
        self.weights = [upload_layer(ctx, lw, e4m3) for lw in layers]
        ops = _Products(g, e4m3, cfg.eps, weights=True)
        ws = [{k: g.input(v) if k in ("g1", "g2") else ops.weight(v) for k, v in dev.items()} for dev in self.weights]
        xres = g.temp((B, d))                 # residual stream
        pending = None                        # sublayer output not yet added into the stream
        for li, w in enumerate(ws):
            kv = g.input(self.kv[li])
            if li == 0:
                h = ops.norm(x_in, w["g1"], B, d)
            else:
                h = ops.norm(pending, w["g1"], B, d, residual=xres)
            qkv = g.temp((B, W))
            ops.matmul(h, w["wqkv"], qkv)
            g.rope_append(qkv, pos, kv, Hq, Hkv, cfg.rope_base)
            attn = g.temp((B, Hq * hd))
            g.attention_decode(qkv, kv, pos, attn, Hq, Hkv, len_hint=len_hint)
            ao = g.temp((B, d))
            ops.matmul(ops.operand(attn, B, Hq * hd), w["wo"], ao)
            if li == 0:
                g.add(x_in, ao, xres)
                h2 = ops.norm(xres, w["g2"], B, d)
            else:
                h2 = ops.norm(ao, w["g2"], B, d, residual=xres)
            gu = g.temp((B, 2 * F))
            ops.matmul(h2, w["wgu"], gu)
            act = ops.swiglu(gu, B, F)
            fo = g.temp((B, d))
            ops.matmul(act, w["wd"], fo)
            pending = fo
        g.add(xres, pending, out)
        if advance:
            g.advance(pos, 1)
        self.arena, _ = g.plan()
        self.captured = False

    def set_pos(self, pos: int):
        import ctypes as C
        from .model_ir import _lib
        a = np.array([pos], np.int32)
        self.ctx._check(_lib.hb_upload(self.ctx._h, C.c_void_p(self.pos.ptr), a.ctypes.data_as(C.c_void_p), 4))
        self.ctx.sync()

    def step(self):
        if self.captured:
            self.graph.replay()
        else:
            self.graph.run()

    def capture(self):
        """Replay from now on: one eager step first (it sizes the scratch buffers and, like any
        step, advances the position), then the capture."""
        self.graph.run()
        self.ctx.sync()
        self.graph.capture()
        self.captured = True

    def bytes_per_step(self, length: int) -> float:
        """Algorithmic HBM bytes of one step at cache length `length`: every weight once, the
        cached keys and values of every layer once."""
        cfg = self.cfg
        w = sum(t.nbytes for dev in self.weights for v in dev.values() for t in (v if isinstance(v, tuple) else (v,)))
        kvb = len(self.kv) * 2.0 * self.batch * length * cfg.n_kv_heads * cfg.head_dim * 2
        return w + kvb

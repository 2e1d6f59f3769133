"""Cases of the 8-bit path: RMSNorm with the residual's addition, SwiGLU and plain quantisation to e4m3 with one
scale per 128 values, and the matrix product of two such operands.

Each case can be run two ways.  With ``own`` false, ``run`` is the plain form: elementary torch operations in 32
bits, rounded once at the end.  With ``own`` true it makes the calls a user makes of ``habu_b200.Context``.
``exact`` restates every operator in 64 bits from its definition:

    scale  s = max(max|y| / 448, 2^-126) over 128 consecutive values of a row (or a 128 x 128 block)
    value  q = e4m3(y / s), to nearest, ties to even
    norm   y = x * rsqrt(mean(x^2) + eps) * gain, after residual <- bf16(residual + x) where there is one
    swiglu y = silu(x[:, :half]) * x[:, half:]
    matmul c = bf16(epilogue(sum over 128-wide k-blocks of sa * sb * sum(qa * qb)))
"""
import math

import torch

own = False

G = 128                 # values per scale
TOP = 448.0             # largest e4m3 value
FLOOR = 2.0 ** -126     # smallest scale
EPS = 1e-5


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one generation step of 16 sequences: latency
        {"name": "norm 16x4096 step", "op": "norm", "rows": 16, "cols": 4096, "residual": True},
        # the residual stream of a 4 x 2048-token prompt
        {"name": "norm 8192x4096 prompt", "op": "norm", "rows": 8192, "cols": 4096, "residual": True},
        # a ragged batch and a width that ends inside a group of 128; the first norm of a model has no residual
        {"name": "norm 777x2056 ragged", "op": "norm", "rows": 777, "cols": 2056, "residual": False},
        # attention outputs of a prompt before the output projection
        {"name": "quant 8192x4096 rows", "op": "quant", "rows": 8192, "cols": 4096, "block": 1, "dtype": "bf16"},
        # the gate/up weights of one layer, laid out once from fp32 masters
        {"name": "quant 28672x4096 blocks", "op": "quant", "rows": 28672, "cols": 4096, "block": 128, "dtype": "f32"},
        # the feed-forward activation of a generation step and of a prompt
        {"name": "swiglu 16x14336 step", "op": "swiglu", "rows": 16, "half": 14336},
        {"name": "swiglu 8192x14336 prompt", "op": "swiglu", "rows": 8192, "half": 14336},
        # one token through the QKV projection: the smallest product
        {"name": "matmul 1x6144x4096", "op": "matmul", "m": 1, "n": 6144, "k": 4096, "epilogue": "none"},
        # 16 sequences through the gate/up projection: bound by reading the weights
        {"name": "matmul 16x28672x4096", "op": "matmul", "m": 16, "n": 28672, "k": 4096, "epilogue": "none"},
        # a ragged batch; N and K end inside a block, the output adds the residual stream
        {"name": "matmul 333x1000x2056 ragged", "op": "matmul", "m": 333, "n": 1000, "k": 2056, "epilogue": "residual"},
        # a prompt through the down projection
        {"name": "matmul 8192x4096x14336", "op": "matmul", "m": 8192, "n": 4096, "k": 14336, "epilogue": "none"},
        # a prompt through the gate/up projection, SwiGLU in the epilogue: the largest product
        {"name": "matmul 8192x28672x4096 swiglu", "op": "matmul", "m": 8192, "n": 28672, "k": 4096, "epilogue": "swiglu"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "quant", "swiglu", "matmul", "matmul"])
    if op == "norm":
        return {"op": op, "rows": _log(rng, 1, 16384), "cols": 8 * _log(rng, 8, 2048), "residual": rng.random() < 0.7}
    if op == "quant":
        return {"op": op, "rows": _log(rng, 1, 16384), "cols": _log(rng, 32, 16384), "block": rng.choice([1, 128]),
                "dtype": rng.choice(["bf16", "f32"])}
    if op == "swiglu":
        return {"op": op, "rows": _log(rng, 1, 8192), "half": 8 * _log(rng, 8, 1792)}
    epilogue = rng.choice(["none", "none", "residual", "gelu", "swiglu"])
    n = _log(rng, 64, 28672)
    return {"op": op, "m": _log(rng, 1, 8192), "n": n + (n & 1 if epilogue == "swiglu" else 0), "k": _log(rng, 64, 14336) if rng.random() < 0.5
            else 128 * _log(rng, 1, 112), "epilogue": epilogue}


# ---------------------------------------------------------------- inputs
def _blocks(n, b):
    return -(-n // b)


def _wide(v, n, dim):
    """One value per group of 128 along `dim` -> one per element, cut to n."""
    return v.repeat_interleave(G, dim).narrow(dim, 0, n)


def _pack(y, block):
    """(q as e4m3 in rows padded to 16 bytes, scales) of fp32 values: operands for the product."""
    rows, cols = y.shape
    rb, cb = _blocks(rows, block), _blocks(cols, G)
    p = torch.zeros(rb * block, cb * G, device=y.device)
    p[:rows, :cols] = y
    s = (p.view(rb, block, cb, G).abs().amax((1, 3)) / TOP).clamp_min(FLOOR)
    q = torch.zeros(rows, _blocks(cols, 16) * 16, dtype=torch.float8_e4m3fn, device=y.device)
    full = (p.view(rb, block, cb, G) / s[:, None, :, None]).view(rb * block, cb * G)[:rows, :cols]
    q[:, :cols] = full.clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return q[:, :cols], s


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    def activations(rows, cols):
        """Normal values with a few strong channels, as a residual stream has."""
        x = normal(rows, cols)
        strong = torch.rand(cols, generator=gen, device=dev) < 0.01
        return x.mul_(torch.where(strong, 12.0, 1.0))

    def empty_q(rows, cols):
        return torch.empty(rows, _blocks(cols, 16) * 16, dtype=torch.float8_e4m3fn, device=dev)[:, :cols]

    st = {"case": case}
    op = case["op"]
    if op == "norm":
        rows, cols = case["rows"], case["cols"]
        st["x"] = activations(rows, cols).bfloat16()
        st["gain"] = (1 + 0.1 * normal(cols)).bfloat16()
        st["residual"] = activations(rows, cols).mul_(2).bfloat16() if case["residual"] else None
        st["q"], st["scale"] = empty_q(rows, cols), torch.empty(rows, _blocks(cols, G), device=dev)
    elif op == "quant":
        rows, cols, block = case["rows"], case["cols"], case["block"]
        x = activations(rows, cols) if block == 1 else normal(rows, cols).mul_(cols ** -0.5)
        st["x"] = x.bfloat16() if case["dtype"] == "bf16" else x
        st["q"], st["scale"] = empty_q(rows, cols), torch.empty(_blocks(rows, block), _blocks(cols, G), device=dev)
    elif op == "swiglu":
        rows, half = case["rows"], case["half"]
        st["x"] = normal(rows, 2 * half).mul_(1.5).bfloat16()
        st["q"], st["scale"] = empty_q(rows, half), torch.empty(rows, _blocks(half, G), device=dev)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        st["a"], st["sa"] = _pack(activations(m, k), 1)
        st["b"], st["sb"] = _pack(normal(n, k).mul_(k ** -0.5), G)
        st["residual"] = normal(m, n).bfloat16() if case["epilogue"] == "residual" else None
        st["c"] = torch.empty(m, n // 2 if case["epilogue"] == "swiglu" else n, dtype=torch.bfloat16, device=dev)
    return st


# ---------------------------------------------------------------- the calls of a user's program
_ctx = None


def _views(st):
    """The state's buffers as the framework's tensors, made once as a program does that keeps its buffers."""
    global _ctx
    import habu_b200 as hb
    if _ctx is None:
        _ctx = hb.Context(torch.cuda.current_device())
    kinds = {torch.bfloat16: hb.HB_BF16, torch.float32: hb.HB_F32, torch.float8_e4m3fn: hb.HB_E4M3}
    v = {k: _ctx.wrap(t.data_ptr(), t.shape, kinds[t.dtype], t.stride(), t) for k, t in st.items() if torch.is_tensor(t)}
    for k in ("b", "sb"):                       # weights are kept [out, in]: the product takes [in, out]
        if k in v:
            v[k] = v[k].T
    st["views"] = v
    if "c" in v:
        st["epilogue"] = {"none": hb.HB_EPI_NONE, "gelu": hb.HB_EPI_GELU, "swiglu": hb.HB_EPI_SWIGLU,
                          "residual": hb.HB_EPI_RESIDUAL}[st["case"]["epilogue"]]
    return v


def _run_own(st):
    v = st.get("views") or _views(st)
    op = st["case"]["op"]
    if op == "norm":
        _ctx.rmsnorm_quant(v["x"], v["gain"], v["q"], v["scale"], EPS, v.get("residual"))
        return {"q": st["q"], "scale": st["scale"], "residual": st["residual"]}
    if op == "quant":
        _ctx.quantize(v["x"], v["q"], v["scale"], st["case"]["block"])
        return {"q": st["q"], "scale": st["scale"]}
    if op == "swiglu":
        _ctx.swiglu_quant(v["x"], v["q"], v["scale"])
        return {"q": st["q"], "scale": st["scale"]}
    _ctx.matmul_scaled(v["a"], v["sa"], v["b"], v["sb"], v["c"], st["epilogue"], v.get("residual"), weights=True)
    return {"c": st["c"]}


# ---------------------------------------------------------------- the plain form
def _plain_quant(y, block):
    rows, cols = y.shape
    rb, cb = _blocks(rows, block), _blocks(cols, G)
    p = y
    if rb * block != rows or cb * G != cols:
        p = torch.zeros(rb * block, cb * G, device=y.device)
        p[:rows, :cols] = y
    p = p.view(rb, block, cb, G)
    s = (p.abs().amax((1, 3)) / TOP).clamp_min(FLOOR)
    q = (p / s[:, None, :, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return q.view(rb * block, cb * G)[:rows, :cols], s


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    if op == "norm":
        x = st["x"].float()
        if st["residual"] is not None:
            st["residual"].copy_(st["residual"].float() + x)
            x = st["residual"].float()
        y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * st["gain"].float()
        q, s = _plain_quant(y, 1)
        return {"q": q, "scale": s, "residual": st["residual"]}
    if op == "quant":
        q, s = _plain_quant(st["x"].float(), case["block"])
        return {"q": q, "scale": s}
    if op == "swiglu":
        x = st["x"].float()
        g, u = x[:, :case["half"]], x[:, case["half"]:]
        q, s = _plain_quant(g / (1 + torch.exp(-g)) * u, 1)
        return {"q": q, "scale": s}
    m, n, k = case["m"], case["n"], case["k"]
    a = st["a"].float() * _wide(st["sa"], k, 1)
    b = st["b"].float() * _wide(_wide(st["sb"], n, 0), k, 1)
    c = a @ b.t()
    if case["epilogue"] == "gelu":
        c = 0.5 * c * (1 + torch.erf(c * 0.5 ** 0.5))
    elif case["epilogue"] == "swiglu":          # columns interleave (gate, up)
        g, u = c[:, 0::2], c[:, 1::2]
        c = g / (1 + torch.exp(-g)) * u
    elif case["epilogue"] == "residual":
        c = c + st["residual"].float()
    return {"c": c.bfloat16()}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "norm":
        n = case["rows"] * case["cols"]
        groups = case["rows"] * _blocks(case["cols"], G)
        return {"bytes": n * (2 + 1 + (4 if case["residual"] else 0)) + 4 * groups + 2 * case["cols"], "flops": 6 * n}
    if op == "quant":
        n = case["rows"] * case["cols"]
        groups = _blocks(case["rows"], case["block"]) * _blocks(case["cols"], G)
        return {"bytes": n * ((2 if case["dtype"] == "bf16" else 4) + 1) + 4 * groups, "flops": 2 * n}
    if op == "swiglu":
        n = case["rows"] * case["half"]
        return {"bytes": 5 * n + 4 * case["rows"] * _blocks(case["half"], G), "flops": 6 * n}
    m, n, k = case["m"], case["n"], case["k"]
    out = n // 2 if case["epilogue"] == "swiglu" else n
    nbytes = m * k + n * k + 4 * _blocks(k, G) * (m + _blocks(n, G)) + 2 * m * out
    return {"bytes": nbytes + (2 * m * n if case["epilogue"] == "residual" else 0), "flops": 2 * m * n * k}


# ---------------------------------------------------------------- the definition in 64 bits
def _e4m3(v):
    """Nearest e4m3 value of each 64-bit value, ties to even, as a 64-bit value."""
    a = v.abs()
    step = torch.ldexp(torch.ones_like(a), (torch.frexp(a).exponent - 1).clamp_min(-6) - 3)
    return torch.copysign((torch.round(a / step) * step).clamp_max(TOP), v)


def _exact_quant(y, block):
    rows, cols = y.shape
    q = torch.empty_like(y)
    s = torch.empty(_blocks(rows, block), _blocks(cols, G), dtype=torch.float64, device=y.device)
    for j in range(_blocks(cols, G)):
        part = y[:, j * G:(j + 1) * G]
        top = part.abs().amax(1)
        if block > 1:
            top = torch.cat([top, top.new_zeros(-rows % block)]).view(-1, block).amax(1)
        s[:, j] = (top / TOP).clamp_min(FLOOR)
        q[:, j * G:(j + 1) * G] = _e4m3(part / s[:, j].repeat_interleave(block)[:rows, None])
    return q, s


def _silu(v):
    return v * torch.sigmoid(v)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        x, residual = st["x"].double(), st["residual"]
        if residual is not None:
            residual = (residual.double() + x).bfloat16()      # the sum of two bf16 values, stored in bf16
            x = residual.double()
        y = x / (x.square().mean(1, keepdim=True) + EPS).sqrt() * st["gain"].double()
        q, s = _exact_quant(y, 1)
        return {"q": q, "scale": s, "residual": residual}
    if op == "quant":
        q, s = _exact_quant(st["x"].double(), case["block"])
        return {"q": q, "scale": s}
    if op == "swiglu":
        gate, up = st["x"].double().chunk(2, 1)
        q, s = _exact_quant(_silu(gate) * up, 1)
        return {"q": q, "scale": s}
    m, n, k = case["m"], case["n"], case["k"]
    c = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    for j in range(_blocks(k, G)):
        part = st["a"][:, j * G:(j + 1) * G].double() @ st["b"][:, j * G:(j + 1) * G].double().t()
        c.addcmul_(part.mul_(st["sa"][:, j, None].double()), st["sb"][:, j].double().repeat_interleave(G)[None, :n])
    if case["epilogue"] == "gelu":
        c = c * 0.5 * torch.special.erfc(-c / math.sqrt(2.0))
    elif case["epilogue"] == "swiglu":
        c = _silu(c.view(m, n // 2, 2)[..., 0]) * c.view(m, n // 2, 2)[..., 1]
    elif case["epilogue"] == "residual":
        c = c + st["residual"].double()
    return {"c": c}

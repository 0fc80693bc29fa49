"""Operators of 8-bit inference: products of 8-bit integers with a scale for each token and each channel (dense, with a gated activation, and
grouped by expert), and the norms on both sides of a sublayer fused with its gate and its residual scale, whose rows the products read.

A row x of K entries becomes q = round(127 x / max|x|), ties to the even one, and the scale max|x| / 127; a weight matrix holds such rows, one
an output channel.  The product is the sum of q_x q_w over k, whole numbers, times the token's scale, times the channel's.  Gate and up rows
of a gated product alternate in groups of 16.  The plain form forms the same in elementary torch operations; `exact` does it in 64 bits.
"""
import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TYPES = {"bfloat16": BF16, "float32": F32}
EPS = 1e-5
LIMIT, SLOPE = 7.0, 1.702            # of the clamped gated activation
ACTS = ("silu", "gelu_tanh", "clamped")
HEAVIEST = 2048 * 28672 * 4096       # multiply-adds of the largest listed case


def _linear(name, tokens, k, n, out="bfloat16", pad=0, glu=""):
    """`pad`: the rows are a column slice of a tensor that is so much wider; `glu`: a gate/up product of n rows, n / 2 features out."""
    c = {"kind": "linear", "tokens": tokens, "k": k, "n": n, "out": out, "pad": pad, "glu": glu}
    return {"name": name, **c} if name else c


def _experts(name, direction, tokens, width, ff, experts, top, glu="silu"):
    c = {"kind": "experts", "direction": direction, "tokens": tokens, "width": width, "ff": ff, "experts": experts, "top": top, "glu": glu}
    return {"name": name, **c} if name else c


def _norm(name, tokens, width, post=True, gate="float32", scale=True, y="bfloat16", rows="bfloat16"):
    c = {"kind": "norm", "tokens": tokens, "width": width, "post": post, "gate": gate, "scale": scale, "y": y, "rows": rows}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one request decodes: the down projection of the 8B decoder
        _linear("down, 1 token", 1, 14336, 4096),
        # eight requests decode: its fused query, key and value projection
        _linear("qkv, 8 tokens", 8, 4096, 6144),
        # eight requests decode: its gate/up product with the activation
        _linear("gate/up, 8 tokens", 8, 4096, 28672, glu="silu"),
        # a short portion whose sizes fill no tile, float32 sums out of a column slice (a small low-rank product)
        _linear("odd sizes, 77 tokens", 77, 1001, 777, out="float32", pad=23),
        # a portion of 512 tokens beside decoded ones: the down projection of the 13B decoder
        _linear("down, 512 tokens", 512, 13824, 5120),
        # a prompt of 2,048 tokens: the 8B decoder's gate/up product
        _linear("gate/up, 2048 tokens", 2048, 4096, 28672, glu="silu"),
        # eight requests decode with routed experts: their gate/up matrices, a few rows an expert
        _experts("experts up, 8 tokens", "up", 8, 2048, 1408, 64, 6),
        # a prompt of 2,048 tokens through the same experts, up and down
        _experts("experts up, 2048 tokens", "up", 2048, 2048, 1408, 64, 6),
        _experts("experts down, 2048 tokens", "down", 2048, 2048, 1408, 64, 6),
        # between two sublayers, eight requests decoding
        _norm("norms, 8 tokens", 8, 4096),
        # between two sublayers, a prompt of 2,048 tokens at the 13B decoder's width
        _norm("norms, 2048 tokens", 2048, 5120, gate="bfloat16"),
        # a feed-forward as a model runs it: norms that leave 8-bit rows, the gate/up product, the down product
        {"name": "feed-forward, 32 tokens", "kind": "layer", "tokens": 32, "width": 4096, "ff": 14336, "glu": "silu"},
    ]


def _log(rng, least, most, step=1):
    v = math.exp(rng.uniform(math.log(least), math.log(most)))
    return max(least, min(most, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(("linear", "linear", "glu", "experts", "experts", "norm", "layer"))
    while True:
        if kind == "linear":
            c = _linear("", _log(rng, 1, 2048), _log(rng, 64, 14336, rng.choice((1, 8, 128))), _log(rng, 48, 28672, rng.choice((1, 16, 128))),
                        rng.choice(("bfloat16", "float32")), rng.choice((0, 0, 1, 8, 64)))
            cost = c["tokens"] * c["k"] * c["n"]
        elif kind == "glu":
            c = _linear("", _log(rng, 1, 2048), _log(rng, 64, 8192, rng.choice((1, 8, 128))), 2 * _log(rng, 32, 14336, 16), "bfloat16",
                        rng.choice((0, 0, 8)), rng.choice(ACTS))
            cost = c["tokens"] * c["k"] * c["n"]
        elif kind == "experts":
            e = rng.randint(4, 64)
            c = _experts("", rng.choice(("up", "down")), _log(rng, 1, 2048), _log(rng, 256, 2048, rng.choice((8, 128))), _log(rng, 64, 1408, 16), e,
                         rng.randint(1, min(e, 8)), rng.choice(ACTS))
            cost = c["tokens"] * c["top"] * c["width"] * 2 * c["ff"]
        elif kind == "norm":
            c = _norm("", _log(rng, 1, 2048), _log(rng, 64, 8192, rng.choice((1, 8, 128))), rng.random() < 0.7, rng.choice(("none", "float32", "bfloat16")),
                      rng.random() < 0.7, rng.choice(("bfloat16", "float32")), rng.choice(("bfloat16", "float32")))
            cost = 0
        else:
            c = {"kind": "layer", "tokens": _log(rng, 1, 512), "width": _log(rng, 256, 4096, 8), "ff": _log(rng, 256, 14336, 16), "glu": rng.choice(ACTS)}
            cost = 3 * c["tokens"] * c["width"] * c["ff"]
        if cost <= HEAVIEST:
            return c


# ------------------------------------------------------------------ inputs

class _Maker:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, std=1.0, mean=0.0, dtype=F32):
        return (torch.randn(shape, generator=self.g, device="cuda", dtype=F32) * std + mean).to(dtype)

    def stream(self, tokens, width, dtype, std=1.0):
        """Rows as a decoder has them: some channels several times as large as the rest, a few tokens small as a whole."""
        x = self.normal(tokens, width, std=std)
        x *= torch.where(torch.rand(width, generator=self.g, device="cuda") < 0.01, 8.0, 1.0)
        x *= torch.where(torch.rand(tokens, 1, generator=self.g, device="cuda") < 0.05, 0.01, 1.0)
        return x.to(dtype)

    def weight(self, *shape):
        """8-bit rows of a normal matrix and their scales."""
        q = torch.empty(shape, device="cuda", dtype=torch.int8)
        for part in (q.split(1) if q.dim() == 3 else (q,)):        # a matrix at a time: the normal numbers need four times its room
            part.copy_((torch.randn(part.shape, generator=self.g, device="cuda", dtype=F32) * 32).round_().clamp_(-127, 127))
        scale = self.normal(*shape[:-1], std=0.2).exp_() * (1.0 / (32 * math.sqrt(shape[-1])))
        return q, scale


def _grouping(m, case):
    """Who goes to which expert, skewed as routers are: the rows in the experts' order."""
    t, e, top = case["tokens"], case["experts"], case["top"]
    logits = m.normal(t, e) + m.normal(e, std=0.5)
    expert, order = logits.topk(top, dim=1).indices.reshape(-1).sort(stable=True)
    counts = torch.bincount(expert, minlength=e)
    first = counts.cumsum(0) - counts
    slot = torch.arange(t * top, device="cuda") - first[expert]
    return {"expert": expert, "slot": slot, "row_token": (order // top).to(torch.int32), "counts": counts.tolist(), "most": int(counts.max())}


def prepare(case, seed):
    m = _Maker(seed)
    s = {"case": case}
    kind = case["kind"]
    if kind == "linear":
        wide = m.stream(case["tokens"], case["k"] + case["pad"], BF16)
        s["x"] = wide[:, case["pad"]:]
        s["w"], s["w_scale"] = m.weight(case["n"], case["k"])
    elif kind == "experts":
        s.update(_grouping(m, case))
        up = case["direction"] == "up"
        rows = case["tokens"] if up else case["tokens"] * case["top"]
        s["x"] = m.stream(rows, case["width"] if up else case["ff"], BF16)
        s["w"], s["w_scale"] = m.weight(case["experts"], *((2 * case["ff"], case["width"]) if up else (case["width"], case["ff"])))
    else:
        t, d = case["tokens"], case["width"]
        layer = kind == "layer"
        gate, scale = ("float32", True) if layer else (case["gate"], case["scale"])
        s["residual"] = m.stream(t, d, F32, std=2.0)
        s["y"] = m.stream(t, d, BF16 if layer else TYPES[case["y"]])
        s["post"] = m.normal(d, std=0.1, mean=1.0) if layer or case["post"] else None
        s["gate"] = m.normal(t, d, dtype=TYPES[gate]) if gate != "none" else None
        s["bias"] = m.normal(d, std=0.5) if gate != "none" else None
        s["scale"] = m.normal(d, std=0.1, mean=0.7) if scale else None
        s["next"] = m.normal(d, std=0.1, mean=1.0)
        if layer:
            s["w"], s["w_scale"] = m.weight(2 * case["ff"], d)
            s["w2"], s["w2_scale"] = m.weight(d, case["ff"])
    if own:
        from qorvix_b200.csrc import ops
        if "w" in s:                       # laid out for the kernels, as a program does when it loads a model
            s["weight"] = ops.pack_int8(s["w"], s["w_scale"])
        if "w2" in s:
            s["weight2"] = ops.pack_int8(s["w2"], s["w2_scale"])
        if kind == "experts":
            s["tile_rows"] = ops.moe_int8_tile_rows(case["tokens"] * case["top"], case["experts"])
            s["tiles"] = _tile_table(s["counts"], s["tile_rows"], ops.moe_max_tiles(case["tokens"] * case["top"], case["experts"], s["tile_rows"]))
    return s


def _tile_table(counts, tile_rows, tiles):
    """(expert, first row, rows) of each tile of grouped rows, as the framework's grouping lists them."""
    table, first = [], 0
    for e, n in enumerate(counts):
        table += [(e, first + r, min(tile_rows, n - r)) for r in range(0, n, tile_rows)]
        first += n
    table += [(-1, 0, 0)] * (tiles - len(table))
    return torch.tensor(table, dtype=torch.int32, device="cuda").reshape(-1)


# ------------------------------------------------------------------ one pass

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from qorvix_b200.csrc import ops
    case = s["case"]
    kind = case["kind"]
    acts = {"silu": ops.GLU_SILU, "gelu_tanh": ops.GLU_GELU_TANH, "clamped": ops.GLU_CLAMPED}
    if kind == "linear":
        out = torch.empty((case["tokens"], case["n"] // 2 if case["glu"] else case["n"]), device="cuda", dtype=TYPES[case["out"]])
        if case["glu"]:
            ops.gemm_int8_glu(out, s["x"], s["weight"], acts[case["glu"]], LIMIT, SLOPE)
        else:
            ops.gemm_int8(out, s["x"], s["weight"])
        return out
    if kind == "experts":
        up = case["direction"] == "up"
        n = case["tokens"] * case["top"]
        rows = ops.int8_rows(n, s["x"].shape[1], s["x"].device)
        ops.quantize_rows(rows, s["x"], row_idx=s["row_token"] if up else None)
        out = torch.empty((n, case["ff"] if up else case["width"]), device="cuda", dtype=BF16 if up else F32)
        ops.moe_experts_int8(up, out, rows, s["weight"], s["tiles"], act=acts[case["glu"]], limit=LIMIT, slope=SLOPE, tile_rows=s["tile_rows"])
        return out
    stream = torch.empty_like(s["residual"])
    t, d = stream.shape
    rows = ops.int8_rows(t, d, stream.device) if kind == "layer" else torch.empty((t, d), device="cuda", dtype=TYPES[case["rows"]])
    ops.norm_gate_add(s["residual"], s["y"], post_weight=s["post"], post_eps=EPS, gate=s["gate"], gate_bias=s["bias"], scale=s["scale"],
                      next_weight=s["next"], next_eps=EPS, out=rows, into=stream)
    if kind == "norm":
        return {"stream": stream, "rows": rows}
    act = torch.empty((t, case["ff"]), device="cuda", dtype=BF16)
    ops.gemm_int8_glu(act, rows, s["weight"], acts[case["glu"]], LIMIT, SLOPE)
    out = torch.empty((t, d), device="cuda", dtype=BF16)
    ops.gemm_int8(out, act, s["weight2"])
    return {"stream": stream, "out": out}


def _quantized(x):
    """Rows in whole numbers and their scales; the quotient in 64 bits, since values lie next to the border between two numbers."""
    most = x.float().abs().amax(dim=1, keepdim=True)
    q = torch.where(most > 0, (x.double() * 127 / most.double()).round(), 0)
    return q.float(), most / 127


def _gated(z, act):
    """[T, 2f] -> [T, f]: 16 gate features, the 16 up features that go with them, and so on."""
    z = z.view(z.shape[0], -1, 2, 16)
    g, u = z[:, :, 0].reshape(z.shape[0], -1), z[:, :, 1].reshape(z.shape[0], -1)
    if act == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u
    if act == "clamped":
        g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
        return g / (1 + torch.exp(-SLOPE * g)) * (u + 1)
    return g / (1 + torch.exp(-g)) * u


def _product(x, w, w_scale):
    q, scale = _quantized(x)
    return q @ w.float().T * scale * w_scale


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "linear":
        z = _product(s["x"], s["w"], s["w_scale"])
        return (_gated(z, case["glu"]) if case["glu"] else z).to(TYPES[case["out"]])
    if kind == "experts":
        q, scale = _quantized(s["x"])
        if case["direction"] == "up":
            q, scale = q[s["row_token"].long()], scale[s["row_token"].long()]
        padded = torch.zeros(case["experts"], s["most"], q.shape[1], device="cuda")
        padded[s["expert"], s["slot"]] = q
        z = torch.bmm(padded, s["w"].float().transpose(1, 2))[s["expert"], s["slot"]] * scale * s["w_scale"][s["expert"]]
        return _gated(z, case["glu"]).to(BF16) if case["direction"] == "up" else z
    z = s["y"].float()
    if s["post"] is not None:
        z = z * torch.rsqrt(z.square().mean(dim=1, keepdim=True) + EPS) * s["post"]
    if s["gate"] is not None:
        z = z / (1 + torch.exp(-(s["gate"].float() + s["bias"])))
    if s["scale"] is not None:
        z = z * s["scale"]
    stream = s["residual"] + z
    rows = stream * torch.rsqrt(stream.square().mean(dim=1, keepdim=True) + EPS) * s["next"]
    if kind == "norm":
        return {"stream": stream, "rows": rows.to(TYPES[case["rows"]])}
    act = _gated(_product(rows.to(BF16), s["w"], s["w_scale"]), case["glu"]).to(BF16)
    return {"stream": stream, "out": _product(act, s["w2"], s["w2_scale"]).to(BF16)}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind = case["kind"]
    size = {"bfloat16": 2, "float32": 4, "none": 0}
    if kind == "linear":
        t, k, n = case["tokens"], case["k"], case["n"]
        feats = n // 2 if case["glu"] else n
        return {"bytes": t * k * 2 + n * k + 4 * n + t * feats * size[case["out"]], "flops": 2 * t * n * k}
    if kind == "experts":
        t, top, e = case["tokens"], case["top"], case["experts"]
        d, ff, r = case["width"], case["ff"], t * top
        used = e * (1 - (1 - top / e) ** t)                      # experts that get any row, were all alike
        if case["direction"] == "up":
            return {"bytes": t * d * 2 + used * 2 * ff * (d + 4) + r * ff * 2, "flops": 4 * r * ff * d}
        return {"bytes": r * ff * 2 + used * d * (ff + 4) + r * d * 4, "flops": 2 * r * ff * d}
    t, d = case["tokens"], case["width"]
    if kind == "norm":
        per = 8 + size[case["y"]] + size[case["gate"]] + size[case["rows"]]
        return {"bytes": t * d * per + 4 * d * (1 + case["post"] + (case["gate"] != "none") + case["scale"]), "flops": 15 * t * d}
    f = case["ff"]
    return {"bytes": t * d * (8 + 2 + 4 + 2) + 16 * d + 3 * d * f + 4 * (2 * f + d), "flops": 6 * t * d * f}


# ------------------------------------------------------------------ the same from the definitions, in 64 bits

def _rows64(x):
    x = x.to(F64)
    top = x.abs().max(dim=1).values
    step = torch.where(top == 0, torch.ones_like(top), top)
    return torch.round(127 * x / step[:, None]), top / 127


def _glu64(gate, up, act):
    if act == "silu":
        return gate * torch.sigmoid(gate) * up
    if act == "gelu_tanh":
        return gate * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate.pow(3))) * up
    gate, up = torch.minimum(gate, torch.full_like(gate, LIMIT)), torch.clamp(up, min=-LIMIT, max=LIMIT)
    return gate * torch.sigmoid(SLOPE * gate) * (up + 1)


def _split64(z, act):
    """The two kinds of rows of a gated product, picked by their number."""
    n = torch.arange(z.shape[1], device=z.device)
    return _glu64(z[:, n % 32 < 16], z[:, n % 32 >= 16], act)


def _matmul64(x, w, w_scale):
    q, step = _rows64(x)
    return torch.einsum("tk,nk->tn", q, w.to(F64)) * torch.outer(step, w_scale.to(F64))


def _rms64(x, weight):
    return x / torch.sqrt((x * x).sum(dim=1, keepdim=True) / x.shape[1] + EPS) * weight.to(F64)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "linear":
        z = _matmul64(s["x"], s["w"], s["w_scale"])
        return _split64(z, case["glu"]) if case["glu"] else z
    if kind == "experts":
        up = case["direction"] == "up"
        out, at = [], 0
        for e, n in enumerate(s["counts"]):
            x = s["x"][s["row_token"][at:at + n].long()] if up else s["x"][at:at + n]
            if n:
                z = _matmul64(x, s["w"][e], s["w_scale"][e])
                out.append(_split64(z, case["glu"]) if up else z)
            at += n
        return torch.cat(out)
    z = s["y"].to(F64)
    if s["post"] is not None:
        z = _rms64(z, s["post"])
    if s["gate"] is not None:
        z = z * torch.sigmoid(s["gate"].to(F64) + s["bias"].to(F64))
    if s["scale"] is not None:
        z = z * s["scale"].to(F64)
    stream = s["residual"].to(F64) + z
    rows = _rms64(stream, s["next"])
    if kind == "norm":
        return {"stream": stream, "rows": rows}
    act = _split64(_matmul64(rows.to(BF16), s["w"], s["w_scale"]), case["glu"])
    return {"stream": stream, "out": _matmul64(act.to(BF16), s["w2"], s["w2_scale"])}

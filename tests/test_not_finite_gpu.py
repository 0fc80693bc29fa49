"""Numbers that are not finite through the activations: a NaN stays one through every clamp and every relu, so that a token's fault is seen where
the token is; infinities do what the formulas say."""
import pytest
import torch

import int8_plain as plain
from qorvix_b200.csrc import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
GLU = (ops.GLU_SILU, ops.GLU_GELU_TANH, ops.GLU_CLAMPED)
LIMIT, SLOPE = 7.0, 1.702
NAN, INF = float("nan"), float("inf")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def marked(g, tokens, k, dtype=BF16):
    """Rows of which the second holds a NaN, the fourth an infinity and the last one both; and which rows these are."""
    x = normal(g, tokens, k, dtype=dtype)
    bad = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    for row, entries in ((1, (NAN,)), (3, (INF,)), (tokens - 1, (-INF, NAN))):
        x[row, : len(entries)] = torch.tensor(entries, device="cuda", dtype=dtype)
        bad[row] = True
    return x, bad


# ------------------------------------------------------------------ 8-bit rows: a scale that is NaN makes every product NaN

@pytest.mark.parametrize("act", GLU)
@pytest.mark.parametrize("out", (BF16, F32))
@pytest.mark.parametrize("tokens,k,f", [(5, 128, 16), (8, 4096, 1040), (16, 512, 96), (64, 512, 208), (300, 384, 704), (700, 256, 2048)])
def test_8_bit_gated_product(tokens, k, f, out, act):
    g = gen(tokens + k + f)
    x, bad = marked(g, tokens, k)
    w = ops.quantize_weight(normal(g, 2 * f, k, dtype=BF16))
    rows = ops.int8_rows(tokens, k, "cuda")
    ops.quantize_rows(rows, x)
    for given in (x, rows):
        got = torch.zeros((tokens, f), device="cuda", dtype=out)
        ops.gemm_int8_glu(got, given, w, act, LIMIT, SLOPE)
        assert got[bad].isnan().all() and torch.isfinite(got[~bad]).all()
    ops.check_kernel_errors()


@pytest.mark.parametrize("act", GLU)
@pytest.mark.parametrize("tile_rows", (32, 64, 128, 256))
def test_8_bit_experts(tile_rows, act):
    g = gen(tile_rows)
    counts, k, f = (70, 0, 300, 9), 256, 48
    x, bad = marked(g, sum(counts), k)
    w = ops.quantize_weight(normal(g, len(counts), 2 * f, k, dtype=BF16))
    rows = ops.int8_rows(x.shape[0], k, "cuda")
    ops.quantize_rows(rows, x)
    tiles = plain.tile_table(counts, tile_rows, ops.moe_max_tiles(x.shape[0], len(counts), tile_rows), "cuda")
    for out in (BF16, F32):
        got = torch.zeros((x.shape[0], f), device="cuda", dtype=out)
        ops.moe_experts_int8(True, got, rows, w, tiles, act=act, limit=LIMIT, slope=SLOPE, tile_rows=tile_rows)
        assert got[bad].isnan().all() and torch.isfinite(got[~bad]).all()
    ops.check_kernel_errors()


# ------------------------------------------------------------------ the same activations over 16 and 32-bit products

def formula(g, u, act):
    g, u = g.double(), u.double()
    if act == ops.GLU_GELU_TANH:
        return 0.5 * g * (1 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g ** 3)).float().double()) * u       # (32 bits: -1 for gates of -7, and 0 times an infinite u)
    if act == ops.GLU_CLAMPED:
        g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
        return g / (1 + torch.exp(-SLOPE * g)) * (u + 1)
    return g / (1 + torch.exp(-g)) * u


@pytest.mark.parametrize("act", GLU)
@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("interleaved", (False, True))
def test_gated_activation_of_every_pair(act, dtype, interleaved):
    """Every pair of a NaN, infinities, the clamp's borders and ordinary numbers: the formula's NaN and infinities, and its numbers within the type's
    rounding and 64 steps of 2^-24 (the exponential's argument, up to 12, moves it by that many steps; the rest is a few)."""
    v = torch.tensor([NAN, INF, -INF, 0.0, -0.0, LIMIT, -LIMIT, 6.5, -7.5, 8.0, 1.0, -1.25], device="cuda", dtype=dtype)
    g, u = v.repeat_interleave(len(v)), v.repeat(len(v))
    assert g.numel() % 16 == 0
    gu = torch.stack([g.view(-1, 16), u.view(-1, 16)], dim=1).reshape(1, -1) if interleaved else torch.cat([g, u]).reshape(1, -1)
    out = torch.empty((1, g.numel()), device="cuda", dtype=dtype)
    ops.glu_act(out, gu.contiguous(), act, interleaved=interleaved, limit=LIMIT, slope=SLOPE)
    want, got = formula(g, u, act), out[0].double()
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf])
    ok = torch.isfinite(want)
    # tanh near -1 loses all but an absolute 2^-24 of what is multiplied by g u
    bound = want.abs() * (torch.finfo(dtype).eps / 2 + 64 * 2.0 ** -24) + (g.double() * u.double()).abs().nan_to_num(0, 0, 0) * 2.0 ** -23 + 1e-30
    assert ((got - want).abs()[ok] <= bound[ok]).all()


@pytest.mark.parametrize("act", GLU)
@pytest.mark.parametrize("tokens,k,f,dtype", [(5, 128, 64, BF16), (90, 256, 128, BF16), (300, 512, 256, BF16), (5, 132, 48, BF16), (6, 96, 32, F32), (70, 256, 64, F32)])
def test_gated_product(tokens, k, f, dtype, act):
    g = gen(tokens + k + f)
    x = normal(g, tokens, k, dtype=dtype)
    x[1, 0] = NAN
    w = normal(g, 2 * f, k, dtype=dtype, std=k ** -0.5)
    bad = torch.arange(tokens, device="cuda") == 1
    for packed in ((None, ops.pack_weight(w)) if dtype == BF16 and k % 8 == 0 else (None,)):
        got = torch.zeros((tokens, f), device="cuda", dtype=dtype)
        ops.gemm_swiglu(got, x, w if packed is None else None, packed, 2 * f, act=act, limit=LIMIT, slope=SLOPE)
        assert got[bad].isnan().all() and torch.isfinite(got[~bad]).all()
    ops.check_kernel_errors()


@pytest.mark.parametrize("mode", GLU + ("relu2",))
@pytest.mark.parametrize("dtype,tensor_cores", [(F32, False), (BF16, False), (BF16, True)])
@pytest.mark.parametrize("tokens", (6, 200))
def test_experts(tokens, dtype, tensor_cores, mode):
    g = gen(tokens)
    E, top, k, f = 4, 2, 128, 64
    x = normal(g, tokens, k, dtype=dtype)
    x[1, 0] = NAN
    w = [normal(g, E, f, k, dtype=dtype, std=k ** -0.5) for _ in range(1 if mode == "relu2" else 2)]
    top_idx = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:top] for t in range(tokens)]).to(torch.int32).cuda()
    R = tokens * top
    tile_rows = ops.moe_tile_rows(tensor_cores, tokens, R, E)
    row_token, slot_row, scratch = (torch.empty(R, device="cuda", dtype=torch.int32) for _ in range(3))
    tiles = torch.empty(3 * ops.moe_max_tiles(R, E, tile_rows), device="cuda", dtype=torch.int32)
    ops.moe_group(row_token, slot_row, tiles, top_idx, scratch, E, tile_rows)
    out = torch.zeros((R, f), device="cuda", dtype=dtype)
    up, kw = (2, {}) if mode == "relu2" else (True, dict(act=mode, limit=LIMIT, slope=SLOPE))
    if tensor_cores:
        p = [ops.moe_pack_experts(m) for m in w]
        ops.moe_experts_tc(up, out, x, p[0], p[1] if len(p) > 1 else None, row_token, tiles, tile_rows=tile_rows,
                           room=torch.empty(R * k, device="cuda", dtype=F32), **kw)
    else:
        ops.moe_experts(up, out, x, w[0], w[1] if len(w) > 1 else None, row_token, tiles, **kw)
    bad = row_token == 1
    assert bad.sum() == top and out[bad].isnan().all() and torch.isfinite(out[~bad]).all()
    ops.check_kernel_errors()


# ------------------------------------------------------------------ the square of relu

@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("cols", (8, 7))
def test_ungated_activations(dtype, cols):
    x = normal(gen(cols), 3, cols, dtype=dtype)
    x[0, 0], x[1, 1], x[1, 2], x[2, 0] = NAN, INF, -INF, -0.0
    for kind in (ops.ACT_RELU2, ops.ACT_GELU_TANH):
        out = torch.empty_like(x)
        ops.activation(out, x, kind)
        z = x.double()
        want = torch.relu(z) ** 2 if kind == ops.ACT_RELU2 else 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z ** 3)))
        assert torch.equal(out.isnan(), want.isnan()) and out[0, 0].isnan() and out[1, 1] == INF


@pytest.mark.parametrize("act", (ops.ACT_RELU2, ops.ACT_GELU_TANH))
@pytest.mark.parametrize("tokens,k,n,dtype", [(5, 128, 64, BF16), (90, 256, 128, BF16), (300, 512, 256, BF16), (5, 132, 48, BF16), (6, 96, 32, F32)])
def test_ungated_product(tokens, k, n, dtype, act):
    g = gen(tokens + k + n)
    x = normal(g, tokens, k, dtype=dtype)
    x[1, 0] = NAN
    w = normal(g, n, k, dtype=dtype, std=k ** -0.5)
    bad = torch.arange(tokens, device="cuda") == 1
    for packed in ((None, ops.pack_weight(w)) if dtype == BF16 and k % 8 == 0 else (None,)):
        got = torch.zeros((tokens, n), device="cuda", dtype=dtype)
        ops.gemm_act(got, x, w if packed is None else None, packed, n, act)
        assert got[bad].isnan().all() and torch.isfinite(got[~bad]).all()
    ops.check_kernel_errors()

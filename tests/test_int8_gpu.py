"""Rows in 8 bits and the products over them against whole numbers: values and float32 products equal to the bit, rounded outputs and
activations within the rounding of their type."""
import pytest
import torch

import int8_plain as plain
from qorvix_b200.csrc import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
ACTS = (ops.GLU_SILU, ops.GLU_GELU_TANH, ops.GLU_CLAMPED)
LIMIT, SLOPE = 7.0, 1.702


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device="cuda", dtype=F32).to(dtype)


def whole(g, *shape, low=-127):
    return torch.randint(low, 128, shape, generator=g, device="cuda", dtype=torch.int32).to(torch.int8)


def weight(g, *shape, low=-127):
    q = whole(g, *shape, low=low)
    s = torch.rand(shape[:-1], generator=g, device="cuda") + 0.5
    return q, s / (64 * shape[-1] ** 0.5), None


def quantized(x, row_idx=None, rows=None):
    n = x.shape[0] if row_idx is None else row_idx.numel()
    r = rows or ops.int8_rows(n, x.shape[1], x.device)
    ops.quantize_rows(r, x, row_idx=row_idx)
    return r


def assert_rows(r, x):
    q, s = plain.rows(x)
    assert torch.equal(r.values.long(), q)
    assert torch.equal(r.scale.view(torch.int32)[~s.isnan()], s.view(torch.int32)[~s.isnan()])
    assert torch.equal(r.scale.isnan(), s.isnan())


# ------------------------------------------------------------------ rows

@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("tokens,k", [(1, 1), (1, 64), (3, 7), (8, 4096), (5, 1001), (2, 14336), (300, 128), (33, 2056), (2, 40000), (1, 131071)])
def test_rows_equal_the_definition(tokens, k, dtype):
    x = normal(gen(tokens * k), tokens, k, dtype=dtype)
    assert_rows(quantized(x), x)
    ops.check_kernel_errors()


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_rows_next_to_the_border(dtype):
    """Quotients that are half-integers exactly, and the numbers on both sides of them."""
    n = torch.arange(-127, 127, device="cuda", dtype=torch.float64) + 0.5
    got = []
    for top in (127.0, 1.0, 254.0, 1.9921875, 3.0e-30, 2.5e30, 1.0e-38, 3.0e38):
        at = (n * top / 127.0).to(dtype)
        row = torch.cat([at.cpu(), torch.nextafter(at.cpu(), torch.full_like(at, float("inf")).cpu()),
                         torch.nextafter(at.cpu(), torch.full_like(at, float("-inf")).cpu()), torch.tensor([top], dtype=dtype)]).cuda()
        row = torch.where(row.abs() > row[-1].abs(), row[-1], row)
        got.append(row)
    x = torch.stack(got)
    assert_rows(quantized(x), x)


def test_rows_of_all_bfloat16_quotients():
    """Every pair of 8-bit numbers at every distance that leaves anything of the smaller: the quotient is rounded exactly for all of them."""
    m = torch.arange(128, 256, device="cuda", dtype=F32)
    entries = torch.cat([m * 2.0 ** -e for e in range(10)])                  # below 2^-8 of the largest nothing but zeros is left
    for shift in (0, -100, 100):
        x = torch.where(entries[None] <= m[:, None], entries[None], 0.0)
        x = torch.cat([m[:, None], x, -x], dim=1) * 2.0 ** shift
        assert (x.to(BF16).float() == x).all()
        assert_rows(quantized(x.to(BF16)), x.to(BF16))


@pytest.mark.parametrize("k", (64, 77))
def test_rows_that_are_not_ordinary(k):
    x = normal(gen(1), 12, k)
    x[0] = 0
    x[1, k - 1] = float("inf")
    x[2, 0] = float("-inf")
    x[3, k // 2] = float("nan")
    x[4] *= 1e-42                       # below the smallest normal number
    x[5] = torch.finfo(F32).tiny * 2 ** -23
    x[6] *= 1e38 / x[6].abs().max()
    x[7] = torch.finfo(F32).max
    x[8] = -x[8].abs() - 1
    x[9, 1:] = 0
    x[10, 3] = torch.finfo(F32).max
    assert_rows(quantized(x), x)


@pytest.mark.parametrize("dtype,pad,ld", [(BF16, 1, 200), (BF16, 8, 208), (F32, 3, 199), (F32, 4, 204), (BF16, 0, 193)])
def test_rows_out_of_a_wider_tensor(dtype, pad, ld):
    x = normal(gen(2), 9, ld, dtype=dtype)[:, pad:pad + 190]
    assert_rows(quantized(x), x)


def test_rows_gathered_and_what_lies_behind_them():
    g = gen(3)
    x = normal(g, 6, 100, dtype=BF16)
    idx = torch.tensor([5, 0, 0, 3, -1, 6, 2 ** 31 - 1, 1], device="cuda", dtype=torch.int32)
    room = ops.int8_rows(10, 100, x.device)
    room.values.fill_(77)
    room.scale.fill_(-3.0)
    part = ops.Int8Rows(room.values[:8], room.scale[:8])
    quantized(x, idx, part)
    q, s = plain.rows(x)
    for r, src in enumerate(idx.tolist()):
        want_q, want_s = (q[src], s[src]) if 0 <= src < 6 else (torch.zeros_like(q[0]), torch.zeros_like(s[0]))
        assert torch.equal(part.values[r].long(), want_q) and part.scale[r] == want_s
    assert (room.values[8:] == 77).all() and (room.scale[8:] == -3.0).all()


# ------------------------------------------------------------------ dense products

@pytest.mark.parametrize("tokens,k,n", [(1, 1, 1), (1, 128, 128), (2, 130, 129), (8, 4096, 384), (16, 257, 100), (17, 1001, 777), (31, 384, 128), (33, 640, 256),
                                        (64, 512, 2048), (65, 512, 200), (77, 1001, 777), (129, 96, 384), (256, 256, 256), (257, 1024, 520),
                                        (1000, 320, 1336), (4, 14336, 256), (700, 130, 19000)])
@pytest.mark.parametrize("out", (F32, BF16))
def test_product_is_whole_sums_times_scales(tokens, k, n, out):
    g = gen(tokens + k + n)
    x = normal(g, tokens, k, dtype=BF16)
    q, s, _ = weight(g, n, k)
    w = ops.pack_int8(q, s)
    got = torch.full((tokens, n), 7.0, device="cuda", dtype=out)
    ops.gemm_int8(got, x, w)
    qx, sx = plain.rows(x)
    want = plain.product32(qx, sx, q, s).to(out)
    assert torch.equal(got, want)
    again = torch.empty_like(got)
    ops.gemm_int8(again, quantized(x), w)
    assert torch.equal(again, want)
    ops.check_kernel_errors()


@pytest.mark.parametrize("dtype,pad", [(BF16, 0), (BF16, 3), (BF16, 8), (F32, 0), (F32, 1)])
@pytest.mark.parametrize("tokens,k,n", [(1, 14336, 4096), (1, 1, 1), (2, 100, 3000), (7, 4096, 6144), (16, 1001, 777), (40, 640, 1000), (100, 257, 515), (3, 9000, 130)])
def test_product_of_rows_as_they_come(tokens, k, n, dtype, pad):
    """Rows of either type out of a wider tensor, some of zeros and some that are not finite, by whichever kernel puts them into 8 bits."""
    g = gen(tokens + k + n + pad)
    x = normal(g, tokens, k + pad, dtype=dtype)[:, pad:]
    if tokens > 2:
        x[1] = 0
        x[2, k - 1] = float("inf")
    q, s, _ = weight(g, n, k)
    got = torch.empty((tokens, n), device="cuda", dtype=F32)
    ops.gemm_int8(got, x, ops.pack_int8(q, s))
    qx, sx = plain.rows(x)
    want = plain.product32(qx, sx, q, s)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    ops.check_kernel_errors()


def test_sums_that_pass_24_and_nearly_31_bits():
    """All values at their largest: the sum of 131,071 products of -128 by -128 is 2^31 - 2^14."""
    for k in (2000, 131071):
        for low, value in ((-128, -128), (127, 127)):
            q = torch.full((3, k), value, device="cuda", dtype=torch.int8)
            rows = ops.int8_rows(2, k, q.device)
            rows.values.fill_(value)
            rows.scale.fill_(1.0)
            got = torch.empty((2, 3), device="cuda", dtype=F32)
            ops.gemm_int8(got, rows, ops.pack_int8(q, torch.ones(3, device="cuda")))
            assert (got == float(k * value * value)).all() or torch.equal(got, torch.full_like(got, k * value * value))


def test_product_into_part_of_a_tensor():
    g = gen(5)
    x = normal(g, 70, 300, dtype=BF16)
    q, s, _ = weight(g, 200, 300)
    w = ops.pack_int8(q, s)
    room = torch.full((72, 260), 3.0, device="cuda", dtype=BF16)
    ops.gemm_int8(room[1:71, 17:217], x, w)
    qx, sx = plain.rows(x)
    assert torch.equal(room[1:71, 17:217], plain.product32(qx, sx, q, s).to(BF16))
    room[1:71, 17:217] = 3.0
    assert (room == 3.0).all()


def test_tokens_that_are_not_finite_stay_by_themselves():
    g = gen(6)
    x = normal(g, 20, 256, dtype=BF16)
    x[3, 5] = float("nan")
    x[11, 0] = float("inf")
    x[12] = 0
    q, s, _ = weight(g, 130, 256)
    got = torch.empty((20, 130), device="cuda", dtype=F32)
    ops.gemm_int8(got, x, ops.pack_int8(q, s))
    qx, sx = plain.rows(x)
    want = plain.product32(qx, sx, q, s)
    bad = torch.zeros(20, dtype=torch.bool, device="cuda")
    bad[3] = bad[11] = True
    assert got[bad].isnan().all() and torch.equal(got[~bad], want[~bad]) and (got[12] == 0).all()


def glu_bound(z, act, out):
    """How far a gated output may be off, from the sums z in 64 bits (one step: 2^-24 of the value).  g and u carry two roundings each.  With
    gate(g) = g / (1 + exp(-a)): a = c (g + b g^3) has 6 steps from g, and one each from b, its two products, the sum, c and its product: 12 of
    itself; the exponential as a power of 2 adds two (the constant and the product).  That moves the quotient by 14 |a| steps; the functions,
    the sum, the quotient and the products are within 16 steps.  The clamped form adds 1 to u, whose error of 3 steps stays while the sum may
    be small.  Then the output's rounding, half a step of its type."""
    n = torch.arange(z.shape[1], device=z.device) % 32
    g, u = z[:, n < 16], z[:, n >= 16]
    arg = g if act == 0 else 2 * 0.7978845608 * (g + 0.044715 * g ** 3) if act == 1 else SLOPE * g.clamp(max=LIMIT)
    want = plain.gated64(z, act, LIMIT, SLOPE)
    bound = want.abs() * (torch.finfo(out).eps / 2 + (16 + 14 * arg.abs()) * 2.0 ** -24) + 1e-30
    if act == 2:
        bound = bound + g.clamp(max=LIMIT).abs() * u.abs().clamp(max=LIMIT) * 3 * 2.0 ** -24
    return want, bound


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("tokens,k,f", [(1, 128, 16), (8, 1024, 208), (33, 130, 16), (64, 512, 1040), (65, 200, 336), (300, 384, 704)])
def test_gated_product(tokens, k, f, act):
    g = gen(tokens + k + f + act)
    x = normal(g, tokens, k, dtype=BF16)
    q, s, _ = weight(g, 2 * f, k)
    w = ops.pack_int8(q, s)
    qx, sx = plain.rows(x)
    z = plain.product64(qx, sx, q, s)
    for out in (BF16, F32):
        want, bound = glu_bound(z, act, out)
        got = torch.empty((tokens, f), device="cuda", dtype=out)
        ops.gemm_int8_glu(got, x, w, act, LIMIT, SLOPE)
        assert ((got.double() - want).abs() <= bound).all()
    ops.check_kernel_errors()


# ------------------------------------------------------------------ grouped by expert

@pytest.mark.parametrize("tile_rows", (32, 64, 128, 256))
@pytest.mark.parametrize("counts,k,n", [((0, 5, 0, 1, 40), 200, 96), ((300, 0, 17, 64, 65), 384, 160), ((1,), 128, 32), ((0, 0, 33), 1001, 288)])
def test_experts(counts, k, n, tile_rows):
    g = gen(sum(counts) + k + n)
    R, E = sum(counts), len(counts)
    spare = 3                                      # rows that no tile lists
    x = normal(g, R + spare, k, dtype=BF16)
    q, s, _ = weight(g, E, n, k)
    w = ops.pack_int8(q, s)
    rows = quantized(x)
    tiles = plain.tile_table(counts, tile_rows, ops.moe_max_tiles(R + spare, E, tile_rows), "cuda")
    qx, sx = plain.rows(x)
    down = torch.full((R + spare, n), 5.0, device="cuda", dtype=F32)
    ops.moe_experts_int8(False, down, rows, w, tiles, tile_rows=tile_rows)
    up = torch.full((R + spare, n // 2), 5.0, device="cuda", dtype=BF16)
    ops.moe_experts_int8(True, up, rows, w, tiles, act=ops.GLU_CLAMPED, limit=LIMIT, slope=SLOPE, tile_rows=tile_rows)
    at = 0
    for e, c in enumerate(counts):
        here = slice(at, at + c)
        assert torch.equal(down[here], plain.product32(qx[here], sx[here], q[e], s[e]))
        want, bound = glu_bound(plain.product64(qx[here], sx[here], q[e], s[e]), ops.GLU_CLAMPED, BF16)
        assert ((up[here].double() - want).abs() <= bound).all()
        at += c
    assert (down[R:] == 5.0).all() and (up[R:] == 5.0).all()
    ops.check_kernel_errors()

"""Tables of tiles with entries that name no expert or no rows, ahead of, between and behind the tiles that there are, over more items than the card
has pairs of SMs."""
import pytest
import torch

import int8_plain as plain
from qorvix_b200.csrc import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
NONE = [(-1, 0, 0), (-7, 3, 9), (5, 0, 32), (2 ** 31 - 1, 1, 1), (0, -1, 4), (1, 2, 0), (1, 2, -3), (2, 10 ** 6, 5), (-1, 5, 32)]


@pytest.mark.parametrize("n", (4000, 250))
@pytest.mark.parametrize("tile_rows", (32, 64, 256))
@pytest.mark.parametrize("up", (False, True))
@pytest.mark.parametrize("where", ("ahead", "between", "behind", "far between"))
def test_entries_without_tiles_are_passed_over(where, up, tile_rows, n):
    g = torch.Generator(device="cuda").manual_seed(n + tile_rows)
    n, k, E = n // 32 * 32, 160, 5
    counts = (90, 0, 33, 300, 64)
    R = sum(counts)
    x = torch.randn((R, k), generator=g, device="cuda").to(BF16)
    q = torch.randint(-127, 128, (E, n, k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    s = torch.rand((E, n), generator=g, device="cuda") / (64 * k ** 0.5)
    rows = ops.int8_rows(R, k, "cuda")
    ops.quantize_rows(rows, x)
    table, first = [], 0
    for e, c in enumerate(counts):
        table += [(e, first + r, min(tile_rows, c - r)) for r in range(0, c, tile_rows)]
        first += c
    if where == "ahead":
        table = NONE + table
    elif where == "behind":
        table = table + 3 * NONE
    elif where == "between":
        table = [t for i, tile in enumerate(table) for t in (NONE[i % len(NONE)], tile, NONE[(5 * i + 1) % len(NONE)])]
    else:                                                 # more of them in a row than a warp looks at in one go
        table = table[:2] + 90 * NONE + table[2:5] + 41 * NONE + table[5:]
    tiles = torch.tensor(table, dtype=torch.int32, device="cuda").reshape(-1)
    out = torch.full((R + 4, n // 2 if up else n), 9.0, device="cuda", dtype=F32)
    ops.moe_experts_int8(up, out[:R], rows, ops.pack_int8(q, s), tiles, tile_rows=tile_rows)
    qx, sx = plain.rows(x)
    at = 0
    for e, c in enumerate(counts):
        here = slice(at, at + c)
        if up:
            z = plain.product64(qx[here], sx[here], q[e], s[e])
            want = plain.gated64(z, 0, 0.0, 0.0)
            gate = z.view(c, -1, 2, 16)[:, :, 0].reshape(c, n // 2) if c else z[:, : n // 2]
            assert ((out[here].double() - want).abs() <= want.abs() * (16 + 14 * gate.abs()) * 2.0 ** -24 + 1e-30).all()
        else:
            assert torch.equal(out[here], plain.product32(qx[here], sx[here], q[e], s[e]))
        at += c
    assert (out[R:] == 9.0).all()
    ops.check_kernel_errors()


def test_tables_without_any_tile():
    R, n, k = 10, 4096, 64
    rows = ops.int8_rows(R, k, "cuda")
    ops.quantize_rows(rows, torch.ones((R, k), device="cuda"))
    w = ops.quantize_weight(torch.ones((2, n, k), device="cuda"))
    out = torch.full((R, n), 9.0, device="cuda", dtype=F32)
    for entries in (1, 40, 700):
        table = torch.tensor((NONE * entries)[:entries], dtype=torch.int32, device="cuda").reshape(-1)
        table[0::3] = torch.where(table[0::3] < 2, table[0::3], -1)
        table[0::3][(table[0::3] >= 0) & (table[1::3] >= 0)] = -1
        ops.moe_experts_int8(False, out, rows, w, table, tile_rows=32)
    assert (out == 9.0).all()
    ops.check_kernel_errors()


def test_more_items_than_a_warp_looks_at_in_one_go():
    """More than 32 items a pair of SMs, of a table with empty entries and of a dense product."""
    g = torch.Generator(device="cuda").manual_seed(1)
    n, k, counts = 4000, 64, (2500, 0, 700, 3333, 1)
    R = sum(counts)
    x = torch.randn((R, k), generator=g, device="cuda").to(BF16)
    q = torch.randint(-127, 128, (len(counts), n, k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    s = torch.rand((len(counts), n), generator=g, device="cuda") / (64 * k ** 0.5)
    rows = ops.int8_rows(R, k, "cuda")
    ops.quantize_rows(rows, x)
    table, first = [], 0
    for e, c in enumerate(counts):
        table += [t for r in range(0, c, 32) for t in ((e, first + r, min(32, c - r)), NONE[r // 32 % len(NONE)])]
        first += c
    assert len(table) * 16 > 2 * 32 * 74
    out = torch.full((R, n), 9.0, device="cuda", dtype=F32)
    ops.moe_experts_int8(False, out, rows, ops.pack_int8(q, s), torch.tensor(table, dtype=torch.int32, device="cuda").reshape(-1), tile_rows=32)
    qx, sx = plain.rows(x)
    at = 0
    for e, c in enumerate(counts):
        assert torch.equal(out[at: at + c], plain.product32(qx[at: at + c], sx[at: at + c], q[e], s[e]))
        at += c
    x = torch.randn((45000, 32), generator=g, device="cuda").to(BF16)
    q, s = q[0, :, :32].contiguous(), s[0]
    out = torch.empty((45000, n), device="cuda", dtype=BF16)
    ops.gemm_int8(out, x, ops.pack_int8(q, s))
    qx, sx = plain.rows(x)
    for part in range(0, 45000, 5000):
        here = slice(part, part + 5000)
        assert torch.equal(out[here], plain.product32(qx[here], sx[here], q, s).to(BF16))
    ops.check_kernel_errors()

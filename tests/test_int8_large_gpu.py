"""Operands whose offsets pass 31 and 32 bits: the far ends equal what the same rows or channels give by themselves."""
import pytest
import torch

import int8_plain as plain
from qorvix_b200.csrc import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 60 GB")
    yield
    torch.cuda.empty_cache()


def whole(*shape):
    return torch.randint(-127, 128, shape, device="cuda", dtype=torch.int8)


def quantized(x, row_idx=None):
    r = ops.int8_rows(x.shape[0] if row_idx is None else row_idx.numel(), x.shape[1], x.device)
    ops.quantize_rows(r, x, row_idx=row_idx)
    return r


def product(x, w, n, dtype=F32):
    T = x.shape[0]
    out = torch.empty((T, n), device="cuda", dtype=dtype)
    ops.gemm_int8(out, x, w)
    return out


@pytest.mark.parametrize("tokens,k", [(40000, 120000), (1200000, 4096)])
def test_rows(tokens, k):
    x = torch.empty((tokens, k), device="cuda", dtype=BF16).normal_()
    r = quantized(x)
    for part in (slice(0, 3), slice(tokens - 3, tokens)):
        q, s = plain.rows(x[part])
        assert torch.equal(r.values[part].long(), q) and torch.equal(r.scale[part], s)
    last = quantized(x, torch.tensor([tokens - 1, 0, tokens - 1], device="cuda", dtype=torch.int32))      # one row twice, the far one
    assert torch.equal(last.values[0], r.values[-1]) and torch.equal(last.values[2], r.values[-1]) and torch.equal(last.values[1], r.values[0])


def test_outputs():
    tokens, k, n = 140000, 200, 32768                         # 4.6e9 entries of output
    x = torch.randn((tokens, k), device="cuda").to(BF16)
    w = ops.pack_int8(whole(n, k), torch.rand(n, device="cuda") + 0.5)
    out = product(x, w, n, BF16)
    for part in (slice(0, 5), slice(tokens - 5, tokens)):
        assert torch.equal(out[part], product(x[part], w, n, BF16))
    ops.check_kernel_errors()


def test_matrices():
    n, k = 280064, 16384                                      # 4.6e9 bytes
    q, s = whole(n, k), torch.rand(n, device="cuda") + 0.5
    w, far = ops.pack_int8(q, s), ops.pack_int8(q[-384:], s[-384:])
    for tokens in (1, 20, 300):                               # clusters that put the row into 8 bits, clusters, pairs
        x = torch.randn((tokens, k), device="cuda").to(BF16)
        assert torch.equal(product(x, w, n)[:, -384:], product(x, far, 384))
    ops.check_kernel_errors()


def test_experts():
    E, n, k = 40, 28672, 4096                                 # 4.7e9 bytes
    q, s = whole(E, n, k), torch.rand((E, n), device="cuda") + 0.5
    x = quantized(torch.randn((70, k), device="cuda").to(BF16))
    tiles = torch.tensor([0, 0, 32, 39, 32, 32, 39, 64, 6], device="cuda", dtype=torch.int32)
    out = torch.zeros((70, n), device="cuda")
    ops.moe_experts_int8(False, out, x, ops.pack_int8(q, s), tiles, tile_rows=32)
    for e, part in ((0, slice(0, 32)), (39, slice(32, 70))):
        rows = ops.Int8Rows(x.values[part], x.scale[part])
        assert torch.equal(out[part], product(rows, ops.pack_int8(q[e], s[e]), n))
    ops.check_kernel_errors()


@pytest.mark.parametrize("d", (4096, 4100))                   # rows on whole 16 bytes of every operand, and not
def test_pass(d):
    tokens = 1100000                                          # 4.5e9 entries
    stream = torch.empty((tokens, d), device="cuda").normal_()
    y = torch.empty((tokens, d), device="cuda", dtype=BF16).normal_()
    weights = [torch.rand(d, device="cuda") + 0.5 for _ in range(2)]
    rows = ops.int8_rows(tokens, d, "cuda")
    parts = (slice(0, 2), slice(tokens - 2, tokens))
    old = [stream[p].clone() for p in parts]
    ops.norm_gate_add(stream, y, weights[0], 1e-5, next_weight=weights[1], next_eps=1e-5, out=rows)
    for p, o in zip(parts, old):
        stream64, rows64 = plain.norm_gate64(residual=o, y=y[p], post_weight=weights[0], post_eps=1e-5, gate=None, gate_bias=None, scale=None,
                                             next_weight=weights[1], next_eps=1e-5)
        # float32 sums, roots and products of the chain: 64 half steps and fewer of the larger term
        assert ((stream[p].double() - stream64).abs() <= 64 * 2.0 ** -24 * (o.double().abs() + (stream64 - o.double()).abs())).all()
        # 8 bits: half a step of a 127th of the row's largest, the bfloat16 row's half step (2^-8 of the entry, and of the largest in the scale) and the chain
        most = rows64.abs().amax(dim=1, keepdim=True)
        got = rows.values[p].double() * rows.scale[p].double()[:, None]
        assert ((got - rows64).abs() <= most / 254 * (1 + 2.0 ** -7) + 2.0 ** -8 * rows64.abs() + 128 * 2.0 ** -24 * most).all()
    ops.check_kernel_errors()

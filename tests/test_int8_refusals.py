"""What the 8-bit operators refuse, on the CPU: nothing is launched and nothing written."""
import pytest
import torch

from qorvix_b200 import LLM, ModelRunner
from qorvix_b200.csrc import ops

BF16, F32, I8 = torch.bfloat16, torch.float32, torch.int8


def rows(t, k):
    return ops.int8_rows(t, k, "cpu")


def weight(n=64, k=64, experts=0):
    return ops.Int8Weight(torch.zeros(16384, dtype=I8), torch.zeros(max(experts, 1) * n), n, k, experts)


def refused(match, f, *a, **kw):
    with pytest.raises(ops.KernelError, match=match):
        f(*a, **kw)


def test_room_for_rows():
    r = rows(5, 100)
    assert tuple(r.shape) == (5, 100) and r.values.stride() == (112, 1) and r.scale.shape == (5,)
    assert rows(3, 128).values.is_contiguous() and tuple(rows(0, 7).shape) == (0, 7)


def test_rows():
    x = torch.zeros(4, 64, dtype=BF16)
    refused("4 rows do not fill 5", ops.quantize_rows, rows(5, 64), x)
    refused("64 entries", ops.quantize_rows, rows(4, 64), torch.zeros(4, 65, dtype=BF16))
    refused("whole in memory", ops.quantize_rows, rows(64, 4), torch.zeros(4, 64, dtype=BF16).T)
    refused("row_idx", ops.quantize_rows, rows(2, 64), x, row_idx=torch.zeros(2, dtype=torch.int64))
    refused("2 row indices do not fill 3", ops.quantize_rows, rows(3, 64), x, row_idx=torch.zeros(2, dtype=torch.int32))
    refused("CUDA device", ops.quantize_rows, rows(4, 64), x)
    r = rows(4, 64)
    refused("contiguous float32 scale", ops.Int8Rows, r.values, r.scale.double())
    refused("contiguous float32 scale", ops.Int8Rows, r.values, r.scale[:3])
    refused("contiguous float32 scale", ops.Int8Rows, r.values.float(), r.scale)
    refused("16 bytes", ops.Int8Rows, torch.zeros(4, 100, dtype=I8), r.scale)
    refused("16 bytes", ops.Int8Rows, torch.zeros(4, 144, dtype=I8)[:, 1:65], r.scale)
    refused("16 bytes", ops.Int8Rows, torch.zeros(1, 64, dtype=I8).expand(4, 64), r.scale)


def test_packing():
    refused("CUDA device", ops.pack_int8, torch.zeros(4, 4, dtype=I8), torch.zeros(4))
    refused("matrix", ops.quantize_weight, torch.zeros(4))


def test_packing_shapes(monkeypatch):
    monkeypatch.setattr(ops, "_on_current", lambda *a: 0)
    refused("int8 values", ops.pack_int8, torch.zeros(4, 4), torch.zeros(4))
    refused("int8 values", ops.pack_int8, torch.zeros(4, 4, dtype=I8), torch.zeros(5))
    refused("int8 values", ops.pack_int8, torch.zeros(2, 4, 4, dtype=I8), torch.zeros(2))
    refused("int8 values", ops.pack_int8, torch.zeros(4, 4, dtype=I8), torch.zeros(4, dtype=torch.float64))
    refused("131071", ops.pack_int8, torch.zeros(1, 131072, dtype=I8), torch.zeros(1))
    refused("131071", ops.pack_int8, torch.zeros(1, 0, dtype=I8), torch.zeros(1))


def test_products():
    x, out = torch.zeros(3, 64, dtype=BF16), torch.zeros(3, 64, dtype=BF16)
    refused("do not give", ops.gemm_int8, out, torch.zeros(3, 63, dtype=BF16), weight())
    refused("do not give", ops.gemm_int8, out[:2], x, weight())
    refused("do not give", ops.gemm_int8, out[:, :63], x, weight())
    refused("do not give", ops.gemm_int8_glu, out, x, weight())
    refused("moe_experts_int8", ops.gemm_int8, out, x, weight(experts=2))
    refused("groups of 16", ops.gemm_int8_glu, out[:, :24], x, weight(n=48))
    refused("groups of 16", ops.gemm_int8_glu, out[:, :32], x, weight(), 3)
    refused("whole in memory", ops.gemm_int8, torch.zeros(64, 3, dtype=BF16).T, x, weight())
    refused("whole in memory", ops.gemm_int8, out, torch.zeros(64, 3, dtype=BF16).T, weight())
    refused("overlap", ops.gemm_int8, torch.zeros(1, 64, dtype=BF16).expand(3, 64), x, weight())
    refused("CUDA device", ops.gemm_int8, out, x, weight())
    ops.gemm_int8(out[:0], x[:0], weight())                                   # no rows: nothing to do


def test_experts():
    r, out, tiles = rows(8, 64), torch.zeros(8, 32, dtype=BF16), torch.zeros(9, dtype=torch.int32)
    w = weight(experts=2)
    refused("experts' matrices", ops.moe_experts_int8, True, out, r, weight(), tiles, tile_rows=32)
    refused("32, 64, 128 or 256", ops.moe_experts_int8, True, out, r, w, tiles)
    refused("32, 64, 128 or 256", ops.moe_experts_int8, True, out, r, w, tiles, tile_rows=48)
    refused("three numbers", ops.moe_experts_int8, True, out, r, w, tiles[:8], tile_rows=32)
    refused("tiles must be", ops.moe_experts_int8, True, out, r, w, tiles.long(), tile_rows=32)
    refused("groups of 16", ops.moe_experts_int8, True, out, r, w, tiles, act=5, tile_rows=32)
    refused("do not go with", ops.moe_experts_int8, True, out, rows(8, 63), w, tiles, tile_rows=32)
    refused("out must be", ops.moe_experts_int8, False, out, r, w, tiles, tile_rows=32)
    refused("CUDA device", ops.moe_experts_int8, True, out, r, w, tiles, tile_rows=32)
    assert [ops.moe_int8_tile_rows(n, 64) for n in (1, 1536, 1537, 6144, 6145, 10 ** 6)] == [32, 32, 64, 128, 256, 256]


def test_norms(monkeypatch):
    s, y, w = torch.zeros(3, 16), torch.zeros(3, 16, dtype=BF16), torch.zeros(16)
    refused("CUDA device", ops.norm_gate_add, s, y)
    monkeypatch.setattr(ops, "_on_current", lambda *a: 0)
    refused("float32", ops.norm_gate_add, s.to(BF16), y)
    refused("float32", ops.norm_gate_add, s[:, :8], y[:, :8])
    refused("needs a y", ops.norm_gate_add, s, None, post_weight=w, out=y)
    refused("needs a y", ops.norm_gate_add, s, None, gate=y, out=y)
    refused("needs a gate", ops.norm_gate_add, s, y, gate_bias=w)
    refused("rows to write", ops.norm_gate_add, s, y, next_weight=w)
    refused("y must be", ops.norm_gate_add, s, y[:2])
    refused("gate must be", ops.norm_gate_add, s, y, gate=torch.zeros(16, 3).T)
    refused("out must be", ops.norm_gate_add, s, y, out=torch.zeros(1, 16).expand(3, 16))
    refused("out must be", ops.norm_gate_add, s, y, out=rows(2, 16))
    refused("float32 \\[16\\]", ops.norm_gate_add, s, y, scale=w[:15])
    refused("float32 \\[16\\]", ops.norm_gate_add, s, y, post_weight=w.to(BF16))
    refused("new residual stream", ops.norm_gate_add, s, y, into=torch.zeros(3, 17)[:, :16])
    both = torch.zeros(100)
    refused("partly over", ops.norm_gate_add, both[:48].view(3, 16), y, into=both[16:64].view(3, 16))
    ops.norm_gate_add(s[:0], y[:0], out=y[:0])                                # no rows: nothing to do


def test_models():
    with pytest.raises(ValueError, match="weights must be one of stored, int8"):
        ModelRunner("/nowhere", weights="int4")
    with pytest.raises(ValueError, match="go with dtype bfloat16"):
        LLM("/nowhere", dtype="float32", weights="int8")

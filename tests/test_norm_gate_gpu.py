"""The pass between two sublayers against 64 bits."""
import pytest
import torch

import int8_plain as plain
from qorvix_b200.csrc import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def inputs(tokens, d, seed, y=BF16, gate=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def n(*shape, mean=0.0, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std + mean

    return dict(residual=n(tokens, d, std=2.0), y=n(tokens, d).to(y), post_weight=n(d, mean=1.0, std=0.1), gate=n(tokens, d).to(gate),
                gate_bias=n(d, std=0.5), scale=n(d, mean=0.7, std=0.1), next_weight=n(d, mean=1.0, std=0.1), post_eps=1e-5, next_eps=1e-6)


def assert_close(got, want, steps, size):
    # float32: each of the chain's operations is off by at most 2^-24 of its result (sums of squares of d terms: a tree of at most 40
    # additions, halved by the root), `steps` of them in all, relative to the largest term of the sum they end in; then the type's rounding
    bound = size * steps * 2.0 ** -24 + want.abs() * (torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else 0.0) + 1e-30
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("parts", ("all", "no post", "no gate", "no scale", "no bias", "sum alone", "no y", "no next"))
@pytest.mark.parametrize("tokens,d,y,gate,out", [(1, 1, F32, F32, F32), (300, 4096, BF16, BF16, BF16), (301, 72, F32, F32, BF16), (700, 2056, BF16, F32, F32), (330, 8192, F32, F32, F32), (310, 5120, F32, F32, F32), (1500, 1024, F32, F32, BF16), (3, 64, BF16, F32, BF16), (8, 4096, BF16, F32, BF16), (5, 1001, F32, BF16, F32),
                                                 (70, 2056, BF16, BF16, BF16), (2, 20000, BF16, F32, F32)])
def test_pass(tokens, d, y, gate, out, parts):
    a = inputs(tokens, d, tokens + d, y, gate)
    drop = {"all": (), "no post": ("post_weight",), "no gate": ("gate", "gate_bias"), "no scale": ("scale",), "no bias": ("gate_bias",),
            "sum alone": ("post_weight", "gate", "gate_bias", "scale"), "no y": ("y", "post_weight", "gate", "gate_bias", "scale"), "no next": ("next_weight",)}
    for name in drop[parts]:
        a[name] = None
    stream64, rows64 = plain.norm_gate64(**a)
    old = a["residual"].clone()
    rows = torch.empty((tokens, d), device="cuda", dtype=out)
    into = torch.full_like(old, 9.0)
    ops.norm_gate_add(out=rows, into=into, **a)
    assert torch.equal(a["residual"], old)
    size = old.double().abs() + (stream64 - old.double()).abs()
    assert_close(into, stream64, 64, size)
    ratio = (rows64 / torch.where(stream64 == 0, 1.0, stream64)).abs()
    assert_close(rows, rows64, 128, size * ratio + rows64.abs())
    rows2 = torch.empty_like(rows)
    ops.norm_gate_add(out=rows2, **a)                                        # in place
    assert torch.equal(a["residual"], into) and torch.equal(rows2, rows)


@pytest.mark.parametrize("tokens,d", [(1, 64), (8, 4096), (3, 1001), (40, 5120), (2, 20000), (310, 1024), (1300, 136), (297, 8192), (900, 2560), (610, 5120), (3000, 520)])
def test_rows_in_8_bits_are_those_of_the_bfloat16_rows(tokens, d):
    a = inputs(tokens, d, 7 * tokens + d)
    a["residual"][0] *= 1e-3
    rows = torch.empty((tokens, d), device="cuda", dtype=BF16)
    stream = torch.empty_like(a["residual"])
    ops.norm_gate_add(out=rows, into=stream, **a)
    r8 = ops.int8_rows(tokens, d, "cuda")
    stream8 = torch.empty_like(stream)
    ops.norm_gate_add(out=r8, into=stream8, **a)
    q, s = plain.rows(rows)
    assert torch.equal(r8.values.long(), q) and torch.equal(r8.scale, s) and torch.equal(stream8, stream)


def test_strided_and_unaligned_operands():
    a = inputs(6, 203, 3)
    wide_y = torch.zeros((6, 300), device="cuda", dtype=BF16)
    wide_g = torch.zeros((6, 301), device="cuda", dtype=F32)
    wide_y[:, 5:208], wide_g[:, 3:206] = a["y"], a["gate"]
    a["y"], a["gate"] = wide_y[:, 5:208], wide_g[:, 3:206]
    stream64, rows64 = plain.norm_gate64(**a)
    room = torch.full((6, 220), 4.0, device="cuda", dtype=BF16)
    into = torch.empty_like(a["residual"])
    ops.norm_gate_add(out=room[:, 1:204], into=into, **a)
    size = a["residual"].double().abs() + (stream64 - a["residual"].double()).abs()
    assert_close(into, stream64, 64, size)
    assert_close(room[:, 1:204], rows64, 128, size * (rows64 / stream64).abs() + rows64.abs())
    room[:, 1:204] = 4.0
    assert (room == 4.0).all()


def test_values_that_are_not_finite_stay_in_their_token():
    a = inputs(4, 96, 11)
    a["y"][1, 7] = float("nan")
    a["gate"][2] = -200.0                                                    # a closed gate: the sum is the stream
    a["gate"][3] = 200.0
    stream64, rows64 = plain.norm_gate64(**a)
    r8 = ops.int8_rows(4, 96, "cuda")
    into = torch.empty_like(a["residual"])
    ops.norm_gate_add(out=r8, into=into, **a)
    assert r8.scale[1].isnan() and (r8.values[1] == 0).all() and torch.equal(into[2], a["residual"][2])
    ok = [0, 2, 3]
    assert torch.isfinite(r8.scale[ok]).all() and torch.isfinite(into[ok]).all()

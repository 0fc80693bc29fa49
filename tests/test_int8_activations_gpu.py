"""Activations behind 8-bit products: the float32 sums go into them as they are; gates far below zero keep what bfloat16 can hold of them."""
from types import SimpleNamespace

import pytest
import torch

import int8_plain as plain
from qorvix_b200.csrc import ops
from qorvix_b200.parts import Runtime, build_part, linear
from qorvix_b200.parts.spec import ActMLPSpec
from qorvix_b200.weights import TensorSource

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
DEV = torch.device("cuda")


@pytest.mark.parametrize("activation", ("relu2", "gelu_tanh"))
@pytest.mark.parametrize("tokens,d,ff", [(1, 64, 96), (7, 128, 100), (300, 72, 48)])
def test_ungated_feed_forward(tokens, d, ff, activation, monkeypatch):
    """bias and activation over the product's float32 sums, one rounding: with a bias that nearly cancels the sum an earlier rounding to bfloat16 would
    be the whole value."""
    monkeypatch.setattr(linear, "INT8_LEAST", 1)
    g = torch.Generator().manual_seed(tokens + d)
    spec = ActMLPSpec(d, ff, "up", "down", activation=activation, bias=True)
    x = torch.randn(tokens, d, generator=g).to(BF16)
    w = {"up": torch.randn(ff, d, generator=g).to(BF16), "down": (torch.randn(d, ff, generator=g) / ff ** 0.5).to(BF16)}
    z = plain.product64(*plain.rows(x), *plain.rows(w["up"]))
    w["up.b"], w["down.b"] = (-z[0] + torch.randn(ff, generator=g, dtype=torch.float64) * 0.02).float(), torch.zeros(d)
    with linear.int8_weights():
        part = build_part("feed_forward", spec, TensorSource(tensors=w, device=DEV, compute_dtype=BF16), Runtime(DEV, BF16, 64, weights="int8"))
    assert part.up.int8 is not None and part.down.int8 is not None
    acts, down = [], part.down

    class Down:
        int8 = down.int8

        def __call__(self, act, out_dtype=None):
            acts.append(act.clone())
            return down(act, out_dtype=out_dtype)

    part.down = Down()
    got = part.forward(x.to(DEV), SimpleNamespace())
    bias = w["up.b"].double()
    v = z + bias
    # one step: 2^-24 of a value.  The sum has two roundings, of |z| each, and the addition's; relu's square doubles the relative error; GELU's slope is under
    # 1.2 and its functions are within 16 steps of the argument
    err = (2 * z.abs() + v.abs()) * 2.0 ** -24
    if activation == "relu2":
        want = torch.relu(v) ** 2
        bound = 2 * torch.relu(v) * err + err ** 2 + want * 2.0 ** -23
    else:
        want = 0.5 * v * (1 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v ** 3)))
        bound = 1.2 * err + v.abs() * 16 * 2.0 ** -24
    bound = bound + (want.abs() + bound) * 2.0 ** -8 + 1e-30
    assert ((acts[0].double().cpu() - want).abs() <= bound).all()
    qa, sa = plain.rows(acts[0].cpu())
    down64 = plain.product64(qa, sa, *plain.rows(w["down"]))
    assert ((got.double().cpu() - down64).abs() <= down64.abs() * 2.0 ** -8 + 1e-30).all()
    ops.check_kernel_errors()


@pytest.mark.parametrize("tokens", (1, 40, 300))
@pytest.mark.parametrize("act", (ops.GLU_SILU, ops.GLU_GELU_TANH, ops.GLU_CLAMPED))
def test_gates_far_below_zero(act, tokens):
    """g sigmoid(a) times a large u is an ordinary number where sigmoid(a) is not far above the smallest normal one, 2^-126, and down to the smallest
    there are: bfloat16 outputs keep it."""
    f, slope = 512, 1.702
    ar = torch.linspace(-101.0, -60.0, f, dtype=torch.float64)                 # the exponential's arguments
    g = ar / slope if act == ops.GLU_CLAMPED else ar
    if act == ops.GLU_GELU_TANH:                                              # 2 c (g + 0.044715 g^3) = ar, by Newton's method
        g = torch.full_like(ar, -6.0)
        for _ in range(60):
            g = g - (1.5957691216057308 * (g + 0.044715 * g ** 3) - ar) / (1.5957691216057308 * (1 + 3 * 0.044715 * g ** 2))
    limit = 1e30
    u = torch.full((f,), 1e30, dtype=torch.float64)
    z = torch.stack([g.view(-1, 16), u.view(-1, 16)], dim=1).reshape(-1)
    # one entry a row: the sum is 127 * 127, the token's scale 1 / 127, the channel's the value over 127
    q = torch.where(z < 0, -127, 127).to(torch.int8).reshape(-1, 1).cuda()
    s = (z.abs() / 127).float().cuda()
    x = torch.ones((tokens, 1), device="cuda", dtype=BF16)
    out = torch.empty((tokens, f), device="cuda", dtype=BF16)
    ops.gemm_int8_glu(out, x, ops.pack_int8(q, s), act, limit, slope)
    z64 = plain.product64(*plain.rows(x), q, s)
    zz = z64.view(tokens, -1, 2, 16)
    g64, u64 = zz[:, :, 0].reshape(tokens, f), zz[:, :, 1].reshape(tokens, f)
    a64 = slope * g64 if act == ops.GLU_CLAMPED else 1.5957691216057308 * (g64 + 0.044715 * g64 ** 3) if act == ops.GLU_GELU_TANH else g64
    e = torch.exp(a64)
    want = g64 * e / (1 + e) * (u64.clamp(-limit, limit) + 1 if act == ops.GLU_CLAMPED else u64)
    # as for ordinary gates (16 + 14 |a| steps of 2^-24, half a step of bfloat16), and below the smallest normal exponentials two of their steps
    bound = want.abs() * (2.0 ** -8 + (16 + 14 * a64.abs()) * 2.0 ** -24) + g64.abs() * u64 * 2.0 ** -148
    assert ((out.double() - want).abs() <= bound).all()
    ops.check_kernel_errors()

"""Activations behind 8-bit products: the float32 sums go into them as they are."""
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

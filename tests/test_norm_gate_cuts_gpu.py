"""The pass between two sublayers: a row is the same to the bit whatever the other rows of the step are; its gate is as accurate as its types."""
import pytest
import torch

import test_int8_engine_gpu as engine
from helpers import random_tokens
from qorvix_b200 import ModelRunner, StepEntry
from qorvix_b200.config import register_architecture, unregister_architecture
from qorvix_b200.csrc import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
ROWS = 640                                               # more than two rows an SM


def inputs(tokens, d, seed, y, gate):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def n(*shape, mean=0.0, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std + mean

    return dict(residual=n(tokens, d, std=2.0), y=n(tokens, d).to(y), post_weight=n(d, mean=1.0, std=0.1), gate=n(tokens, d).to(gate),
                gate_bias=n(d, std=0.5), scale=n(d, mean=0.7, std=0.1), next_weight=n(d, mean=1.0, std=0.1), post_eps=1e-5, next_eps=1e-6)


def bits(t):
    return t.view(torch.int32 if t.dtype == F32 else torch.int16 if t.dtype == BF16 else torch.int8)


def the_pass(a, out, rows):
    a = {k: v[rows] if torch.is_tensor(v) and v.dim() == 2 else v for k, v in a.items()}
    T, d = a["residual"].shape
    into = torch.empty((T, d), device="cuda", dtype=F32)
    if out == "int8":
        r = ops.int8_rows(T, d, "cuda")
        ops.norm_gate_add(out=r, into=into, **a)
        return [bits(into), r.values, bits(r.scale)]
    r = torch.empty((T, d), device="cuda", dtype=out)
    ops.norm_gate_add(out=r, into=into, **a)
    return [bits(into), bits(r)]


@pytest.mark.parametrize("y,gate,out,drop", [(F32, F32, F32, ()), (BF16, F32, BF16, ()), (BF16, BF16, "int8", ()), (F32, F32, F32, ("gate", "gate_bias", "scale")),
                                             (BF16, F32, "int8", ("post_weight", "gate", "gate_bias", "scale")), (F32, F32, F32, ("y", "post_weight", "gate", "gate_bias", "scale")),
                                             (BF16, F32, F32, ("next_weight", "post_weight"))])
@pytest.mark.parametrize("d", (1, 4, 36, 128, 520, 1000, 1001, 1024, 2048, 2056, 4096, 4100, 5120, 8192, 8200, 20000))
def test_a_row_does_not_depend_on_its_neighbours(d, y, gate, out, drop):
    a = inputs(ROWS, d, d, y, gate)
    for name in drop:
        a[name] = None
    a["residual"][5, 0] = -0.0
    if a["y"] is not None:
        a["y"][5, 0] = -0.0
    whole = the_pass(a, out, slice(0, ROWS))
    # alone, a few, as many as take a thread for every group of four, one more, and the rest
    cuts = (0, 1, 8, 304, 601, ROWS)
    for first, last in zip(cuts, cuts[1:]):
        for w, part in zip(whole, the_pass(a, out, slice(first, last))):
            assert torch.equal(w[first:last], part), (first, last)


def test_logits_of_a_float32_model_do_not_depend_on_the_cut():
    """Gates and scales around the sublayers, 32-bit path: two prompts in one step of 500 tokens, alone, and in portions."""
    spec = engine.sandwich_spec
    g = torch.Generator().manual_seed(8)
    tensors = {}
    for name, (shape, _) in spec(None).tensor_table().items():
        t = torch.randn(shape, generator=g)
        tensors[name] = (1 + 0.1 * t if len(shape) == 1 and not name.endswith(".b") else t if name.endswith(".b") else 0.03 * t if shape[0] != engine.VOCAB else 0.5 * t).to(BF16)
    a, b = random_tokens(engine.VOCAB, 250, 5), random_tokens(engine.VOCAB, 250, 6)
    every = list(range(250))
    register_architecture("SandwichGateLM", lambda raw: engine.ToyCfg("SandwichGateLM"), spec)
    try:
        r = ModelRunner(config=engine.ToyCfg("SandwichGateLM"), tensors=tensors, dtype="float32", max_tokens=1024, max_requests=4)
        both = r.step([StepEntry("a", a, every), StepEntry("b", b, every)], end=["a", "b"])
        alone = torch.cat([r.step([StepEntry(n, t, every)], end=[n]) for n, t in (("a", a), ("b", b))])
        cut = [r.step([StepEntry("c", a[:200], every[:200])]), r.step([StepEntry("c", a[200:249], every[:49])]), r.step([StepEntry("c", a[249:], [0])], end=["c"])]
    finally:
        unregister_architecture("SandwichGateLM")
    assert torch.equal(both, alone)
    assert torch.equal(torch.cat(cut), both[:250])


# ------------------------------------------------------------------ the gate

@pytest.mark.parametrize("tokens", (3, 700))
@pytest.mark.parametrize("y", (F32, BF16))
@pytest.mark.parametrize("gate", (F32, BF16))
def test_gates_and_biases_that_nearly_cancel(tokens, y, gate):
    """sigmoid(g + b) where both are large: what counts is the sum x, rounded once (half a step of x, which moves the sigmoid by |x| / 2 steps of
    2^-23 at most); the exponential's argument in base 2 has three roundings more for bfloat16 y (1.5 |x| steps of 2^-24), the functions, the quotient and
    the products a few."""
    d = 512
    g = torch.Generator(device="cuda").manual_seed(tokens)
    b = (torch.randn(d, generator=g, device="cuda") * 3e3).to(BF16).float()
    x = torch.randn((tokens, d), generator=g, device="cuda") * 4
    pre = (x - b).to(gate)
    a = inputs(tokens, d, 3, y, gate)
    into = torch.empty_like(a["residual"])
    ops.norm_gate_add(torch.zeros_like(into), a["y"], gate=pre, gate_bias=b, into=into)
    arg = pre.double() + b.double()
    want = a["y"].double() * torch.sigmoid(arg)
    assert ((into.double() - want).abs() <= want.abs() * (16 + 3 * arg.abs()) * 2.0 ** -24).all()


@pytest.mark.parametrize("tokens", (3, 700))
def test_a_closed_gate_of_32_bits(tokens):
    """32-bit y: the accurate functions, within 12 steps of 2^-24 however closed the gate is (the exponential 2 ulp = 4 steps, the sum and the quotient, the
    products); bfloat16 y: the argument's rounding too, 1.5 |x| steps.  Results below 2^-126 lie 2^-149 apart."""
    d = 640
    x = torch.linspace(-85, 20, d, device="cuda").repeat(tokens, 1)
    a = inputs(tokens, d, 5, F32, F32)
    for y in (F32, BF16):
        v = a["y"].to(y)
        into = torch.empty_like(a["residual"])
        ops.norm_gate_add(torch.zeros_like(into), v, gate=x, into=into)
        want = v.double() * torch.sigmoid(x.double())
        steps = 12 if y == F32 else 16 + 3 * x.double().abs()
        assert ((into.double() - want).abs() <= want.abs() * steps * 2.0 ** -24 + 2.0 ** -149).all()

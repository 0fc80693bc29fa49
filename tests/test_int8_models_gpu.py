"""Every architecture with its layers' matrices in 8 bits: which products are, and that each of them is the exact one over the 8-bit rows; Tubazen's
logits against its plain decoder with those products; and how far 8-bit weights move a decoder's logits."""
import pytest
import torch

import darovik_helpers
import deganex_helpers
import int8_plain
import lotirax_helpers
import lugizen_helpers
import nedasun_helpers
import plain_tubazen
import test_int8_engine_gpu as engine
import tubazen_helpers
from helpers import PlainModel, make_model_dir, random_tokens
from qorvix_b200 import ModelRunner, StepEntry
from qorvix_b200.csrc import ops
from qorvix_b200.parts import linear
from qorvix_b200.parts.shared_io import SharedIOMixer
from qorvix_b200.parts.side_by_side import SideBySide

pytestmark = pytest.mark.gpu
HELPERS = {"tubazen": tubazen_helpers, "lugizen": lugizen_helpers, "nedasun": nedasun_helpers, "lotirax": lotirax_helpers, "darovik": darovik_helpers,
           "deganex": deganex_helpers}
WITH_SHARED = ("tubazen", "lugizen", "nedasun")          # whose configurations have mixers with projections that can be shared


def tokens(vocab, n, seed):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def shared_mixers(model):
    """The mixers that own an input and an output product for themselves or for a pair."""
    found = []

    def look(m):
        if isinstance(m, SideBySide) and not m.shared:
            look(m.left), look(m.right)
        elif isinstance(m, SharedIOMixer):
            found.append(m)
        elif hasattr(m, "inner"):
            look(m.inner)

    for b in model.blocks:
        look(b.mixer)
    return found


@pytest.fixture
def small_too(monkeypatch):
    """The tests' matrices are small: all of them go into 8 bits."""
    monkeypatch.setattr(linear, "INT8_LEAST", 1)


@pytest.fixture
def checked(monkeypatch):
    """Every 8-bit product of a dense matrix is compared, as it runs, with the whole sums of the 8-bit rows."""
    whole, product, seen = ops.quantize_weight, ops.gemm_int8, {"matrices": {}, "products": 0}

    def quantize(w):
        q = whole(w)
        if w.dim() == 2:
            seen["matrices"][id(q)] = (q, *int8_plain.rows(w))
        return q

    def gemm(out, x, weight):
        product(out, x, weight)
        qw, sw = seen["matrices"][id(weight)][1:]
        qx, sx = (x.values.long(), x.scale) if isinstance(x, ops.Int8Rows) else int8_plain.rows(x)
        assert torch.equal(out, int8_plain.product32(qx, sx, qw, sw).to(out.dtype))
        seen["products"] += 1

    monkeypatch.setattr(ops, "quantize_weight", quantize)
    monkeypatch.setattr(ops, "gemm_int8", gemm)
    return seen


@pytest.mark.parametrize("config", ("CONFIG_A", "CONFIG_C", "CONFIG_D"))
@pytest.mark.parametrize("name", sorted(HELPERS))
def test_all_products_of_the_layers(name, config, small_too, checked):
    h = HELPERS[name]
    if not hasattr(h, config):
        pytest.skip("no such configuration")
    cfg = getattr(h, config)
    r = ModelRunner(str(h.make_model_dir(cfg, 3)), dtype="bfloat16", max_tokens=256, max_requests=2, page_size=16, weights="int8", use_graphs=False)
    mixers = shared_mixers(r.model)
    assert bool(mixers) == any(isinstance(getattr(b.mixer, "inner", b.mixer), SharedIOMixer) for b in r.model.blocks)
    if config == "CONFIG_A" and name in WITH_SHARED:
        assert mixers
    for m in mixers:                                      # when the model is loaded, not at a first step
        assert m._in is not None and m._in.int8 is not None and m._out.int8 is not None, type(m).__name__
    toks = tokens(cfg["vocab"], 40, 9)
    out = [r.step([StepEntry("a", toks[:33], list(range(33)))])] + [r.step([StepEntry("a", [t], [0])]) for t in toks[33:]]
    assert all(torch.isfinite(o).all() for o in out)
    assert checked["products"] >= 8 * 2 * len(mixers)     # eight steps
    ops.check_kernel_errors()


@pytest.mark.parametrize("name", sorted(WITH_SHARED))
def test_models_as_stored_have_nothing_in_8_bits(name, checked, small_too):
    h = HELPERS[name]
    r = ModelRunner(str(h.make_model_dir(h.CONFIG_A, 3)), dtype="bfloat16", max_tokens=128, max_requests=2, page_size=16)
    r.step([StepEntry("a", tokens(h.CONFIG_A["vocab"], 9, 9), [8])])
    assert all(m._in.int8 is None and m._out.int8 is None for m in shared_mixers(r.model)) and not checked["matrices"]


class Rows8:
    """A matrix whose products run over the 8-bit rows of the other side: h @ w.T."""

    def __init__(self, w):
        self.w = w

    def is_floating_point(self):
        return False

    @property
    def T(self):
        return self

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        h, rows = args
        qx, sx = int8_plain.rows(h.to(torch.bfloat16))
        qw, sw = int8_plain.rows(rows.w)
        return int8_plain.product64(qx, sx, qw, sw)


@pytest.mark.parametrize("config", ("CONFIG_A", "CONFIG_B", "CONFIG_C"))
def test_logits_of_a_model_with_shared_projections(config, small_too):
    cfg = getattr(tubazen_helpers, config)
    path = tubazen_helpers.make_model_dir(cfg, 5)
    W = tubazen_helpers.as_float64(tubazen_helpers.model_weights(cfg, 5))
    product = ("q", "k", "v", "g", "o", "a1", "r", "a", "w1", "gate", "up", "down")
    W = {n: Rows8(w) if n.startswith("l") and (n.split(".")[-1] in product or n.endswith(("rg1", "rg2"))) else w for n, w in W.items()}
    toks = tokens(cfg["vocab"], 95, 4)
    want = plain_tubazen.forward(cfg, W, toks)
    r = ModelRunner(str(path), dtype="bfloat16", max_tokens=256, max_requests=3, page_size=16, weights="int8")
    whole = r.step([StepEntry("w", toks, list(range(95)))], end=["w"])
    cut = [r.step([StepEntry("a", toks[:60], list(range(60)))]), r.step([StepEntry("a", toks[60:90], list(range(30)))])]
    cut += [r.step([StepEntry("a", [t], [0])]) for t in toks[90:]]
    # rows that differ by a bfloat16 rounding differ, of entries that are half a step of a row of max / rms r apart, by r / 127 in a quarter of the
    # entries: 0.5 r / 127 of the product's rms, r = 3 for rows of 20 to 100 numbers.  Four products in a chain a layer, in squares, and twice that
    # for the slopes of decays, softmax and norms: 2 * sqrt(4 * 4) * 0.5 * 3 / 127 = 9.4 % of the logits' rms in a usual row; four times
    # that in the worst
    for got, what in ((whole, "whole"), (torch.cat(cut), "in portions and single tokens")):
        d = got.double().cpu() - want
        rel = d.pow(2).mean(dim=-1).sqrt() / want.pow(2).mean().sqrt()
        assert float(rel.median()) < 0.094 and float(rel.max()) < 0.38, (what, float(rel.median()), float(rel.max()))
    ops.check_kernel_errors()


def test_logits_beside_those_of_the_model_as_stored():
    """A row of 1,024 normal numbers has its largest at 3.3 times their rms: a step is 3.3 / 127 of it and rounding to whole numbers of steps loses a uniform error,
    its rms 1 / sqrt(12) of a step, 0.75 % of the row's.  Rows and matrix each do that to a product, 1.06 %; eight products of two layers, in squares,
    3.0 % of the logits' rms.  No more than twice that, and no less than a quarter (or nothing was rounded)."""
    path = make_model_dir(engine.CFG, seed=4)
    toks = random_tokens(engine.CFG.vocab_size, 150, 3)
    ref = PlainModel(path).logits(toks).double()
    off = {}
    for weights in ("stored", "int8"):
        r = ModelRunner(str(path), dtype="bfloat16", max_tokens=512, max_requests=2, weights=weights)
        got = r.step([StepEntry("w", toks, list(range(150)))], end=["w"]).double().cpu()
        off[weights] = float((got - ref).pow(2).mean().sqrt() / ref.pow(2).mean().sqrt())
    print(off)
    assert 0.0075 < off["int8"] < 0.06 and off["stored"] < off["int8"], off

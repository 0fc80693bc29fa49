"""Models whose layers keep their matrices in 8 bits: logits against the plain decoder with every product of a layer formed from 8-bit rows,
routed experts and sandwich-norm blocks with gates and scales against float64."""
from dataclasses import dataclass
from types import SimpleNamespace

import pytest
import torch

import int8_plain
import plain_llama as plain
from helpers import ARCH, CallCounter, PlainModel, assert_close_logits, make_model_dir, random_tokens
from qorvix_b200 import LLM, LlamaConfig, ModelRunner, SamplingParams, StepEntry
from qorvix_b200.config import ModelConfig, register_architecture, unregister_architecture
from qorvix_b200.csrc import ops
from qorvix_b200.parts import (AttentionSpec, LayerSpec, ModelSpec, RMSNormSpec, RotarySpec, Runtime, SwiGLUSpec, build_part)
from qorvix_b200.parts.linear import Linear, int8_weights
from qorvix_b200.parts.spec import MoESpec
from qorvix_b200.weights import TensorSource

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")

# every layer's matrices have 2^20 entries or more (the fused query, key and value projection as a whole), the head's has not
CFG = LlamaConfig(architecture=ARCH, vocab_size=301, hidden_size=1024, intermediate_size=2048, num_hidden_layers=2, num_attention_heads=8,
                  num_key_value_heads=2, head_dim=128, max_position_embeddings=256, rms_norm_eps=1e-5, rope_theta=40000.0, tie_word_embeddings=False)


def linear8(x, w):
    """A product over the 8-bit rows of the bfloat16 rows, in 64 bits."""
    flat = x.reshape(-1, x.shape[-1])
    qx, sx = int8_plain.rows(flat.to(torch.bfloat16))
    qw, sw = int8_plain.rows(w)
    return int8_plain.product64(qx, sx, qw, sw).reshape(*x.shape[:-1], w.shape[0])


def assert_close8(got, ref, products, what):
    """The engine's rows and the plain decoder's differ by bfloat16 rounding, 2^-8 of an entry, up to half a step of the 8-bit row for its
    largest entries and an eighth for usual ones: at most a quarter of the entries go to another whole number, a step away.  A step is r / 127
    of the row's root mean square, r = max / rms, 4 at the most for rows of 1,024 normal numbers: a product is off by sqrt(1/4) * 4 / 127 = 1.6 % of its rms.  `products`
    in a chain add in squares; the largest of some 10^4.7 errors is 4.3 times their rms, the largest logit at least 4 times the logits'."""
    got, ref = got.detach().double().cpu(), ref.double()
    bound = 0.5 * 4 / 127 * products ** 0.5 * 4.3 / 4 * float(ref.abs().max())
    err = float((got - ref).abs().max())
    assert got.shape == ref.shape and err <= bound, (what, err, bound)


@pytest.fixture(scope="module")
def model_dir():
    return make_model_dir(CFG, seed=4)


@pytest.fixture
def plain8(model_dir, monkeypatch):
    """The plain decoder whose layers' products run over 8-bit rows (the head's do not)."""
    whole = plain.linear
    monkeypatch.setattr(plain, "linear", lambda x, w: whole(x, w) if w.shape[0] == CFG.vocab_size else linear8(x, w))
    return PlainModel(model_dir)


def test_a_decoder_in_8_bits(model_dir, plain8, monkeypatch):
    counts = CallCounter(monkeypatch, "gemm_int8", "gemm_int8_glu", "norm_gate_add")
    toks = random_tokens(CFG.vocab_size, 150, 3)
    ref = plain8.logits(toks)
    r = ModelRunner(str(model_dir), dtype="bfloat16", max_tokens=512, max_requests=3, weights="int8")
    assert r.model.blocks[0].mixer.qkv_proj.int8 is not None and r.model.lm_head.int8 is None
    whole = r.step([StepEntry("w", toks, list(range(150)))], end=["w"])
    assert_close8(whole, ref, 8, "whole")
    got = [r.step([StepEntry("a", toks[:70], list(range(70)))]), r.step([StepEntry("a", toks[70:140], list(range(70)))])]
    got += [r.step([StepEntry("a", [toks[i]], [0])]) for i in range(140, 150)]           # captured steps
    assert_close8(torch.cat(got), ref, 8, "in portions and single tokens")
    assert counts["gemm_int8_glu"] > 0 and counts["gemm_int8"] > 0 and counts["norm_gate_add"] > 0
    ops.check_kernel_errors()


def test_generation_in_8_bits_follows_the_plain_decoder(model_dir, plain8):
    from helpers import assert_greedy_follows_plain
    prompts = [random_tokens(CFG.vocab_size, n, n) for n in (5, 40)]
    llm = LLM(str(model_dir), dtype="bfloat16", max_tokens=512, weights="int8")
    out = llm.generate(prompts, SamplingParams.greedy_params(max_new_tokens=6))
    compared = [assert_greedy_follows_plain(plain8, p, o.tokens, at_least=0) for p, o in zip(prompts, out)]
    assert all(len(o.tokens) == 6 for o in out) and max(compared) >= 1


def test_the_matrices_take_half_the_room(model_dir):
    def room(weights):
        before = torch.cuda.memory_allocated()
        r = ModelRunner(str(model_dir), dtype="bfloat16", max_tokens=64, weights=weights)
        return torch.cuda.memory_allocated() - before, r

    stored, a = room("stored")
    del a
    int8, b = room("int8")
    matrices = 2 * (1536 * 1024 + 1024 * 1024 + 3 * 2048 * 1024)
    assert stored - int8 > 0.9 * matrices                                                # a byte an entry less, but for the scales


def test_the_command_line_takes_them(model_dir, capsys):
    from qorvix_b200.cli.main import main
    assert main(["generate", str(model_dir), "--tokens", "1,2,3", "--max", "3", "--temp", "0", "--weights", "int8"]) == 0
    assert "3 prompt tokens, 3 generated" in capsys.readouterr().out
    assert main(["bench", str(model_dir), "--prompt", "4", "--gen", "2", "--runs", "1", "--weights", "int8", "--json"]) == 0
    assert main(["generate", str(model_dir), "--tokens", "1,2,3", "--weights", "int9"]) == 1


# ------------------------------------------------------------------ routed experts

@pytest.mark.parametrize("tokens", (1, 7, 70, 400))
def test_routed_experts_in_8_bits(tokens):
    d, ff, E, top = 1024, 1040, 5, 2
    g = torch.Generator().manual_seed(tokens)
    spec = MoESpec(hidden_size=d, experts=E, top=top, expert_ff=ff, router="r", expert_prefix="e", activation="clamped", limit=7.0, slope=1.702)
    tensors = {n: (torch.randn(shape, generator=g) * (0.2 if n == "r" else 0.03)).to(torch.bfloat16) for n, (shape, _) in spec.tensors().items()}
    with int8_weights():
        part = build_part("feed_forward", spec, TensorSource(tensors=tensors, device=DEV, compute_dtype=torch.bfloat16),
                          Runtime(DEV, torch.bfloat16, 64, weights="int8"))
    assert part.int8 is not None
    x = torch.randn(tokens, d, generator=g).to(torch.bfloat16)
    got = part.forward(x.to(DEV), SimpleNamespace())
    w = {n: t.double() for n, t in tensors.items()}
    logits = x.double() @ w["r"].T
    val, idx = logits.topk(top, dim=1)
    weight = torch.softmax(val, dim=1)
    want = torch.zeros(tokens, d, dtype=torch.float64)
    for t in range(tokens):
        for j in range(top):
            e = int(idx[t, j])
            h = x[t:t + 1].double()
            gate, up = linear8(h, w[f"e{e}.gate"]).clamp(max=7.0), linear8(h, w[f"e{e}.up"]).clamp(-7.0, 7.0)
            act = (gate * torch.sigmoid(1.702 * gate) * (up + 1)).to(torch.bfloat16).double()
            want[t] += weight[t, j] * linear8(act, w[f"e{e}.down"])[0]
    # act's entries, equal up to float32 rounding, may round to neighbouring bfloat16 numbers (one in 2^14 or fewer: 2^-24 times some tens of steps
    # against 2^-9) and then to neighbouring whole numbers: of 1,040 entries at most a few, each a step of 1/127 of the largest times a weight of
    # some 4 rms; an output's largest value is over 2.5 rms of 1,040 such terms
    assert (got.double().cpu() - want).abs().max() <= 3 * (4 / 127) * 4 / 1040 ** 0.5 / 2.5 * want.abs().max()
    ops.check_kernel_errors()


# ------------------------------------------------------------------ sandwich norms with gates and scales

@dataclass(frozen=True)
class ToyCfg(ModelConfig):
    def to_dict(self):
        return {"architectures": [self.architecture]}


D, F, VOCAB, HD = 1024, 1056, 211, 64


def sandwich_spec(cfg):
    layers = []
    for i in range(3):
        p = f"l{i}."
        # the second layer has a gate and no scale, the third neither
        layers.append(LayerSpec(
            mixer=AttentionSpec(hidden_size=D, num_heads=16, num_kv_heads=4, head_dim=HD, scale=HD ** -0.5, q_proj=p + "q", k_proj=p + "k", v_proj=p + "v",
                                o_proj=p + "o", position=RotarySpec(HD, HD, 10000.0)),
            feed_forward=SwiGLUSpec(D, F, p + "gate", p + "up", p + "down"), block="sandwich_norm",
            mixer_norm=RMSNormSpec(D, 1e-5, p + "n1"), mixer_post_norm=RMSNormSpec(D, 1e-5, p + "n1b"), ffn_norm=RMSNormSpec(D, 1e-5, p + "n2"),
            ffn_post_norm=RMSNormSpec(D, 1e-5, p + "n2b"), mixer_gate=p + "mg" if i < 2 else None, ffn_gate=p + "fg" if i < 2 else None,
            mixer_scale=p + "ms" if i < 1 else None, ffn_scale=p + "fs" if i < 1 else None))
    return ModelSpec(architecture="SandwichGateLM", vocab_size=VOCAB, hidden_size=D, embedding="emb", layers=layers, final_norm=RMSNormSpec(D, 1e-5, "fn"),
                     lm_head="head", max_position=256)


def sandwich_plain(w, tokens, product):
    pos, inv = torch.arange(len(tokens)), plain.plain_inv_freq(HD, 10000.0)
    x = w["emb"][torch.tensor(tokens)]
    for i in range(3):
        p = f"l{i}."

        def add(x, y, h, gate, scale, norm):
            z = plain.rmsnorm(y, w[p + norm], 1e-5)
            if p + gate in w:
                z = z * torch.sigmoid(product(h, w[p + gate]) + w[p + gate + ".b"])
            return x + z * (w[p + scale] if p + scale in w else 1.0)

        h = plain.rmsnorm(x, w[p + "n1"], 1e-5)
        q = plain.rope(product(h, w[p + "q"]).reshape(-1, 16, HD), pos, inv)
        k = plain.rope(product(h, w[p + "k"]).reshape(-1, 4, HD), pos, inv)
        a = plain.attention(q, k, product(h, w[p + "v"]).reshape(-1, 4, HD)).reshape(-1, 16 * HD)
        x = add(x, product(a, w[p + "o"]), h, "mg", "ms", "n1b")
        h = plain.rmsnorm(x, w[p + "n2"], 1e-5)
        y = product(plain.swiglu(product(h, w[p + "gate"]), product(h, w[p + "up"])), w[p + "down"])
        x = add(x, y, h, "fg", "fs", "n2b")
    return plain.rmsnorm(x, w["fn"], 1e-5) @ w["head"].T


@pytest.mark.parametrize("dtype,weights", [("float32", "stored"), ("bfloat16", "stored"), ("bfloat16", "int8")])
def test_sandwich_norms_with_gates_and_scales(dtype, weights):
    g = torch.Generator().manual_seed(8)
    tensors = {}
    for name, (shape, _) in sandwich_spec(None).tensor_table().items():
        t = torch.randn(shape, generator=g)
        t = 1 + 0.1 * t if len(shape) == 1 and not name.endswith(".b") else t if name.endswith(".b") else 0.03 * t if shape[0] != VOCAB else 0.5 * t
        tensors[name] = t.to(torch.bfloat16)
    w = {k: v.double() for k, v in tensors.items()}
    toks = random_tokens(VOCAB, 120, 5)
    ref = sandwich_plain(w, toks, linear8 if weights == "int8" else plain.linear)
    register_architecture("SandwichGateLM", lambda raw: ToyCfg("SandwichGateLM"), sandwich_spec)
    try:
        r = ModelRunner(config=ToyCfg("SandwichGateLM"), tensors=tensors, dtype=dtype, max_tokens=512, max_requests=2, weights=weights)
        whole = r.step([StepEntry("w", toks, list(range(120)))], end=["w"])
        close = (lambda got, what: assert_close8(got, ref, 3 * 4 + 4, what)) if weights == "int8" else (lambda got, what: assert_close_logits(got, ref, dtype, what))
        close(whole, "whole")
        got = [r.step([StepEntry("a", toks[:90], list(range(90)))]), r.step([StepEntry("a", toks[90:114], list(range(24)))])]
        got += [r.step([StepEntry("a", [toks[i]], [0])]) for i in range(114, 120)]
        close(torch.cat(got), "in portions and single tokens")
        ops.check_kernel_errors()
    finally:
        unregister_architecture("SandwichGateLM")


def test_small_matrices_and_marked_ones_stay_as_stored():
    w = torch.randn(1024, 1024, device=DEV).to(torch.bfloat16)
    with int8_weights():
        assert Linear(w).int8 is not None and Linear(w[:1023]).int8 is None and Linear(w, as_stored=True).int8 is None and Linear(w.float()).int8 is None
    assert Linear(w).int8 is None

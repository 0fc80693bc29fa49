"""The 8-bit operators as they are used: one after the other, captured and replayed, on a stream of their own, over matrices that were laid out
a moment ago, beside rows that belong to others."""
import pytest
import torch

import int8_plain as plain
from qorvix_b200.csrc import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)


def matrix(g, n, k):
    return torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8), torch.rand(n, generator=g, device="cuda") / (64 * k ** 0.5)


class Sublayer:
    """Norms with a gate and a scale, a gate/up product over their 8-bit rows, a down product."""

    def __init__(self, d, f, seed):
        g = gen(seed)
        self.d, self.f = d, f
        self.q1, self.s1 = matrix(g, 2 * f, d)
        self.q2, self.s2 = matrix(g, d, f)
        self.w1, self.w2 = ops.pack_int8(self.q1, self.s1), ops.pack_int8(self.q2, self.s2)
        self.vectors = dict(post_weight=normal(g, d, std=0.1, mean=1.0), post_eps=1e-5, gate_bias=normal(g, d), scale=normal(g, d, std=0.1, mean=0.7),
                            next_weight=normal(g, d, std=0.1, mean=1.0), next_eps=1e-5)

    def inputs(self, tokens, seed):
        g = gen(seed)
        return dict(residual=normal(g, tokens, self.d, std=2.0), y=normal(g, tokens, self.d, dtype=BF16), gate=normal(g, tokens, self.d))

    def __call__(self, residual, y, gate):
        tokens = residual.shape[0]
        stream, rows = torch.empty_like(residual), ops.int8_rows(tokens, self.d, residual.device)
        ops.norm_gate_add(residual, y, gate=gate, out=rows, into=stream, **self.vectors)
        act = torch.empty((tokens, self.f), device="cuda", dtype=BF16)
        ops.gemm_int8_glu(act, rows, self.w1)
        out = torch.empty((tokens, self.d), device="cuda", dtype=BF16)
        ops.gemm_int8(out, act, self.w2)
        return stream, rows.values.clone(), rows.scale.clone(), act, out

    def check(self, got, residual, y, gate):
        """Each step against 64 bits from what the step before gave."""
        stream, q, s, act, out = got
        want, rows = plain.norm_gate64(residual, y, gate=gate, **self.vectors)
        assert ((stream.double() - want).abs() <= (residual.abs() + (want - residual).abs()) * 64 * 2.0 ** -24).all()
        # the rows are those of bfloat16 rows that are within a rounding (and float32's errors) of the exact ones
        step = s.double()[:, None]
        assert ((q.double() * step - rows).abs() <= step * 0.51 + rows.abs() * 2.0 ** -8).all()
        z = plain.gated64(plain.product64(q, s, self.q1, self.s1), 0, 0.0, 0.0)
        arg = plain.product64(q, s, self.q1, self.s1).abs().max()
        assert ((act.double() - z).abs() <= z.abs() * (2.0 ** -8 + (16 + 14 * arg) * 2.0 ** -24) + 1e-30).all()
        qa, sa = plain.rows(act)
        assert torch.equal(out, plain.product32(qa, sa, self.q2, self.s2).to(BF16))


@pytest.mark.parametrize("tokens,d,f", [(1, 512, 96), (5, 1024, 528), (33, 264, 80), (300, 512, 1040)])
def test_a_sublayer_and_its_replays(tokens, d, f):
    layer = Sublayer(d, f, tokens + d)
    first = layer.inputs(tokens, 1)
    layer.check(layer(**first), **first)
    held = {k: v.clone() for k, v in first.items()}
    graphs = []
    for _ in range(2):                                # two graphs of the same calls live side by side
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = layer(**held)
        graphs.append((g, got))
    for seed in (2, 3):
        new = layer.inputs(tokens, seed)
        for k, v in new.items():
            held[k].copy_(v)
        for g, _ in graphs + graphs[:1]:
            g.replay()
        torch.cuda.synchronize()
        for _, got in graphs:
            layer.check(got, **new)
    ops.check_kernel_errors()


def test_on_two_streams_at_once():
    """Two streams run different sublayers; nothing that a call needs is shared between them."""
    layers = [Sublayer(1024, 512, 5), Sublayer(768, 1040, 6)]
    inputs = [[layer.inputs(t, 10 * t) for t in (3, 40, 200)] for layer in layers]
    streams = [torch.cuda.Stream() for _ in layers]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for i, (layer, s) in enumerate(zip(layers, streams)):
            with torch.cuda.stream(s):
                got[i] = [layer(**x) for x in inputs[i]]
    torch.cuda.synchronize()
    for layer, xs, gs in zip(layers, inputs, got):
        for x, g in zip(xs, gs):
            layer.check(g, **x)
    ops.check_kernel_errors()


@pytest.mark.parametrize("tokens", (1, 4, 30, 100))
def test_matrices_that_were_laid_out_a_moment_ago(tokens):
    """The products ask for weights before they wait for the kernel ahead: it must not matter that the matrix, in memory that held another one, was
    written just before."""
    g = gen(tokens)
    x = normal(g, tokens, 640, dtype=BF16)
    qx, sx = plain.rows(x)
    mats = [matrix(g, 1000, 640) for _ in range(6)]
    outs = []
    for q, s in mats:
        out = torch.empty((tokens, 1000), device="cuda", dtype=F32)
        w = ops.pack_int8(q, s)
        ops.gemm_int8(out, x, w)
        del w                                         # its memory goes to the next one
        outs.append(out)
    for (q, s), out in zip(mats, outs):
        assert torch.equal(out, plain.product32(qx, sx, q, s))
    w = torch.randn(1000, 640, generator=g, device="cuda").to(BF16)
    out = torch.empty((tokens, 1000), device="cuda", dtype=F32)
    ops.gemm_int8(out, x, ops.quantize_weight(w))
    qw, sw = plain.rows(w)
    assert torch.equal(out, plain.product32(qx, sx, qw, sw))
    ops.check_kernel_errors()


def test_tables_that_do_not_fit_write_nothing_outside():
    """Entries that name no expert or no rows are passed over; tiles are cut at the rows there are and at the tiles' rows."""
    g = gen(9)
    R, E, n, k, tr = 70, 3, 64, 128, 32
    x = normal(g, R, k, dtype=BF16)
    q, s = zip(*(matrix(g, n, k) for _ in range(E)))
    w = ops.pack_int8(torch.stack(q), torch.stack(s))
    rows = ops.int8_rows(R, k, "cuda")
    ops.quantize_rows(rows, x)
    qx, sx = plain.rows(x)
    room = torch.full((R + 20, n), 9.0, device="cuda")
    table = [(0, 0, 32), (2, 60, 500), (1, 40, 200), (E, 33, 3), (-1, 34, 2), (0, -5, 3), (0, 35, 0)]       # the second and third are longer than what is left or a tile
    ops.moe_experts_int8(False, room[:R], rows, w, torch.tensor(table, dtype=torch.int32, device="cuda").reshape(-1), tile_rows=tr)
    got = room.clone()
    assert (room[32:40] == 9.0).all() and (room[R:] == 9.0).all()
    assert torch.equal(got[:32], plain.product32(qx[:32], sx[:32], q[0], s[0]))
    assert torch.equal(got[40:60], plain.product32(qx[40:60], sx[40:60], q[1], s[1]))
    ops.check_kernel_errors()


def test_a_first_call_inside_a_capture_is_refused_or_prepared(monkeypatch):
    monkeypatch.setattr(ops, "_err_words", {})
    monkeypatch.setattr(ops, "_tc_state", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(ops.KernelError, match="prepare_products"):
        ops._err_word(torch.cuda.current_device())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert ops._err_word(torch.cuda.current_device()) > 0


def test_other_types_are_refused():
    x = torch.zeros(2, 64, device="cuda", dtype=torch.float16)
    w = ops.pack_int8(torch.zeros(64, 64, device="cuda", dtype=torch.int8), torch.zeros(64, device="cuda"))
    out = torch.zeros(2, 64, device="cuda", dtype=BF16)
    for call in (lambda: ops.quantize_rows(ops.int8_rows(2, 64, "cuda"), x), lambda: ops.gemm_int8(out, x, w), lambda: ops.gemm_int8(x, out, w),
                 lambda: ops.norm_gate_add(torch.zeros(2, 64, device="cuda"), x), lambda: ops.gemm_int8(out.cpu(), out, w),
                 lambda: ops.gemm_int8(out, out.cpu(), w)):
        with pytest.raises(ops.KernelError):
            call()

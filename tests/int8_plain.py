"""The 8-bit operators from their definitions, in whole numbers and 64 bits, on the CPU or wherever the tensors are."""
import math

import torch


def rows(x):
    """(q int64, scale float32) of the rows of x: the quotient 127 x / top in 64 bits is exact enough to tell on which side of a border it
    lies (a quotient of a 31-bit and a 24-bit number that is no half-integer differs from it by 2^-25 of itself or more)."""
    x = x.double()
    top = x.abs().amax(dim=1, keepdim=True) if x.shape[1] else x.new_zeros(x.shape[0], 1)
    bad = ~torch.isfinite(x).all(dim=1, keepdim=True)
    q = torch.where(bad | (top == 0), 0.0, (127.0 * x / torch.where(top == 0, 1.0, top)).round())
    q = torch.where(torch.isfinite(q), q, 0.0)
    scale = torch.where(bad, float("nan"), top / 127.0).float()
    return q.long(), scale[:, 0]


def sums(qx, qw):
    """The whole sums, exactly (float64 holds them: they stay below 2^31)."""
    return (qx.double() @ qw.double().T).round()


def product32(qx, sx, qw, sw):
    """The product as the operator rounds it, in float32: the sum, times the token's scale, times the channel's."""
    return sums(qx, qw).float() * sx[:, None] * sw[None, :]


def product64(qx, sx, qw, sw):
    return sums(qx, qw) * sx.double()[:, None] * sw.double()[None, :]


def gated64(z, act, limit, slope):
    """[T, 2f] -> [T, f], 16 gate features and the 16 up features that go with them in turn; act 0 SiLU, 1 tanh GELU, 2 clamped."""
    z = z.double().view(z.shape[0], z.shape[1] // 32, 2, 16)
    g, u = z[:, :, 0].reshape(z.shape[0], z.shape[1] * 16), z[:, :, 1].reshape(z.shape[0], z.shape[1] * 16)
    if act == 1:
        return g / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u     # (1 + tanh x) / 2, also where that is tiny
    if act == 2:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        return g / (1 + torch.exp(-slope * g)) * (u + 1)
    return g / (1 + torch.exp(-g)) * u


def norm_gate64(residual, y=None, post_weight=None, post_eps=0.0, gate=None, gate_bias=None, scale=None, next_weight=None, next_eps=0.0):
    """(new stream, rows) in 64 bits."""
    def rms(v, eps):
        return (v.square().mean(dim=1, keepdim=True) + eps).sqrt()

    stream = residual.double()
    if y is not None:
        z = y.double()
        if post_weight is not None:
            z = z / rms(z, post_eps) * post_weight.double()
        if gate is not None:
            z = z * torch.sigmoid(gate.double() + (gate_bias.double() if gate_bias is not None else 0.0))
        if scale is not None:
            z = z * scale.double()
        stream = stream + z
    return stream, stream if next_weight is None else stream / rms(stream, next_eps) * next_weight.double()


def tile_table(counts, tile_rows, tiles, device):
    """(expert, first row, rows) of every tile, padded with (-1, 0, 0)."""
    table, first = [], 0
    for e, n in enumerate(counts):
        table += [(e, first + r, min(tile_rows, n - r)) for r in range(0, n, tile_rows)]
        first += n
    table += [(-1, 0, 0)] * (tiles - len(table))
    return torch.tensor(table, dtype=torch.int32, device=device).reshape(-1)

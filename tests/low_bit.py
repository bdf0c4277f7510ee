"""Plain 64-bit forms of the 4-bit and mixture-of-experts entry points, and the error bounds their results are held to.

Bounds.  A result is fl(y) with y computed in 32 bits: half a step of the 16-bit type, plus the summation.  Products of
a 16-bit number and a small integer are exact in 32 bits.  A group of 128 is summed in at most 8 steps of a matrix
instruction, each of which may lose up to 2 units of 2^-23 of the sum of magnitudes; the groups follow in a chain of
ceil(k / 128) additions and at most 16 more across warps and blocks, half a unit of 2^-23 each.  Together
    |err| <= eps / 2 |y| + (48 + k / 128) 2^-24 sum |terms|    (and the 16-bit type's smallest step below its normal range).
"""
import math

import torch

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}


def chain(k):
    return (48 + k / 128) * 2.0 ** -24


def make_w4(gen, m, k, group, zeros, dt):
    """codes (m, k) as numbers, scales and zero points, on the CPU."""
    g = -(-k // group)
    codes = torch.randint(0, 16, (m, k), generator=gen, dtype=torch.uint8)
    scales = (0.002 + 0.01 * torch.rand(m, g, generator=gen)).to(dt)
    zps = torch.randint(0, 16, (m, g), generator=gen, dtype=torch.uint8) if zeros else None
    return codes, scales, zps


def two_a_byte(codes):
    m, k = codes.shape
    if k % 2:
        codes = torch.cat((codes, torch.full((m, 1), 9, dtype=torch.uint8)), dim=1)
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous()


def weights64(codes, scales, zps, group):
    grp = torch.arange(codes.shape[1]) // group
    z = 8.0 if zps is None else zps.double()[:, grp]
    return (codes.double() - z) * scales.double()[:, grp]


def pack(mm, dtype, codes, scales, zps, group, device="cuda"):
    m, k = codes.shape
    g = scales.shape[1]
    out = torch.full((mm.w4_bytes(m, k, group, zps is not None) + 64,), 0xA5, dtype=torch.uint8, device=device)
    c = two_a_byte(codes).to(device)
    mm.w4_pack(dtype, m, k, group, c, c.shape[1], scales.to(device), g, None if zps is None else zps.to(device), g, out)
    torch.cuda.synchronize()
    assert (out[-64:] == 0xA5).all(), "written past the packed matrix"
    return out


def padded(t, ld, dt, fill=float("nan")):
    """(columns, rows) tensor -> device buffer with leading dimension ld and a guard on both sides; returns (buffer, view)."""
    n, k = t.shape
    buf = torch.full((n * ld + 128,), fill, dtype=dt, device="cuda")
    view = buf[64:64 + n * ld].view(n, ld)
    view[:, :k].copy_(t)
    return buf, view


def round64(w, group, zeros, dt):
    """The 4-bit round trip of (m, k) 16-bit weights, in 64 bits: the values that come back (unrounded)."""
    out = torch.empty(w.shape, dtype=torch.float64)
    for lo in range(0, w.shape[1], group):
        x = w[:, lo:lo + group].double()
        if zeros:
            bot, top = x.min(1, keepdim=True).values.clamp(max=0), x.max(1, keepdim=True).values.clamp(min=0)
            s = ((top - bot) / 15).to(dt).double()
            z = torch.where(s > 0, torch.round(-bot / s).clamp(0, 15), torch.zeros_like(s))
        else:
            s = (x.abs().max(1, keepdim=True).values / 7).to(dt).double()
            z = torch.full_like(s, 8)
        q = torch.where(s > 0, (torch.round(x / torch.where(s > 0, s, torch.ones_like(s))) + z).clamp(0, 15), z)
        out[:, lo:lo + group] = (q - z) * s
    return out


def score_gaps(x, router, topk):
    """Per token: the smallest difference between scores whose order decides anything (infinite where there is none),
    and the error of a score summed in 32 bits."""
    scores = x @ router.t()
    slack = chain(x.shape[1]) * (x.abs() @ router.abs().t()).max(1).values
    s = torch.sort(scores, dim=1, descending=True).values[:, :topk + 1]
    if s.shape[1] < 2:
        return torch.full_like(slack, float("inf")), slack
    return (s[:, :-1] - s[:, 1:]).min(1).values, slack


def moe64(x, router, gate, up, down, topk, renorm):
    """x (tokens, d), router (E, d), gate / up (E, f, d), down (E, d, f), all 64-bit.  Returns y, ids, gates, a
    bound on the error of a 32-bit evaluation of y (without the final rounding), and one on the gates' (relative)."""
    tokens, d = x.shape
    f = gate.shape[1]
    scores = x @ router.t()
    slack = chain(d) * (x.abs() @ router.abs().t()).max(1).values  # of a score
    p = torch.softmax(scores, 1)
    order = torch.argsort(scores, dim=1, descending=True, stable=True)
    ids = order[:, :topk]
    gates = torch.gather(p, 1, ids)
    if renorm:
        gates = gates / gates.sum(1, keepdim=True)
    # exp(v - max): both shift by slack; exp, sum and division lose a few units of 2^-24 each
    grel = 4 * slack + (16 + scores.shape[1] / 16) * 2.0 ** -24
    y = torch.zeros_like(x)
    bound = torch.zeros_like(x)
    for t in range(tokens):
        for j in range(topk):
            e = int(ids[t, j])
            g, u = gate[e] @ x[t], up[e] @ x[t]
            eg, eu = chain(d) * (gate[e].abs() @ x[t].abs()), chain(d) * (up[e].abs() @ x[t].abs())
            sig = torch.sigmoid(g)
            h = g * sig * u
            # |silu'| <= 1.1; exp and the division lose a few 2^-24; h is held to 2^-16 of itself or better, and to
            # 2^-18 absolutely where it is stored scaled down by 2^6 in half precision
            eh = 1.1 * eg * u.abs() + (g * sig).abs() * eu + 1.1 * eg * eu + h.abs() * 2.0 ** -16 + 2.0 ** -18
            o = down[e] @ h
            y[t] += gates[t, j] * o
            bound[t] += gates[t, j] * (down[e].abs() @ (eh + chain(f) * h.abs()) + (grel[t] + 2.0 ** -20) * o.abs())
    return y, ids, gates, bound, grel


def check16(got, want, bound, dtype):
    """|got - want| <= bound + half a step of the 16-bit type (of the larger neighbour)."""
    eps = torch.finfo(TYPES[dtype]).eps
    lim = bound + eps / 2 * (want.abs() + bound) + TINY[dtype]
    err = (got.double() - want).abs()
    worst = (err / lim).max().item() if err.numel() else 0.0
    assert torch.isfinite(got.double()).all() and worst <= 1.0, f"error {worst:.3g} times the bound"
    return worst

"""A whole mixture-of-experts layer for a few tokens against its formula in 64 bits."""
import math
import pathlib
import subprocess
import sys

import pytest
import torch

from low_bit import TYPES, check16, make_w4, moe64, pack, padded, round64, score_gaps, weights64

pytestmark = pytest.mark.gpu


class Layer:
    def __init__(self, mm, dtype, tokens, d, f, experts, topk, renorm=False, group=0, zeros=False, seed=0, pads=(0, 0, 0),
                 x=None):
        gen = torch.Generator().manual_seed(seed * 7 + tokens * 1009 + d * 31 + f)
        dt = TYPES[dtype]
        self.__dict__.update(mm=mm, dtype=dtype, dt=dt, tokens=tokens, d=d, f=f, experts=experts, topk=topk, renorm=renorm,
                             group=group, zeros=zeros)
        self.x = torch.randn(tokens, d, generator=gen).to(dt) if x is None else x.to(dt)
        self.router = (torch.randn(experts, d, generator=gen) * 2 / math.sqrt(d)).to(dt)
        for _ in range(200):  # tokens whose choice of experts hangs on the last bits are drawn again
            gap, slack = score_gaps(self.x.double(), self.router.double(), topk)
            close = ~(gap > 8 * slack)
            if x is not None or not close.any():
                break
            self.x[close] = torch.randn(int(close.sum()), d, generator=gen).to(dt)
        pw, pr, px = pads
        self.dev, self.ref = {}, {}
        for name, r, c in (("gate", f, d), ("up", f, d), ("down", d, f)):
            if group:
                parts = [make_w4(gen, r, c, group, zeros, dt) for _ in range(experts)]
                self.ref[name] = torch.stack([weights64(*p, group) for p in parts])
                self.dev[name] = torch.stack([pack(mm, dtype, *p, group) for p in parts])  # 64 spare bytes each
            else:
                w = (torch.randn(experts, r, c, generator=gen) / math.sqrt(c)).to(dt)
                self.ref[name] = w.double()
                buf = torch.full((experts, r, c + pw), float("nan"), dtype=dt, device="cuda")
                buf[:, :, :c] = w
                self.dev[name] = buf
        self.router_dev = torch.full((experts, d + pr), float("nan"), dtype=dt, device="cuda")
        self.router_dev[:, :d] = self.router
        self.xbuf, self.xdev = padded(self.x, d + px, dt)

    def call(self, Y, beta=0.0, ids=None, gates=None, ws=None, stream=None, tokens=None):
        g, dn = self.dev["gate"], self.dev["down"]
        if self.group:
            st = dict(ldg=0, strideG=g.stride(0), ldd=0, strideD=dn.stride(0))
        else:
            st = dict(ldg=g.stride(1), strideG=g.stride(0), ldd=dn.stride(1), strideD=dn.stride(0))
        tokens = self.tokens if tokens is None else tokens
        if ws is None:
            ws = torch.full((self.mm.moe_workspace_bytes(self.dtype, tokens, self.d, self.f, self.experts, self.topk),),
                            0xFF, dtype=torch.uint8, device="cuda")
        self.mm.moe(self.dtype, tokens, self.d, self.f, self.experts, self.topk, self.xdev, self.xdev.shape[1],
                    self.router_dev, self.router_dev.shape[1], g, self.dev["up"], down=dn, Y=Y, ldy=Y.shape[1],
                    group=self.group, zeros=self.zeros, renorm=self.renorm, beta=beta, ids=ids, gates=gates, workspace=ws,
                    stream=stream, **st)
        return ws

    def check(self, beta=0.0, ldy=None):
        y, want_ids, want_gates, bound, grel = moe64(self.x.double(), self.router.double(), self.ref["gate"],
                                                     self.ref["up"], self.ref["down"], self.topk, self.renorm)
        gap, slack = score_gaps(self.x.double(), self.router.double(), self.topk)
        assert (gap > 4 * slack).all(), "the inputs leave the choice of experts open"
        c = torch.randn(self.tokens, self.d, generator=torch.Generator().manual_seed(1)).to(self.dt)
        buf, Y = padded(c if beta else torch.full_like(c, float("nan")), ldy or self.d, self.dt)
        before = buf.clone()
        ids = torch.full((self.tokens, self.topk), -1, dtype=torch.int32, device="cuda")
        gates = torch.full((self.tokens, self.topk), float("nan"), device="cuda")
        self.call(Y, beta, ids, gates)
        torch.cuda.synchronize()
        assert self.mm.device_status() == 0
        win = lambda b: b[64:64 + Y.numel()].view(Y.shape)[:, :self.d]
        got = win(buf).cpu()
        win(before).zero_(), win(buf).zero_()
        assert torch.equal(before.view(torch.int16), buf.view(torch.int16)), "written outside Y"
        assert torch.equal(ids.cpu().long(), want_ids)
        assert ((gates.cpu().double() - want_gates).abs() <= grel[:, None] * want_gates + 1e-37).all()
        check16(got, y + beta * c.double() if beta else y, bound + (2.0 ** -23 * c.double().abs() if beta else 0), self.dtype)


# (tokens, d, f, experts, topk)
SIZES = [(1, 64, 32, 4, 1), (1, 256, 384, 8, 2), (2, 130, 70, 5, 5), (3, 200, 120, 16, 4), (8, 512, 200, 8, 3),
         (9, 129, 257, 3, 2), (17, 256, 128, 4, 2), (40, 136, 144, 2, 1), (64, 64, 48, 33, 6), (1, 1, 1, 1, 1),
         (5, 1030, 40, 7, 2), (70, 96, 80, 3, 2)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("group,zeros", [(0, False), (32, True), (64, False), (128, True)])
def test_layer(cuda, mm, dtype, group, zeros):
    for i, s in enumerate(SIZES):
        Layer(mm, dtype, *s, renorm=bool(i % 2), group=group, zeros=zeros, seed=i).check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("group", [0, 32, 128])
def test_long_rows(cuda, mm, dtype, group):
    """Rows of several pieces with a ragged last one, experts with more tokens than a group takes, many rows of units to a
    block and blocks without any."""
    for i, s in enumerate(((20, 1096, 1544, 3, 1), (7, 2048, 520, 5, 3), (1, 3000, 2056, 2, 2), (64, 640, 1032, 2, 1),
                           (33, 513, 1025, 4, 2), (3, 5000, 16, 3, 1))):
        Layer(mm, dtype, *s, renorm=bool(i % 2), group=group, zeros=group == 32, seed=40 + i).check()


def test_the_widest_layers(cuda, mm):
    Layer(mm, "f16", 2, 65536, 24, 2, 1).check()
    Layer(mm, "f16", 2, 24, 65536, 2, 1).check()
    Layer(mm, "bf16", 1, 65536, 40, 2, 2, group=64).check()
    Layer(mm, "bf16", 1, 40, 65536, 2, 2, group=128).check()


def test_the_most_tokens(cuda, mm):
    """Four passes of 64 tokens, with one expert and with several."""
    Layer(mm, "f16", 256, 64, 48, 1, 1).check()
    Layer(mm, "bf16", 256, 72, 40, 3, 2, renorm=True, group=32).check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("group", [0, 64])
def test_layer_strides_and_beta(cuda, mm, dtype, group):
    for pads, s in (((8, 8, 8), (5, 264, 136, 6, 2)), ((3, 1, 5), (5, 265, 137, 6, 2)), ((1, 3, 0), (12, 100, 60, 4, 4))):
        Layer(mm, dtype, *s, renorm=True, group=group, pads=pads, seed=3).check(beta=-0.5, ldy=s[1] + pads[2])


def test_every_token_at_one_expert_and_none_at_others(cuda, mm):
    """All tokens equal: every expert but topk of them stays empty, those get the whole batch."""
    x = torch.randn(1, 160, generator=torch.Generator().manual_seed(21)).expand(33, 160).contiguous()
    Layer(mm, "f16", 33, 160, 96, 64, 2, renorm=True, x=x).check()
    Layer(mm, "bf16", 33, 160, 96, 64, 2, renorm=True, x=x, group=32, zeros=True).check()


@pytest.mark.parametrize("group", [0, 128])
def test_the_largest_selections(cuda, mm, group):
    """As many experts and choices as a call may have, with more tokens than one pass takes."""
    Layer(mm, "bf16", 20, 64, 16, 1024, 32, renorm=True, group=group).check()
    Layer(mm, "f16", 130, 32, 24, 9, 7, group=group).check()


def test_equal_scores_go_to_the_lowest_index(cuda, mm):
    for experts, topk in ((8, 3), (70, 32), (256, 9)):
        layer = Layer(mm, "f16", 4, 64, 32, experts, topk)
        layer.router_dev.zero_()
        ids = torch.empty(4, topk, dtype=torch.int32, device="cuda")
        gates = torch.empty(4, topk, device="cuda")
        layer.call(torch.empty(4, 64, dtype=torch.float16, device="cuda"), ids=ids, gates=gates)
        assert torch.equal(ids.cpu(), torch.arange(topk, dtype=torch.int32).expand(4, topk))
        assert ((gates.cpu() - 1 / experts).abs() <= 2.0 ** -20 / experts).all()


def test_nan_token_spoils_itself_only(cuda, mm):
    layer = Layer(mm, "bf16", 6, 128, 64, 8, 2, renorm=True)
    want = torch.empty(6, 128, dtype=torch.bfloat16, device="cuda")
    layer.call(want)
    for bad in (float("nan"), float("inf")):
        layer.xdev.copy_(layer.x)
        layer.xdev[2, 5] = bad
        ids = torch.full((6, 2), -1, dtype=torch.int32, device="cuda")
        Y = torch.empty_like(want)
        layer.call(Y, ids=ids)
        keep = torch.arange(6) != 2
        assert torch.equal(Y[keep], want[keep])
        assert torch.isnan(Y[2]).all()
        assert ((ids >= 0) & (ids < 8)).all() and (ids[:, 0] != ids[:, 1]).all()


def test_wide_scores(cuda, mm):
    """Scores hundreds apart: the far experts' gates vanish without a NaN."""
    layer = Layer(mm, "f16", 3, 64, 32, 6, 3)
    layer.router_dev.mul_(400)
    layer.router.mul_(400)
    layer.check()


@pytest.mark.parametrize("group", [0, 128])
def test_same_bits_every_time_and_any_workspace_contents(cuda, mm, group):
    layer = Layer(mm, "f16", 7, 300, 260, 12, 4, group=group)
    out = []
    for fill in (0, 255, 17):
        ws = torch.full((mm.moe_workspace_bytes("f16", 7, 300, 260, 12, 4),), fill, dtype=torch.uint8, device="cuda")
        Y = torch.empty(7, 300, dtype=torch.float16, device="cuda")
        layer.call(Y, ws=ws)
        out.append(Y)
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])


def test_rows_of_other_tokens_are_left(cuda, mm):
    """A padded batch: the call is told of five tokens, the rows behind them keep their contents."""
    layer = Layer(mm, "f16", 9, 96, 64, 4, 2)
    Y = torch.full((9, 96), 3.0, dtype=torch.float16, device="cuda")
    layer.call(Y, tokens=5)
    full = torch.empty_like(Y)
    layer.call(full)
    assert (Y[5:] == 3).all() and torch.allclose(Y[:5].float(), full[:5].float(), atol=2e-3, rtol=2e-3)


@pytest.mark.parametrize("group", [0, 64])
def test_captured_and_replayed(cuda, mm, group):
    layer = Layer(mm, "bf16", 4, 256, 192, 8, 2, renorm=True, group=group)
    Y = torch.empty(4, 256, dtype=torch.bfloat16, device="cuda")
    ws = layer.call(Y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.call(Y, ws=ws)
        layer.call(Y, ws=ws, beta=1.0)
    for seed in range(3):
        layer.xdev.copy_(torch.randn(4, 256, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        want = torch.empty_like(Y)
        layer.call(want)
        layer.call(want, beta=1.0)
        torch.cuda.synchronize()
        assert torch.equal(Y, want)


def test_two_streams_with_a_workspace_each(cuda, mm):
    layer = Layer(mm, "f16", 6, 512, 300, 16, 4)
    want = torch.empty(6, 512, dtype=torch.float16, device="cuda")
    ws = [layer.call(want), layer.call(want)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [torch.empty_like(want) for _ in range(30)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        layer.call(o, ws=ws[i % 2], stream=streams[i % 2])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_decoding_step(cuda, mm):
    """As a decoder would use them together: a 4-bit projection, the expert layer with 4-bit experts added to it (beta = 1),
    and a 4-bit head; the experts' weights rounded on the device by w4_quantize."""
    gen = torch.Generator().manual_seed(8)
    t, d, f, E, topk, vocab, group = 5, 256, 160, 6, 2, 500, 64

    def rounded(m, k):
        w = (torch.randn(m, k, generator=gen) / math.sqrt(k)).half()
        p = torch.empty(mm.w4_bytes(m, k, group, True), dtype=torch.uint8, device="cuda")
        mm.w4_quantize("f16", m, k, group, True, w.cuda(), k, p)
        return p, round64(w, group, True, torch.float16)

    proj, proj_w = rounded(d, d)
    head, head_w = rounded(vocab, d)
    packs = {n: [rounded(r, c) for _ in range(E)] for n, r, c in (("gate", f, d), ("up", f, d), ("down", d, f))}
    router = (torch.randn(E, d, generator=gen) * 2 / math.sqrt(d)).half()
    while True:  # a token's choice of experts must not hang on the rounding of the projection
        x = torch.randn(t, d, generator=gen).half()
        h = x.double() @ proj_w.t()
        if (score_gaps(h, router.double(), topk)[0] > 0.02).all():
            break
    hidden = torch.empty(t, d, dtype=torch.float16, device="cuda")
    logits = torch.empty(t, vocab, dtype=torch.float16, device="cuda")
    mm.gemm_w4("f16", d, t, d, 1.0, proj, group, True, x.cuda(), d, 0.0, hidden, d)
    dev = {n: torch.stack([p for p, _ in v]) for n, v in packs.items()}
    ws = torch.empty(mm.moe_workspace_bytes("f16", t, d, f, E, topk), dtype=torch.uint8, device="cuda")
    out = hidden.clone()
    mm.moe("f16", t, d, f, E, topk, hidden, d, router.cuda(), d, dev["gate"], dev["up"], ldg=0,
           strideG=dev["gate"].shape[1], down=dev["down"], ldd=0, strideD=dev["down"].shape[1], Y=out, ldy=d, group=group,
           zeros=True, renorm=True, beta=1.0, workspace=ws)
    mm.gemm_w4("f16", vocab, t, d, 1.0, head, group, True, out, d, 0.0, logits, vocab)
    torch.cuda.synchronize()
    ref = {n: torch.stack([w for _, w in v]) for n, v in packs.items()}
    y = moe64(h, router.double(), ref["gate"], ref["up"], ref["down"], topk, True)[0]
    want = (h + y) @ head_w.t()
    # three results rounded to half precision (2^-11 of their size each), each passing through a product whose rows
    # have norm about one: eight half steps of the largest logit
    assert (logits.cpu().double() - want).abs().max() <= 8 * 2.0 ** -11 * want.abs().max()


FIRST_CALLS = """
import torch
import gemm_mmbo_b200 as mm
t, d, f, E, k, g = 3, 320, 200, 6, 2, 64
gen = torch.Generator().manual_seed(0)
r = lambda *s: (torch.randn(*s, generator=gen) * 0.1).half().cuda()
x, router, W = r(t, d), r(E, d), r(E * f, d)
gate, up, down = r(E, f, d), r(E, f, d), r(E, d, f)
per, perd = mm.w4_bytes(f, d, g, True), mm.w4_bytes(d, f, g, True)
pg, pu, pd = [torch.zeros(E * b, dtype=torch.uint8, device="cuda") for b in (per, per, perd)]
packed = torch.zeros(mm.w4_bytes(E * f, d, g, True), dtype=torch.uint8, device="cuda")
ws = torch.empty(mm.moe_workspace_bytes("f16", t, d, f, E, k), dtype=torch.uint8, device="cuda")
many = r(40, d)
outs = [torch.zeros(t, d).half().cuda(), torch.zeros(t, d).half().cuda(), torch.zeros(1, E * f).half().cuda(),
        torch.zeros(40, E * f).half().cuda(), torch.zeros(E * f, d).half().cuda()]
def step(o):
    mm.w4_quantize("f16", E * f, d, g, True, W, d, packed)
    for e in range(E):
        mm.w4_quantize("f16", f, d, g, True, gate[e], d, pg[e * per:])
        mm.w4_quantize("f16", f, d, g, True, up[e], d, pu[e * per:])
        mm.w4_quantize("f16", d, f, g, True, down[e], f, pd[e * perd:])
    mm.moe("f16", t, d, f, E, k, x, d, router, d, gate, up, d, f * d, down, f, d * f, o[0], d, workspace=ws)
    mm.moe("f16", t, d, f, E, k, x, d, router, d, pg, pu, 0, per, pd, 0, perd, o[1], d, group=g, zeros=True, workspace=ws)
    mm.gemm_w4("f16", E * f, 1, d, 1.0, packed, g, True, x, d, 0.0, o[2], E * f)
    mm.gemm_w4("f16", E * f, 40, d, 1.0, packed, g, True, many, d, 0.0, o[3], E * f)
    mm.w4_unpack("f16", E * f, d, g, True, packed, o[4], d)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    step(outs)
graph.replay()
torch.cuda.synchronize()
eager = [torch.zeros_like(o) for o in outs]
step(eager)
torch.cuda.synchronize()
assert all(torch.equal(a, b) and bool(a.abs().sum() > 0) for a, b in zip(outs, eager))
assert mm.device_status() == 0
"""


def test_first_calls_of_a_process_captured(cuda):
    """Nothing has to run before it can be captured."""
    subprocess.run([sys.executable, "-c", FIRST_CALLS], check=True, timeout=300,
                   cwd=pathlib.Path(__file__).resolve().parent.parent)

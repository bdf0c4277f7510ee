"""Inputs on which the 4-bit and mixture-of-experts entry points could lose what their formulas keep: values far apart, sums near
the ends of a type's range, codes equal to their zero points, results that nearly cancel."""
import pytest
import torch

from low_bit import TYPES, chain, check16, make_w4, moe64, pack, weights64

pytestmark = pytest.mark.gpu


def expert_layer(mm, dtype, x, router, experts, group, topk, renorm=False, beta=0.0, Y=None):
    """One call with packed experts (a dict of lists of (codes, scales, zero points)); returns Y, ids and gates on the CPU."""
    (tokens, d), E = x.shape, router.shape[0]
    f = experts["gate"][0][0].shape[0]
    zeros = experts["gate"][0][2] is not None
    dev = {n: torch.stack([pack(mm, dtype, *p, group) for p in v]) for n, v in experts.items()}
    Y = torch.full((tokens, d), float("nan"), dtype=TYPES[dtype], device="cuda") if Y is None else Y
    ids = torch.full((tokens, topk), -1, dtype=torch.int32, device="cuda")
    gates = torch.full((tokens, topk), float("nan"), device="cuda")
    ws = torch.full((mm.moe_workspace_bytes(dtype, tokens, d, f, E, topk),), 0xFF, dtype=torch.uint8, device="cuda")
    mm.moe(dtype, tokens, d, f, E, topk, x.cuda(), d, router.cuda(), d, dev["gate"], dev["up"], ldg=0,
           strideG=dev["gate"].stride(0), down=dev["down"], ldd=0, strideD=dev["down"].stride(0), Y=Y, ldy=d, group=group,
           zeros=zeros, renorm=renorm, beta=beta, ids=ids, gates=gates, workspace=ws)
    torch.cuda.synchronize()
    assert mm.device_status() == 0
    return Y.cpu(), ids.cpu(), gates.cpu()


def expert_weights(gen, E, d, f, group, zeros, dt):
    return {n: [make_w4(gen, r, c, group, zeros, dt) for _ in range(E)] for n, r, c in (("gate", f, d), ("up", f, d), ("down", d, f))}


def in64(experts, group):
    return [torch.stack([weights64(*p, group) for p in experts[n]]) for n in ("gate", "up", "down")]


@pytest.mark.parametrize("zeros", [False, True])
def test_packed_layer_with_activations_near_the_end_of_the_range(cuda, mm, zeros):
    """A bfloat16 token of 2^123 whose gate and up weights bring it back to ordinary hidden values."""
    gen = torch.Generator().manual_seed(31)
    tokens, d, f, E, group, dt = 3, 96, 64, 4, 32, torch.bfloat16
    x = torch.randn(tokens, d, generator=gen).to(dt)
    x[1] = 0
    x[1, 40] = 2.0 ** 123
    router = torch.randn(E, d, generator=gen).to(dt)
    router[:, 40] = 0
    experts = expert_weights(gen, E, d, f, group, zeros, dt)
    for n in ("gate", "up"):
        for codes, scales, zps in experts[n]:
            scales[:, 1] = 2.0 ** -122  # the group of column 40
            codes[::3, 32:64] = 8 if zps is None else zps[::3, 1:2]  # some rows have no weight there
    Y, ids, _ = expert_layer(mm, "bf16", x, router, experts, group, 2)
    y, want_ids, _, bound, _ = moe64(x.double(), router.double(), *in64(experts, group), 2, False)
    assert torch.equal(ids.long(), want_ids)
    check16(Y, y, bound, "bf16")


def test_contractions_past_the_32_bit_words_of_a_row_block(cuda, mm):
    """One row of 1.82e9 weights in groups of 32 with zero points: 2.16e9 64-bit words of packed tiles.  B is zero but for 200
    places on both sides of word 2^31 and at the ends, so that at most 200 groups' sums are inexact additions."""
    k, n, group = 1_820_000_000, 9, 32
    if torch.cuda.mem_get_info()[0] < 60 * 2 ** 30:
        pytest.skip("needs 60 GB")
    g, gen = k // group, torch.Generator().manual_seed(3)
    edge = 2 ** 31 // 152 * 128  # first column of the tile with word 2^31
    at = torch.cat([torch.arange(a, a + 50) * 3 for a in (0, edge // 3 - 60, edge // 3 + 200, k // 3 - 50)])
    codes = torch.randint(0, 256, (1, k // 2), dtype=torch.uint8, device="cuda")
    scales = (0.002 + 0.01 * torch.rand(1, g, device="cuda")).half()
    zps = torch.randint(0, 16, (1, g), dtype=torch.uint8, device="cuda")
    packed = torch.empty(mm.w4_bytes(1, k, group, True), dtype=torch.uint8, device="cuda")
    mm.w4_pack("f16", 1, k, group, codes, k // 2, scales, g, zps, g, packed)
    x = torch.randn(n, at.numel(), generator=gen).half()
    B = torch.zeros(n, k, dtype=torch.float16, device="cuda")
    B[:, at.cuda()] = x.cuda()
    C = torch.empty(n, 1, dtype=torch.float16, device="cuda")
    mm.gemm_w4("f16", 1, n, k, 1.0, packed, group, True, B, k, 0.0, C, 1)
    torch.cuda.synchronize()
    assert mm.device_status() == 0
    both, where = codes[0, at.cuda() // 2].cpu(), at // group
    q = torch.where(at % 2 == 0, both & 15, both >> 4).double()
    w = (q - zps[0, where.cuda()].cpu().double()) * scales[0, where.cuda()].cpu().double()
    check16(C[:, 0].cpu(), x.double() @ w, chain(200 * 128) * (x.double().abs() @ w.abs()), "f16")


@pytest.mark.parametrize("n", [1, 8, 9, 70, 300])
@pytest.mark.parametrize("group", [32, 128])
def test_group_sums_past_the_largest_float(cuda, mm, n, group):
    """bfloat16 activations around 2^120 with equal signs and the largest codes: a group's sum of (q - z) x passes 2^128, its
    product with the scale does not."""
    gen = torch.Generator().manual_seed(n + group)
    m, k, dt = 150, 520, torch.bfloat16
    codes, scales, zps = make_w4(gen, m, k, group, True, dt)
    codes[::2], zps[::2] = 15, 0
    x = (torch.randn(n, k, generator=gen).abs() * 2.0 ** 120).to(dt)
    packed = pack(mm, "bf16", codes, scales, zps, group)
    C = torch.empty(n, m, dtype=dt, device="cuda")
    mm.gemm_w4("bf16", m, n, k, 1.0, packed, group, True, x.cuda(), k, 0.0, C, m)
    w = weights64(codes, scales, zps, group)
    check16(C.cpu(), x.double() @ w.t(), chain(k) * (x.double().abs() @ w.abs().t()), "bf16")


@pytest.mark.parametrize("n", [1, 9, 70])
def test_results_near_the_smallest_bfloat16(cuda, mm, n):
    """The other end: results around 2^-126, where a step is 2^-133."""
    gen = torch.Generator().manual_seed(n)
    m, k, group, dt = 150, 520, 64, torch.bfloat16
    codes, scales, zps = make_w4(gen, m, k, group, True, dt)
    x = (torch.randn(n, k, generator=gen) * 2.0 ** -123).to(dt)
    packed = pack(mm, "bf16", codes, scales, zps, group)
    C = torch.empty(n, m, dtype=dt, device="cuda")
    mm.gemm_w4("bf16", m, n, k, 1.0, packed, group, True, x.cuda(), k, 0.0, C, m)
    w = weights64(codes, scales, zps, group)
    # 9 groups and the joints of their sums, each rounded to steps of 2^-138
    check16(C.cpu(), x.double() @ w.t(), chain(k) * (x.double().abs() @ w.abs().t()) + 30 * 2.0 ** -139, "bf16")


def test_packed_hidden_vectors_near_the_end_of_the_range(cuda, mm):
    """Hidden values of 2^116 and more that down's scales bring back."""
    gen = torch.Generator().manual_seed(9)
    tokens, d, f, E, group, dt = 4, 64, 128, 2, 128, torch.bfloat16
    x = torch.randn(tokens, d, generator=gen).abs().to(dt)
    router = torch.randn(E, d, generator=gen).to(dt)
    experts = expert_weights(gen, E, d, f, group, True, dt)
    for e in range(E):
        for n, size in (("gate", 2.0 ** 50), ("up", 2.0 ** 50), ("down", 2.0 ** -118)):
            codes, scales, zps = experts[n][e]
            scales.fill_(size)
            zps.fill_(0)
            codes.clamp_(min=1)
            if n == "down":
                codes[::2] = 15
    Y, ids, _ = expert_layer(mm, "bf16", x, router, experts, group, 1)
    y, want_ids, _, bound, _ = moe64(x.double(), router.double(), *in64(experts, group), 1, False)
    assert torch.equal(ids.long(), want_ids)
    check16(Y, y, bound, "bf16")

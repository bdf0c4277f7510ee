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


LOUD = [("f16", 60000.0), ("bf16", 2.0 ** 17), ("bf16", 2.0 ** 30), ("bf16", 2.0 ** 120)]


@pytest.mark.parametrize("dtype,loud", LOUD)
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_loud_activations_at_weights_of_zero(cuda, mm, dtype, loud, group, zeros):
    """A weight whose code is its zero point is zero: what it meets drops out, however large.  The same columns give the same
    accuracy alone, in a call of 8 and in one of 9, and rows of zeros give zeros."""
    gen = torch.Generator().manual_seed(group)
    m, k, dt = 150, 1100, TYPES[dtype]
    codes, scales, zps = make_w4(gen, m, k, group, zeros, dt)
    for j in (3, 700, k - 1):
        codes[:, j] = 8 if zps is None else zps[:, j // group]
    for i in (0, 77, m - 1):
        codes[i] = 8 if zps is None else zps[i, torch.arange(k) // group]
    packed = pack(mm, dtype, codes, scales, zps, group)
    w = weights64(codes, scales, zps, group)
    x = torch.randn(70, k, generator=gen).to(dt)
    x[:, 3], x[::2, 700], x[1::2, k - 1] = loud, -loud, loud
    for n in (1, 2, 8, 9, 33, 70):
        C = torch.full((n, m), float("nan"), dtype=dt, device="cuda")
        mm.gemm_w4(dtype, m, n, k, 1.0, packed, group, zeros, x.cuda(), k, 0.0, C, m)
        check16(C.cpu(), x[:n].double() @ w.t(), chain(k) * (x[:n].double().abs() @ w.abs().t()), dtype)
        assert (C[:, [0, 77, m - 1]] == 0).all()


@pytest.mark.parametrize("n", [1, 8, 9])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_small_results_beside_large_ones(cuda, mm, dtype, n):
    """One large weight-activation pair in a column of B leaves the other rows' small sums alone."""
    gen = torch.Generator().manual_seed(n)
    m, k, group, dt = 64, 384, 128, TYPES[dtype]
    codes, scales, zps = make_w4(gen, m, k, group, True, dt)
    codes[1:, 5] = zps[1:, 0]  # only row 0 has a weight in column 5
    packed = pack(mm, dtype, codes, scales, zps, group)
    x = (torch.randn(n, k, generator=gen) * 2.0 ** -10).to(dt)
    x[:, 5] = 2.0 ** 14
    C = torch.empty(n, m, dtype=dt, device="cuda")
    mm.gemm_w4(dtype, m, n, k, 1.0, packed, group, True, x.cuda(), k, 0.0, C, m)
    w = weights64(codes, scales, zps, group)
    check16(C.cpu(), x.double() @ w.t(), chain(k) * (x.double().abs() @ w.abs().t()), dtype)


@pytest.mark.parametrize("dtype,loud", LOUD)
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_packed_layer_with_loud_activations_at_weights_of_zero(cuda, mm, dtype, loud, group, zeros):
    gen = torch.Generator().manual_seed(group + 1)
    tokens, d, f, E, topk, dt = 11, 300, 96, 4, 2, TYPES[dtype]
    x = torch.randn(tokens, d, generator=gen).to(dt)
    router = (torch.randn(E, d, generator=gen) / 8).to(dt)
    experts = expert_weights(gen, E, d, f, group, zeros, dt)
    for j in (1, 200, d - 1):
        x[:, j] = loud if j != 200 else -loud
        router[:, j] = 0
        for n in ("gate", "up"):
            for codes, scales, zps in experts[n]:
                codes[:, j] = 8 if zps is None else zps[:, j // group]
    Y, ids, _ = expert_layer(mm, dtype, x, router, experts, group, topk, renorm=True)
    y, want_ids, _, bound, _ = moe64(x.double(), router.double(), *in64(experts, group), topk, True)
    assert torch.equal(ids.long(), want_ids)
    check16(Y, y, bound, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_spoilt_column_beside_others_costs_nothing(cuda, mm, dtype):
    """A column with a NaN and one with an infinity among eight: they come out as NaN and infinities, and the call takes as
    long as without them (it took some milliseconds when such columns were summed again element by element)."""
    gen = torch.Generator().manual_seed(2)
    m, k, n, group, dt = 512, 16384, 8, 128, TYPES[dtype]
    codes, scales, zps = make_w4(gen, m, k, group, True, dt)
    codes[:, 7] = (zps[:, 0] + 1) % 16
    packed = pack(mm, dtype, codes, scales, zps, group)
    x = torch.randn(n, k, generator=gen).to(dt)
    times = []
    for spoilt in (False, True):
        if spoilt:
            x[2, 9], x[5, 7] = float("nan"), float("inf")
        X, C = x.cuda(), torch.empty(n, m, dtype=dt, device="cuda")
        marks = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        best = float("inf")
        for _ in range(8):  # the shortest of several: another process may take the host for a while
            marks[0].record()
            for _ in range(20):
                mm.gemm_w4(dtype, m, n, k, 1.0, packed, group, True, X, k, 0.0, C, m)
            marks[1].record()
            torch.cuda.synchronize()
            best = min(best, marks[0].elapsed_time(marks[1]))
        times.append(best)
    got = C.cpu()
    assert torch.isnan(got[2]).all() and torch.isinf(got[5]).all()
    assert torch.isfinite(got[[0, 1, 3, 4, 6, 7]]).all()
    assert times[1] < 5 * times[0]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k,ldb", [(2600, 8, 6001, 6008), (2600, 8, 5500, 5504), (5000, 3, 20002, 20008)])
def test_columns_staged_again_for_every_batch_of_rows(cuda, mm, dtype, m, n, k, ldb):
    """Columns that do not fit a block's shared memory and rows of several rounds: what plain stores left of one staging (the
    ragged end of a column) is overwritten by the bulk copies of the next."""
    gen = torch.Generator().manual_seed(m + k)
    group, dt = 128, TYPES[dtype]
    codes, scales, zps = make_w4(gen, m, k, group, True, dt)
    packed = pack(mm, dtype, codes, scales, zps, group)
    x = torch.randn(n, k, generator=gen).to(dt)
    B = torch.full((n, ldb), float("nan"), dtype=dt, device="cuda")
    B[:, :k] = x.cuda()
    out = [torch.empty(n, m, dtype=dt, device="cuda") for _ in range(30)]
    for C in out:
        mm.gemm_w4(dtype, m, n, k, 1.0, packed, group, True, B, ldb, 0.0, C, m)
    torch.cuda.synchronize()
    w = weights64(codes, scales, zps, group).cuda()
    X = x.cuda().double()
    check16(out[0].cpu(), (X @ w.t()).cpu(), (chain(k) * (X.abs() @ w.abs().t())).cpu(), dtype)
    assert all(torch.equal(out[0], C) for C in out[1:])


@pytest.mark.parametrize("n", [1, 3, 5, 7, 8])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_joins_whose_units_do_not_fill_a_warp(cuda, mm, dtype, n):
    """Few rows and a long contraction: clusters cut k, and the halves of a warp have different numbers of sums to hand over."""
    gen = torch.Generator().manual_seed(n)
    group, dt = 64, TYPES[dtype]
    for m, k in ((16, 8192), (17, 16384), (144, 12288), (1000, 8200), (4112, 4096)):
        codes, scales, zps = make_w4(gen, m, k, group, True, dt)
        packed = pack(mm, dtype, codes, scales, zps, group)
        x = torch.randn(n, k, generator=gen).to(dt)
        C = torch.empty(n, m, dtype=dt, device="cuda")
        mm.gemm_w4(dtype, m, n, k, 1.0, packed, group, True, x.cuda(), k, 0.0, C, m)
        torch.cuda.synchronize()
        assert mm.device_status() == 0
        w = weights64(codes, scales, zps, group).cuda()
        X = x.cuda().double()
        check16(C.cpu(), (X @ w.t()).cpu(), (chain(k) * (X.abs() @ w.abs().t())).cpu(), dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("experts,topk", [(5, 2), (70, 32), (300, 7)])
def test_choices_without_a_number(cuda, mm, dtype, experts, topk):
    """A NaN or +inf among a token's scores makes all its probabilities NaN: equal ones, so the lowest experts.  One -inf is a
    probability of zero."""
    gen = torch.Generator().manual_seed(experts)
    tokens, d, f, group, dt = 6, 64, 32, 32, TYPES[dtype]
    x = torch.randn(tokens, d, generator=gen).to(dt)
    x[:, 0] = torch.tensor([1.0, -1.0, 1.0, -1.0, 0.0, -1.0])
    x[3, 9] = float("nan")
    router = torch.randn(experts, d, generator=gen).to(dt)
    router[3, 0] = float("inf")  # scores of +inf, -inf, +inf, NaN, NaN, -inf
    one = expert_weights(gen, 1, d, f, group, False, dt)
    packs = {n: v * experts for n, v in one.items()}
    Y, ids, gates = expert_layer(mm, dtype, x, router, packs, group, topk)
    lowest = torch.arange(topk, dtype=torch.int32)
    for t in (0, 2, 3, 4):
        assert torch.equal(ids[t], lowest), t
        assert torch.isnan(gates[t]).all() and torch.isnan(Y[t]).all()
    scores = x.double() @ router.double().t()
    for t in (1, 5):
        p = torch.softmax(scores[t], 0)
        assert 3 not in ids[t].tolist() and torch.isfinite(gates[t]).all() and torch.isfinite(Y[t]).all()
        assert ((gates[t].double() - p[ids[t].long()]).abs() <= 2.0 ** -12 * p[ids[t].long()]).all()


def to_bits(value, bits):
    """A positive Fraction rounded to that many significant bits, ties to even."""
    from fractions import Fraction
    e = value.numerator.bit_length() - value.denominator.bit_length()
    if Fraction(2) ** e > value:
        e -= 1
    unit = Fraction(2) ** (e - bits + 1)
    q = value / unit
    n, rest = divmod(q.numerator, q.denominator)
    twice = 2 * rest - q.denominator
    return (n + (twice > 0 or (twice == 0 and n % 2))) * unit


def spans_beside_ties():
    """(h, -l) of half precision whose span in 32 bits is 15 times a tie between two half-precision scales although the
    span itself is not."""
    from fractions import Fraction
    found = []
    for h in range(1024, 2048):
        x = Fraction(h, 15)
        unit = to_bits(x, 1) / 2 ** 11 if to_bits(x, 1) <= x else to_bits(x, 1) / 2 ** 12
        for n in range(int(x / unit), int(x / unit) + 3):
            gap = 15 * n * unit - h
            if n % 2 == 0 or gap <= 0:
                continue
            low = to_bits(gap, 11)
            ulp = to_bits(low, 1) / 2 ** 10 if to_bits(low, 1) <= low else to_bits(low, 1) / 2 ** 11
            for j in range(-8, 9):
                l = low + j * ulp
                if l > 0 and to_bits(l, 11) == l and to_bits(to_bits(h + l, 24) / 15, 11) != to_bits((h + l) / 15, 11):
                    found.append((h, l))
    return found


def test_scales_of_spans_beside_a_tie(cuda, mm):
    """Groups whose ends need more than 24 bits together: the scale is the rounded quotient of the exact span."""
    pairs = spans_beside_ties()
    assert len(pairs) > 50
    k, m = 32, len(pairs)
    for exponent in (0, 4):
        w = torch.zeros(m, k, dtype=torch.float64)
        for i, (h, l) in enumerate(pairs):
            w[i, 3], w[i, 17] = float(h) * 2.0 ** exponent, -float(l) * 2.0 ** exponent
        W = w.half()
        assert torch.equal(W.double(), w)
        packed = torch.empty(mm.w4_bytes(m, k, 32, True), dtype=torch.uint8, device="cuda")
        mm.w4_quantize("f16", m, k, 32, True, W.cuda(), k, packed)
        back = torch.empty(m, k, dtype=torch.float16, device="cuda")
        mm.w4_unpack("f16", m, k, 32, True, packed, back, k)
        # the small end rounds to no step at all, so that the zero point is 0 and the large end 15 steps
        want = torch.tensor([float(to_bits(15 * to_bits((h + l) / 15, 11), 11)) for h, l in pairs], dtype=torch.float64)
        assert torch.equal(back[:, 3].cpu().double(), want * 2.0 ** exponent)
        assert (back[:, 17] == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("group", [0, 64])
def test_hidden_vectors_keep_what_a_16_bit_rounding_leaves(cuda, mm, dtype, group):
    """Tokens with one element each, so that scores, gates and hidden values come from single exact products; Y holds the
    negative of the rounded result and beta is one, so that what is left shows the sums to 32 bits.  A hidden value may be off
    by 2^-17 of itself (two bfloat16) or 2^-22 and 2^-30 (two halves), and by 2^-21 for exp, division and product; dropping
    the second half would be off by more than the bound."""
    from test_gpu_moe import Layer
    tokens, d, f, E, topk, dt = 6, 64, 40, 4, 2, TYPES[dtype]
    gen = torch.Generator().manual_seed(77)
    x = torch.zeros(tokens, d)
    x[torch.arange(tokens), torch.arange(tokens) * 9] = 1 + torch.rand(tokens, generator=gen)
    layer = Layer(mm, dtype, tokens, d, f, E, topk, renorm=True, group=group, x=x, seed=5)
    halves = dtype == "f16" and group == 0
    rel, floor = (2.0 ** -22, 2.0 ** -30) if halves else (2.0 ** -17, 0.0)
    scores = layer.x.double() @ layer.router.double().t()
    p, order = torch.sort(torch.softmax(scores, 1), dim=1, descending=True)
    assert ((p[:, :-1] - p[:, 1:]) > 1e-4).all(), "the inputs leave the choice of experts open"
    gates = p[:, :topk] / p[:, :topk].sum(1, keepdim=True)
    y, lost, bound = (torch.zeros(tokens, d, dtype=torch.float64) for _ in range(3))
    for t in range(tokens):
        for j in range(topk):
            e = int(order[t, j])
            g, u = layer.ref["gate"][e] @ layer.x[t].double(), layer.ref["up"][e] @ layer.x[t].double()
            h, down = g * torch.sigmoid(g) * u, layer.ref["down"][e]
            y[t] += gates[t, j] * (down @ h)
            lost[t] += gates[t, j] * (down @ h.to(dt if group == 0 else torch.bfloat16).double())
            bound[t] += gates[t, j] * (down.abs() @ (h.abs() * (rel + 2.0 ** -21 + chain(f)) + floor) + 2.0 ** -19 * (down @ h).abs())
    assert ((lost - y).abs() / bound).max() > 3, "the bound would not notice"
    Y = -y.to(dt)
    rest = y + Y.double()
    Y = Y.cuda()
    layer.call(Y, beta=1.0)
    torch.cuda.synchronize()
    check16(Y.cpu(), rest, bound, dtype)


@pytest.mark.parametrize("n,ldb_pad", [(1, 0), (8, 0), (8, 3)])
def test_long_contractions_of_few_rows(cuda, mm, n, ldb_pad):
    """Two rows of 6e8 weights: more than a million tiles for each of a few blocks, whose feeding warps' waits add up.  B is zero but for 150 places, so that the other additions are exact."""
    k, m, group = 600_000_000, 2, 128
    if torch.cuda.mem_get_info()[0] < 40 * 2 ** 30:
        pytest.skip("needs 40 GB")
    g, gen = k // group, torch.Generator().manual_seed(3)
    at = torch.cat([torch.arange(a, a + 50) * 5 for a in (0, k // 11, k // 5 - 50)])
    codes = torch.randint(0, 256, (m, k // 2), dtype=torch.uint8, device="cuda")
    scales = (0.002 + 0.01 * torch.rand(m, g, device="cuda")).bfloat16()
    packed = torch.empty(mm.w4_bytes(m, k, group, False), dtype=torch.uint8, device="cuda")
    mm.w4_pack("bf16", m, k, group, codes, k // 2, scales, g, None, 0, packed)
    x = torch.randn(n, at.numel(), generator=gen).bfloat16()
    B = torch.zeros(n, k + ldb_pad, dtype=torch.bfloat16, device="cuda")
    B[:, at.cuda()] = x.cuda()
    C = torch.empty(n, m, dtype=torch.bfloat16, device="cuda")
    mm.gemm_w4("bf16", m, n, k, 1.0, packed, group, False, B, k + ldb_pad, 0.0, C, m)
    torch.cuda.synchronize()
    assert mm.device_status() == 0
    both = codes[:, at.cuda() // 2].cpu()
    q = torch.where(at % 2 == 0, both & 15, both >> 4).double()
    w = (q - 8) * scales[:, (at // group).cuda()].cpu().double()
    check16(C.cpu(), x.double() @ w.t(), chain(200 * 128) * (x.double().abs() @ w.abs().t()), "bf16")

"""4-bit weights with group scales: packing, rounding and the product, against plain forms in 64 bits."""
import pytest
import torch

from low_bit import TYPES, chain, check16, make_w4, pack, padded, round64, weights64

pytestmark = pytest.mark.gpu

# (m, k, n): one element, exact and ragged blocks, tiles and groups, every number of columns at which the work is cut
# differently, long and short contractions
SIZES = [(1, 1, 1), (16, 128, 1), (17, 129, 1), (5, 31, 2), (130, 1000, 3), (40, 33, 7), (257, 515, 8), (300, 2050, 9),
         (64, 8200, 2), (48, 640, 15), (2048, 512, 16), (333, 700, 17), (129, 260, 31), (128, 384, 32), (200, 1111, 33),
         (100, 4100, 48), (513, 640, 64), (390, 900, 65), (256, 1024, 128), (131, 300, 130), (70, 260, 257)]


def product(mm, dtype, m, n, k, group, zeros, alpha=1.0, beta=0.0, ldb=None, ldc=None, seed=0, stream=None):
    gen = torch.Generator().manual_seed(seed * 1000003 + m * 7919 + n * 104729 + k)
    dt = TYPES[dtype]
    codes, scales, zps = make_w4(gen, m, k, group, zeros, dt)
    x = torch.randn(n, k, generator=gen).to(dt)
    c = torch.randn(n, m, generator=gen).to(dt)
    packed = pack(mm, dtype, codes, scales, zps, group)
    bufb, B = padded(x, ldb or k, dt)
    bufc, C = padded(c if beta else torch.full_like(c, float("nan")), ldc or m, dt)
    before = bufc.clone()
    torch.cuda.synchronize()
    mm.gemm_w4(dtype, m, n, k, alpha, packed, group, zeros, B, B.shape[1], beta, C, C.shape[1], stream=stream)
    torch.cuda.synchronize()
    assert mm.device_status() == 0
    # everything outside the window of C keeps its bits
    before[64:64 + C.numel()].view(C.shape)[:, :m] = 0
    after = bufc.clone()
    after[64:64 + C.numel()].view(C.shape)[:, :m] = 0
    assert torch.equal(before.view(torch.int16), after.view(torch.int16)), "written outside C"
    w = weights64(codes, scales, zps, group)
    want = alpha * (x.double() @ w.t()) + (beta * c.double() if beta else 0)
    terms = abs(alpha) * (x.double().abs() @ w.abs().t()) + abs(beta) * c.double().abs()
    return check16(C[:, :m].cpu(), want, chain(k) * terms, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (64, True), (128, False), (128, True)])
def test_product_sizes(cuda, mm, dtype, group, zeros):
    for m, k, n in SIZES:
        product(mm, dtype, m, n, k, group, zeros)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("group,zeros", [(32, False), (64, True), (128, False)])
@pytest.mark.parametrize("n,pad", [(600, 0), (777, 8), (530, 1)])
def test_product_with_enough_columns_for_wide_tiles(cuda, mm, dtype, group, zeros, n, pad):
    """Several rounds of 128-column tiles, ragged in both directions."""
    product(mm, dtype, 3001, n, 520, group, zeros, alpha=0.5, beta=1.0, ldb=520 + pad, ldc=3001 + pad)


@pytest.mark.parametrize("n", [1, 5, 12, 40, 150])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_product_strides_alpha_beta(cuda, mm, dtype, n):
    """Leading dimensions that leave columns 16-byte aligned, 2-byte aligned only, and scalars."""
    for pad_b, pad_c in ((8, 8), (3, 1), (1, 5)):
        product(mm, dtype, 203, n, 708, 64, True, alpha=1.5, beta=-0.25, ldb=708 + pad_b, ldc=203 + pad_c, seed=1)
        product(mm, dtype, 203, n, 708, 128, False, alpha=-0.5, beta=0.0, ldb=708 + pad_b, ldc=203 + pad_c, seed=2)


@pytest.mark.parametrize("n", [1, 6, 16, 30, 100])
def test_product_operands_at_odd_addresses(cuda, mm, n):
    """B and C that start on a 2-byte boundary only."""
    gen = torch.Generator().manual_seed(n)
    m, k, group = 150, 392, 32
    codes, scales, zps = make_w4(gen, m, k, group, True, torch.float16)
    packed = pack(mm, "f16", codes, scales, zps, group)
    x = torch.randn(n, k, generator=gen).half()
    B = torch.full((n * k + 3,), float("nan"), dtype=torch.float16, device="cuda")[3:]
    B.view(n, k).copy_(x)
    C = torch.empty(n * m + 1, dtype=torch.float16, device="cuda")[1:]
    mm.gemm_w4("f16", m, n, k, 1.0, packed, group, True, B, k, 0.0, C, m)
    w = weights64(codes, scales, zps, group)
    check16(C.view(n, m).cpu(), x.double() @ w.t(), chain(k) * (x.double().abs() @ w.abs().t()), "f16")


@pytest.mark.parametrize("n", [1, 9, 20, 70])
def test_product_empty_contraction_and_empty_results(cuda, mm, n):
    C = torch.ones(n, 40, dtype=torch.bfloat16, device="cuda")
    mm.gemm_w4("bf16", 40, n, 0, 1.0, None, 64, False, None, 0, 0.5, C, 40)
    assert (C == 0.5).all()
    C.fill_(float("nan"))
    mm.gemm_w4("bf16", 40, n, 0, 1.0, None, 64, False, None, 0, 0.0, C, 40)
    assert (C == 0).all()
    before = mm.launch_count()
    mm.gemm_w4("bf16", 0, n, 64, 1.0, None, 64, False, None, 64, 0.0, None, 0)
    mm.gemm_w4("bf16", 64, 0, 64, 1.0, None, 64, False, None, 64, 0.0, None, 64)
    assert mm.launch_count() == before


@pytest.mark.parametrize("n", [1, 4, 16, 24, 200])
def test_infinities_and_nans_stay_in_their_column(cuda, mm, n):
    """A column of B with an infinity or a NaN spoils that column of C and no other one; the columns behind k do not."""
    gen = torch.Generator().manual_seed(5)
    m, k, group = 100, 330, 128
    codes, scales, zps = make_w4(gen, m, k, group, True, torch.float16)
    codes[:, 7] = (zps[:, 0] + 1) % 16  # no weight of column 7 is zero
    packed = pack(mm, "f16", codes, scales, zps, group)
    x = torch.randn(n, k, generator=gen).half()
    x[n // 2, 7] = float("inf")
    _, B = padded(x, k + 5, torch.float16)  # NaN behind every column
    C = torch.empty(n, m, dtype=torch.float16, device="cuda")
    mm.gemm_w4("f16", m, n, k, 1.0, packed, group, True, B, k + 5, 0.0, C, m)
    got = C.cpu()
    keep = torch.arange(n) != n // 2
    assert torch.isfinite(got[keep]).all()
    assert torch.isinf(got[n // 2]).all()
    x[n // 2, 7] = float("nan")
    B[:, :k].copy_(x)
    mm.gemm_w4("f16", m, n, k, 1.0, packed, group, True, B, k + 5, 0.0, C, m)
    got = C.cpu()
    assert torch.isfinite(got[keep]).all() and torch.isnan(got[n // 2]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_results_beyond_the_type_become_infinite(cuda, mm, dtype):
    m, k = 32, 256
    codes = torch.full((m, k), 15, dtype=torch.uint8)
    big = 6e4 if dtype == "f16" else 3e38
    scales = torch.full((m, 2), big).to(TYPES[dtype])
    packed = pack(mm, dtype, codes, scales, None, 128)
    for n in (1, 20):
        x = torch.ones(n, k, dtype=TYPES[dtype], device="cuda")
        C = torch.zeros(n, m, dtype=TYPES[dtype], device="cuda")
        mm.gemm_w4(dtype, m, n, k, 1.0, packed, 128, False, x, k, 0.0, C, m)
        assert torch.isinf(C).all()


@pytest.mark.parametrize("n", [1, 8, 13, 50, 140])
def test_same_bits_every_time(cuda, mm, n):
    gen = torch.Generator().manual_seed(3)
    m, k = 700, 5000
    codes, scales, zps = make_w4(gen, m, k, 64, True, torch.float16)
    packed = pack(mm, "f16", codes, scales, zps, 64)
    x = torch.randn(n, k, generator=gen).half().cuda()
    out = []
    for _ in range(5):
        C = torch.empty(n, m, dtype=torch.float16, device="cuda")
        mm.gemm_w4("f16", m, n, k, 1.0, packed, 64, True, x, k, 0.0, C, m)
        out.append(C)
    assert all(torch.equal(out[0], c) for c in out[1:])


def test_offsets_past_32_bits(cuda, mm):
    """A packed matrix of more than 2^32 bytes: its first, middle and last rows."""
    m, k, group = 70000, 131072, 128
    g = k // group
    gen = torch.Generator(device="cuda").manual_seed(11)
    codes = torch.randint(0, 256, (m, k // 2), generator=gen, dtype=torch.uint8, device="cuda")
    scales = (0.001 + 0.01 * torch.rand(m, g, generator=gen, device="cuda")).half()
    packed = torch.empty(mm.w4_bytes(m, k, group, False), dtype=torch.uint8, device="cuda")
    assert packed.numel() > 2 ** 32
    mm.w4_pack("f16", m, k, group, codes, k // 2, scales, g, None, 0, packed)
    for n in (1, 20):
        x = torch.randn(n, k, generator=gen, device="cuda").half()
        C = torch.empty(n, m, dtype=torch.float16, device="cuda")
        mm.gemm_w4("f16", m, n, k, 1.0, packed, group, False, x, k, 0.0, C, m)
        for r in (0, 12345, 65536, m - 1):
            both = torch.stack((codes[r] & 15, codes[r] >> 4), dim=-1).flatten().double()
            w = (both - 8) * scales[r].double().repeat_interleave(group)
            want = x.double() @ w
            check16(C[:, r].cpu(), want.cpu(), (chain(k) * (x.double().abs() @ w.abs())).cpu(), "f16")


# ---------------------------------------------------------------- packing and rounding --

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", [(40, 8, 70001), (24, 5, 40000), (17, 1, 200000), (20001, 8, 256), (150000, 3, 64),
                                   (1024, 1, 16384), (16, 16, 60000), (40000, 9, 130)])
def test_product_of_long_and_tall_matrices(cuda, mm, dtype, m, n, k):
    """Activations that do not fit a block's shared memory, contractions cut over blocks, several batches of rows a block."""
    product(mm, dtype, m, n, k, 128, True)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("group,zeros", [(32, True), (32, False), (64, True), (128, False), (128, True)])
def test_round_trip_is_the_formula(cuda, mm, dtype, group, zeros):
    """Rounding and unpacking against 64 bits: equal to the last bit, ties and short last groups included."""
    dt = TYPES[dtype]
    for m, k, pad in ((1, 1, 0), (16, 128, 0), (33, 300, 4), (50, 1025, 7), (128, 512, 8)):
        gen = torch.Generator().manual_seed(m + k)
        w = (torch.randn(m, k, generator=gen) * 0.02).to(dt)
        w[0, :min(k, 20)] = 0
        if m > 2:
            w[1] = 0                                                     # empty groups: scale zero
            w[2, :] = (torch.randint(-14, 15, (k,), generator=gen) * 0.25).to(dt)  # multiples of half a step: ties
            w[2, ::group] = 3.5
            w[2, 1::group] = -3.5 if k > 1 else 3.5
            w[3 % m] = w[3 % m].abs()                                    # one sign only
        ld = k + pad
        buf, W = padded(w, ld, dt)
        packed = torch.full((mm.w4_bytes(m, k, group, zeros) + 32,), 0x5A, dtype=torch.uint8, device="cuda")
        mm.w4_quantize(dtype, m, k, group, zeros, W, ld, packed)
        obuf, out = padded(torch.zeros(m, k, dtype=dt), ld, dt)
        before = obuf.clone()
        mm.w4_unpack(dtype, m, k, group, zeros, packed, out, ld)
        torch.cuda.synchronize()
        assert (packed[-32:] == 0x5A).all()
        want = round64(w, group, zeros, dt).to(dt)
        assert torch.equal(out[:, :k].cpu(), want), (m, k)
        before[64:64 + out.numel()].view(out.shape)[:, :k] = out[:, :k]
        assert torch.equal(before.view(torch.int16), obuf.view(torch.int16)), "written outside W"


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("ld", [700, 701, 702, 704])
def test_round_trip_with_rows_at_any_address(cuda, mm, dtype, ld):
    """Rows that start on any 2-byte boundary, tiles inside the rows and at their ends; the columns between them stay."""
    dt, m, k, group = TYPES[dtype], 19, 700, 64
    w = (torch.randn(m, k, generator=torch.Generator().manual_seed(ld)) * 0.02).to(dt)
    want = round64(w, group, True, dt).to(dt)
    for off in range(8):
        flat = torch.full((m * ld + 16,), float("nan"), dtype=dt, device="cuda")
        flat[off:off + m * ld].view(m, ld)[:, :k] = w.cuda()
        packed = torch.zeros(mm.w4_bytes(m, k, group, True), dtype=torch.uint8, device="cuda")
        mm.w4_quantize(dtype, m, k, group, True, flat[off:], ld, packed)
        back = torch.full_like(flat, float("nan"))
        mm.w4_unpack(dtype, m, k, group, True, packed, back[off:], ld)
        out = back[off:off + m * ld].view(m, ld)
        assert torch.equal(out[:, :k].cpu(), want), off
        out[:, :k] = float("nan")
        assert torch.isnan(back.float()).all(), "written outside W"


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_round_trip_of_every_value(cuda, mm, dtype):
    """All finite 16-bit patterns, in groups with a common largest value: from the smallest subnormal up."""
    dt = TYPES[dtype]
    pat = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dt)
    pat = pat[torch.isfinite(pat.float())]
    pat = pat[torch.argsort(pat.float().abs())]
    k = 64
    w = pat[:pat.numel() // k * k].view(-1, k).contiguous()
    m = w.shape[0]
    for zeros in (False, True):
        packed = torch.empty(mm.w4_bytes(m, k, 64, zeros), dtype=torch.uint8, device="cuda")
        mm.w4_quantize(dtype, m, k, 64, zeros, w.cuda(), k, packed)
        out = torch.empty(m, k, dtype=dt, device="cuda")
        mm.w4_unpack(dtype, m, k, 64, zeros, packed, out, k)
        want = round64(w, 64, zeros, dt).to(dt)
        assert torch.equal(out.cpu(), want)


def test_non_finite_weights_poison_their_group_only(cuda, mm):
    w = torch.randn(20, 256, generator=torch.Generator().manual_seed(1)).half()
    w[3, 5], w[4, 200] = float("inf"), float("nan")
    for zeros in (False, True):
        packed = torch.empty(mm.w4_bytes(20, 256, 64, zeros), dtype=torch.uint8, device="cuda")
        mm.w4_quantize("f16", 20, 256, 64, zeros, w.cuda(), 256, packed)
        out = torch.empty(20, 256, dtype=torch.float16, device="cuda")
        mm.w4_unpack("f16", 20, 256, 64, zeros, packed, out, 256)
        bad = torch.isnan(out.cpu())
        want = torch.zeros(20, 256, dtype=torch.bool)
        want[3, :64] = True
        want[4, 192:] = True
        assert torch.equal(bad, want)
        x = torch.ones(3, 256).half().cuda()
        C = torch.empty(3, 20, dtype=torch.float16, device="cuda")
        mm.gemm_w4("f16", 20, 3, 256, 1.0, packed, 64, zeros, x, 256, 0.0, C, 20)
        assert torch.isnan(C[:, 3:5]).all() and torch.isfinite(C[:, :3]).all() and torch.isfinite(C[:, 5:]).all()


@pytest.mark.parametrize("zeros", [False, True])
def test_pack_and_unpack_agree(cuda, mm, zeros):
    gen = torch.Generator().manual_seed(9)
    for m, k, group in ((1, 1, 32), (31, 257, 64), (100, 1000, 128), (17, 96, 32)):
        codes, scales, zps = make_w4(gen, m, k, group, zeros, torch.bfloat16)
        packed = pack(mm, "bf16", codes, scales, zps, group)
        out = torch.empty(m, k, dtype=torch.bfloat16, device="cuda")
        mm.w4_unpack("bf16", m, k, group, zeros, packed, out, k)
        assert torch.equal(out.cpu(), weights64(codes, scales, zps, group).to(torch.bfloat16))


# ---------------------------------------------------------------- streams and graphs ---

@pytest.mark.parametrize("n", [1, 16, 40])
def test_captured_and_replayed(cuda, mm, n):
    """Round, multiply and unpack captured into one graph; replayed on new inputs it gives what eager calls give."""
    m, k, group = 300, 1024, 128
    gen = torch.Generator().manual_seed(2)
    w = torch.empty(m, k, dtype=torch.float16, device="cuda")
    x = torch.empty(n, k, dtype=torch.float16, device="cuda")
    packed = torch.empty(mm.w4_bytes(m, k, group, True), dtype=torch.uint8, device="cuda")
    C = torch.empty(n, m, dtype=torch.float16, device="cuda")
    back = torch.empty_like(w)

    def step(c, b):
        mm.w4_quantize("f16", m, k, group, True, w, k, packed)
        mm.gemm_w4("f16", m, n, k, 1.0, packed, group, True, x, k, 0.0, c, m)
        mm.w4_unpack("f16", m, k, group, True, packed, b, k)

    w.zero_(), x.zero_()
    step(C, back)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(C, back)
    for _ in range(3):
        w.copy_(torch.randn(m, k, generator=gen) * 0.02)
        x.copy_(torch.randn(n, k, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        c2, b2 = torch.empty_like(C), torch.empty_like(back)
        step(c2, b2)
        torch.cuda.synchronize()
        assert torch.equal(C, c2) and torch.equal(back, b2)


def test_two_streams_at_once(cuda, mm):
    """The same weights used from two streams at the same time, many times over."""
    gen = torch.Generator().manual_seed(4)
    m, k = 2000, 4000
    codes, scales, zps = make_w4(gen, m, k, 128, False, torch.float16)
    packed = pack(mm, "f16", codes, scales, zps, 128)
    want, xs, outs = [], [], []
    for n in (1, 7, 16, 33):
        x = torch.randn(n, k, generator=gen).half().cuda()
        c = torch.empty(n, m, dtype=torch.float16, device="cuda")
        mm.gemm_w4("f16", m, n, k, 1.0, packed, 128, False, x, k, 0.0, c, m)
        xs.append(x), want.append(c)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(40):
        j = i % 4
        c = torch.empty_like(want[j])
        outs.append((j, c))
    torch.cuda.synchronize()
    for i, (j, c) in enumerate(outs):
        mm.gemm_w4("f16", m, xs[j].shape[0], k, 1.0, packed, 128, False, xs[j], k, 0.0, c, m,
                   stream=streams[i // 4 % 2])
    torch.cuda.synchronize()
    assert all(torch.equal(want[j], c) for j, c in outs)

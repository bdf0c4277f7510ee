"""Workloads of the low-bit and mixture-of-experts products: 4-bit weights with group scales times a few (or many)
columns of activations, the round trip of a weight matrix through that format, and a whole mixture-of-experts layer
for a few tokens.

Every workload has two forms.  With `own` false, `run` computes it with elementary torch operations in 32 bits (the
router's scores in 64, because a selection hangs on their order) and rounds once at the end.  With `own` true it makes
the calls of `gemm_mmbo_b200`.  Matrices follow the library's convention: column-major, so that a torch tensor of
shape (columns, leading dimension) holds one, and the weights are the transposed operand (k contiguous).

The 4-bit format.  A weight matrix of m rows and k columns has one code 0..15 per element, one scale per row and group
of `group` consecutive columns (the last group may be short), in the activations' type, and either one zero point
0..15 per row and group or the fixed zero point 8.  The weight is (code - zero point) * scale.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # One token of a small model's square projection: 2 MB of codes, so the launch and the latency of one trip to
        # memory are what a decoder of that size pays some hundred times per token.
        dict(name="gemm_w4_one_token_small", op="gemm_w4", dtype="f16", m=2048, k=2048, n=1, group=128, zeros=False,
             pad=0),
        # One token of a wide up projection with zero points, as asymmetric checkpoints store them.
        dict(name="gemm_w4_one_token_wide", op="gemm_w4", dtype="bf16", m=14336, k=4096, n=1, group=128, zeros=True,
             pad=0),
        # One token of a long down projection of a large model: 117 MB of codes, pure bandwidth.
        dict(name="gemm_w4_one_token_long", op="gemm_w4", dtype="f16", m=8192, k=28672, n=1, group=128, zeros=False,
             pad=0),
        # A handful of sequences, finer groups, ragged sizes and padded leading dimensions: a projection cut over
        # three devices, whose blocks are no multiple of anything.
        dict(name="gemm_w4_few_ragged", op="gemm_w4", dtype="f16", m=3669, k=11005, n=5, group=64, zeros=True, pad=3),
        # A decoding batch of sixteen sequences.
        dict(name="gemm_w4_batch16", op="gemm_w4", dtype="bf16", m=8192, k=8192, n=16, group=128, zeros=False, pad=0),
        # Speculative decoding or a larger batch: 48 columns, still close to the bound by bytes.
        dict(name="gemm_w4_batch48", op="gemm_w4", dtype="f16", m=8192, k=8192, n=48, group=128, zeros=True, pad=0),
        # A prompt of 512 tokens through the same weights: bound by the products.
        dict(name="gemm_w4_prompt512", op="gemm_w4", dtype="bf16", m=8192, k=4096, n=512, group=128, zeros=False,
             pad=0),
        # Weights rounded to the format and back, as a training step with quantised forward weights or an export
        # check does it: one projection of a middle-sized model.
        dict(name="w4_round_square", op="w4_round", dtype="f16", m=4096, k=4096, group=128, zeros=False, pad=0),
        # The same with zero points, a fine group and ragged sizes, larger than the second-level cache.
        dict(name="w4_round_ragged", op="w4_round", dtype="bf16", m=11001, k=8200, group=32, zeros=True, pad=8),
        # One token through a layer of many small experts: latency of the chain router -> up -> down.
        dict(name="moe_one_token", op="moe", dtype="bf16", tokens=1, d=2048, f=1408, experts=64, topk=6, renorm=True,
             group=0, zeros=False, pad=0),
        # A few sequences through a layer with 4-bit experts, ragged expert width.
        dict(name="moe_few_w4", op="moe", dtype="f16", tokens=8, d=4096, f=1800, experts=32, topk=4, renorm=True,
             group=128, zeros=True, pad=0),
        # A decoding batch that reaches nearly every expert: the whole layer's weights are read.
        dict(name="moe_batch", op="moe", dtype="f16", tokens=48, d=2048, f=1408, experts=64, topk=8, renorm=False,
             group=0, zeros=False, pad=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges.  Sizes are spread over their logarithm and mostly odd."""
    op = rng.choice(["gemm_w4", "gemm_w4", "gemm_w4", "w4_round", "moe", "moe"])
    dtype = rng.choice(["f16", "bf16"])
    group = rng.choice([32, 64, 128])
    zeros = rng.random() < 0.5
    pad = rng.choice([0, 0, 8, 3])
    if op == "gemm_w4":
        while True:
            m, k, n = _log(rng, 200, 20000), _log(rng, 200, 28672), _log(rng, 1, 512)
            if rng.random() < 0.5:
                m, k = (m + 63) // 64 * 64, (k + 63) // 64 * 64
            if m * k <= 8192 * 28672 and m * k * n <= 8192 * 4096 * 512 and m * k * n >= 1 << 20:
                break
        return dict(op=op, dtype=dtype, m=m, k=k, n=n, group=group, zeros=zeros, pad=pad)
    if op == "w4_round":
        while True:
            m, k = _log(rng, 200, 20000), _log(rng, 200, 20000)
            if m * k <= 11001 * 8200:
                break
        return dict(op=op, dtype=dtype, m=m, k=k, group=group, zeros=zeros, pad=pad)
    w4 = rng.random() < 0.5
    while True:
        tokens, experts = _log(rng, 1, 64), _log(rng, 4, 128)
        topk = rng.randint(1, min(8, experts))
        d, f = _log(rng, 500, 5000), _log(rng, 300, 4000)
        if rng.random() < 0.7:
            d, f = (d + 31) // 32 * 32, (f + 31) // 32 * 32
        if 3 * experts * d * f <= 600e6 and 3 * tokens * topk * d * f <= 4e9:
            break
    return dict(op=op, dtype=dtype, tokens=tokens, d=d, f=f, experts=experts, topk=topk, renorm=rng.random() < 0.5,
                group=group if w4 else 0, zeros=zeros if w4 else False, pad=pad)


# ---------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFFFFFFFFF)
    return g


def _activations(gen, n, k, pad, dt):
    """n columns of k activations, `pad` unused elements behind each; one channel in a hundred is ten times as large,
    as hidden states of language models have it."""
    buf = torch.randn(n, k + pad, generator=gen, device="cuda")
    loud = torch.rand(1, k + pad, generator=gen, device="cuda") < 0.01
    return torch.where(loud, buf * 10, buf).to(dt)


def _w4(gen, m, k, group, zeros, dt):
    """Codes, two a byte (element 2i in the low half; the last half of an odd row is unused), scales and zero points
    of one matrix: codes of normally distributed weights, scales around 0.005."""
    g = -(-k // group)
    k2 = (k + 1) // 2
    codes = torch.empty(m, k2, dtype=torch.uint8, device="cuda")
    for lo in range(0, m, 4096):
        hi = min(m, lo + 4096)
        c = (torch.randn(hi - lo, 2 * k2, generator=gen, device="cuda") * 2.7 + 8).round_().clamp_(0, 15)
        c = c.to(torch.uint8)
        codes[lo:hi] = c[:, 0::2] | (c[:, 1::2] << 4)
    scales = (0.005 * (0.5 + torch.rand(m, g, generator=gen, device="cuda"))).to(dt)
    zps = torch.randint(5, 11, (m, g), generator=gen, device="cuda", dtype=torch.uint8) if zeros else None
    return dict(codes=codes, scales=scales, zps=zps)


def _inputs(case, seed):
    gen = _gen(seed)
    dt = TYPES[case["dtype"]]
    if case["op"] == "gemm_w4":
        w = _w4(gen, case["m"], case["k"], case["group"], case["zeros"], dt)
        return dict(w=w, x=_activations(gen, case["n"], case["k"], case["pad"], dt))
    if case["op"] == "w4_round":
        w = torch.empty(case["m"], case["k"] + case["pad"], dtype=dt, device="cuda")
        for lo in range(0, case["m"], 4096):
            part = w[lo:lo + 4096]
            part.copy_(torch.randn(part.shape, generator=gen, device="cuda") * 0.02)
        return dict(w=w)
    E, d, f = case["experts"], case["d"], case["f"]
    s = dict(x=_activations(gen, case["tokens"], d, case["pad"], dt),
             router=(torch.randn(E, d, generator=gen, device="cuda") / math.sqrt(d)).to(dt))
    for name, rows, cols in (("gate", f, d), ("up", f, d), ("down", d, f)):
        if case["group"]:
            s[name] = [_w4(gen, rows, cols, case["group"], case["zeros"], dt) for _ in range(E)]
        else:
            w = torch.empty(E, rows, cols, dtype=dt, device="cuda")
            for e in range(E):
                w[e] = torch.randn(rows, cols, generator=gen, device="cuda") / math.sqrt(cols)
            s[name] = w
    return s


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if case["op"] == "moe" and case["group"]:  # one tensor for all experts, to index with their numbers
        for name in ("gate", "up", "down"):
            per = state[name]
            state[name] = {k: (None if per[0][k] is None else torch.stack([p[k] for p in per])) for k in per[0]}
    dt = TYPES[case["dtype"]]
    if own:
        import gemm_mmbo_b200 as mm
        state["mm"] = mm

        def packed(w, m, k):
            buf = torch.empty(mm.w4_bytes(m, k, case["group"], case["zeros"]), dtype=torch.uint8, device="cuda")
            g = -(-k // case["group"])
            mm.w4_pack(case["dtype"], m, k, case["group"], w["codes"], w["codes"].shape[-1], w["scales"], g, w["zps"],
                       g, buf)
            return buf

        if case["op"] == "gemm_w4":
            state["packed"] = packed(state["w"], case["m"], case["k"])
            state["y"] = torch.empty(case["n"], case["m"] + case["pad"], dtype=dt, device="cuda")
        elif case["op"] == "w4_round":
            state["packed"] = torch.empty(mm.w4_bytes(case["m"], case["k"], case["group"], case["zeros"]),
                                          dtype=torch.uint8, device="cuda")
            state["back"] = torch.empty_like(state["w"])
        else:
            E, d, f, t = case["experts"], case["d"], case["f"], case["tokens"]
            if case["group"]:
                for name, rows, cols in (("gate", f, d), ("up", f, d), ("down", d, f)):
                    per = [packed({k: (None if v is None else v[e]) for k, v in state[name].items()}, rows, cols)
                           for e in range(E)]
                    state[name + "_packed"] = torch.stack(per)
            state["y"] = torch.empty(t, d + case["pad"], dtype=dt, device="cuda")
            state["ids"] = torch.empty(t, case["topk"], dtype=torch.int32, device="cuda")
            state["gates"] = torch.empty(t, case["topk"], dtype=torch.float32, device="cuda")
            state["ws"] = torch.empty(mm.moe_workspace_bytes(case["dtype"], t, d, f, E, case["topk"]),
                                      dtype=torch.uint8, device="cuda")
    return state


# ---------------------------------------------------------------------------------------------------- one pass

def _dequantised(w, k, group):
    """(..., m, k) weights in 32 bits from packed codes."""
    both = torch.stack((w["codes"] & 15, w["codes"] >> 4), dim=-1)
    codes = both.flatten(-2)[..., :k].float()
    grp = torch.arange(k, device=codes.device) // group
    zero = 8.0 if w["zps"] is None else w["zps"].float()[..., grp]
    return (codes - zero) * w["scales"].float()[..., grp]


def _round_plain(w, group, zeros):
    m, k = w.shape
    g = -(-k // group)
    x = w.float()
    if g * group != k:
        x = torch.cat((x, x.new_zeros(m, g * group - k)), dim=1)
    x = x.view(m, g, group)
    if zeros:
        lo, hi = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
        scale = ((hi - lo) / 15).to(w.dtype).float()
        live = torch.where(scale > 0, scale, torch.ones_like(scale))
        zero = torch.where(scale > 0, torch.round(-lo / live).clamp(0, 15), torch.zeros_like(lo))
    else:
        scale = (x.abs().amax(-1, keepdim=True) / 7).to(w.dtype).float()
        live = torch.where(scale > 0, scale, torch.ones_like(scale))
        zero = torch.full_like(scale, 8)
    code = torch.where(scale > 0, (torch.round(x / live) + zero).clamp(0, 15), zero)
    return ((code - zero) * scale).view(m, g * group)[:, :k].to(w.dtype)


def _moe_plain(s, case):
    d, k, dt = case["d"], case["topk"], TYPES[case["dtype"]]
    x = s["x"][:, :d].float()
    scores = x.double() @ s["router"].double().t()
    prob = torch.softmax(scores, dim=-1)
    order = torch.argsort(prob, dim=-1, descending=True, stable=True)[:, :k]
    gate = torch.gather(prob, 1, order)
    if case["renorm"]:
        gate = gate / gate.sum(-1, keepdim=True)
    gate = gate.float()

    def weights(name, ids, cols):
        if case["group"]:
            w = s[name]
            return _dequantised({n: (None if v is None else v[ids]) for n, v in w.items()}, cols, case["group"])
        return s[name][ids].float()

    y = torch.zeros_like(x)
    for j in range(k):  # the j-th expert of every token
        ids = order[:, j]
        for t0 in range(0, ids.numel(), 16):
            part, xp = ids[t0:t0 + 16], x[t0:t0 + 16].unsqueeze(-1)
            g = torch.bmm(weights("gate", part, d), xp)
            u = torch.bmm(weights("up", part, d), xp)
            h = g * torch.sigmoid(g) * u
            y[t0:t0 + 16] += gate[t0:t0 + 16, j:j + 1] * torch.bmm(weights("down", part, case["f"]), h).squeeze(-1)
    return dict(y=y.to(dt), ids=order.int(), gates=gate)


def run(state):
    case = state["case"]
    op, dt = case["op"], case["dtype"]
    if not own:
        if op == "gemm_w4":
            w = _dequantised(state["w"], case["k"], case["group"])
            return (state["x"][:, :case["k"]].float() @ w.t()).to(TYPES[dt])
        if op == "w4_round":
            return _round_plain(state["w"][:, :case["k"]], case["group"], case["zeros"])
        return _moe_plain(state, case)
    mm = state["mm"]
    if op == "gemm_w4":
        y, x = state["y"], state["x"]
        mm.gemm_w4(dt, case["m"], case["n"], case["k"], 1.0, state["packed"], case["group"], case["zeros"], x,
                   x.shape[1], 0.0, y, y.shape[1])
        return y[:, :case["m"]]
    if op == "w4_round":
        w, back = state["w"], state["back"]
        mm.w4_quantize(dt, case["m"], case["k"], case["group"], case["zeros"], w, w.shape[1], state["packed"])
        mm.w4_unpack(dt, case["m"], case["k"], case["group"], case["zeros"], state["packed"], back, back.shape[1])
        return back[:, :case["k"]]
    E, d, f = case["experts"], case["d"], case["f"]
    x, y, suffix = state["x"], state["y"], "_packed" if case["group"] else ""
    gate, up, down = (state[n + suffix] for n in ("gate", "up", "down"))
    if case["group"]:
        strides = dict(ldg=0, strideG=gate.shape[1], ldd=0, strideD=down.shape[1])
    else:
        strides = dict(ldg=d, strideG=f * d, ldd=f, strideD=d * f)
    mm.moe(dt, case["tokens"], d, f, E, case["topk"], x, x.shape[1], state["router"], d, gate, up, down=down,
           group=case["group"], zeros=case["zeros"], renorm=case["renorm"], beta=0.0, Y=y, ldy=y.shape[1],
           ids=state["ids"], gates=state["gates"], workspace=state["ws"], **strides)
    return dict(y=y[:, :d], ids=state["ids"], gates=state["gates"])


# ---------------------------------------------------------------------------------------------------- floor

def _w4_bytes(m, k, group, zeros):
    g = -(-k // group)
    return m * ((k + 1) // 2) + m * g * (2 + (0.5 if zeros else 0))


def work(case):
    """Each input read once, each output written once.  A mixture-of-experts pass reads the experts that its tokens
    choose; their number depends on the inputs, and what is counted is its expectation for independent, even
    choices."""
    if case["op"] == "gemm_w4":
        m, n, k = case["m"], case["n"], case["k"]
        return dict(bytes=int(_w4_bytes(m, k, case["group"], case["zeros"]) + 2 * n * (m + k)), flops=2 * m * n * k)
    if case["op"] == "w4_round":
        m, k = case["m"], case["k"]
        return dict(bytes=4 * m * k, flops=4 * m * k)
    t, d, f, E, top = case["tokens"], case["d"], case["f"], case["experts"], case["topk"]
    touched = E * (1 - (1 - top / E) ** t)
    if case["group"]:
        expert = 2 * _w4_bytes(f, d, case["group"], case["zeros"]) + _w4_bytes(d, f, case["group"], case["zeros"])
    else:
        expert = 6 * d * f
    return dict(bytes=int(touched * expert + 2 * E * d + 4 * t * d + 8 * t * top),
                flops=6 * t * top * d * f + 2 * t * E * d)


# ---------------------------------------------------------------------------------------------------- 64 bits

def _exact_weights(w, k, group):
    c = torch.empty(w["codes"].shape[0], 2 * w["codes"].shape[1], dtype=torch.float64, device=w["codes"].device)
    c[:, 0::2] = w["codes"] % 16
    c[:, 1::2] = torch.div(w["codes"], 16, rounding_mode="floor")
    c = c[:, :k]
    for g in range(w["scales"].shape[1]):
        cols = slice(g * group, min(k, (g + 1) * group))
        c[:, cols] -= 8 if w["zps"] is None else w["zps"][:, g:g + 1].double()
        c[:, cols] *= w["scales"][:, g:g + 1].double()
    return c


def exact(case, seed):
    s = _inputs(case, seed)
    dt = TYPES[case["dtype"]]
    if case["op"] == "gemm_w4":
        x = s["x"][:, :case["k"]].double()
        return torch.einsum("nk,mk->nm", x, _exact_weights(s["w"], case["k"], case["group"]))
    if case["op"] == "w4_round":
        k, group = case["k"], case["group"]
        out = torch.empty(case["m"], k, dtype=torch.float64, device="cuda")
        for lo in range(0, k, group):
            w = s["w"][:, lo:min(k, lo + group)].double()
            if case["zeros"]:
                bottom, top = w.min(1).values.clamp(max=0), w.max(1).values.clamp(min=0)
                scale = ((top - bottom) / 15).to(dt).double()
                zero = torch.nan_to_num(torch.round(-bottom / scale), nan=0.0).clamp(0, 15)
            else:
                scale = (w.abs().max(1).values / 7).to(dt).double()
                zero = torch.full_like(scale, 8)
            steps = torch.nan_to_num(torch.round(w / scale[:, None]), nan=0.0, posinf=0.0, neginf=0.0)
            code = (steps + zero[:, None]).clamp(0, 15)
            out[:, lo:lo + w.shape[1]] = (code - zero[:, None]) * scale[:, None]
        return out
    d, top = case["d"], case["topk"]
    x = s["x"][:, :d].double()
    scores = torch.einsum("td,ed->te", x, s["router"].double())
    prob = (scores - scores.max(1, keepdim=True).values).exp()
    prob = prob / prob.sum(1, keepdim=True)
    gates, ids = torch.sort(prob, dim=1, descending=True, stable=True)
    gates, ids = gates[:, :top], ids[:, :top]
    if case["renorm"]:
        gates = gates / gates.sum(1, keepdim=True)
    y = torch.zeros_like(x)
    for e in range(case["experts"]):
        rows, slots = torch.nonzero(ids == e, as_tuple=True)
        if rows.numel() == 0:
            continue
        if case["group"]:
            gate, up, down = (_exact_weights(s[n][e], c, case["group"])
                              for n, c in (("gate", d), ("up", d), ("down", case["f"])))
        else:
            gate, up, down = (s[n][e].double() for n in ("gate", "up", "down"))
        g, u = x[rows] @ gate.t(), x[rows] @ up.t()
        y.index_add_(0, rows, gates[rows, slots, None] * ((g / (1 + (-g).exp()) * u) @ down.t()))
    return dict(y=y, ids=ids.int(), gates=gates)

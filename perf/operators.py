"""What the embedding and optimiser operators are measured on: the cases, their inputs, their plain
form in elementary torch operations, and their values in 64 bits.

Three kinds of case: "lookup" (rows of a table by token, scaled), "gradient" (the table's gradient,
summed by token) and "adamw" (one AdamW step over many tensors, optionally clipped by the norm of all
their gradients, states in 32 or 8 bits).
"""
import importlib
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
MOST_FEATURES = 3355443 * 64  # rows x features of the largest listed lookup
MOST_VALUES = 150_000_000     # values of the largest listed optimiser step

LR, BETA1, BETA2, EPS, DECAY, STEP, SEED = 1e-3, 0.9, 0.999, 1e-8, 0.01, 100, 12345
BLOCK = 256  # values that share a scale where the states have 8 bits


def _abi():
    return importlib.import_module("sparseconvnet-archived_b200").abi


# ------------------------------------------------------------------------------------------ cases
def listed():
    lookup = dict(op="lookup", table="f32", out="f32", pad=0)
    grad = dict(op="gradient", dout="f32", pad=0, accumulate=False, hot=0.0)
    adam = dict(op="adamw", net=0, tensors=0, values=0, bits=32, grad="f32", copy="", clip=0.0)
    return [
        # one picture of strokes (about 200 sites): what a single request looks up
        dict(lookup, name="lookup one picture", n=203, vocab=128, C=32),
        # a batch of 64 voxelised surfaces, 3.5 k sites each, every site a material code; 16-bit table, odd row stride
        # (the features go into columns of a wider matrix)
        dict(lookup, name="lookup surfaces strided", n=224101, vocab=5003, C=96, table="bf16", pad=3),
        # the space-time volume's batch of 512 (6.5 k sites a sample), 64 features a site
        dict(lookup, name="lookup volume batch", n=3355443, vocab=65536, C=64),
        # training on one picture
        dict(grad, name="gradient one picture", n=203, vocab=128, C=32),
        # a small vocabulary with one code on a third of the sites
        dict(grad, name="gradient surfaces hot", n=224101, vocab=5003, C=96, hot=0.3),
        # gradient accumulation over parts of a batch, odd width and stride
        dict(grad, name="gradient odd accumulated", n=50021, vocab=30011, C=33, pad=5, accumulate=True),
        # the space-time volume's batch of 512, 16-bit gradients, a large table
        dict(grad, name="gradient volume batch", n=3355443, vocab=131072, C=64, dout="bf16"),
        # the strokes network (14 tensors, 0.2 M values): launch-bound
        dict(adam, name="adamw strokes network", net=1),
        # the same with 8-bit states
        dict(adam, name="adamw strokes 8-bit", net=1, bits=8),
        # the DeepCNet(5,100) benchmark network (2.8 M values), clipped by the norm over all gradients
        dict(adam, name="adamw DeepCNet clipped", net=2, clip=1.0),
        # a large model: matrices and vectors of odd sizes, 16-bit gradients and a 16-bit copy of the weights
        dict(adam, name="adamw large", tensors=200, values=MOST_VALUES, grad="bf16", copy="bf16"),
        # the same model with 8-bit states
        dict(adam, name="adamw large 8-bit", tensors=200, values=MOST_VALUES, grad="bf16", copy="bf16", bits=8),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["lookup", "gradient", "adamw"])
    if op == "adamw":
        values = _log(rng, 1, MOST_VALUES)
        return dict(op=op, net=0, tensors=max(1, min(_log(rng, 1, 400), values)), values=values, bits=rng.choice([32, 8]),
                    grad=rng.choice(["f32", "bf16", "f16"]), copy=rng.choice(["", "bf16", "f16"]), clip=rng.choice([0.0, 1.0]))
    C = _log(rng, 1, 1024)
    n = _log(rng, 1, min(3355443, MOST_FEATURES // C))
    vocab = min(_log(rng, 2, 262144), MOST_FEATURES // C)
    pad = rng.choice([0, 0, 1, 3, 8])
    n = max(1, min(n, MOST_FEATURES // (C + pad)))
    if op == "lookup":
        return dict(op=op, n=n, vocab=vocab, C=C, pad=pad, table=rng.choice(["f32", "bf16", "f16"]), out=rng.choice(["f32", "f32", "bf16", "f16"]))
    return dict(op=op, n=n, vocab=vocab, C=C, pad=pad, dout=rng.choice(["f32", "bf16", "f16"]), accumulate=rng.choice([False, True]), hot=rng.choice([0.0, 0.3]))


def _sizes(case):
    """The sizes of the tensors of an optimiser step: a network's weights and biases, or matrices and vectors of odd sizes."""
    nets = {1: (3, 3, (32, 64, 96, 128, 160), 10), 2: (3, 3, (100, 200, 300, 400, 500, 600), 10)}
    if case["net"]:
        nin, first, widths, classes = nets[case["net"]]
        out = []
        for i, w in enumerate(widths):
            k = nin * (first if i == 0 else 2) ** 2
            out += [k * w, w]
            nin = w
        return out + [nin * classes, classes]
    T, total = case["tensors"], case["values"]
    r = random.Random(T * 1000003 + total)
    share = [4.0 ** r.uniform(0, 3) if i % 2 == 0 else 4.0 ** r.uniform(-6, -4) for i in range(T)]
    left, all_ = total - T, sum(share)
    size = [1 + int(left * s / all_) for s in share]
    size[0] += total - sum(size)
    return size


# ------------------------------------------------------------------------------------------ inputs
def _tokens(case, gen):
    """Tokens as they come: few frequent ones, many rare ones (the k-th in frequency about 1 / k), in no order of frequency;
    one row in 512 a background row (-1); with `hot`, that share of the rows has one and the same token."""
    n, V = case["n"], case["vocab"]
    u = torch.rand(n, device="cuda", generator=gen, dtype=torch.float64)
    rank = (torch.exp(u * math.log(V + 1)) - 1).long().clamp_(0, V - 1)
    tok = torch.randperm(V, device="cuda", generator=gen)[rank].int()
    if case.get("hot"):
        tok[torch.rand(n, device="cuda", generator=gen) < case["hot"]] = V // 3
    tok[torch.rand(n, device="cuda", generator=gen) < 1 / 512] = -1
    return tok


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    if case["op"] == "lookup":
        out = torch.empty((case["n"], case["C"] + case["pad"]), device="cuda", dtype=TYPES[case["out"]])[:, case["pad"]:]
        return dict(case=case, tokens=_tokens(case, gen), table=randn(case["vocab"], case["C"]).to(TYPES[case["table"]]), out=out,
                    scale=math.sqrt(case["C"]))
    if case["op"] == "gradient":
        state = dict(case=case, tokens=_tokens(case, gen), dout=randn(case["n"], case["C"] + case["pad"]).to(TYPES[case["dout"]])[:, case["pad"]:],
                     scale=math.sqrt(case["C"]))
        if case["accumulate"]:
            state["dtable"] = randn(case["vocab"], case["C"])
        else:
            state["dtable"] = torch.empty((case["vocab"], case["C"]), device="cuda")
        if own:
            state["workspace"] = _abi().embedding_backward_workspace(case["n"], case["vocab"], case["C"], torch.device("cuda"))
        return state
    # adamw: all tensors lie in flat buffers, each at a multiple of BLOCK values
    sizes = _sizes(case)
    start, at = [], 0
    for s in sizes:
        start.append(at)
        at += -(-s // BLOCK) * BLOCK
    inside = torch.zeros(at, device="cuda")
    decay = torch.zeros(at, device="cuda")
    for i, (o, s) in enumerate(zip(start, sizes)):
        inside[o:o + s] = 1
        decay[o:o + s] = _decay(i)
    spread = torch.exp(2 * randn(at))  # gradients of one tensor differ by orders of magnitude
    w = randn(at) * 0.05 * inside
    g = (randn(at) * spread * 1e-3 * inside).to(TYPES[case["grad"]])
    m = randn(at) * spread * 3e-4 * inside
    v = (spread * 1e-3) ** 2 * torch.rand(at, device="cuda", generator=gen) * inside
    state = dict(case=case, w=w, g=g, decay=decay, copy=torch.zeros(at, device="cuda", dtype=TYPES[case["copy"]]) if case["copy"] else None)
    if case["bits"] == 8:
        half = torch.full((at,), 32767.5 / 65536, device="cuda")
        state["m"], state["ms"] = _encode_m(m, half)
        state["v"], state["vs"] = _encode_v(v, half)
    else:
        state["m"], state["v"] = m, v
    del inside, spread
    if own:
        state["optimiser"] = _optimiser(state, start, sizes)
    return state


def _decay(i):
    return DECAY if i % 2 == 0 else 0.0  # matrices decay, vectors do not


def _optimiser(state, start, sizes):
    """The framework's handle on the tensors: views of the flat buffers."""
    abi, tensors = _abi(), []
    for i, (o, s) in enumerate(zip(start, sizes)):
        part = lambda t, d=1: None if t is None else t[o // d:o // d + -(-s // d)]  # noqa: E731
        tensors.append(dict(w=part(state["w"]), g=part(state["g"]), m=part(state["m"]), v=part(state["v"]), weight_decay=_decay(i),
                            w16=part(state["copy"]), m_scale=part(state.get("ms"), BLOCK), v_scale=part(state.get("vs"), BLOCK)))
    return abi.AdamW(tensors)


# ------------------------------------------------------------------------------------------ the operators
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    case, abi = state["case"], _abi()
    if case["op"] == "lookup":
        return abi.embedding_forward(state["table"], state["tokens"], state["scale"], out=state["out"])
    if case["op"] == "gradient":
        return abi.embedding_backward(state["dout"], state["tokens"], state["dtable"], state["scale"], accumulate=case["accumulate"],
                                      workspace=state["workspace"])
    opt = state["optimiser"]
    norm = opt.grad_norm() if case["clip"] else None
    opt.step(LR, STEP, beta1=BETA1, beta2=BETA2, eps=EPS, seed=SEED, norm=norm, max_norm=case["clip"])
    if case["bits"] == 8:
        m, v = abi.adamw_decode(state["m"], state["ms"]), abi.adamw_decode(state["v"], state["vs"])
    else:
        m, v = state["m"], state["v"]
    return dict(w=state["w"], m=m, v=v, copy=state["copy"], norm=norm)


def _run_plain(state):
    case = state["case"]
    if case["op"] == "lookup":
        tok = state["tokens"]
        rows = state["table"][tok.clamp(min=0).long()].float() * state["scale"]
        rows[tok < 0] = 0
        state["out"].copy_(rows)
        return state["out"]
    if case["op"] == "gradient":
        tok, V = state["tokens"], case["vocab"]
        total = torch.zeros((V + 1, case["C"]), device="cuda", dtype=torch.float64)  # 64 bits: sums of up to millions of rows
        total.index_add_(0, torch.where(tok < 0, V, tok), state["dout"].double())
        total = (total[:V] * state["scale"])
        if case["accumulate"]:
            state["dtable"].copy_(state["dtable"] + total)
        else:
            state["dtable"].copy_(total)
        return state["dtable"]
    b1, b2, n1, n2 = _f32(BETA1), _f32(BETA2), _f32(1 - BETA1), _f32(1 - BETA2)
    c1, c2 = _f32(1 / (1 - BETA1 ** STEP)), _f32(1 / math.sqrt(1 - BETA2 ** STEP))
    w, g = state["w"], state["g"].float()
    norm = None
    if case["clip"]:
        norm = g.double().square().sum().sqrt().float()
        g = g * torch.clamp(case["clip"] / norm, max=1.0)
    eight = case["bits"] == 8
    m = _decode_m(state["m"], state["ms"]) if eight else state["m"]
    v = _decode_v(state["v"], state["vs"]) if eight else state["v"]
    m = m * b1 + g * n1
    v = v * b2 + (g * g) * n2
    w.sub_((m / (v.sqrt() * c2 + _f32(EPS)) * c1 + w * state["decay"]) * _f32(LR))
    if eight:
        u_m, u_v = _dither(w.numel(), SEED)
        codes, scale = _encode_m(m, u_m)
        state["m"].copy_(codes), state["ms"].copy_(scale)
        codes, scale = _encode_v(v, u_v)
        state["v"].copy_(codes), state["vs"].copy_(scale)
        m, v = _decode_m(state["m"], state["ms"]), _decode_v(state["v"], state["vs"])
    else:
        state["m"].copy_(m), state["v"].copy_(v)
    if state["copy"] is not None:
        state["copy"].copy_(w)
    return dict(w=w, m=m if eight else state["m"], v=v if eight else state["v"], copy=state["copy"], norm=norm)


def _f32(x):
    return float(torch.tensor(x, dtype=torch.float64).float())


# ---- the 8-bit states: blocks of BLOCK values with a power of two s as their scale; a first moment is q |q| s with q in
# -127..127, a second one q^4 s with q in 0..255
def _decode_m(codes, scale):
    q = codes.float().view(-1, BLOCK)
    return (q * q.abs() * scale[:, None]).view(-1)


def _decode_v(codes, scale):
    q = codes.float().view(-1, BLOCK)
    p = q * q
    return (p * p * scale[:, None]).view(-1)


def _power(e):
    """2^e for whole e in -126..127."""
    return ((e + 127) << 23).int().view(torch.float32)


def _scale(most, top, bits):
    """The smallest 2^e, e >= -126, with most <= top 2^e, and 2^-e; top lies between 2^bits and 2^(bits + 1)."""
    e = (torch.frexp(most)[1].long() - 1 - bits).clamp(-126, 127)
    e = torch.where(most > top * _power(e), e + 1, e)
    scale = torch.where(most > 0, _power(e), 0.0)
    return torch.where(torch.isfinite(most), scale, math.nan), _power(-e)


def _encode_m(m, u):
    m, u = m.view(-1, BLOCK), u.view(-1, BLOCK)
    scale, inverse = _scale(m.abs().amax(1), 127.0 ** 2, 13)
    x = m.abs() * inverse[:, None]
    q = x.sqrt().floor()
    q = torch.where(q * q > x, q - 1, q)
    q = torch.where((q + 1) * (q + 1) <= x, q + 1, q)
    up = (x - q * q) > u * (2 * q + 1)
    q = torch.where(up, q + 1, q) * torch.sign(m)
    return q.to(torch.int8).view(-1), scale


def _encode_v(v, u):
    v, u = v.view(-1, BLOCK), u.view(-1, BLOCK)
    fourth = lambda q: (q * q) * (q * q)  # noqa: E731
    scale, inverse = _scale(v.amax(1), float(255 ** 4 - 1), 31)
    y = v * inverse[:, None]
    q = y.sqrt().sqrt().floor()
    q = torch.where(fourth(q) > y, q - 1, q)
    q = torch.where(fourth(q + 1) <= y, q + 1, q)
    up = (y - fourth(q)) > u * (fourth(q + 1) - fourth(q))
    q = torch.where(up, q + 1, q)
    q = torch.where(v > 0, q.clamp(min=1), q)
    return q.to(torch.uint8).view(-1), scale


def _dither(n, seed):
    """Two numbers in (0, 1) for each place, from the place and the seed: 16 bits each of a 32-bit mix."""
    full = 0xFFFFFFFF
    at = torch.arange(n, device="cuda")
    h = ((at & full) * 0x6A09E667 + (((seed * 0xBB67AE85) & full) + (at >> 32) * 0xA54FF53B)) & full
    h = h ^ (h >> 16)
    h = (h * 0xBB67AE85) & full
    h = h ^ (h >> 15)
    h = (h * 0x3C6EF373) & full
    h = h ^ (h >> 16)
    return ((h & 0xFFFF).float() + 0.5) * 2.0 ** -16, ((h >> 16).float() + 0.5) * 2.0 ** -16


# ------------------------------------------------------------------------------------------ costs, values in 64 bits
def _distinct(case):
    """Rows of the table that the tokens of _tokens() name, about: each token's chance to come up at all."""
    n, V = case["n"], case["vocab"]
    step = max(1, V // 4096)
    seen = 0.0
    for k in range(0, V, step):
        p = math.log((k + 2) / (k + 1)) / math.log(V + 1)
        seen += (1 - math.exp(n * math.log1p(-min(p, 0.999999)))) * min(step, V - k)
    return max(1.0, min(n, V, seen))


def work(case):
    if case["op"] == "lookup":
        n, C = case["n"], case["C"]
        return {"bytes": 4 * n + _distinct(case) * C * BYTES[case["table"]] + n * C * BYTES[case["out"]], "flops": n * C}
    if case["op"] == "gradient":
        n, C = case["n"], case["C"]
        table = 8 * _distinct(case) * C if case["accumulate"] else 4 * case["vocab"] * C
        return {"bytes": 4 * n + n * C * BYTES[case["dout"]] + table, "flops": n * C}
    sizes = _sizes(case)
    n, blocks = sum(sizes), sum(-(-s // BLOCK) for s in sizes)
    each = 8 + BYTES[case["grad"]] + (BYTES[case["copy"]] if case["copy"] else 0)
    states = 16 * n if case["bits"] == 32 else (4 + 8) * n + 16 * blocks  # 8 bits: read, written, and returned as the values they stand for
    return {"bytes": each * n + states, "flops": (14 if case["bits"] == 32 else 40) * n + (2 * n if case["clip"] else 0)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lookup":
        keep = s["tokens"] >= 0
        out = torch.zeros((case["n"], case["C"]), device="cuda", dtype=torch.float64)
        out[keep] = torch.index_select(s["table"].double().mul_(s["scale"]), 0, s["tokens"][keep])
        return out
    if case["op"] == "gradient":
        tok, order = torch.sort(s["tokens"].long(), stable=True)
        running = torch.zeros((case["n"] + 1, case["C"]), device="cuda", dtype=torch.float64)
        torch.cumsum(s["dout"][order].double(), 0, out=running[1:])
        at = torch.arange(case["vocab"], device="cuda")
        first, last = torch.searchsorted(tok, at), torch.searchsorted(tok, at, right=True)
        total = torch.where((last > first)[:, None], running[last] - running[first], 0.0) * s["scale"]
        return total + s["dtable"].double() if case["accumulate"] else total
    w, g = s["w"].double(), s["g"].double()
    norm = None
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        g *= min(1.0, case["clip"] / float(norm))
    eight = case["bits"] == 8
    if eight:
        q, p = s["m"].double().view(-1, BLOCK), s["v"].double().view(-1, BLOCK)
        m, v = (q.abs() * q * s["ms"].double()[:, None]).view(-1), (p.pow(4) * s["vs"].double()[:, None]).view(-1)
    else:
        m, v = s["m"].double(), s["v"].double()
    m, v = torch.lerp(g, m, BETA1), torch.lerp(g * g, v, BETA2)
    hat = (m / (1 - BETA1 ** STEP)) / (torch.sqrt(v / (1 - BETA2 ** STEP)) + EPS)
    w = w * (1 - LR * s["decay"].double()) - LR * hat
    return dict(w=w, m=None if eight else m, v=None if eight else v, copy=w if case["copy"] else None, norm=norm)

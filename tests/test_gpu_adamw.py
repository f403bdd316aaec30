"""GPU tests of the AdamW step over many tensors, with 32-bit and 8-bit states, and of the gradients' norm, against plain
64-bit arithmetic, and of the 8-bit codes against a restatement in single 32-bit roundings.

Tolerances count roundings to 32 bits (U = 2^-24 of the value each) and to 16 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
B1, B2, EPS = 0.9, 0.999, 1e-8
BLOCK = 256


# ------------------------------------------------------------------ the 8-bit states, restated in numpy (each operation one rounding)
f32 = np.float32


def np_scale(most, top, bits):
    if most == 0:
        return f32(0), f32(1)
    e = max(math.frexp(float(most))[1] - 1 - bits, -126)
    if most > f32(top) * f32(2.0 ** e):
        e += 1
    return f32(2.0 ** e), f32(2.0 ** -e)


def np_mix(at, seed):
    mask = np.uint64(0xFFFFFFFF)
    h = (np.uint64(0x6A09E667) * (at & mask) + (np.uint64(seed) * np.uint64(0xBB67AE85) & mask) + (at >> np.uint64(32)) * np.uint64(0xA54FF53B)) & mask
    h ^= h >> np.uint64(16)
    h = h * np.uint64(0xBB67AE85) & mask
    h ^= h >> np.uint64(15)
    h = h * np.uint64(0x3C6EF373) & mask
    h ^= h >> np.uint64(16)
    u = lambda b: ((b.astype(f32) + f32(0.5)) * f32(2.0 ** -16))  # noqa: E731
    return u(h & np.uint64(0xFFFF)), u(h >> np.uint64(16))


def np_decode(codes, scale, second):
    q = codes.astype(f32)
    s = np.repeat(scale, BLOCK)[:len(q)]
    return (q * q) * (q * q) * s if second else q * np.abs(q) * s


def np_encode(x, u, second):
    power = (lambda q: (q * q) * (q * q)) if second else (lambda q: q * q)
    codes, scales = np.zeros(len(x), f32), []
    for b in range(0, len(x), BLOCK):
        v = np.abs(x[b:b + BLOCK])
        s, inv = np_scale(v.max(), 4228250624.0 if second else 16129.0, 31 if second else 13)
        y = v * inv
        q = np.floor(y.astype(np.float64) ** (0.25 if second else 0.5)).astype(f32)
        q = np.where(power(q) > y, q - 1, q)
        q = np.where(power(q + 1) <= y, q + 1, q)
        q = np.where(y - power(q) > u[b:b + BLOCK] * (power(q + 1) - power(q)), q + 1, q)
        if second:
            q = np.where((v > 0) & (q < 1), f32(1), q)
        codes[b:b + BLOCK] = q * np.sign(x[b:b + BLOCK])
        scales.append(s)
    return codes.astype(np.uint8 if second else np.int8), np.array(scales, f32)


def np_moments(m, v, g, gs=1.0, b1=B1, b2=B2):
    g = g.astype(f32) * f32(gs)
    m = m * f32(b1) + g * f32(1 - b1)
    v = v * f32(b2) + (g * g) * f32(1 - b2)
    return m, v


# ------------------------------------------------------------------ helpers
def make(abi, rng, sizes, bits=32, g_type=torch.float32, w16=None, decay=0.01, w_min=-math.inf, offset=0, fresh=False):
    """Entries of a list; offset: values by which each array starts behind an aligned address."""
    def put(a, dtype=None):
        a = torch.from_numpy(np.ascontiguousarray(a))
        a = a if dtype is None else a.to(dtype)
        whole = torch.empty(len(a) + offset, dtype=a.dtype, device="cuda")
        whole[offset:] = a
        return whole[offset:]
    out = []
    for k, n in enumerate(sizes):
        spread = np.exp(2 * rng.standard_normal(n))
        t = dict(w=put((rng.standard_normal(n) * 0.05).astype(f32)), g=put((rng.standard_normal(n) * spread * 1e-3).astype(f32), g_type),
                 weight_decay=decay if k % 2 == 0 else 0.0, w_min=w_min)
        m, v = (rng.standard_normal(n) * spread * 3e-4).astype(f32), (spread ** 2 * 1e-6 * rng.random(n)).astype(f32)
        if bits == 32:
            t.update(m=put(m), v=put(v))
        else:
            half = np.full(n, 0.5, f32)
            mq, ms = np_encode(m, half, False) if n else (np.zeros(0, np.int8), np.zeros(0, f32))
            vq, vs = np_encode(v, half, True) if n else (np.zeros(0, np.uint8), np.zeros(0, f32))
            t.update(m=put(mq), v=put(vq), m_scale=torch.from_numpy(ms).cuda(), v_scale=torch.from_numpy(vs).cuda())
        if w16 is not None:
            t["w16"] = put(np.zeros(n, f32), w16)
        out.append(t)
    return out


def snapshot(tensors):
    return [{k: (x.clone() if torch.is_tensor(x) else x) for k, x in t.items()} for t in tensors]


def moments_before(t):
    if t.get("m_scale") is None:
        return t["m"].double(), t["v"].double()
    return tuple(torch.from_numpy(np_decode(t[k].cpu().numpy(), t[k + "_scale"].cpu().numpy(), k == "v")).cuda().double() for k in ("m", "v"))


def check_step(before, after, lr=1e-3, step=3, gs=1.0, b1=B1, b2=B2, eps=EPS):
    """The updated parameters (and 32-bit moments) within the roundings of the formula."""
    lr, eps = float(f32(lr)), float(f32(eps))
    for t, a in zip(before, after):
        g = t["g"].double() * gs
        m0, v0 = moments_before(t)
        m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
        # m: the two factors, the gradient's scale, two products and the addition: at most 4 U on either term, U on the sum
        merr = 5 * U * ((b1 * m0).abs() + ((1 - b1) * g).abs())
        # v: no cancellation; its terms carry up to 2 (gradient scale, twice) + 1 + 1 + 1 roundings, the sum one more
        verr = 7 * U * v
        if t.get("m_scale") is None:
            assert ((a["m"].double() - m).abs() <= merr + 1e-44).all()
            assert ((a["v"].double() - v).abs() <= verr + 1e-44).all()
        c1, c2 = 1 / (1 - b1 ** step), 1 / math.sqrt(1 - b2 ** step)
        den = v.sqrt() * c2 + eps
        hat = m * c1 / den
        decay = float(f32(t["weight_decay"]))
        # hat: m's error, and relative roundings of bias1 (2), v (3.5), root, bias2 (2), the sum (2), the quotient and its approximation
        # (an ulp is 2 U: root and quotient at most 2 ulps each): below 20 U.  Then lr (1), the decay term (2) and the last sum
        err = lr * (merr * c1 / den + 20 * U * hat.abs()) + 3 * U * lr * (hat.abs() + (decay * t["w"].double()).abs())
        want = t["w"].double() - lr * (hat + decay * t["w"].double())
        want = torch.clamp(want, min=float(f32(t["w_min"])))
        assert ((a["w"].double() - want).abs() <= err + U * want.abs() + 1e-44).all()
        if t.get("w16") is not None:
            assert torch.equal(a["w16"], a["w"].to(a["w16"].dtype))


def check_codes(before, after, seed, gs=1.0):
    """8-bit states: exactly the codes and scales of the restatement (each of its operations is one rounding, as the kernel's)."""
    block = 0
    for t, a in zip(before, after):
        n = len(t["w"])
        if n and t.get("m_scale") is not None:
            m, v = (np_decode(t[k].cpu().numpy(), t[k + "_scale"].cpu().numpy(), k == "v") for k in ("m", "v"))
            m, v = np_moments(m, v, t["g"].float().cpu().numpy(), gs)
            um, uv = np_mix(np.arange(n, dtype=np.uint64) + np.uint64(block * BLOCK), seed)
            for k, x, u in (("m", m, um), ("v", v, uv)):
                codes, scale = np_encode(x, u, k == "v")
                assert np.array_equal(a[k + "_scale"].cpu().numpy(), scale), k
                assert np.array_equal(a[k].cpu().numpy(), codes), k
        block += -(-n // BLOCK)


SIZES = [1, 2, 255, 256, 257, 2047, 2048, 2049, 4096, 100003, 7, 0, 31, 33]


# ------------------------------------------------------------------ steps
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("g_type", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("w16", [None, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [0, 1, 2])
def test_step(abi, bits, g_type, w16, offset):
    """Sizes around warps, blocks and chunks; arrays at aligned and odd addresses; types of gradient and copy."""
    ts = make(abi, np.random.default_rng(bits + offset), SIZES, bits, g_type, w16, offset=offset)
    before = snapshot(ts)
    abi.AdamW(ts).step(1e-3, 3, seed=77)
    check_step(before, ts)
    check_codes(before, ts, 77)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(abi, bits):
    """More tensors than one launch takes, most of them small."""
    rng = np.random.default_rng(3)
    ts = make(abi, rng, [int(x) for x in np.exp(rng.uniform(0, 8, 700))], bits)
    before = snapshot(ts)
    abi.AdamW(ts).step(1e-3, 3, seed=5)
    check_step(before, ts)
    check_codes(before, ts, 5)


@pytest.mark.parametrize("count", [1, 15, 16, 17, 48, 49, 319, 320, 321])
def test_list_lengths(abi, count):
    ts = make(abi, np.random.default_rng(count), [100 + 37 * i % 611 for i in range(count)], 8)
    before = snapshot(ts)
    abi.AdamW(ts).step(1e-3, 3, seed=5)
    check_step(before, ts)
    check_codes(before, ts, 5)


def test_mixed_states(abi):
    """A list with both kinds of state, types and sizes: places of the dither are counted over the whole list."""
    rng = np.random.default_rng(8)
    ts = []
    for i, n in enumerate([300, 5, 5000, 1, 256, 77777, 12, 2048] * 3):
        ts += make(abi, rng, [n], 8 if i % 3 else 32, [torch.float32, torch.bfloat16, torch.float16][i % 3], [None, torch.bfloat16][i % 2])
    before = snapshot(ts)
    abi.AdamW(ts).step(1e-3, 3, seed=1234567890)
    check_step(before, ts)
    check_codes(before, ts, 1234567890)


@pytest.mark.parametrize("bits", [32, 8])
def test_from_zero_states_over_several_steps(abi, bits):
    """A run from its start: each step checked on the states the one before left; seeds follow the step numbers."""
    rng = np.random.default_rng(4)
    ts = []
    for n in (1000, 33):
        ts.append(dict(w=torch.from_numpy(rng.standard_normal(n).astype(f32)).cuda(), g=torch.empty(n, device="cuda"), **abi.adamw_states(n, "cuda", bits)))
    opt = abi.AdamW(ts)
    for step in range(1, 8):
        for t in ts:
            t["g"].copy_(torch.from_numpy(rng.standard_normal(len(t["g"])).astype(f32)))
            if step == 2:
                t["g"].zero_()
        before = [dict(t, weight_decay=0.0, w_min=-math.inf) for t in snapshot(ts)]
        opt.step(1e-2, step)
        check_step(before, ts, lr=1e-2, step=step)
        check_codes(before, ts, step)


def test_zero_gradients_from_zero_states_change_nothing(abi):
    for bits in (32, 8):
        t = dict(w=torch.randn(700, device="cuda"), g=torch.zeros(700, device="cuda"), **abi.adamw_states(700, "cuda", bits))
        before = snapshot([t])
        abi.AdamW([t]).step(1e-2, 1)
        assert all(torch.equal(t[k], before[0][k]) for k in t)


def test_lower_bound_and_grad_scale(abi):
    ts = make(abi, np.random.default_rng(2), [5000, 300], 32, w_min=0.001)
    before = snapshot(ts)
    abi.AdamW(ts).step(1e-2, 3, grad_scale=1 / 64)
    check_step(before, ts, lr=1e-2, gs=1 / 64)
    assert min(t["w"].min().item() for t in ts) == f32(0.001)


@pytest.mark.parametrize("betas", [(0.0, 0.0), (0.0, 0.999), (0.95, 0.9)])
def test_other_betas(abi, betas):
    ts = make(abi, np.random.default_rng(2), [5000, 300])
    before = snapshot(ts)
    abi.AdamW(ts).step(1e-2, 10, beta1=betas[0], beta2=betas[1], eps=1e-3)
    check_step(before, ts, 1e-2, 10, 1.0, betas[0], betas[1], 1e-3)


# ------------------------------------------------------------------ norm, clipping
@pytest.mark.parametrize("g_type", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [0, 1])
def test_norm(abi, g_type, offset):
    """64-bit sums: what is left is the rounding of the result to 32 bits."""
    rng = np.random.default_rng(1)
    for sizes in (SIZES, [1], [0, 3], [3000001], [17] * 400):
        ts = make(abi, rng, sizes, 32, g_type, offset=offset)
        want = math.sqrt(sum((t["g"].double() ** 2).sum().item() for t in ts))
        opt = abi.AdamW(ts)
        got = opt.grad_norm().item()
        assert abs(got - want) <= 1.001 * U * want
        assert opt.grad_norm().item() == got


def test_norm_of_large_and_small_values(abi):
    """Squares past 32 bits' range on either side."""
    for x in (1e30, 1e-30):
        t = dict(w=torch.zeros(1000, device="cuda"), g=torch.full((1000,), x, device="cuda"), **abi.adamw_states(1000, "cuda", 32))
        want = math.sqrt(1000) * float(f32(x))
        assert abs(abi.AdamW([t]).grad_norm().item() - want) <= 1.001 * U * want


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [0.01, 1e6])
def test_clipping(abi, bits, max_norm):
    ts = make(abi, np.random.default_rng(6), SIZES, bits)
    before = snapshot(ts)
    opt = abi.AdamW(ts)
    norm = opt.grad_norm()
    opt.step(1e-3, 3, seed=9, grad_scale=0.5, norm=norm, max_norm=max_norm)
    total = f32(norm.item()) * f32(0.5)
    gs = f32(0.5) * (f32(max_norm) / total if total > f32(max_norm) else f32(1))
    assert (gs == f32(0.5)) == (max_norm > 1)
    check_step(before, ts, gs=float(gs))
    check_codes(before, ts, 9, gs)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_norm_that_is_not_finite_changes_nothing(abi, bits, bad):
    ts = make(abi, np.random.default_rng(6), [300, 5000], bits, w16=torch.bfloat16)
    ts[1]["g"][4999] = bad
    before = snapshot(ts)
    opt = abi.AdamW(ts)
    opt.step(1e-3, 3, norm=opt.grad_norm(), max_norm=1.0)
    opt.step(1e-3, 3, norm=opt.grad_norm())  # also without clipping
    for t, b in zip(ts, before):
        assert all(torch.equal(t[k], b[k]) for k in ("w", "m", "v", "w16"))


# ------------------------------------------------------------------ values that are not finite, without a norm
def test_nan_stays_in_its_value_or_block(abi):
    """32 bits: the value itself.  8 bits: no code stands for it, the states of its block read as NaN; the parameters of the others are right."""
    for bits in (32, 8):
        ts = make(abi, np.random.default_rng(6), [1000], bits)
        clean = snapshot(ts)
        ts[0]["g"][300] = math.nan
        abi.AdamW(ts).step(1e-3, 3, seed=1)
        abi.AdamW(clean).step(1e-3, 3, seed=1)
        a, c = ts[0], clean[0]
        others = torch.arange(1000, device="cuda") != 300
        assert a["w"][300].isnan() and torch.equal(a["w"][others], c["w"][others])
        if bits == 32:
            assert a["m"][300].isnan() and a["v"][300].isnan() and torch.equal(a["m"][others], c["m"][others])
        else:
            block = torch.arange(1000, device="cuda") // BLOCK
            for k in ("m", "v"):
                got, want = abi.adamw_decode(a[k], a[k + "_scale"]), abi.adamw_decode(c[k], c[k + "_scale"])
                assert got[block == 1].isnan().all() and torch.equal(got[block != 1], want[block != 1])


@pytest.mark.parametrize("size", [1e-30, 1e-17, 1e-10, 1.0, 1e10, 1e18])
def test_8_bit_codes_over_the_range(abi, size):
    """Gradients near both ends of 32 bits, with spreads that reach the smallest codes and beyond."""
    rng = np.random.default_rng(3)
    n = 4096
    t = dict(w=torch.zeros(n, device="cuda"), g=torch.from_numpy((size * rng.standard_normal(n) * 10.0 ** rng.uniform(-7, 0, n)).astype(f32)).cuda(),
             weight_decay=0.0, w_min=-math.inf, **abi.adamw_states(n, "cuda", 8))
    for step in range(1, 4):
        before = snapshot([t])
        abi.AdamW([t]).step(1e-3, step, seed=step)
        check_codes(before, [t], step)
        assert torch.isfinite(t["w"]).all()


# ------------------------------------------------------------------ what the 8 bits are worth
def test_rounding_of_8_bit_states_has_the_right_mean(abi):
    """One step with beta = 0 stores g and g^2: over S seeds the mean of what the codes stand for is the value, within six standard
    errors (a code step's half over sqrt(S) at most) and the dither's own step (2^-17 of a code step)."""
    rng = np.random.default_rng(12)
    n, S = 512, 4000
    g = torch.from_numpy((rng.standard_normal(n) * 10.0 ** rng.uniform(-2, 0, n)).astype(f32)).cuda()
    t = dict(w=torch.zeros(n, device="cuda"), g=g, **abi.adamw_states(n, "cuda", 8))
    opt = abi.AdamW([t])
    mean_m, mean_v = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    for seed in range(S):
        opt.step(1e-3, 1, beta1=0.0, beta2=0.0, seed=seed)
        mean_m += abi.adamw_decode(t["m"], t["m_scale"]).double() / S
        mean_v += abi.adamw_decode(t["v"], t["v_scale"]).double() / S
    for mean, x, power, scale in ((mean_m, g.double(), 2, t["m_scale"]), (mean_v, g.double() ** 2, 4, t["v_scale"])):
        s = scale.double().repeat_interleave(BLOCK)
        q = torch.floor((x.abs() / s) ** (1 / power))
        width = ((q + 2) ** power - (q - 1).clamp(min=0) ** power) * s  # a code step, and room for q being one off
        keep = q >= 1 if power == 4 else q >= 0  # a second moment below the smallest code is stored as that code
        assert ((mean - x).abs() <= width * (6 * 0.5 / math.sqrt(S) + 2.0 ** -17))[keep].all()


def test_8_bit_moving_average_does_not_stand_still(abi):
    """g^2 constant at four times the stored v: after k steps v is g^2 (1 - 0.75 beta2^k) in the mean, though one step moves it by
    less than a code.  Over 4096 values the mean of v must come within 3 %: code noise is below 20 % a value (a code step at
    q >= 100 is 4 %, and a random walk forgets after 1 / (1 - beta2) steps), so the mean of 4096 is known to 0.3 %."""
    n, k = 4096, 1500
    t = dict(w=torch.zeros(n, device="cuda"), g=torch.full((n,), 1e-3, device="cuda"), **abi.adamw_states(n, "cuda", 8))
    opt = abi.AdamW([t])
    opt.step(0.0, 1, beta2=0.75, seed=0)  # v = g^2 / 4
    for step in range(1, k + 1):
        opt.step(0.0, step, seed=step)
    want = 1e-6 * (1 - 0.75 * B2 ** k)
    got = abi.adamw_decode(t["v"], t["v_scale"]).double().mean().item()
    assert abs(got / want - 1) < 0.03


# ------------------------------------------------------------------ graphs, streams
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_and_replayed_with_device_scalars(abi, bits):
    """Norm and step captured once, replayed with other gradients, step numbers and rates: the same bits as the plain calls."""
    ts = make(abi, np.random.default_rng(5), [5000, 33, 70001], bits, w16=torch.bfloat16)
    plain = snapshot(ts)
    opt, other = abi.AdamW(ts), abi.AdamW(plain)
    scalars = torch.zeros(12, dtype=torch.int32, device="cuda")
    start = snapshot(ts)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    scalars.copy_(abi.adamw_scalars(1e-3, 1))
    with torch.cuda.stream(s):
        opt.step(norm=opt.grad_norm(), scalars=scalars)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step(norm=opt.grad_norm(), scalars=scalars)
    for t, b in zip(ts, start):  # back to where it was
        for k in ("w", "m", "v", "w16", "m_scale", "v_scale"):
            if t.get(k) is not None:
                t[k].copy_(b[k])
    for step in range(1, 5):
        for t, p in zip(ts, plain):
            p["g"].normal_(std=0.01 * step)
            t["g"].copy_(p["g"])
        scalars.copy_(abi.adamw_scalars(1e-3 / step, step, max_norm=1.0))
        g.replay()
        other.step(1e-3 / step, step, norm=other.grad_norm(), max_norm=1.0)
        for t, p in zip(ts, plain):
            assert all(torch.equal(t[k], p[k]) for k in ("w", "m", "v", "w16"))


def test_runs_on_the_current_stream(abi):
    """The step waits for what its stream holds: the gradients arrive late on a side stream."""
    ts = make(abi, np.random.default_rng(5), [100000])
    late = torch.randn(100000, device="cuda")
    opt, s = abi.AdamW(ts), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            big = big @ big * 1e-2
        ts[0]["g"].copy_(late)
        before = snapshot(ts)
        opt.step(1e-3, 3, norm=opt.grad_norm())
    s.synchronize()
    assert torch.equal(before[0]["g"], late)
    check_step(before, ts)


# ------------------------------------------------------------------ decode, refusals
@pytest.mark.parametrize("n", [1, 255, 256, 257, 100003])
def test_decode(abi, n):
    rng = np.random.default_rng(n)
    scale = (2.0 ** rng.integers(-100, 60, -(-n // BLOCK))).astype(f32)
    for second, dtype in ((False, np.int8), (True, np.uint8)):
        codes = rng.integers(0 if second else -127, 256 if second else 128, n).astype(dtype)
        got = abi.adamw_decode(torch.from_numpy(codes).cuda(), torch.from_numpy(scale).cuda())
        assert np.array_equal(got.cpu().numpy(), np_decode(codes, scale, second))


def test_refusals_of_the_binding(abi):
    ok = lambda n=8, bits=32: dict(w=torch.zeros(n, device="cuda"), g=torch.zeros(n, device="cuda"), **abi.adamw_states(n, "cuda", bits))  # noqa: E731
    t = ok()
    for bad in [dict(t, g=torch.zeros(7, device="cuda")), dict(t, m=torch.zeros(8, dtype=torch.int8, device="cuda")), dict(t, w=t["w"].double()),
                dict(t, g=t["g"].cpu()), dict(t, w16=torch.zeros(8, device="cuda")), dict(t, what=1), dict(t, m=t["w"]), dict(t, w=torch.zeros(16, device="cuda")[::2]),
                dict(t, m_scale=torch.zeros(1, device="cuda")), dict(t, g=t["w"]), {k: v for k, v in t.items() if k != "v"}]:
        with pytest.raises(abi.ScnError):
            abi.AdamW([bad])
    with pytest.raises(abi.ScnError, match="overlap"):
        abi.AdamW([t, t])
    opt = abi.AdamW([ok(), ok(300, 8)])
    for kw in [dict(), dict(lr=1e-3), dict(lr=1e-3, step=0), dict(lr=1e-3, step=1, max_norm=1.0), dict(lr=math.nan, step=1), dict(lr=1e-3, step=1, beta1=1.0),
               dict(lr=1e-3, step=1, eps=0.0), dict(lr=1e-3, step=1, norm=torch.zeros(2, device="cuda")),
               dict(scalars=abi.adamw_scalars(1e-3, 1)), dict(lr=1e-3, step=1, scalars=abi.adamw_scalars(1e-3, 1).cuda())]:
        with pytest.raises(abi.ScnError):
            opt.step(**kw)
    with pytest.raises(abi.ScnError):
        abi.adamw_decode(torch.zeros(300, dtype=torch.int8, device="cuda"), torch.zeros(1, device="cuda"))
    with pytest.raises(abi.ScnError):
        abi.adamw_decode(torch.zeros(300, dtype=torch.int16, device="cuda"), torch.zeros(2, device="cuda"))


def test_more_than_32_bits_of_values(abi):
    """A tensor of more than 2^32 values with 8-bit states: offsets and the dither's places past 32 bits, at both ends."""
    n = (1 << 32) + 1000
    t = dict(w=torch.zeros(n, device="cuda"), g=torch.zeros(n, device="cuda", dtype=torch.bfloat16), weight_decay=0.0, w_min=-math.inf, **abi.adamw_states(n, "cuda", 8))
    ends = [slice(0, 3 * BLOCK), slice((1 << 32) - 2 * BLOCK, (1 << 32) + 2 * BLOCK), slice(n - 1000 + 2 * BLOCK, n)]
    for e in ends:
        t["g"][e] = torch.randn(e.stop - e.start, device="cuda").to(torch.bfloat16)
    opt = abi.AdamW([t])
    norm = opt.grad_norm().item()
    want = math.sqrt(sum((t["g"][e].double() ** 2).sum().item() for e in ends))
    assert abs(norm - want) <= 1.001 * U * want
    opt.step(1e-3, 1, seed=7)
    for e in ends:
        at = np.arange(e.start, e.stop, dtype=np.uint64)
        m, v = np_moments(np.zeros(len(at), f32), np.zeros(len(at), f32), t["g"][e].float().cpu().numpy())
        um, uv = np_mix(at, 7)
        for k, x, u in (("m", m, um), ("v", v, uv)):
            codes, scale = np_encode(x, u, k == "v")
            assert np.array_equal(t[k][e].cpu().numpy(), codes) and np.array_equal(t[k + "_scale"][e.start // BLOCK:-(-e.stop // BLOCK)].cpu().numpy(), scale)
    assert t["w"][4096].item() == 0 and t["m"][1 << 31].item() == 0


# ------------------------------------------------------------------ many codes: the restatement in torch, on the GPU
def torch_scale(most, top, bits):
    e = (torch.frexp(most)[1].long() - 1 - bits).clamp(min=-126)
    power = lambda e: ((e + 127) << 23).int().view(torch.float32)  # noqa: E731
    e = torch.where(most > top * power(e), e + 1, e)
    return torch.where(most > 0, power(e), 0.0), power(-e)


def torch_encode(x, u, second):
    x, u = x.view(-1, BLOCK), u.view(-1, BLOCK)
    power = (lambda q: (q * q) * (q * q)) if second else (lambda q: q * q)
    scale, inverse = torch_scale(x.abs().amax(1), 4228250624.0 if second else 16129.0, 31 if second else 13)
    y = x.abs() * inverse[:, None]
    q = torch.floor(y.double() ** (0.25 if second else 0.5)).float()
    q = torch.where(power(q) > y, q - 1, q)
    q = torch.where(power(q + 1) <= y, q + 1, q)
    q = torch.where(y - power(q) > u * (power(q + 1) - power(q)), q + 1, q)
    if second:
        q = torch.where((x > 0) & (q < 1), 1.0, q)
    return (q * torch.sign(x)).to(torch.uint8 if second else torch.int8).view(-1), scale


def test_codes_of_a_large_tensor(abi):
    """2^26 values over three steps, codes and scales exactly those of single roundings.  (A moment computed with one fused
    multiply-add differs in the last bit of some values, which turns about one code in ten million over: too rarely for
    the smaller tests to see.)"""
    n = 1 << 26
    gen = torch.Generator(device="cuda").manual_seed(3)
    t = dict(w=torch.zeros(n, device="cuda"), g=torch.empty(n, device="cuda", dtype=torch.bfloat16), **abi.adamw_states(n, "cuda", 8))
    opt = abi.AdamW([t])
    at = torch.arange(n, device="cuda")
    m = v = torch.zeros(n, device="cuda")
    one = lambda x: float(f32(x))  # noqa: E731
    for step in (1, 2, 3):
        t["g"].copy_(torch.randn(n, device="cuda", generator=gen) * torch.exp(2 * torch.randn(n, device="cuda", generator=gen)) * 1e-3)
        opt.step(1e-3, step)
        g = t["g"].float()
        m, v = m * one(B1) + g * one(1 - B1), v * one(B2) + (g * g) * one(1 - B2)
        full = 0xFFFFFFFF
        h = (at * 0x6A09E667 + ((step * 0xBB67AE85) & full)) & full
        h = ((h ^ (h >> 16)) * 0xBB67AE85) & full
        h = ((h ^ (h >> 15)) * 0x3C6EF373) & full
        h = h ^ (h >> 16)
        for k, x, bits in (("m", m, h & 0xFFFF), ("v", v, h >> 16)):
            codes, scale = torch_encode(x, (bits.float() + 0.5) * 2.0 ** -16, k == "v")
            assert torch.equal(t[k + "_scale"], scale) and int((t[k] != codes).sum()) == 0, k
        m, v = abi.adamw_decode(t["m"], t["m_scale"]), abi.adamw_decode(t["v"], t["v_scale"])


def test_numbers_after_a_refused_step(abi):
    """A step with numbers that are none raises and leaves nothing behind: the next one takes its own."""
    def run(spoil):
        w, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
        opt = abi.AdamW([dict(w=w, g=g, **abi.adamw_states(300, "cuda", 32))])
        opt.step(0.1, 1)
        if spoil:
            with pytest.raises(TypeError):
                opt.step(0.7, "two", seed=0)
        opt.step(0.1, 1)
        return w
    assert torch.equal(run(False), run(True))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("size,gs,max_norm", [
    (1e20, 5e18, 0.0), (1e30, 1e10, 1e-3), (1e30, -1e10, 1e-3), (1e8, 1e30, 1e-7), (1e-30, 1e38, 1.0), (1e15, 1e-30, 1.0), (1e37, 1.0, 1e-2)])
def test_finite_norms_that_grad_scale_takes_out_of_32_bits(abi, bits, size, gs, max_norm):
    """norm |grad_scale|, or max_norm over it, leaves 32 bits or all but does: the step is taken, with the gradients' norm scaled to
    max_norm.  Only a norm that is itself not finite stops it."""
    rng = np.random.default_rng(17)
    n = 3000
    x = rng.standard_normal(n)
    g = torch.from_numpy((x / np.sqrt((x ** 2).sum()) * size).astype(f32)).cuda()
    t = dict(w=torch.zeros(n, device="cuda"), g=g, **abi.adamw_states(n, "cuda", bits))
    opt = abi.AdamW([t])
    norm = opt.grad_norm()
    assert math.isfinite(norm.item()) and abs(norm.item() / size - 1) < 1e-3
    gs, max_norm = float(f32(gs)), float(f32(max_norm))
    clipped = max_norm > 0 and norm.item() * abs(gs) > max_norm
    scaled = g.double() * (math.copysign(max_norm / norm.item(), gs) if clipped else gs)
    # the scale: three roundings (a product, a quotient, a product), or 2^-150 where it lies below the normal range; then the gradient's
    # product (beta1 = 1/2 is exact)
    err = 4.1 * U * scaled.abs() + g.double().abs() * 2.0 ** -150 + 2.0 ** -149
    opt.step(1e-3, 1, beta1=0.5, beta2=0.0, grad_scale=gs, norm=norm, max_norm=max_norm)
    m = 0.5 * scaled
    if bits == 32:
        assert ((t["m"].double() - m).abs() <= err).all()
    elif max_norm == 0:  # squares past 32 bits: no code stands for them
        assert t["m_scale"].isnan().all() and t["v_scale"].isnan().all()
    else:  # a code that stands for at least a quarter of its block's largest value is at least 45: within a step of (2 q + 1) / q^2 < 0.05
        got, large = abi.adamw_decode(t["m"], t["m_scale"]).double(), m.abs() > 0.25 * m.abs().max()
        assert ((got - m).abs() <= 0.05 * m.abs())[large].all()
    if max_norm > 0:  # beta2 = 0: v = g'^2, and the bias corrections leave g' / (|g'| + eps); roundings behind g' as in check_step, below 20 U
        eps = float(f32(EPS))
        hat = scaled / (scaled.abs() + eps)
        assert ((t["w"].double() + float(f32(1e-3)) * hat).abs() <= 1e-3 * (24 * U * hat.abs() + err / (scaled.abs() + eps)) + 1e-44).all()


def test_norm_depends_on_the_gradients_alone(abi):
    """The norm reads d_g, g_type and n: whatever else an entry holds, the squares are added in the same order.  The values make another
    order show: 1 + 2 (2^-12)^2 + (2^-24)^2 is (1 + 2^-24)^2, whose root lies halfway between two numbers of 32 bits; seven squares of
    0.99 2^-53 vanish one by one beside the 1, but tip the balance once two of them are added up first."""
    n = 2048
    g = torch.zeros(n, device="cuda")
    g[0], g[1:8], g[8:10], g[16] = 1.0, math.sqrt(0.99) * 2.0 ** -26.5, 2.0 ** -12, 2.0 ** -24
    L, s = abi.lib(), torch.cuda.current_stream().cuda_stream
    norm, ws = torch.empty(1, device="cuda"), torch.empty(L.scn_grad_norm_workspace_bytes(), dtype=torch.uint8, device="cuda")
    results = set()
    for other in (dict(), dict(d_w=4), dict(d_m=1, d_v=3), dict(d_m_scale=4), dict(d_w16=2), dict(d_w=1, d_m=7, w16_type=9, weight_decay=math.nan)):
        e = abi.AdamWTensor(d_g=g.data_ptr(), n=n, g_type=abi.F32, **other)  # (none of the other pointers is read)
        abi.check(L.scn_grad_norm((abi.AdamWTensor * 1)(e), 1, norm.data_ptr(), ws.data_ptr(), ws.numel(), s))
        results.add(norm.item())
    assert len(results) == 1 and abs(results.pop() - 1) <= 2.0 ** -23


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("eps", [1.2e-38, 1e-30, 1e-20, 1e-15, 2e-12, 3e-12, 1e-8])
def test_second_moments_below_the_normal_range(abi, bits, offset, eps):
    """Gradients from 1e-23 to 1e-15: second moments from nothing over 2^-149 and 2^-126 up, beside an eps that hides their roots or is
    dwarfed by them.  The moments in single 32-bit roundings, then the step from them in 64 bits."""
    rng = np.random.default_rng(23)
    n, lr, b1, b2 = 5000, 1e-3, 0.5, 0.5
    t = make(abi, rng, [n], bits, offset=offset, decay=0.0)[0]
    g = (rng.choice([-1, 1], n) * 10.0 ** rng.uniform(-23, -15, n)).astype(f32)
    t["g"].copy_(torch.from_numpy(g))
    for k in ("w", "m", "v", "m_scale", "v_scale"):
        if t.get(k) is not None:
            t[k].zero_()
    abi.AdamW([t]).step(lr, 1, beta1=b1, beta2=b2, eps=eps)
    m, v = np_moments(np.zeros(n, f32), np.zeros(n, f32), g, 1.0, b1, b2)
    assert (v == 0).any() and ((v > 0) & (v < 2.0 ** -126)).any() and (v > 2.0 ** -126).any()
    if bits == 32:
        assert np.array_equal(t["m"].cpu().numpy(), m) and np.array_equal(t["v"].cpu().numpy(), v)
    m, v, eps = m.astype(np.float64), v.astype(np.float64), float(f32(eps))
    want = -float(f32(lr)) * 2.0 * m / (np.sqrt(v) * math.sqrt(2.0) + eps)
    # behind the moments below 20 U (see check_step), one more where eps hides a root that is left out, lr's product and the result
    assert (np.abs(t["w"].cpu().numpy().astype(np.float64) - want) <= 23 * U * np.abs(want) + 1e-44).all()


def test_every_step_takes_its_own_numbers(abi):
    """Nothing is kept of the step before, also where the numbers are the same."""
    w, g = torch.zeros(300, device="cuda"), torch.ones(300, device="cuda")
    opt = abi.AdamW([dict(w=w, g=g, **abi.adamw_states(300, "cuda", 32))])
    opt.step(0.125, 1, eps=1e-12)
    opt.h.lr = 7.0  # (what the C call last read)
    opt.step(0.125, 1, eps=1e-12)
    # step 1 twice: m = 0.1, then 0.19, v = 0.001, then 0.001999: lr times 1, then 1.9 / sqrt(1.999)
    assert (w.double() + 0.125 * (1 + 1.9 / math.sqrt(1.999))).abs().max() < 1e-6


@pytest.mark.parametrize("bits", [8, 32])
def test_a_large_list_of_several_tensors(abi, bits):
    """Above some 30 M values a CTA takes several turns of a chunk (of the norm's too).  Tensors that end at a chunk's end, within one, one
    value on either side, at an address that allows single values only, with and without a copy: every code, scale, moment and parameter, and the norm."""
    chunk = 8 * 8 * BLOCK  # of 8-bit states
    sizes = [20_000_003, chunk, 3 * chunk + 1, 5 * chunk - 1, 777, 6_000_001, 1, 8 * chunk + 12 * BLOCK, 5_000_000, 4 * chunk]
    odd, types = {1, 5, 7}, [torch.bfloat16, torch.float32, torch.float16]
    assert sum(sizes) > 100 * 148 * 8 * BLOCK
    gen = torch.Generator(device="cuda").manual_seed(8)
    dither, ts, block = [], [], 0

    def put(n, dtype, k):
        return torch.zeros(n + 1, device="cuda", dtype=dtype)[1:] if k in odd else torch.zeros(n, device="cuda", dtype=dtype)

    for k, n in enumerate(sizes):
        t = dict(w=put(n, torch.float32, k), g=put(n, types[k % 3], k), weight_decay=0.0, w_min=-math.inf)
        states = abi.adamw_states(n, "cuda", bits)
        t.update(m=put(n, states["m"].dtype, k), v=put(n, states["v"].dtype, k), **{x: states[x] for x in states if x.endswith("scale")})
        if k % 2:
            t["w16"] = put(n, torch.bfloat16, k)
        t["w"].normal_(generator=gen)
        ts.append(t)
        dither.append(block * BLOCK)
        block += -(-n // BLOCK)
    opt, one, full = abi.AdamW(ts), lambda x: float(f32(x)), 0xFFFFFFFF
    moments = [[torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")] for n in sizes]
    for step in (1, 2):
        for t in ts:
            n = len(t["g"])
            t["g"].copy_(torch.randn(n, device="cuda", generator=gen) * torch.exp(2 * torch.randn(n, device="cuda", generator=gen)) * 1e-3)
        before = snapshot(ts)
        want = math.sqrt(sum((t["g"].double() ** 2).sum().item() for t in ts))
        norm = opt.grad_norm()
        assert abs(norm.item() - want) <= 1.001 * U * want
        opt.step(1e-3, step)
        check_step(before, ts, step=step)
        for t, mv, start in zip(ts, moments, dither):
            g, n = t["g"].float(), len(t["g"])
            mv[0], mv[1] = mv[0] * one(B1) + g * one(1 - B1), mv[1] * one(B2) + (g * g) * one(1 - B2)
            if bits == 32:
                assert torch.equal(t["m"], mv[0]) and torch.equal(t["v"], mv[1])
                continue
            h = ((start + torch.arange(n, device="cuda")) * 0x6A09E667 + ((step * 0xBB67AE85) & full)) & full
            h = ((h ^ (h >> 16)) * 0xBB67AE85) & full
            h = ((h ^ (h >> 15)) * 0x3C6EF373) & full
            h = h ^ (h >> 16)
            pad = torch.nn.functional.pad
            for i, (k, bits_of) in enumerate((("m", h & 0xFFFF), ("v", h >> 16))):
                fill = (0, -n % BLOCK)
                codes, scale = torch_encode(pad(mv[i], fill), pad((bits_of.float() + 0.5) * 2.0 ** -16, fill, value=0.5), k == "v")
                assert torch.equal(t[k + "_scale"], scale) and torch.equal(t[k], codes[:n])
                mv[i] = abi.adamw_decode(t[k], t[k + "_scale"])

"""GPU tests of the embedding lookup and its gradient by sorted tokens against plain 64-bit arithmetic.

Tolerances: a rounding to 32 bits is off by at most 2^-24 of the value (U), to bfloat16 by 2^-8, to half by 2^-11 (or half its
smallest step, 2^-25)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def tokens_like(rng, n, vocab, kind):
    if kind == "uniform":
        t = rng.integers(0, vocab, n)
    elif kind == "frequent":  # the k-th in frequency about 1 / k
        t = np.minimum(np.exp(rng.random(n) * math.log(vocab + 1)) - 1, vocab - 1).astype(np.int64)
        t = (t * 7919) % vocab
    elif kind == "one":
        t = np.full(n, vocab // 2)
    elif kind == "half":  # one token on half of the rows, between all the others
        t = np.where(rng.random(n) < 0.5, vocab // 3, rng.integers(0, vocab, n))
    elif kind == "none":
        return torch.full((n,), -1, dtype=torch.int32, device="cuda")
    elif kind == "descending":
        t = (vocab - 1 - np.arange(n) % vocab)
    t = t.astype(np.int32)
    t[rng.random(n) < 0.05] = -1
    return torch.from_numpy(t).cuda()


# widths and strides that allow whole 16-byte accesses, some of them, none
LAYOUTS = [(64, 0, 0), (96, 32, 32), (1, 0, 0), (3, 0, 0), (33, 5, 2), (100, 4, 4), (128, 1, 1), (256, 0, 0), (515, 0, 0), (1024, 8, 0), (2, 0, 0), (40, 0, 0), (4100, 0, 0)]


def strided(n, C, extra, first, dtype):
    """A [n, C] view whose rows lie C + extra values apart, starting at column `first`, and the whole buffer."""
    whole = torch.full((n, C + extra), 7.0, device="cuda", dtype=dtype)
    return whole[:, first:first + C] if extra else whole, whole


def check_lookup(table, tok, scale, out):
    V, s = table.shape[0], float(np.float32(scale))
    t = tok.long()
    want = table.double()[t.clamp(0, V - 1)] * s
    want[(t < 0) | (t >= V)] = 0
    # one product in 32 bits, one rounding to the output's type
    bound = want.abs() * (U + HALF[out.dtype] * (1 + U)) + (2.0 ** -25 if out.dtype == torch.float16 else 1e-44)
    assert ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("table_type", TYPES)
@pytest.mark.parametrize("out_type", TYPES)
@pytest.mark.parametrize("C,extra,first", LAYOUTS)
def test_lookup(abi, table_type, out_type, C, extra, first):
    rng = np.random.default_rng(C + extra)
    V, n = 301, 1237
    table = torch.from_numpy(rng.standard_normal((V, C))).cuda().to(table_type)
    tok = tokens_like(rng, n, V, "uniform")
    out, whole = strided(n, C, extra, first, out_type)
    got = abi.embedding_forward(table, tok, 1.7, out=out)
    assert got is out
    check_lookup(table, tok, 1.7, out)
    keep = torch.ones(C + extra, dtype=torch.bool, device="cuda")
    keep[first:first + C] = False
    assert (whole[:, keep] == 7.0).all()  # nothing between the rows is written


@pytest.mark.parametrize("n", [0, 1, 2, 31, 33, 255, 257, 4097])
@pytest.mark.parametrize("V", [1, 2, 65537])
def test_lookup_sizes(abi, n, V):
    rng = np.random.default_rng(n)
    table = torch.from_numpy(rng.standard_normal((V, 20)).astype(np.float32)).cuda()
    tok = tokens_like(rng, n, V, "uniform")
    out = abi.embedding_forward(table, tok, 0.5)
    assert out.shape == (n, 20) and out.dtype == torch.float32
    check_lookup(table, tok, 0.5, out)


def test_lookup_unaligned_table(abi):
    """A table that starts at no 16-byte boundary."""
    whole = torch.randn(1 + 50 * 64, device="cuda")
    table = whole[1:].view(50, 64)
    tok = torch.arange(50, device="cuda", dtype=torch.int32).flip(0).repeat(9)
    check_lookup(table, tok, 3.0, abi.embedding_forward(table, tok, 3.0))


def test_tokens_outside_the_table(abi):
    """Negative: a zero row, no error.  Too large: a zero row, no gradient, and the error bit (or-ed in, never cleared)."""
    table = torch.randn(10, 8, device="cuda")
    errors = torch.zeros(1, dtype=torch.int32, device="cuda")
    tok = torch.tensor([0, -1, 9, -2147483648], dtype=torch.int32, device="cuda")
    check_lookup(table, tok, 1.0, abi.embedding_forward(table, tok, errors=errors))
    dt = abi.embedding_backward(torch.ones(4, 8, device="cuda"), tok, torch.empty(10, 8, device="cuda"), errors=errors)
    assert errors.item() == 0 and dt.sum().item() == 16
    tok = torch.tensor([0, 10, 9, 2147483647], dtype=torch.int32, device="cuda")
    check_lookup(table, tok, 1.0, abi.embedding_forward(table, tok, errors=errors))
    assert errors.item() == abi.DEV_ERR_KEY
    errors.fill_(8)
    dt = abi.embedding_backward(torch.ones(4, 8, device="cuda"), tok, torch.empty(10, 8, device="cuda"), errors=errors)
    assert errors.item() == 8 | abi.DEV_ERR_KEY and dt.sum().item() == 16
    assert abi.embedding_backward(torch.ones(4, 8, device="cuda"), tok, torch.empty(10, 8, device="cuda")).sum().item() == 16  # no place for the bit


def check_gradient(dout, tok, V, scale, got, before=None):
    t, s = tok.long(), float(np.float32(scale))
    ok = (t >= 0) & (t < V)
    C = dout.shape[1]
    want = torch.zeros(V, C, dtype=torch.float64, device="cuda").index_add_(0, t[ok], dout.double()[ok] * s)
    size = torch.zeros(V, C, dtype=torch.float64, device="cuda").index_add_(0, t[ok], (dout.double()[ok] * s).abs())
    count = torch.zeros(V, dtype=torch.float64, device="cuda").index_add_(0, t[ok], torch.ones_like(t[ok], dtype=torch.float64))
    # k terms: k - 1 additions in any order, each off by U of a partial sum that the sum of absolute values bounds, then the scale's
    # product; with accumulation one more addition
    bound = size * U * (count[:, None] + 1) * 1.01
    if before is not None:
        want = want + before.double()
        bound = bound + want.abs() * U
    assert ((got.double() - want).abs() <= bound + 1e-44).all()
    return count


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("C,extra,first", LAYOUTS)
def test_gradient(abi, dtype, accumulate, C, extra, first):
    rng = np.random.default_rng(C + extra)
    V, n = 301, 3001
    tok = tokens_like(rng, n, V, "frequent")
    dout, whole = strided(n, C, extra, first, dtype)
    dout.copy_(torch.from_numpy(rng.standard_normal((n, C))))
    before = torch.from_numpy(rng.standard_normal((V, C)).astype(np.float32)).cuda()
    dt = before.clone() if accumulate else torch.full((V, C), math.nan, device="cuda")
    assert abi.embedding_backward(dout, tok, dt, 1.7, accumulate=accumulate) is dt
    count = check_gradient(dout, tok, V, 1.7, dt, before if accumulate else None)
    assert torch.equal(dt[count == 0], before[count == 0] if accumulate else torch.zeros_like(dt[count == 0]))


@pytest.mark.parametrize("kind", ["uniform", "frequent", "one", "half", "none", "descending"])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 203, 1000, 4095, 4096, 4097, 50021, 300007])
@pytest.mark.parametrize("V", [1, 2, 100, 1023, 1024, 70001])
def test_gradient_tokens(abi, kind, n, V):
    """Sizes around the sort's tiles and digits; tokens spread, repeated, all the same, or none; rows without tokens."""
    rng = np.random.default_rng(n + V)
    tok = tokens_like(rng, n, V, kind)
    C = 12
    dout = torch.from_numpy(rng.standard_normal((n, C)).astype(np.float32)).cuda()
    dt = abi.embedding_backward(dout, tok, torch.full((V, C), math.nan, device="cuda"), 0.25)
    check_gradient(dout, tok, V, 0.25, dt)
    again = abi.embedding_backward(dout, tok, torch.full((V, C), math.nan, device="cuda"), 0.25)
    assert torch.equal(dt, again)  # the order of the additions depends on the tokens alone
    added = abi.embedding_backward(dout, tok, dt.clone(), 0.25, accumulate=True)
    check_gradient(dout, tok, V, 0.25, added, dt)


def test_gradient_large_vocabularies(abi):
    """Tables of more rows than tokens, up to the sort's third digit; the rows between are zero or left as they are."""
    rng = np.random.default_rng(5)
    for V, n, C in [(3000017, 999, 4), (1 << 21, 70000, 5), ((1 << 20) - 1, 5000, 3)]:
        tok = tokens_like(rng, n, V, "uniform")
        tok[0], tok[-1] = V - 1, 0
        dout = torch.from_numpy(rng.standard_normal((n, C)).astype(np.float32)).cuda()
        dt = abi.embedding_backward(dout, tok, torch.full((V, C), math.nan, device="cuda"))
        check_gradient(dout, tok, V, 1.0, dt)
        before = torch.randn(V, C, device="cuda")
        check_gradient(dout, tok, V, 1.0, abi.embedding_backward(dout, tok, before.clone(), accumulate=True), before)


def test_gradient_empty(abi):
    tok = torch.empty(0, dtype=torch.int32, device="cuda")
    dt = torch.ones(5, 4, device="cuda")
    abi.embedding_backward(torch.empty(0, 4, device="cuda"), tok, dt, accumulate=True)
    assert (dt == 1).all()
    abi.embedding_backward(torch.empty(0, 4, device="cuda"), tok, dt)
    assert (dt == 0).all()
    assert abi.embedding_forward(dt, tok).shape == (0, 4)


def test_infinities_and_nan_stay_in_their_rows(abi):
    table = torch.randn(6, 8, device="cuda")
    table[2, 3], table[4, 0] = math.inf, math.nan
    tok = torch.tensor([2, 1, 4, -1, 5], dtype=torch.int32, device="cuda")
    out = abi.embedding_forward(table, tok, -2.0)
    assert out[0, 3] == -math.inf and out[2, 0].isnan() and torch.isfinite(out).sum() == 38
    dout = torch.ones(5, 8, device="cuda")
    dout[3] = math.nan  # the row of a negative token: contributes nothing
    dout[1, 1] = math.inf
    dt = abi.embedding_backward(dout, tok, torch.empty(6, 8, device="cuda"))
    assert dt[1, 1] == math.inf and torch.isfinite(dt).sum() == 47 and dt[0].sum() == 0


def test_offsets_past_32_bits(abi):
    """More than 2^32 values in the output's rows and in the table."""
    V, C = 2100007, 2048  # 4.3e9 values: 8.6 GB in 16 bits
    table = torch.zeros(V, C, device="cuda", dtype=torch.bfloat16)
    rows = torch.tensor([0, 1, V // 2, V - 2, V - 1], device="cuda")
    table[rows] = torch.randn(5, C, device="cuda").to(torch.bfloat16)
    tok = torch.tensor([V - 1, V // 2, 0, V - 2, 1], dtype=torch.int32, device="cuda")
    check_lookup(table[rows], torch.tensor([4, 2, 0, 3, 1], dtype=torch.int32, device="cuda"), 2.0, abi.embedding_forward(table, tok, 2.0))
    n = V
    small = torch.randn(3, C, device="cuda")
    tok = (torch.arange(n, device="cuda") % 3).int()
    out = abi.embedding_forward(small, tok, out=table)  # the same memory as an output of n rows
    assert out is table
    at = torch.tensor([0, 1, 2, n // 2, n - 3, n - 2, n - 1], device="cuda")
    check_lookup(small, tok[at], 1.0, out[at])
    del out
    tok.fill_(-1)
    tok[n - 5:] = 1
    table[n - 5:] = torch.randn(5, C, device="cuda").to(torch.bfloat16)
    dt = abi.embedding_backward(table, tok, torch.empty(3, C, device="cuda"))
    check_gradient(table[n - 5:], tok[n - 5:], 3, 1.0, dt)


def test_captured_and_replayed(abi):
    """Both calls in one CUDA graph, replayed on other tokens and values in the same memory."""
    V, C, n = 500, 48, 20011
    rng = np.random.default_rng(9)
    table = torch.randn(V, C, device="cuda")
    tok, dout = tokens_like(rng, n, V, "half"), torch.randn(n, C, device="cuda")
    out, dt = torch.empty(n, C, device="cuda"), torch.empty(V, C, device="cuda")
    ws = abi.embedding_backward_workspace(n, V, C, tok.device)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        abi.embedding_forward(table, tok, 2.0, out=out)
        abi.embedding_backward(dout, tok, dt, 2.0, workspace=ws)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        abi.embedding_forward(table, tok, 2.0, out=out)
        abi.embedding_backward(dout, tok, dt, 2.0, workspace=ws)
    for kind in ("uniform", "one", "frequent"):
        tok.copy_(tokens_like(rng, n, V, kind))
        dout.normal_()
        ws.fill_(255)  # nothing is kept in the workspace between calls
        g.replay()
        torch.cuda.synchronize()
        check_lookup(table, tok, 2.0, out)
        check_gradient(dout, tok, V, 2.0, dt)


def test_two_streams_with_a_workspace_each(abi):
    rng = np.random.default_rng(11)
    V, C, n = 3000, 32, 60000
    toks = [tokens_like(rng, n, V, k) for k in ("uniform", "half")]
    douts = [torch.randn(n, C, device="cuda") for _ in range(2)]
    dts = [torch.empty(V, C, device="cuda") for _ in range(2)]
    spaces = [abi.embedding_backward_workspace(n, V, C, toks[0].device) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                abi.embedding_backward(douts[k], toks[k], dts[k], workspace=spaces[k])
    torch.cuda.synchronize()
    for k in range(2):
        check_gradient(douts[k], toks[k], V, 1.0, dts[k])


def test_gradient_against_differences(abi):
    """The gradient of f(table) = sum(out * r): f is linear, so differences of any size give it up to the roundings of f."""
    rng = np.random.default_rng(13)
    V, C, n = 7, 5, 40
    table = torch.from_numpy(rng.integers(-8, 9, (V, C)).astype(np.float32)).cuda()
    r = torch.from_numpy(rng.integers(-8, 9, (n, C)).astype(np.float32)).cuda()
    tok = tokens_like(rng, n, V, "uniform")
    f = lambda t: (abi.embedding_forward(t, tok, 0.5).double() * r.double()).sum().item()  # whole and half numbers: exact  # noqa: E731
    dt = abi.embedding_backward(r, tok, torch.empty(V, C, device="cuda"), 0.5)
    for v in range(V):
        for c in range(C):
            other = table.clone()
            other[v, c] += 4
            assert (f(other) - f(table)) / 4 == dt[v, c].item()


def test_refusals_of_the_binding(abi):
    table, tok = torch.zeros(5, 4, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    dout = torch.zeros(3, 4, device="cuda")
    for bad in [lambda: abi.embedding_forward(table.double(), tok), lambda: abi.embedding_forward(table.t(), tok), lambda: abi.embedding_forward(table, tok.long()),
                lambda: abi.embedding_forward(table, tok.cpu()), lambda: abi.embedding_forward(table, tok, out=torch.zeros(2, 4, device="cuda")),
                lambda: abi.embedding_forward(table, tok, out=torch.zeros(4, 3, device="cuda").t()),
                lambda: abi.embedding_forward(table, tok, out=torch.zeros(1, 4, device="cuda").expand(3, 4)),
                lambda: abi.embedding_forward(table, tok, errors=torch.zeros(1, device="cuda")),
                lambda: abi.embedding_backward(dout[:2], tok, table), lambda: abi.embedding_backward(dout, tok, table.half()),
                lambda: abi.embedding_backward(dout, tok, table, workspace=torch.empty(16, dtype=torch.uint8, device="cuda")),
                lambda: abi.embedding_backward(dout, tok, table, workspace=torch.empty(1 << 20, device="cuda"))]:
        with pytest.raises(abi.ScnError):
            bad()


@pytest.mark.parametrize("C", [1, 64, 100, 300])
@pytest.mark.parametrize("n,starts", [
    (4096, [0]), (4097, [0]), (6143, [0, 1]), (20000, [0]), (20000, [2048]), (20000, [2047]), (20000, [2049]), (20000, [2048, 4096]), (20000, [2047, 4095]),
    (20000, [2049, 4097]), (20000, [1984, 4032]), (20000, [2112, 4160]), (20000, [100, 6000, 14000, 19999]), (20000, [0, 64, 128, 8000]), (70000, [5, 40000]),
    (70000, [33000, 66000]), (700001, [0, 350000]), (700001, [65536, 131072]), (700001, [65535, 131073, 600000]),
])
@pytest.mark.parametrize("missing", [0, 3000])
def test_long_tokens(abi, n, starts, missing, C):
    """Tokens on thousands of rows, that begin at, before and behind the places where their parts are joined (64 to 256 rows a part, then
    32 parts).  Whole numbers of at most 4: the sums of 700 k of them stay below 2^24, so they are exact in whatever order."""
    gen = torch.Generator(device="cuda").manual_seed(n + C)
    at = torch.arange(n, device="cuda")
    tok = torch.bucketize(at, torch.tensor(starts, device="cuda"), right=True).int() * 3
    if missing:
        tok[-missing:] = -1
    order = torch.randperm(n, device="cuda", generator=gen)
    tok = tok[order].contiguous()
    dout = torch.randint(-4, 5, (n, C), device="cuda", generator=gen).float()
    V = 3 * len(starts) + 2
    want = torch.zeros(V, C, dtype=torch.float64, device="cuda").index_add_(0, tok[tok >= 0].long(), dout[tok >= 0].double())
    got = abi.embedding_backward(dout, tok, torch.full((V, C), 7.0, device="cuda"))
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("n", [4096 * 1024, 4096 * 1024 + 1, 4096 * 2048, 4096 * 2048 + 1, 20000003])
def test_many_rows_of_one_value(abi, n):
    """Sorts of thousands of tiles.  Whole numbers whose sums stay below 2^24: exact."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    tok = torch.randint(-5, 100000, (n,), device="cuda", generator=gen, dtype=torch.int32)
    dout = torch.randint(-4, 5, (n, 1), device="cuda", generator=gen).to(torch.bfloat16)
    want = torch.zeros(99990, 1, dtype=torch.float64, device="cuda")
    ok = (tok >= 0) & (tok < 99990)
    want.index_add_(0, tok[ok].long(), dout[ok].double())
    errors = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = abi.embedding_backward(dout, tok, torch.empty(99990, 1, device="cuda"), errors=errors)
    assert torch.equal(got.double(), want) and errors.item() != 0


@pytest.mark.parametrize("n", [5, 1024, 1025])
@pytest.mark.parametrize("V", [2147467264, 2147467265, 2147483647])
def test_gradient_of_the_largest_vocabularies(abi, n, V):
    """As many tokens as 32 bits count, or nearly: few rows are summed in one launch that divides the table among its CTAs, more by the sort."""
    tok = torch.randint(0, V, (n,), device="cuda", dtype=torch.int64).int()
    tok[0], tok[1], tok[2], tok[3], tok[4] = V - 1, 0, -2147483648, V - 1, -1
    dout = torch.randint(1, 5, (n, 1), device="cuda").float()
    ok = tok >= 0
    at, where = torch.unique(tok[ok], return_inverse=True)
    want = torch.zeros(len(at), device="cuda").index_add_(0, where, dout[ok, 0])  # whole numbers: exact
    dt = abi.embedding_backward(dout, tok, torch.full((V, 1), math.nan, device="cuda"))
    assert torch.equal(dt[at.long(), 0], want) and dt.count_nonzero().item() == len(at)
    abi.embedding_backward(dout, tok, dt, accumulate=True)
    assert torch.equal(dt[at.long(), 0], 2 * want) and dt.count_nonzero().item() == len(at)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("C,extra,first", LAYOUTS[:10] + [(48, 1, 1), (65, 0, 0), (130, 0, 0)])
def test_gradient_of_many_tiles(abi, dtype, accumulate, C, extra, first):
    """Some thousands of tiles, so that tokens on 32 of them and more are joined by the tiles' own warps: every width of access and number
    of columns a thread, with a token on a third of the rows, some on a few tiles, and many on a few rows.  Whole numbers whose sums stay
    below 2^24: exact in whatever order."""
    n, V = 300007, 5003
    gen = torch.Generator(device="cuda").manual_seed(C + extra)
    u = torch.rand(n, device="cuda", generator=gen)
    tok = torch.randint(0, V, (n,), device="cuda", generator=gen, dtype=torch.int32)
    tok[u < 0.6] = (torch.randint(0, 9, (n,), device="cuda", generator=gen, dtype=torch.int32) * 500 + 7)[u < 0.6]
    tok[u < 0.33] = V // 3
    tok[u > 0.99] = -1
    dout, whole = strided(n, C, extra, first, dtype)
    dout.copy_(torch.randint(-4, 5, (n, C), device="cuda", generator=gen))
    before = torch.randint(-9, 10, (V, C), device="cuda", generator=gen).float()
    ok = tok >= 0
    want = torch.zeros(V, C, dtype=torch.float64, device="cuda").index_add_(0, tok[ok].long(), dout.double()[ok])
    if accumulate:
        want += before
    dt = before.clone() if accumulate else torch.full((V, C), math.nan, device="cuda")
    assert torch.equal(abi.embedding_backward(dout, tok, dt, accumulate=accumulate).double(), want)

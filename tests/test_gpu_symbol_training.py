"""The embedding and optimiser operators together, as a training run uses them: through the C ABI (a 16-bit table that the
lookup reads, its gradient, the gradients' norm, one step over all tensors), and inside the networks (symbol inputs,
training by AdamW)."""
import math

import numpy as np
import pytest
import torch

from netutil import relerr

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


# ------------------------------------------------------------------ the operators one after the other
@pytest.mark.parametrize("bits", [32, 8])
def test_table_and_matrix_trained_together(abi, bits):
    """out = lookup(tokens) M, loss = sum (out - target)^2 / 2 for three steps; every step is checked against 64 bits from the
    state it began with: the gradients, their norm, and the parameters after the step."""
    rng = np.random.default_rng(3)
    V, C, n, K = 500, 24, 3001, 8
    table = torch.from_numpy(rng.standard_normal((V, C)).astype(np.float32)).cuda()
    table16 = table.to(torch.bfloat16)
    M = torch.from_numpy(rng.standard_normal((C, K)).astype(np.float32) * 0.2).cuda()
    tok = torch.from_numpy(rng.integers(-1, V, n).astype(np.int32)).cuda()
    target = torch.from_numpy(rng.standard_normal((n, K)).astype(np.float32)).cuda()
    dtable, dM = torch.empty(V, C, device="cuda"), torch.empty(C, K, device="cuda")
    opt = abi.AdamW([dict(w=table.view(-1), g=dtable.view(-1), w16=table16.view(-1), weight_decay=0.01, **abi.adamw_states(V * C, "cuda", bits)),
                     dict(w=M.view(-1), g=dM.view(-1), **abi.adamw_states(C * K, "cuda", bits))])
    scale, lr, eps, max_norm = 0.5, 0.01, 1e-6, 1.0
    for step in (1, 2, 3):
        before = [table.double(), M.double()]
        moments = [(abi.adamw_decode(t["m"], t["m_scale"]).double(), abi.adamw_decode(t["v"], t["v_scale"]).double()) if bits == 8 else
                   (t["m"].double(), t["v"].double()) for t in opt.tensors]
        rows = abi.embedding_forward(table16, tok, scale)
        keep = (tok >= 0).double()[:, None]
        assert torch.equal(rows.double(), table16.double()[tok.clamp(min=0).long()] * scale * keep)  # a product with 1/2 is exact
        out = rows.double() @ M.double() - target.double()
        drows = (out @ M.double().t()).float()
        dM.copy_(rows.double().t() @ out)
        abi.embedding_backward(drows, tok, dtable, scale)
        ok = tok >= 0
        exact = torch.zeros(V, C, dtype=torch.float64, device="cuda").index_add_(0, tok[ok].long(), drows[ok].double() * scale)
        size = torch.zeros(V, C, dtype=torch.float64, device="cuda").index_add_(0, tok[ok].long(), (drows[ok].double() * scale).abs())
        assert ((dtable.double() - exact).abs() <= 40 * U * size).all()  # fewer than 38 rows a token: an addition each, and the scale
        assert torch.bincount(tok[ok].long()).max() < 38
        norm = opt.grad_norm()
        total = math.sqrt((dtable.double() ** 2).sum().item() + (dM.double() ** 2).sum().item())
        assert abs(norm.item() - total) <= 1.001 * U * total and total > max_norm
        opt.step(lr, step, eps=eps, norm=norm, max_norm=max_norm)
        for w, w0, g, (m0, v0), decay in ((table, before[0], dtable, moments[0], 0.01), (M, before[1], dM, moments[1], 0.0)):
            g = g.double().view(-1) * (max_norm / total)
            m, v = 0.9 * m0.view(-1) + 0.1 * g, 0.999 * v0.view(-1) + 0.001 * g * g
            den = (v / (1 - 0.999 ** step)).sqrt() + eps
            hat = m / (1 - 0.9 ** step) / den
            want = w0.view(-1) * (1 - lr * decay) - lr * hat
            # as in the optimiser's own tests: m within 5 U of its two terms and the clip's three roundings, the rest below 25 U of hat
            merr = 8 * U * ((0.9 * m0.view(-1)).abs() + 0.1 * g.abs()) / (1 - 0.9 ** step)
            bound = lr * (merr / den + 25 * U * hat.abs()) + 4 * U * want.abs() + 3 * U * lr
            assert ((w.double().view(-1) - want).abs() <= bound).all()
        assert torch.equal(table16, table.to(torch.bfloat16))


# ------------------------------------------------------------------ inside the networks
N_IN, N_CLASSES, V = 5, 4, 37


def build(scn, abi, act, dropout=0.0):
    net = scn.net.Net(2, N_IN, N_CLASSES, 1, 0)
    net.addLeNetLayerMP(32, 3, 1, 2, 2, act, 0.0, 1)
    net.addLeNetLayerMP(64, 2, 1, 2, 2, act, dropout, 1)
    net.addLeNetLayerMP(64, 2, 1, 1, 1, act, 0.0, 1)
    net.addSoftmaxLayer()
    for i, (W, B, pr) in scn.synth.init_weights(net.layers(), 31).items():
        net.set_weights(i, W, B, pr)
    return net


def batch(S, seed, samples=6):
    rng = np.random.default_rng(seed)
    keys, syms, off = [], [], [0]
    for _ in range(samples):
        k = np.unique(rng.integers(0, S * S, 5 * S))
        keys.append(np.concatenate([[-1], k]))
        syms.append(np.concatenate([[-1], np.minimum(rng.geometric(0.15, len(k)) - 1, V - 1)]))
        off.append(off[-1] + len(k) + 1)
    return np.concatenate(keys).astype(np.int32), np.array(off, np.int32), np.concatenate(syms).astype(np.int32), rng.integers(0, N_CLASSES, samples).astype(np.int32)


def features_of(table, syms, scale):
    f = table[np.maximum(syms, 0)] * np.float32(scale)
    f[syms < 0] = 0
    return f


@pytest.fixture()
def table():
    return np.random.default_rng(1).standard_normal((V, N_IN)).astype(np.float32)


def test_symbols_are_their_rows(scn, abi, table):
    """A forward pass of symbols is the forward pass of their scaled rows, bit for bit; plain features still work beside them."""
    net, plain = build(scn, abi, abi.VLEAKYRELU), build(scn, abi, abi.VLEAKYRELU)
    net.set_symbols(table, 1.5)
    keys, off, syms, _ = batch(net.inputSpatialSize, 2)
    f = features_of(table, syms, 1.5)
    want = plain.forward_host(keys, off, f)
    for _ in range(2):
        got = net.forward_host_symbols(keys, off, syms)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        got = net.forward_host(keys, off, f)
        assert np.array_equal(got[0], want[0])


def test_training_on_symbols(scn, abi, table):
    """A step on symbols changes the layers as the step on their rows does (the only difference: the input's gradient is computed too;
    sums by atomics may be ordered differently, so not to the bit), and the table by its gradient, which is the input's
    gradient summed by symbol."""
    net, plain = build(scn, abi, abi.VLEAKYRELU), build(scn, abi, abi.VLEAKYRELU)
    net.set_symbols(table, 1.5)
    keys, off, syms, labels = batch(net.inputSpatialSize, 3)
    lr = 0.01
    _, stats = net.train_batch_symbols(keys, off, syms, labels, lr, 0.0)
    _, pstats = plain.train_batch(keys, off, features_of(table, syms, 1.5), labels, lr, 0.0)
    assert stats == pstats
    for i, L in enumerate(net.layers()):
        if L["type"] == 2:
            for a, b in zip(net.get_weights(i)[:2], plain.get_weights(i)[:2]):
                assert relerr(a, b) < 1e-5
    d = net.dfeatures(0).reshape(-1, N_IN).astype(np.float64)
    assert len(d) == len(syms) and np.abs(d).max() > 0
    exact, size = np.zeros((V, N_IN)), np.zeros((V, N_IN))
    np.add.at(exact, syms[syms >= 0], 1.5 * d[syms >= 0])
    np.add.at(size, syms[syms >= 0], np.abs(1.5 * d[syms >= 0]))
    now, g = net.get_symbols(gradient=True)
    count = np.bincount(syms[syms >= 0], minlength=V)[:, None]
    assert (np.abs(g - exact) <= (count + 1) * U * 1.01 * size).all()
    # momentum 0: w -= lr g, three roundings
    assert (np.abs(now - (table - np.float64(np.float32(lr)) * g)) <= 3 * U * (np.abs(table) + lr * np.abs(g))).all()


def test_table_gradient_against_differences(scn, abi, table):
    """One-sided differences of the batch's negative log-likelihood.  Max pooling makes it piecewise smooth: where a window's two
    largest values lie closer together than h moves them, the quotient of one side mixes two slopes, while the other side
    keeps the slope at the point, which the gradient has to equal.  (Of the thousands of windows some do lie that close: the two
    quotients of an entry differ by up to a tenth of it at any h from 2^-8 down.)  In fp32 the log-likelihoods are known to about
    1e-6, which h = 2^-10 makes 1e-3 in a quotient.  2 % of the largest gradient (0.7) is 14e-3."""
    net = build(scn, abi, abi.TANH)
    net.set_precision(abi.PREC_FP32)
    net.set_symbols(table)
    keys, off, syms, labels = batch(net.inputSpatialSize, 4)
    nll = lambda t: (net.set_symbols(t), -np.log(net.forward_host_symbols(keys, off, syms)[0].astype(np.float64)[np.arange(len(labels)), labels]).sum())[1]  # noqa: E731
    net.train_batch_symbols(keys, off, syms, labels, 0.0, 0.0)  # rate 0: gradients, no change
    t0, g = net.get_symbols(gradient=True)
    assert np.array_equal(t0, table)
    h = 2.0 ** -10
    at = nll(table)
    for v in range(6):
        for c in range(N_IN):
            off_by = []
            for side in (h, -h):
                moved = table.copy()
                moved[v, c] += side
                off_by.append(abs((nll(moved) - at) / (float(moved[v, c]) - float(table[v, c])) - g[v, c]))
            assert min(off_by) < 0.02 * np.abs(g).max()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("act", ["VLEAKYRELU", "PRELU"])
def test_adamw_step_of_a_network(scn, abi, table, act, bits):
    """The first step from zero moments is w - lr (g / (|g| + eps) + decay w), g the mean gradient, which a plain SGD step of rate 1
    without momentum shows as a difference of weights (off by 2 U of the weight, and by the order of atomic sums)."""
    act = getattr(abi, act)
    net, sgd = build(scn, abi, act), build(scn, abi, act)
    for x in (net, sgd):
        x.set_symbols(table)
    keys, off, syms, labels = batch(net.inputSpatialSize, 5)
    lr, eps, decay, B = 0.05, 0.01, 0.1, len(labels)
    net.use_adamw(eps=eps, weight_decay=decay, state_bits=bits)
    learnt = [i for i, L in enumerate(net.layers()) if L["type"] == 2]
    before = {i: net.get_weights(i) for i in learnt}
    _, stats = net.train_batch_symbols(keys, off, syms, labels, lr, 0.9)
    _, sstats = sgd.train_batch_symbols(keys, off, syms, labels, 1.0, 0.0)
    assert stats == sstats and abi.conv_tc_take_error() == 0
    cases = [(before[i][k], net.get_weights(i)[k], sgd.get_weights(i)[k], decay if k == 0 else 0.0, 0.001 if k == 2 else -math.inf)
             for i in learnt for k in range(3) if before[i][k] is not None]
    cases.append((table, net.get_symbols(), sgd.get_symbols(), decay, -math.inf))
    for w, now, stepped, dec, least in cases:
        w, now, g = w.astype(np.float64), now.astype(np.float64), (w.astype(np.float64) - stepped.astype(np.float64)) / B
        if least > 0:
            free = stepped > least * 1.001  # (SGD holds the slopes too: where it did, the difference is not the gradient)
            w, now, g = w[free], now[free], g[free]
        want = np.maximum(w - lr * (g / (np.abs(g) + eps) + dec * w), least)
        gerr = (2 * U * np.abs(w).max() + 2e-5 * np.abs(g).max() * B) / B
        assert np.abs(now - want).max() <= lr * gerr / eps + 30 * U * lr + 2 * U * np.abs(w).max()
        assert np.abs(now - w).max() > 0.1 * lr


def test_clipping_and_return_to_sgd(scn, abi, table):
    """A clip so tight that eps rules the step makes it proportional to the clip; after use_adamw(state_bits=0) a step is SGD's."""
    keys, off, syms, labels = None, None, None, None
    moved = []
    for max_norm in (1e-6, 2e-6):
        net = build(scn, abi, abi.VLEAKYRELU)
        net.set_symbols(table)
        keys, off, syms, labels = batch(net.inputSpatialSize, 6)
        net.use_adamw(eps=1.0, weight_decay=0.0, max_norm=max_norm)
        net.train_batch_symbols(keys, off, syms, labels, 100.0)
        moved.append(net.get_symbols().astype(np.float64) - table)
    # update = lr g / (|g| + 1), |g| <= 2e-6: linear within 2e-6; a weight near 1 is rounded by U, the moves are some 1e-5
    assert np.abs(moved[0]).max() > 1e-6
    assert np.abs(moved[1] - 2 * moved[0]).max() <= 4 * U * np.abs(table).max() + 1e-5 * np.abs(moved[1]).max()
    net, plain = build(scn, abi, abi.VLEAKYRELU), build(scn, abi, abi.VLEAKYRELU)
    f = features_of(table, syms, 1.0)
    net.use_adamw()
    net.use_adamw(state_bits=0)
    net.train_batch(keys, off, f, labels, 0.01, 0.9)
    plain.train_batch(keys, off, f, labels, 0.01, 0.9)
    for i, L in enumerate(net.layers()):
        if L["type"] == 2:
            assert relerr(net.get_weights(i)[0], plain.get_weights(i)[0]) < 1e-5


@pytest.mark.parametrize("bits", [32, 8])
def test_runs_with_dropout_several_steps_and_batches(scn, abi, table, bits):
    """Batches of different sizes, dropout, and both kinds of input in turn: finite, and the table rests while plain features train."""
    net = build(scn, abi, abi.PRELU, dropout=0.5)
    net.set_symbols(table, math.sqrt(N_IN))
    net.use_adamw(state_bits=bits, max_norm=1.0)
    for step in range(6):
        keys, off, syms, labels = batch(net.inputSpatialSize, 10 + step, samples=2 + step)
        was = net.get_symbols()
        if step % 3 == 2:
            net.train_batch(keys, off, features_of(was, syms, 1.0), labels, 1e-3, 0.0)
            assert np.array_equal(net.get_symbols(), was)
        else:
            _, stats = net.train_batch_symbols(keys, off, syms, labels, 1e-3)
            assert math.isfinite(stats["nll"]) and not np.array_equal(net.get_symbols(), was)
        probs, _ = net.forward_host_symbols(keys, off, syms)
        assert np.isfinite(probs).all() and abi.conv_tc_take_error() == 0
    for i, L in enumerate(net.layers()):
        if L["type"] == 2:
            assert all(np.isfinite(x).all() for x in net.get_weights(i) if x is not None)


def test_index_learning_with_adamw(scn, abi):
    net = scn.net.Net(2, 3, 10, 1, 0)
    net.addLeNetLayerMP(32, 3, 1, 2, 2, abi.VLEAKYRELU, 0.0, 1)
    net.addLeNetLayerMP(64, 2, 1, 1, 1, abi.VLEAKYRELU, 0.0, 1)
    net.addIndexLearnerLayer()
    net.use_adamw()
    S = net.inputSpatialSize
    k = np.arange(S * S, dtype=np.int32)
    keys, off = np.concatenate([k, k]), np.array([0, len(k), 2 * len(k)], np.int32)
    f = np.random.default_rng(0).standard_normal((2 * len(k), 3)).astype(np.float32)
    top = len(net.layers()) - 1
    for _ in range(3):
        before = [net.get_weights(i)[0] for i, L in enumerate(net.layers()) if L["type"] in (2, 7)]
        net.index_learner_batch(keys, off, f, np.array([3, 7], np.int32), 0.01, 0.0)
    assert not np.array_equal(before[0], net.get_weights([i for i, L in enumerate(net.layers()) if L["type"] == 2][0])[0])
    W = net.get_weights(top)[0]
    assert np.abs(W[:, [3, 7]]).max() > 0 and not W[:, [0, 1, 2, 4, 5, 6, 8, 9]].any()


def test_weight_files_carry_the_table(scn, abi, table, tmp_path):
    net, other = build(scn, abi, abi.VLEAKYRELU), build(scn, abi, abi.VLEAKYRELU)
    net.set_symbols(table)
    keys, off, syms, labels = batch(net.inputSpatialSize, 7)
    net.use_adamw()
    net.train_batch_symbols(keys, off, syms, labels, 1e-2)
    net.save_weights(str(tmp_path / "w"), 1)
    other.set_symbols(np.zeros_like(table))
    other.load_weights(str(tmp_path / "w"), 1)
    assert np.array_equal(other.get_symbols(), net.get_symbols()) and not np.array_equal(net.get_symbols(), table)
    assert np.array_equal(other.forward_host_symbols(keys, off, syms)[0], net.forward_host_symbols(keys, off, syms)[0])


def test_refusals(scn, abi, table):
    net = build(scn, abi, abi.VLEAKYRELU)
    keys, off, syms, labels = batch(net.inputSpatialSize, 8)
    for bad in [lambda: net.forward_host_symbols(keys, off, syms), lambda: net.train_batch_symbols(keys, off, syms, labels, 0.1), lambda: net.get_symbols(),
                lambda: net.set_symbols(table[:, :3]), lambda: net.set_symbols(table[:0]), lambda: net.use_adamw(beta1=1.0), lambda: net.use_adamw(eps=0.0),
                lambda: net.use_adamw(state_bits=16), lambda: net.use_adamw(max_norm=-1.0), lambda: net.use_adamw(weight_decay=math.nan)]:
        with pytest.raises(abi.ScnError):
            bad()
    net.set_symbols(table)
    with pytest.raises(abi.ScnError):
        net.get_symbols(gradient=True)  # none yet
    wrong = syms.copy()
    wrong[5] = V
    with pytest.raises(abi.ScnError, match="row 5"):
        net.forward_host_symbols(keys, off, wrong)
    net.use_adamw()
    with pytest.raises(abi.ScnError):
        net.set_symbols(table)  # its moments belong to the table that is there
    probs, _ = net.forward_host_symbols(keys, off, syms)
    assert np.isfinite(probs).all()


def test_fewer_symbols_than_rows(scn, abi, table):
    net = build(scn, abi, abi.VLEAKYRELU)
    net.set_symbols(table)
    keys, off, syms, labels = batch(net.inputSpatialSize, 8)
    for k, y in [(keys, syms[:-1]), (keys[:-1], syms)]:
        with pytest.raises(abi.ScnError, match="rows need"):
            net.forward_host_symbols(k, off, y)
        with pytest.raises(abi.ScnError, match="rows need"):
            net.train_batch_symbols(k, off, y, labels, 0.1)


@pytest.mark.parametrize("bits", [32, 8])
def test_dropped_features_stay(scn, abi, table, bits):
    """A first step without weight decay: the weights of the features that the batch drops have gradients of zero and moments of
    zero, so they keep their bits; each of the others with a gradient far above eps moves by the learning rate."""
    net = build(scn, abi, abi.VLEAKYRELU, dropout=0.5)
    at = [i for i, L in enumerate(net.layers()) if L["type"] == 2][1]
    net.set_symbols(table)
    keys, off, syms, labels = batch(net.inputSpatialSize, 5)
    kept = np.arange(0, 64, 2)
    net.set_dropout_features(at, kept)
    net.use_adamw(weight_decay=0.0, state_bits=bits)
    W0, B0 = net.get_weights(at)[:2]
    net.train_batch_symbols(keys, off, syms, labels, 1e-3)
    W1, B1 = net.get_weights(at)[:2]
    dropped = np.setdiff1d(np.arange(64), kept)
    assert np.array_equal(W0[:, dropped], W1[:, dropped]) and np.array_equal(B0[dropped], B1[dropped])
    assert (W0[:, kept] != W1[:, kept]).mean() > 0.5


@pytest.mark.parametrize("rows", ["many", "few"])
@pytest.mark.parametrize("work", ["other kernels", "a forward pass of device arrays"])
@pytest.mark.parametrize("call", ["forward_host_symbols", "forward_host", "train_batch_symbols", "train_batch"])
def test_host_arrays_on_a_busy_stream(scn, abi, table, rows, work, call):
    """Calls from pageable arrays while the stream still holds work that was there before, so that their uploads wait in the queue:
    the results of the same call on an idle stream, bit for bit.  few: fewer rows than there are words in the layers' counts."""
    net = build(scn, abi, abi.VLEAKYRELU)
    net.set_symbols(table, 1.5)
    S = net.inputSpatialSize
    if rows == "many":
        keys, off, syms, labels = batch(S, 2)
    else:
        k = np.arange(3, S * S, S * S // 9)[:8]
        keys, off = np.concatenate([[-1], k[:4], [-1], k[4:]]).astype(np.int32), np.array([0, 5, 10], np.int32)
        syms, labels = np.array([-1, 5, 6, 7, 8, -1, 9, 10, 11, 12], np.int32), np.array([1, 2], np.int32)
        assert len(keys) < 4 * len(net.layers())
    values = syms if call.endswith("symbols") else features_of(table, syms, 1.5)

    def run():
        if call.startswith("forward"):
            return getattr(net, call)(keys, off, values)
        probs, stats = getattr(net, call)(keys, off, values, labels, 0.0, 0.0)  # rate 0: the weights stay as they are
        return probs, np.array([stats["nll"], stats["mistakes"]])

    big = batch(S, 9, samples=400)
    device = [torch.from_numpy(x).cuda() for x in (big[0], big[1], big[1][:-1], features_of(table, big[2], 1.5))]  # a sample's background row is its first
    a, out = torch.ones(8192, 8192, device="cuda", dtype=torch.bfloat16), torch.empty(8192, 8192, device="cuda", dtype=torch.bfloat16)

    def other_work(times):
        for _ in range(times):
            if work == "other kernels":
                torch.matmul(a, a, out=out)
            else:
                net.forward_device(*device, max_sites=int(np.diff(big[1]).max()) - 1)

    other_work(1)
    run()  # (memory is allocated: nothing below waits for the GPU but the call itself)
    torch.cuda.synchronize()
    want = run()
    other_work(60 if work == "other kernels" else 3)
    got = run()
    assert all(np.array_equal(x, y) for x, y in zip(got, want))
    assert abi.conv_tc_take_error() == 0


def test_batches_of_too_many_features(scn, abi):
    """2^16 + 1 rows of 2^16 features: the count of the features, 2^32 + 2^16, would be 2^16 in 32 bits."""
    wide, rows = 1 << 16, (1 << 16) + 1
    net = scn.net.Net(2, wide, N_CLASSES, 1, 0)
    net.addLeNetLayerMP(4, 1, 1, 2, 2, abi.VLEAKYRELU, 0.0, 1)
    net.addSoftmaxLayer()
    net.set_precision(abi.PREC_FP32)  # (no layer of 2^16 inputs has a tensor-core path)
    net.set_symbols(np.ones((1, wide), np.float32))
    keys, off, syms = np.arange(rows, dtype=np.int32), np.array([0, rows], np.int32), np.zeros(rows, np.int32)
    for bad in [lambda: net.forward_host_symbols(keys, off, syms), lambda: net.train_batch_symbols(keys, off, syms, [0], 0.1)]:
        with pytest.raises(abi.ScnError, match="smaller batches"):
            bad()
    probs, _ = net.forward_host_symbols(keys[:1], [0, 1], syms[:1])
    assert np.isfinite(probs).all()


@pytest.mark.parametrize("act", ["VLEAKYRELU", "PRELU"])
def test_weight_files_without_the_table(scn, abi, table, tmp_path, act):
    """Such a file, or one that a byte has been cut off, is refused by a network of symbols before it changes anything."""
    act = getattr(abi, act)
    plain, net = build(scn, abi, act), build(scn, abi, act)
    learnt = [i for i, L in enumerate(plain.layers()) if L["type"] == 2]
    for i in learnt:
        plain.set_weights(i, *[None if x is None else x + np.float32(1) for x in plain.get_weights(i)])
    plain.save_weights(str(tmp_path / "w"), 1)
    plain.set_symbols(table + np.float32(1))
    plain.save_weights(str(tmp_path / "w"), 2)
    whole = (tmp_path / "w_epoch-2.cnn").read_bytes()
    (tmp_path / "w_epoch-3.cnn").write_bytes(whole[:-1])
    net.set_symbols(table)
    before = [net.get_weights(i) for i in learnt]
    for epoch in (1, 3):
        with pytest.raises(abi.ScnError, match="ends early"):
            net.load_weights(str(tmp_path / "w"), epoch)
        assert all(x is None or np.array_equal(x, y) for a, b in zip(before, learnt) for x, y in zip(a, net.get_weights(b)))
        assert np.array_equal(net.get_symbols(), table)
    net.load_weights(str(tmp_path / "w"), 2)
    assert all(x is None or np.array_equal(x, y) for i in learnt for x, y in zip(plain.get_weights(i), net.get_weights(i)))
    assert np.array_equal(net.get_symbols(), table + np.float32(1))


def test_dropped_features_follow_their_moments_and_decay(scn, abi, table):
    """As documented: a batch that drops features gives their weights gradients of zero, so that the moments of earlier batches and the
    weight decay go on moving them.  Step 1 keeps all features: m = 0.1 g and v = 0.001 g^2, the move is the rate times the sign of g (and
    decay).  Step 2 with g = 0: m = 0.09 g, v = 0.000999 g^2, a move by (0.09 / 0.19) / sqrt(0.000999 / 0.001999) of the rate, whatever g."""
    net = build(scn, abi, abi.VLEAKYRELU, dropout=0.5)
    at = [i for i, L in enumerate(net.layers()) if L["type"] == 2][1]
    net.set_symbols(table)
    keys, off, syms, labels = batch(net.inputSpatialSize, 5)
    lr, decay = 1e-3, 0.25
    net.use_adamw(eps=1e-20, weight_decay=decay)
    W = [net.get_weights(at)[0].astype(np.float64)]
    dropped = np.arange(1, 64, 2)
    for present in (np.arange(64), np.arange(0, 64, 2)):
        net.set_dropout_features(at, present)
        net.train_batch_symbols(keys, off, syms, labels, lr)
        W.append(net.get_weights(at)[0].astype(np.float64))
    first, second = (W[1] - W[0] + lr * decay * W[0])[:, dropped] / lr, (W[2] - W[1] + lr * decay * W[1])[:, dropped] / lr
    learnt = np.abs(first) > 0.5  # (a weight without a gradient has only decayed)
    assert learnt.mean() > 0.5
    want = np.sign(first) * (0.09 / 0.19) / np.sqrt(0.000999 / 0.001999)
    # each weight is rounded to 32 bits (U of it, over the rate), the step below 30 U, the rates and betas given in 32 bits
    assert (np.abs(second - want)[learnt] <= 2 * U * np.abs(W[1][:, dropped]).max() / lr + 40 * U + 1e-5).all()
    assert np.abs(second[~learnt]).max(initial=0.0) <= 2 * U * np.abs(W[1]).max() / lr + 1e-5

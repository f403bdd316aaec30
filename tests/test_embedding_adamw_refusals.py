"""CPU checks of the embedding and AdamW entry points: what the C ABI and its Python binding refuse, before any CUDA call,
and the numbers that the host side computes."""
import ctypes
import math

import pytest
import torch

P = 0x1000  # stands for a device pointer in calls that are refused before anything is read


@pytest.fixture(scope="module")
def a(scn):
    scn.abi.lib()
    return scn.abi


def refused(a, status, code, text):
    assert status == code, status
    assert text in a.lib().scn_last_error().decode()


INVALID, WORKSPACE, UNSUPPORTED = 1, 3, 4


def test_rows_too_far_apart(a):
    refused(a, a.lib().scn_embedding_forward(P, 0, 5, 4, P, 7, 1.0, P, 0, 1 << 30, None, None), UNSUPPORTED, "4 GiB")
    refused(a, a.lib().scn_embedding_backward(P, 7, P, 1, 1 << 31, 5, 4, 1.0, 0, P, None, P, 1 << 40, None), UNSUPPORTED, "4 GiB")


@pytest.mark.parametrize("n", [7, 5000])
@pytest.mark.parametrize("C", [4194241, 1 << 23, 1 << 28])
def test_gradient_rows_too_wide(a, n, C):
    """The gradient's kernels take 64 columns and more a slab, at most 65535 slabs."""
    assert a.lib().scn_embedding_backward_workspace_bytes(n, 5, C) == 0
    refused(a, a.lib().scn_embedding_backward(P, n, P, 0, C, 5, C, 1.0, 0, P, None, P, 1 << 40, None), UNSUPPORTED, "4194240")
    assert a.lib().scn_embedding_backward_workspace_bytes(n, 5, 4194240) > 0


@pytest.mark.parametrize("change,text", [
    (dict(vocab=0), "sizes"), (dict(C=0), "sizes"), (dict(n=-1), "sizes"), (dict(n=1 << 31), "sizes"), (dict(stride=3), "row stride"), (dict(C=1 << 29, stride=1 << 29), "sizes"),
    (dict(table_type=3), "type"), (dict(out_type=-1), "type"), (dict(table=None), "null"), (dict(tokens=None), "null"), (dict(out=None), "null"),
])
def test_lookup_refusals(a, change, text):
    k = dict(table=P, table_type=0, vocab=5, C=4, tokens=P, n=7, out=P, out_type=0, stride=4)
    k.update(change)
    refused(a, a.lib().scn_embedding_forward(k["table"], k["table_type"], k["vocab"], k["C"], k["tokens"], k["n"], 1.0, k["out"], k["out_type"], k["stride"],
                                             None, None), INVALID, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(vocab=0), INVALID, "sizes"), (dict(C=0), INVALID, "sizes"), (dict(n=-1), INVALID, "sizes"), (dict(n=(1 << 31) - 1), INVALID, "sizes"),
    (dict(stride=3), INVALID, "row stride"), (dict(type=7), INVALID, "type"), (dict(dtable=None), INVALID, "null"), (dict(tokens=None), INVALID, "null"),
    (dict(dout=None), INVALID, "null"), (dict(ws=None), INVALID, "null"), (dict(ws=P + 8), INVALID, "aligned"), (dict(short=1), WORKSPACE, "workspace"),
])
def test_gradient_refusals(a, change, code, text):
    k = dict(tokens=P, n=7, dout=P, type=0, stride=4, vocab=5, C=4, dtable=P, ws=P, short=0)
    k.update(change)
    need = a.lib().scn_embedding_backward_workspace_bytes(7, 5, 4)
    refused(a, a.lib().scn_embedding_backward(k["tokens"], k["n"], k["dout"], k["type"], k["stride"], k["vocab"], k["C"], 1.0, 0, k["dtable"], None, k["ws"],
                                              need - k["short"], None), code, text)


@pytest.mark.parametrize("at", range(9))
def test_misaligned_pointers(a, at):
    """Each pointer has to be aligned to its own type."""
    L, h, t = a.lib(), parameters(a), (a.AdamWTensor * 1)(entry(a))
    q = [P] * 9
    q[at] += 1 if at < 3 else 2
    if at < 4:  # 16-bit table and values at odd addresses, tokens and errors at half a word
        refused(a, L.scn_embedding_forward(q[0], 1, 5, 4, q[3], 7, 1.0, q[1], 2, 4, q[2], None), INVALID, "misaligned")
    if at in (1, 2, 3, 4):
        refused(a, L.scn_embedding_backward(q[3], 7, q[1], 1, 4, 5, 4, 1.0, 0, q[4], q[2], P, 1 << 20, None), INVALID, "misaligned")
    if at == 5:
        refused(a, L.scn_grad_norm(t, 1, q[5], P, 1 << 20, None), INVALID, "misaligned")
    if at >= 5 and at < 7:
        refused(a, L.scn_adamw_step(t, 1, ctypes.byref(h), q[6] if at == 6 else None, q[5], None), INVALID, "misaligned")
    if at >= 7:
        refused(a, L.scn_adamw_decode(P + 1, q[7], 9, 0, q[8], None), INVALID, "misaligned")


def test_workspace_sizes(a):
    f = a.lib().scn_embedding_backward_workspace_bytes
    assert f(-1, 5, 4) == f(1 << 31, 5, 4) == f(7, 0, 4) == f(7, 5, 0) == 0
    assert f(0, 5, 4) > 0 and f(1000000, 100000, 64) >= 8 * 1000000
    assert f(2147000000, 2147483647, 4) > 8 * 2147000000  # sizes beyond 32 bits


def entry(a, **change):
    k = dict(d_w=P, d_g=P, d_m=P, d_v=P, d_m_scale=None, d_v_scale=None, d_w16=None, n=10, weight_decay=0.0, w_min=-math.inf, g_type=0, w16_type=0)
    k.update(change)
    return a.AdamWTensor(*[k[f] for f, _ in a.AdamWTensor._fields_])


def parameters(a, **change):
    k = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, max_norm=0.0, step=1, seed=0)
    k.update(change)
    return a.AdamWParameters(*[k[f] for f, _ in a.AdamWParameters._fields_])


@pytest.mark.parametrize("change,text", [
    (dict(n=-1), "number of values"), (dict(n=(1 << 40) + 1), "number of values"), (dict(g_type=3), "gradient type"), (dict(d_g=None), "null"),
    (dict(d_w=None), "null"), (dict(d_m=None), "null"), (dict(d_v=None), "null"), (dict(d_m_scale=P), "both scales"), (dict(d_v_scale=P), "both scales"),
    (dict(d_w16=P, w16_type=0), "16-bit copy"), (dict(d_w16=P + 1, w16_type=1), "misaligned"), (dict(weight_decay=math.nan), "weight decay"),
    (dict(weight_decay=math.inf), "weight decay"), (dict(w_min=math.nan), "w_min"), (dict(d_w=P + 2), "misaligned"), (dict(d_g=P + 2), "misaligned"),
    (dict(d_g=P + 1, g_type=2), "misaligned"), (dict(d_m=P + 1), "misaligned"), (dict(d_m_scale=P + 1, d_v_scale=P), "misaligned"),
])
def test_step_refuses_bad_tensors(a, change, text):
    t = (a.AdamWTensor * 2)(entry(a), entry(a, **change))
    h = parameters(a)
    refused(a, a.lib().scn_adamw_step(t, 2, ctypes.byref(h), None, None, None), INVALID, text)


def test_lists_of_too_many_values(a):
    """Several gradients may lie on one another for the norm: the list's values, not the memory, are what bounds it."""
    t = (a.AdamWTensor * 9)(*[entry(a, n=1 << 40) for _ in range(9)])
    h = parameters(a)
    refused(a, a.lib().scn_grad_norm(t, 9, P, P, 1 << 20, None), INVALID, "number of values")
    refused(a, a.lib().scn_adamw_step(t, 9, ctypes.byref(h), None, None, None), INVALID, "number of values")


@pytest.mark.parametrize("change,text", [
    (dict(lr=math.nan), "finite"), (dict(lr=math.inf), "finite"), (dict(grad_scale=math.nan), "finite"), (dict(beta1=1.0), "beta"), (dict(beta1=-0.1), "beta"),
    (dict(beta2=1.0), "beta"), (dict(beta2=math.nan), "beta"), (dict(eps=0.0), "eps"), (dict(eps=1e-60), "eps"), (dict(eps=1e-39), "eps"), (dict(eps=-1.0), "eps"), (dict(step=0), "steps"),
    (dict(max_norm=-1.0), "max_norm"), (dict(max_norm=math.nan), "max_norm"), (dict(max_norm=1.0), "needs the gradients' norm"),
])
def test_step_refuses_bad_parameters(a, change, text):
    t = (a.AdamWTensor * 1)(entry(a))
    h = parameters(a, **change)
    refused(a, a.lib().scn_adamw_step(t, 1, ctypes.byref(h), None, None, None), INVALID, text)


def test_lists_and_empty_calls(a):
    L, h = a.lib(), parameters(a)
    t = (a.AdamWTensor * 1)(entry(a))
    refused(a, L.scn_adamw_step(t, -1, ctypes.byref(h), None, None, None), INVALID, "bad list")
    refused(a, L.scn_adamw_step(None, 1, ctypes.byref(h), None, None, None), INVALID, "bad list")
    refused(a, L.scn_adamw_step(t, 1, None, None, None, None), INVALID, "null")
    need = L.scn_grad_norm_workspace_bytes()
    refused(a, L.scn_grad_norm(t, 1, None, P, need, None), INVALID, "null")
    refused(a, L.scn_grad_norm(t, 1, P, P, need - 1, None), WORKSPACE, "workspace")
    refused(a, L.scn_grad_norm(t, 1, P, P + 4, need, None), INVALID, "aligned")
    # nothing to do: no launch, no device needed
    assert L.scn_adamw_step(None, 0, ctypes.byref(h), None, None, None) == 0
    assert L.scn_adamw_step((a.AdamWTensor * 1)(entry(a, n=0, d_w=None, d_g=None, d_m=None, d_v=None)), 1, ctypes.byref(h), None, None, None) == 0
    assert L.scn_embedding_forward(None, 0, 5, 4, None, 0, 1.0, None, 0, 4, None, None) == 0
    assert L.scn_adamw_decode(None, None, 0, 0, None, None) == 0
    refused(a, L.scn_adamw_decode(None, None, 1, 0, None, None), INVALID, "null")
    refused(a, L.scn_adamw_decode(None, None, -1, 0, None, None), INVALID, "size")


@pytest.mark.parametrize("step", [1, 2, 1000, 10 ** 9])
def test_scalars(a, step):
    """Constants come from 64-bit arithmetic, rounded once: half a step of 32 bits (2^-24), and the power's own rounding
    (about step ulps of 64 bits in beta^step at worst, far below)."""
    s = a.AdamWScalars.from_buffer_copy(a.adamw_scalars(1e-3, step, beta1=0.9, beta2=0.999, eps=1e-8, max_norm=2.0).numpy().tobytes())
    for got, want in [(s.lr, 1e-3), (s.beta1, 0.9), (s.beta2, 0.999), (s.one_minus_beta1, 0.1), (s.one_minus_beta2, 0.001), (s.eps, 1e-8),
                      (s.bias1, 1 / (1 - 0.9 ** step)), (s.bias2, 1 / math.sqrt(1 - 0.999 ** step)), (s.max_norm, 2.0), (s.grad_scale, 1.0)]:
        assert abs(got - want) <= 1.001 * 2.0 ** -24 * want
    assert s.seed == step & 0xFFFFFFFF


def test_python_binding_refuses_cpu_tensors(a):
    table, tok = torch.zeros(5, 4), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(a.ScnError):
        a.embedding_forward(table, tok)
    with pytest.raises(a.ScnError):
        a.embedding_backward(torch.zeros(3, 4), tok, table)
    with pytest.raises(a.ScnError):
        a.adamw_decode(torch.zeros(3, dtype=torch.int8), torch.zeros(1))
    with pytest.raises(a.ScnError):
        a.adamw_states(5, "cpu", bits=16)
    with pytest.raises(a.ScnError, match="w must be"):
        a.AdamW([dict(w=torch.zeros(4), g=torch.zeros(4), **a.adamw_states(4, "cpu", bits=32))])


def test_row_strides(a):
    """A single row has no stride to speak of, however its view was made; several rows must not overlap."""
    assert a._row_stride(torch.empty_strided((1, 4), (1 << 40, 1)), 1, 4, "out") == 4
    assert a._row_stride(torch.empty(0, 4), 0, 4, "out") == 4
    assert a._row_stride(torch.empty(3, 9)[:, 2:6], 3, 4, "out") == 9
    assert a._row_stride(torch.empty(3, 9)[:, 2:3], 3, 1, "out") == 9
    for bad in [torch.empty(1, 4).expand(3, 4), torch.empty(4, 3).t(), torch.empty(3, 8)[:, ::2], torch.empty(3, 4, dtype=torch.float64), torch.empty(12)]:
        with pytest.raises(a.ScnError):
            a._row_stride(bad, 3, 4, "out")


@pytest.mark.parametrize("change,text", [
    (dict(lr=1e39), "finite"), (dict(lr=-1e39), "finite"), (dict(grad_scale=1e39), "finite"), (dict(grad_scale=-4e38), "finite"), (dict(max_norm=1e-46), "max_norm"),
    (dict(max_norm=5e-324), "max_norm")])
def test_numbers_that_32_bits_cannot_hold(a, change, text):
    """The kernel reads 32-bit numbers: infinities in place of a rate or a scale, or a clip that turned into no clip, are refused."""
    t, h = (a.AdamWTensor * 1)(entry(a)), parameters(a, **change)
    refused(a, a.lib().scn_adamw_step(t, 1, ctypes.byref(h), None, P, None), INVALID, text)
    out = a.AdamWScalars()
    refused(a, a.lib().scn_adamw_scalars(ctypes.byref(h), ctypes.byref(out)), INVALID, text)


@pytest.mark.parametrize("change", [dict(lr=3e38), dict(max_norm=1e300), dict(max_norm=1e-44), dict(eps=1e39), dict(lr=1e-50)])
def test_numbers_at_the_ends_of_32_bits(a, change):
    """Rounding these to 32 bits changes no step by more than roundings do."""
    h, out = parameters(a, **change), a.AdamWScalars()
    assert a.lib().scn_adamw_scalars(ctypes.byref(h), ctypes.byref(out)) == 0
    assert out.max_norm > 0 or "max_norm" not in change


def test_parameters_are_packed_in_the_order_of_their_fields(a):
    values = dict(lr=1.5, beta1=0.25, beta2=0.5, eps=2.0, grad_scale=-3.0, max_norm=7.0, step=(1 << 40) + 3, seed=0xFFFFFFFF)
    h = a.AdamWParameters()
    a._PACK_PARAMETERS(h, 0, *values.values())
    assert [f for f, _ in a.AdamWParameters._fields_] == list(values)
    assert all(getattr(h, k) == v for k, v in values.items())

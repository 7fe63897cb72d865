"""CPU checks of the operators of a block in plain rows: what a call refuses
(arguments are checked before anything else, so a call without a context names the
first wrong one), workspaces, and the plain forms the GPU tests use."""
import ctypes as C
import math

import numpy as np
import pytest

import gotransformers_amd as gt
from tests import plain_block as plain

P = 1 << 40  # addresses that are only compared
GAP = 1 << 36
X, W, Y, OFFSETS, D, U, S, WS, A, B, Q, K = (P + i * GAP for i in range(12))
FINE = "context is null"  # nothing else was wrong


def refused(name, *args):
    assert getattr(gt.library(), name)(None, *args) == gt.ERR_INVALID_ARGUMENT
    return gt.library().gtmoe_last_error(None).decode()


def changed(d, changes):
    for k, v in changes.items():
        setattr(d, k, v)
    return d


def packed(**changes):
    return changed(gt.packed_desc(gt.VALUES_BFLOAT16, 10, 100, gt.CODES_INT8, 32), changes)


@pytest.mark.parametrize("changes, text", [
    (dict(values=3), "type of values"), (dict(rows=-1), "rows must be"), (dict(rows=(1 << 30) + 1), "rows must be"),
    (dict(columns=0), "columns must be"), (dict(columns=(1 << 20) + 1), "columns must be"), (dict(codes=0), "type of codes"),
    (dict(codes=3), "type of codes"), (dict(scale_columns=8), "scale columns"), (dict(scale_columns=256), "scale columns"),
    (dict(scale_columns=-16), "scale columns"), (dict(reserved=1), "reserved"), (dict(value_stride=99), "value stride"),
    (dict(code_stride=99), "code stride"), (dict(scale_stride=3), "scale stride"), (dict(value_stride=(1 << 20) + 1), "value stride"),
])
def test_packed_descriptions_that_are_refused(changes, text):
    d = packed(**changes)
    assert text in refused("gtmoe_pack_rows", C.byref(d), X, Q, S, None)
    assert text in refused("gtmoe_unpack_rows", C.byref(d), Q, S, X, None)


def test_packed_buffers_that_are_refused():
    d = C.byref(packed())
    for call, args in (("gtmoe_pack_rows", (X, Q, S)), ("gtmoe_unpack_rows", (Q, S, X))):
        assert FINE in refused(call, d, *args, None)
        assert "description" in refused(call, None, *args, None)
        for i in range(3):
            assert "null" in refused(call, d, *args[:i], None, *args[i + 1:], None)
        assert FINE in refused(call, C.byref(packed(rows=0)), None, None, None, None)
    assert "not aligned" in refused("gtmoe_pack_rows", d, X + 1, Q, S, None)
    assert "scales are not aligned" in refused("gtmoe_pack_rows", d, X, Q, S + 2, None)
    assert FINE in refused("gtmoe_pack_rows", d, X, Q + 1, S, None)
    assert "codes overlap" in refused("gtmoe_pack_rows", d, X, X + 1998, S, None)
    assert FINE in refused("gtmoe_pack_rows", d, X, X + 2000, S, None)
    assert "scales overlap" in refused("gtmoe_pack_rows", d, X, Q, X + 1996, None)
    assert "codes overlap" in refused("gtmoe_pack_rows", d, X, Q, Q + 996, None)
    assert "outputs overlap" in refused("gtmoe_unpack_rows", d, Q, S, Q + 998, None)
    # one scale per row
    assert FINE in refused("gtmoe_pack_rows", C.byref(packed(scale_columns=0, scale_stride=1)), X, Q, S, None)


def norm(**changes):
    return changed(gt.norm_desc(gt.VALUES_FLOAT16, 10, 100, codes=gt.CODES_E4M3), changes)


@pytest.mark.parametrize("changes, text", [
    (dict(values=-1), "type of values"), (dict(rows=-1), "rows must be"), (dict(columns=0), "columns must be"),
    (dict(reserved=2), "reserved"), (dict(epsilon=-1e-9), "epsilon"), (dict(epsilon=math.nan), "epsilon"),
    (dict(epsilon=math.inf), "epsilon"), (dict(codes=7), "type of codes"), (dict(scale_columns=1), "scale columns"),
    (dict(code_stride=1), "code stride"), (dict(input_stride=99), "input stride"), (dict(residual_stride=99), "residual stride"),
    (dict(sum_stride=99), "sum stride"), (dict(output_stride=99), "output stride"),
])
def test_norm_descriptions_that_are_refused(changes, text):
    d = norm(**changes)
    assert text in refused("gtmoe_norm_forward", C.byref(d), X, B, W, D, Y, Q, S, None)
    if "residual" not in text:
        assert text in refused("gtmoe_norm_gradient", C.byref(d), Y, D, W, U, X, None, 0, 0, None, 0, None)


def test_norm_buffers_that_are_refused():
    d = C.byref(norm())
    call = lambda *a: refused("gtmoe_norm_forward", *a, None)
    assert FINE in call(d, X, B, W, D, Y, Q, S)
    assert FINE in call(d, X, None, None, None, None, Q, S)
    assert "inputs are null" in call(d, None, B, W, D, Y, Q, S)
    assert "sums are null" in call(d, X, B, W, None, Y, Q, S)
    assert "codes are null" in call(d, X, B, W, D, Y, None, S)
    assert "outputs are null" in call(C.byref(norm(codes=0, scale_columns=0)), X, B, W, D, None, None, None)
    assert FINE in call(d, X, B, W, X, Y, Q, S) and FINE in call(d, X, B, W, B, Y, Q, S)  # the sums in place
    assert "sums overlap" in call(d, X, B, W, X + 2, Y, Q, S)
    assert "sums overlap" in call(C.byref(norm(sum_stride=101)), X, B, W, B, Y, Q, S)
    assert "outputs overlap" in call(d, X, B, W, D, X, Q, S) and "outputs overlap" in call(d, X, B, W, D, D, Q, S)
    assert "codes overlap" in call(d, X, B, W, D, Y, W, S)
    assert "scales overlap" in call(d, X, B, W, D, Y, Q, Q + 996)
    # unused buffers' strides are not looked at
    assert FINE in call(C.byref(norm(residual_stride=0, sum_stride=0)), X, None, W, None, Y, Q, S)
    n = gt.norm_workspace_bytes(norm())
    back = lambda *a: refused("gtmoe_norm_gradient", *a, None)
    assert FINE in back(d, Y, D, W, U, X, A, 0, 0, WS, n)
    assert FINE in back(d, Y, D, W, U, U, A, 0, 0, WS, n)  # the input gradients in place
    assert FINE in back(d, Y, D, None, None, X, None, 9, 0, None, 0)
    assert "output gradients are null" in back(d, None, D, W, U, X, A, 0, 0, WS, n)
    assert "input gradients are null" in back(d, Y, D, W, U, None, A, 0, 0, WS, n)
    assert "values' type or float32" in back(d, Y, D, W, U, X, A, gt.VALUES_BFLOAT16, 0, WS, n)
    assert "workspace has" in back(d, Y, D, W, U, X, A, 0, 0, WS, n - 1)
    assert "workspace bytes are null" in back(d, Y, D, W, U, X, A, 0, 0, None, n)
    assert "not aligned to 16" in back(d, Y, D, W, U, X, A, 0, 0, WS + 8, n)
    assert "input gradients overlap" in back(d, Y, D, W, U, Y, A, 0, 0, WS, n)
    assert "input gradients overlap" in back(d, Y, D, W, U, D, A, 0, 0, WS, n)
    assert "weight gradients overlap" in back(d, Y, D, W, U, X, W, 0, 0, WS, n)
    assert "workspace's bytes overlap" in back(d, Y, D, W, U, X, A, 0, 0, A, n)
    assert gt.norm_workspace_bytes(norm(rows=0)) == 0
    with pytest.raises(gt.InvalidArgument, match="epsilon"):
        gt.norm_workspace_bytes(norm(epsilon=-1))


def activation(**changes):
    return changed(gt.activation_desc(gt.VALUES_FLOAT32, 10, 100, gt.ACTIVATION_SILU, codes=gt.CODES_INT8), changes)


@pytest.mark.parametrize("changes, text", [
    (dict(values=5), "type of values"), (dict(rows=-1), "rows must be"), (dict(columns=0), "columns must be"),
    (dict(activation=-1), "activation"), (dict(activation=5), "activation"), (dict(limit=-1.0), "limit"),
    (dict(limit=math.nan), "limit"), (dict(limit=1e-60), "limit"), (dict(codes=-1), "type of codes"),
    (dict(scale_columns=0), "scale columns"), (dict(scale_columns=24), "scale columns"), (dict(code_stride=4), "code stride"),
    (dict(gate_stride=99), "gate stride"), (dict(up_stride=99), "up stride"), (dict(output_stride=99), "output stride"),
])
def test_activation_descriptions_that_are_refused(changes, text):
    d = activation(**changes)
    assert text in refused("gtmoe_activation_forward", C.byref(d), X, U, Y, Q, S, K, A, None)
    assert text in refused("gtmoe_activation_gradient", C.byref(d), Y, Q, S, K, A, X, U, D, None)


def test_activation_buffers_that_are_refused():
    d, plainly = C.byref(activation()), C.byref(activation(codes=0, scale_columns=0))
    call = lambda *a: refused("gtmoe_activation_forward", *a, None)
    assert FINE in call(d, X, U, Y, Q, S, K, A) and FINE in call(d, X, None, Y, Q, S, None, None)
    assert FINE in call(plainly, X, U, Y, None, None, None, None)
    assert FINE in call(plainly, X, U, X, None, None, None, None) and FINE in call(plainly, X, U, U, None, None, None, None)
    for i, what in ((1, "gates"), (3, "outputs"), (4, "gate codes"), (5, "gate scales"), (6, "up codes"), (7, "up scales")):
        args = [d, X, U, Y, Q, S, K, A]
        args[i] = None
        assert what + " are null" in call(*args)
    assert "outputs overlap" in call(plainly, X, U, X + 4, None, None, None, None)
    assert "gate codes overlap" in call(d, X, U, Y, X, S, K, A)
    assert "up codes overlap" in call(d, X, U, Y, Q, S, Q + 999, A)
    assert "up scales overlap" in call(d, X, U, Y, Q, S, K, S)
    back = lambda *a: refused("gtmoe_activation_gradient", *a, None)
    assert FINE in back(d, Y, Q, S, K, A, X, U, D) and FINE in back(d, Y, Q, S, K, A, None, None, None)
    assert FINE in back(plainly, Y, X, None, U, None, X, U, Y)  # all in place
    assert FINE in back(d, Y, Q, S, None, None, X, None, Y)
    assert "up gradients without ups" in back(d, Y, Q, S, None, None, X, U, D)
    assert "gate scales are null" in back(d, Y, Q, None, K, A, X, U, D)
    assert "up scales are null" in back(d, Y, Q, S, K, None, X, U, D)
    assert "gate gradients overlap" in back(d, Y, Q, S, K, A, Q, U, D)
    assert "up gradients overlap" in back(plainly, Y, X, None, U, None, D, D, None)
    assert "outputs overlap" in back(plainly, Y, X, None, U, None, D, None, D)


def product(**changes):
    return changed(gt.grouped_desc(gt.VALUES_BFLOAT16, 4, 100, 64, 32), changes)


def test_fused_products_that_are_refused():
    d = C.byref(product())
    full = lambda **c: C.byref(changed(gt.epilogue(gt.ACTIVATION_SILU, A, B, D, S, 32), c))
    call = lambda *a: refused("gtmoe_grouped_fused_forward", *a, None)
    assert FINE in call(d, full(), OFFSETS, X, W, Y)
    assert FINE in call(d, C.byref(gt.epilogue()), OFFSETS, X, W, Y)
    assert "epilogue is null" in call(d, None, OFFSETS, X, W, Y)
    assert "offsets are null" in call(d, full(), None, X, W, Y)
    assert FINE in call(C.byref(product(groups=1)), full(), None, X, W, Y)
    assert "groups must be" in call(C.byref(product(groups=0)), full(), OFFSETS, X, W, Y)
    for changes, text in ((dict(activation=9), "activation"), (dict(reserved=1), "reserved"), (dict(bias_stride=31), "bias stride"),
                          (dict(factor_stride=31), "factor stride"), (dict(residual_stride=31), "residual stride"),
                          (dict(product_stride=31), "product stride"), (dict(factors=B + 1), "factors are not aligned"),
                          (dict(biases=A + 1), "biases are not aligned"), (dict(products=B), "products overlap"),
                          (dict(products=X), "products overlap"), (dict(products=Y), "outputs overlap"),
                          (dict(biases=Y), "outputs overlap"), (dict(factors=Y + 2), "outputs overlap")):
        assert text in call(d, full(**changes), OFFSETS, X, W, Y)
    assert FINE in call(d, full(residuals=Y), OFFSETS, X, W, Y) and FINE in call(d, full(factors=Y), OFFSETS, X, W, Y)
    assert "outputs overlap" in call(d, full(residuals=Y, residual_stride=33), OFFSETS, X, W, Y)
    assert "one launch" in call(C.byref(product(rows=1 << 30, outputs=1 << 20, output_stride=1 << 20, group_stride=1 << 26)),
                                C.byref(gt.epilogue()), OFFSETS, X, W, 1 << 55)
    n = gt.grouped_bias_workspace_bytes(product())
    back = lambda *a: refused("gtmoe_grouped_bias_gradient", *a, None)
    assert FINE in back(d, OFFSETS, Y, A, 0, 0, WS, n)
    assert "bias gradients are null" in back(d, OFFSETS, Y, None, 0, 0, WS, n)
    assert "output gradients are null" in back(d, OFFSETS, None, A, 0, 0, WS, n)
    assert "values' type or float32" in back(d, OFFSETS, Y, A, gt.VALUES_FLOAT16, 0, WS, n)
    assert "workspace has" in back(d, OFFSETS, Y, A, 0, 0, WS, n - 1)
    assert "bias gradients overlap" in back(d, OFFSETS, Y, Y, 0, 0, WS, n)
    assert "workspace's bytes overlap" in back(d, OFFSETS, Y, A, 0, 0, Y, n)
    assert FINE in back(C.byref(product(groups=1)), None, Y, A, 0, 0, WS, n)


def route(**changes):
    return changed(gt.route_desc(gt.VALUES_FLOAT32, 1000, 64, 6, 8, 3, 2), changes)


@pytest.mark.parametrize("changes, text", [
    (dict(values=4), "type of values"), (dict(tokens=-1), "tokens must be"), (dict(tokens=(1 << 24) + 1), "tokens must be"),
    (dict(experts=0), "experts must be"), (dict(experts=1025), "experts must be"), (dict(expert_groups=0), "expert groups must"),
    (dict(expert_groups=65), "expert groups must"), (dict(expert_groups=7), "whole in 7 groups"), (dict(chosen_groups=0), "chosen groups"),
    (dict(chosen_groups=9), "chosen groups"), (dict(experts_per_token=0), "experts per token"),
    (dict(experts_per_token=25), "experts per token"), (dict(group_best=3), "best"), (dict(group_best=0), "best"),
    (dict(scores=2), "unknown scores"), (dict(reserved=1), "reserved"), (dict(scale=math.inf), "scale"), (dict(scale=1e300), "scale"),
    (dict(logit_stride=63), "logit stride"),
])
def test_route_descriptions_that_are_refused(changes, text):
    d = route(**changes)
    assert text in refused("gtmoe_route_forward", C.byref(d), X, B, Q, S, OFFSETS, D, A, WS, 1 << 20, None)
    assert text in refused("gtmoe_route_gradient", C.byref(d), X, Q, S, Y, None)


def test_route_buffers_that_are_refused():
    d = C.byref(route())
    n = gt.route_workspace_bytes(route())
    call = lambda *a: refused("gtmoe_route_forward", *a, None)
    assert FINE in call(d, X, B, Q, S, OFFSETS, D, A, WS, n) and FINE in call(d, X, None, Q, S, None, None, None, None, 0)
    assert FINE in call(d, X, None, Q, S, OFFSETS, None, None, WS, n)
    assert "without expert offsets" in call(d, X, None, Q, S, None, D, None, None, 0)
    assert "without expert offsets" in call(d, X, None, Q, S, None, None, A, None, 0)
    assert "workspace has" in call(d, X, B, Q, S, OFFSETS, D, A, WS, n - 1)
    assert "workspace bytes are null" in call(d, X, B, Q, S, OFFSETS, D, A, None, n)
    for i, what in ((1, "logits"), (3, "chosen"), (4, "gates")):
        args = [d, X, B, Q, S, OFFSETS, D, A, WS, n]
        args[i] = None
        assert what + " are null" in call(*args)
    assert "gates overlap" in call(d, X, B, Q, Q, OFFSETS, D, A, WS, n)
    assert "chosen overlap" in call(d, X, B, X, S, OFFSETS, D, A, WS, n)
    assert "places overlap" in call(d, X, B, Q, S, OFFSETS, D, D, WS, n)
    assert "workspace's bytes overlap" in call(d, X, B, Q, S, OFFSETS, D, A, D, n)
    # few tokens need no workspace
    assert gt.route_workspace_bytes(route(tokens=1)) == 0 and gt.route_workspace_bytes(route(tokens=0)) == 0
    back = lambda *a: refused("gtmoe_route_gradient", *a, None)
    assert FINE in back(d, X, Q, S, Y)
    assert "logit gradients overlap" in back(d, X, Q, S, X)
    assert "gate gradients are null" in back(d, X, Q, None, Y)


def test_workspaces_need_a_place_for_their_size():
    for name in ("gtmoe_norm_workspace", "gtmoe_grouped_bias_workspace", "gtmoe_route_workspace"):
        assert getattr(gt.library(), name)(C.byref(norm()), None) == gt.ERR_INVALID_ARGUMENT
        assert getattr(gt.library(), name)(None, C.byref(C.c_size_t())) == gt.ERR_INVALID_ARGUMENT


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------

def test_plain_codes():
    # every e4m3 value is its own code's; halves go to the even neighbour
    codes = np.arange(256, dtype=np.uint8)
    v = plain.e4m3_decode(codes)
    fine = np.isfinite(v)
    assert fine.sum() == 254 and v[fine].max() == 448
    assert np.array_equal(plain.e4m3_round(v[fine]), v[fine])
    assert np.array_equal(plain.e4m3_round(np.array([17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10])), [16.0, 20.0, 0.0, 2 * 2.0 ** -9])
    rows = np.random.default_rng(0).normal(size=(5, 50))
    own = gt.encode_rows(gt.INT8, rows)
    q, s = plain.packed(rows, "int8", 16)
    assert np.array_equal(q, own.values) and np.array_equal(s, own.scales)


def test_plain_activations():
    z = np.linspace(-6, 6, 41)
    for name in ("silu", "gelu", "gelu_tanh"):
        f = lambda x: plain.activation(x, name)[0]
        assert np.allclose((f(z + 1e-5) - f(z - 1e-5)) / 2e-5, plain.activation(z, name)[1], rtol=0, atol=1e-8)
    assert abs(plain.activation(np.array([1.0]), "gelu")[0][0] - 0.8413447460685429) < 1e-15
    assert np.abs(plain.activation(z, "gelu")[0] - plain.activation(z, "gelu_tanh")[0]).max() < 5e-4


def test_plain_choice():
    l = np.array([[0.0, 2.0, 2.0, -1.0], [1.0, -np.inf, 0.0, 3.0], [-np.inf] * 4])
    chosen, gates = plain.route(l, None, 2, "softmax")
    assert chosen.tolist() == [[1, 2], [3, 0], [0, 1]] and np.allclose(gates[0], 0.5) and np.all(gates[2] == 0)
    chosen, _ = plain.route(l, np.array([0.0, 0.0, 0.0, 9.0]), 2, "sigmoid")
    assert chosen.tolist() == [[3, 1], [3, 0], [0, 1]]
    # groups {0, 1} and {2, 3} by their two best
    chosen, _ = plain.route(l, None, 2, "softmax", 2, 1, 2)
    assert chosen.tolist() == [[1, 0], [3, 2], [0, 1]]
    off, rows, places = plain.lists(np.array([[1, 2], [3, 1], [0, 1]]), 4)
    assert off.tolist() == [0, 1, 4, 5, 6] and rows.tolist() == [2, 0, 1, 2, 0, 1] and places.tolist() == [[1, 4], [5, 2], [0, 3]]


def test_plain_gradients_against_differences():
    rng = np.random.default_rng(2)
    l, dg = rng.normal(size=(2, 6)), rng.normal(size=(2, 3))
    chosen = np.array([[0, 4, 2], [5, 1, 3]])
    for kind in ("softmax", "sigmoid"):
        for renormalize in (False, True):
            def f(v):
                m = np.take_along_axis(plain.scores(v, kind), chosen, axis=1)
                return float((m / (m.sum(axis=1, keepdims=True) if renormalize else 1.0) * dg).sum())
            got, _ = plain.route_gradient(l, chosen, dg, kind, renormalize, 1.0)
            for t in range(2):
                for e in range(6):
                    h = np.zeros((2, 6))
                    h[t, e] = 1e-6
                    assert abs((f(l + h) - f(l - h)) / 2e-6 - got[t, e]) < 1e-8
    s, w, dy = rng.normal(size=(2, 5)), rng.normal(size=5), rng.normal(size=(2, 5))
    dx, dw, _, _ = plain.norm_gradient(dy, s, w, None, 0.1)
    for c in range(5):
        h = np.zeros((2, 5))
        h[1, c] = 1e-6
        f = lambda x: float((plain.norm(x, w, 0.1)[0] * dy).sum())
        assert abs((f(s + h) - f(s - h)) / 2e-6 - dx[1, c]) < 1e-8

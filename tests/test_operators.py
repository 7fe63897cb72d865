"""CPU checks of the operators over plain rows: what a call refuses (arguments
are checked before anything else, so a call without a context names the first
wrong one), the workspace's size, and the plain forms the GPU tests use."""
import ctypes as C

import numpy as np
import pytest

import gotransformers_amd as gt
from tests.plain_rows import adapted, dropout_factor, dropout_threshold, grouped, offsets_of, philox4x32

P = 1 << 40  # addresses that are only compared
GAP = 1 << 36
X, W, Y, OFFSETS, D, U, S, WS, A = (P + i * GAP for i in range(9))


def refused(call, *args):
    code = call(None, *args)
    assert code == gt.ERR_INVALID_ARGUMENT
    return gt.library().gtmoe_last_error(None).decode()


def test_philox_known_answers():
    # the generator's published test vectors
    ones, pi = 0xFFFFFFFF, (0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344)
    for counter, key, want in (((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                               ((ones,) * 4, (ones, ones), (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                               (pi, (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(v) for v in philox4x32(counter, key)) == want


def test_dropout_factor_keeps_the_expected_share():
    f, keep = dropout_factor(300, 1001, 0.25, 7, 9)
    t = dropout_threshold(0.25) / 65536
    n = keep.size
    assert abs(keep.mean() - (1 - t)) < 5 * np.sqrt(t * (1 - t) / n)
    assert np.all(f[keep] == 1 / (1 - t)) and np.all(f[~keep] == 0)
    assert dropout_threshold(0.9999999) == 65535 and dropout_threshold(0.0) == 0


def test_plain_gradients_against_differences():
    rng = np.random.default_rng(0)
    off = offsets_of([3, 0, 2])
    x, w, dy = rng.normal(size=(5, 4)), rng.normal(size=(3, 6, 4)), rng.normal(size=(5, 6))
    y, dx, dw = grouped(off, x, w, dy)
    f = lambda x_, w_: float(np.sum(grouped(off, x_, w_, dy)[0] * dy))
    h = 0.5  # f is linear in x and in w: any step is exact up to rounding
    for index in ((0, 1), (4, 3)):
        e = np.zeros_like(x)
        e[index] = h
        assert abs((f(x + e, w) - f(x - e, w)) / (2 * h) - dx[index]) < 1e-12
    for index in ((0, 2, 1), (1, 0, 0), (2, 5, 3)):
        e = np.zeros_like(w)
        e[index] = h
        assert abs((f(x, w + e) - f(x, w - e)) / (2 * h) - dw[index]) < 1e-12


def test_plain_adapted_is_the_merged_projection():
    rng = np.random.default_rng(1)
    x, w, b = rng.normal(size=(4, 5)), rng.normal(size=(6, 5)), rng.normal(size=6)
    down, up, s = rng.normal(size=(2, 3, 5)), rng.normal(size=(2, 6, 3)), np.array([0.5, 2.0])
    y, _ = adapted(x, w, b, [1, -1, 0, 7], down, up, s)
    for t, a in enumerate([1, None, 0, None]):
        m = w if a is None else w + s[a] * up[a] @ down[a]
        assert np.allclose(y[t], m @ x[t] + b, rtol=0, atol=1e-12)


def grouped_args(**changes):
    d = gt.grouped_desc(gt.VALUES_BFLOAT16, 4, 100, 64, 32)
    for k, v in changes.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("changes, text", [
    (dict(values=3), "type of values"), (dict(values=-1), "type of values"),
    (dict(groups=0), "groups must be"), (dict(groups=4097), "groups must be"),
    (dict(rows=-1), "rows must be"), (dict(rows=(1 << 30) + 1), "rows must be"),
    (dict(inputs=0), "inputs must be"), (dict(outputs=0), "outputs must be"),
    (dict(inputs=(1 << 20) + 1), "inputs must be"), (dict(reserved=1), "reserved"),
    (dict(input_stride=63), "input stride"), (dict(output_stride=31), "output stride"),
    (dict(weight_stride=63), "weight stride"), (dict(input_stride=(1 << 20) + 1), "input stride"),
    (dict(group_stride=64 * 32 - 1), "group stride"), (dict(group_stride=1 << 47), "group stride"),
    (dict(rows=1 << 30, outputs=1 << 20, output_stride=1 << 20, group_stride=1 << 26), "one launch"),
])
def test_grouped_descriptions_that_are_refused(changes, text):
    lib, d = gt.library(), grouped_args(**changes)
    far = 1 << 55
    assert text in refused(lib.gtmoe_grouped_forward, C.byref(d), OFFSETS, X, W, far, None)
    if text != "one launch":
        assert text in refused(lib.gtmoe_grouped_input_gradient, C.byref(d), OFFSETS, far, W, X, None)
        assert text in refused(lib.gtmoe_grouped_weight_gradient, C.byref(d), OFFSETS, Y, X, far, d.values, 0, None)


def test_grouped_pointers_that_are_refused():
    lib, d = gt.library(), grouped_args()
    fwd, dx, dw = lib.gtmoe_grouped_forward, lib.gtmoe_grouped_input_gradient, lib.gtmoe_grouped_weight_gradient
    assert "description" in refused(fwd, None, OFFSETS, X, W, Y, None)
    assert "offsets are null" in refused(fwd, C.byref(d), None, X, W, Y, None)
    assert "offsets are not aligned" in refused(fwd, C.byref(d), OFFSETS + 2, X, W, Y, None)
    assert "inputs are null" in refused(fwd, C.byref(d), OFFSETS, None, W, Y, None)
    assert "weights are null" in refused(fwd, C.byref(d), OFFSETS, X, None, Y, None)
    assert "outputs are null" in refused(fwd, C.byref(d), OFFSETS, X, W, None, None)
    assert "not aligned" in refused(fwd, C.byref(d), OFFSETS, X + 1, W, Y, None)
    assert "output gradients are null" in refused(dx, C.byref(d), OFFSETS, None, W, X, None)
    assert "weight gradients are null" in refused(dw, C.byref(d), OFFSETS, Y, X, None, d.values, 0, None)
    assert "values' type or float32" in refused(dw, C.byref(d), OFFSETS, Y, X, W, gt.VALUES_FLOAT16, 0, None)
    # everything in order but the context
    assert "context is null" in refused(fwd, C.byref(d), OFFSETS, X, W, Y, None)
    assert "context is null" in refused(dx, C.byref(d), OFFSETS, Y, W, X, None)
    assert "context is null" in refused(dw, C.byref(d), OFFSETS, Y, X, W, gt.VALUES_FLOAT32, 1, None)
    # no rows: no row buffers needed
    d0 = grouped_args(rows=0)
    assert "context is null" in refused(fwd, C.byref(d0), OFFSETS, None, None, None, None)
    assert "context is null" in refused(dw, C.byref(d0), OFFSETS, None, None, W, d.values, 0, None)


def test_grouped_buffers_that_overlap_are_refused():
    lib, d = gt.library(), grouped_args()
    fwd = lib.gtmoe_grouped_forward
    last = X + (100 * 64 - 1) * 2
    assert "outputs overlap" in refused(fwd, C.byref(d), OFFSETS, X, W, X, None)
    assert "outputs overlap" in refused(fwd, C.byref(d), OFFSETS, X, W, last, None)
    assert "context is null" in refused(fwd, C.byref(d), OFFSETS, X, W, last + 2, None)
    assert "outputs overlap" in refused(fwd, C.byref(d), OFFSETS, X, W, W + 2 * (4 * 64 * 32 - 1), None)
    assert "outputs overlap" in refused(fwd, C.byref(d), Y + 8, X, W, Y, None)
    # column ranges of one matrix interleave without sharing a value
    side = grouped_args(input_stride=96, output_stride=96)
    assert "context is null" in refused(fwd, C.byref(side), OFFSETS, X, W, X + 64 * 2, None)
    assert "outputs overlap" in refused(fwd, C.byref(side), OFFSETS, X, W, X + 63 * 2, None)
    assert "context is null" in refused(fwd, C.byref(side), OFFSETS, X + 32 * 2, W, X, None)
    assert "outputs overlap" in refused(fwd, C.byref(side), OFFSETS, X + 31 * 2, W, X, None)


def adapted_desc(**changes):
    d = gt.adapted_desc(gt.VALUES_FLOAT16, 50, 64, 32, 6, 13)
    for k, v in changes.items():
        setattr(d, k, v)
    return d


def test_adapted_workspace_size():
    # u, the rows' scales and order (16-byte multiples), the adapters' places
    rest = 2 * 208 + 32
    assert gt.adapted_workspace_bytes(adapted_desc()) == 50 * 16 * 4 + rest
    assert gt.adapted_workspace_bytes(adapted_desc(rank=16)) == 50 * 16 * 4 + rest
    assert gt.adapted_workspace_bytes(adapted_desc(rank=17)) == 50 * 24 * 4 + rest
    assert gt.adapted_workspace_bytes(adapted_desc(rows=0)) > 0
    with pytest.raises(gt.InvalidArgument, match="rank must be"):
        gt.adapted_workspace_bytes(adapted_desc(rank=257))
    assert gt.library().gtmoe_adapted_workspace(C.byref(adapted_desc()), None) == gt.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("changes, text", [
    (dict(values=7), "type of values"), (dict(rows=-1), "rows must be"), (dict(inputs=0), "inputs must be"),
    (dict(outputs=0), "outputs must be"), (dict(adapters=0), "adapters must be"), (dict(rank=0), "rank must be"),
    (dict(rank=257), "rank must be"), (dict(input_stride=63), "input stride"),
    (dict(output_stride=31), "output stride"), (dict(weight_stride=2), "weight stride"),
])
def test_adapted_descriptions_that_are_refused(changes, text):
    d = adapted_desc(**changes)
    assert text in refused(gt.library().gtmoe_adapted_forward, C.byref(d), X, W, None, A, D, U, S, Y, WS, 1 << 20, None)


def test_adapted_pointers_that_are_refused():
    d, f = adapted_desc(), gt.library().gtmoe_adapted_forward
    need = gt.adapted_workspace_bytes(d)
    good = [X, W, None, A, D, U, S, Y, WS]
    assert "context is null" in refused(f, C.byref(d), *good, need, None)
    assert "needs" in refused(f, C.byref(d), *good, need - 1, None)
    names = ["inputs", None, None, "adapters of the rows", "down", "up", "scales", "outputs", "workspace"]
    for i, name in enumerate(names):
        if name:
            args = list(good)
            args[i] = None
            assert name in refused(f, C.byref(d), *args, need, None)
    for i, what in ((1, "weights"), (2, "biases"), (3, "adapters"), (6, "scales"), (8, "workspace")):
        args = list(good)
        args[i] = (args[i] or A + GAP) + 1
        assert what in refused(f, C.byref(d), *args, need, None)
    # no shared product: outputs are added to
    assert "context is null" in refused(f, C.byref(d), X, None, None, A, D, U, S, Y, WS, need, None)
    for at in (X, W, A, D, U, S):
        args = list(good)
        args[7] = at
        assert "outputs overlap" in refused(f, C.byref(d), *args, need, None)
        args = list(good)
        args[8] = at
        assert "overlap" in refused(f, C.byref(d), *args, need, None)
    assert "context is null" in refused(f, C.byref(adapted_desc(rows=0)), *[None] * 9, 0, None)


def test_dropout_calls_that_are_refused():
    lib = gt.library()

    def desc(**changes):
        d = gt.dropout_desc(gt.VALUES_FLOAT32, 20, 30)
        for k, v in changes.items():
            setattr(d, k, v)
        return d

    def text(d, x, base, y, rate):
        return refused(lib.gtmoe_dropout, C.byref(d), x, base, y, rate, 1, 2, None)

    for rate in (-0.1, 1.0, 2.0, float("nan"), float("inf")):
        assert "rate must be" in text(desc(), X, None, Y, rate)
    assert "type of values" in text(desc(values=9), X, None, Y, 0.5)
    assert "rows must be" in text(desc(rows=-1), X, None, Y, 0.5)
    assert "columns must be" in text(desc(columns=0), X, None, Y, 0.5)
    assert "reserved" in text(desc(reserved=5), X, None, Y, 0.5)
    assert "base stride" in text(desc(base_stride=29), X, None, Y, 0.5)
    assert "inputs are null" in text(desc(), None, None, Y, 0.5)
    assert "outputs are null" in text(desc(), X, None, None, 0.5)
    assert "not aligned" in text(desc(), X + 2, None, Y, 0.5)
    # in place: the same address and stride only
    assert "context is null" in text(desc(), X, None, X, 0.5)
    assert "context is null" in text(desc(), X, Y, Y, 0.5)
    assert "overlap" in text(desc(), X, None, X + 4, 0.5)
    assert "overlap" in text(desc(output_stride=31), X, None, X, 0.5)
    assert "overlap" in text(desc(), X, Y + 4, Y, 0.5)
    assert "context is null" in text(desc(rows=0), None, None, None, 0.0)

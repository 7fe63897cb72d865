"""The operators of a block in plain rows on the GPU against plain 64-bit forms
(tests/plain_block.py): norm, products with an epilogue, activations and rows in 8
bits, the choice of experts.

Bounds.  U = 2^-24 is fp32's largest relative rounding error, H that of the output's
type (HALF_STEP) with HALF_LAST_STEP below its normal numbers.  A sum of n terms in
fp32 is off by at most (n + 1) U times the sum of their sizes.  exp, log1p and erfc
of the device's library are good to 16 units (2^-20) by its documentation; a
rounded argument x of an exponential adds |x| U.  The factors below add such terms up
and say how."""
import numpy as np
import pytest
import torch

import gotransformers_amd as gt
from tests import plain_block as plain
from tests.device_rows import SENTINEL, Rows, rounded, say, strides, stream
from tests.plain_rows import HALF_LAST_STEP, HALF_STEP, VALUES, offsets_of

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
CODES = {"int8": gt.CODES_INT8, "e4m3": gt.CODES_E4M3, "none": gt.CODES_NONE}
ACTS = {"none": gt.ACTIVATION_NONE, "relu": gt.ACTIVATION_RELU, "silu": gt.ACTIVATION_SILU, "gelu": gt.ACTIVATION_GELU,
        "gelu_tanh": gt.ACTIVATION_GELU_TANH}
KINDS = ["f32", "bf16", "f16"]


@pytest.fixture(scope="module")
def ctx():
    c = gt.Context(0)
    yield c
    c.close()


def near(got, want, error, kind):
    """got is want, off by `error` before one rounding to the type."""
    error = error + HALF_STEP[kind] * (np.abs(want) + error) + HALF_LAST_STEP[kind]
    off = np.abs(got - want)
    bad = ~(off <= error)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], error[bad][:5])


def workspace(n):
    return torch.full((n + 64,), 0xA5, dtype=torch.uint8, device="cuda")


def same_codes(got, want, codes):
    """Stored bytes against code values."""
    have = got.view(np.int8).astype(np.float64) if codes == "int8" else plain.e4m3_decode(got)
    assert np.array_equal(have, want)


# --------------------------------------------------------------------------
# rows in 8 bits
# --------------------------------------------------------------------------

def spread(rng, rows, columns, kind):
    """Values of many sizes, zeros, blocks of zeros, whole multiples (exact halves of a step)."""
    v = rng.normal(size=(rows, columns)) * 2.0 ** rng.integers(-12, 13, size=(rows, columns))
    v = np.where(rng.random(v.shape) < 0.1, 0.0, v)
    v[::5] = rng.integers(-254, 255, size=v[::5].shape) / 2.0  # max 127: scale 1, halves
    if rows > 3:
        v[3] = 0.0
        v[1, :16] = -v[1, 0]
    top = 60000.0 if kind == "f16" else 3e38
    return rounded(np.clip(v, -top, top), kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("scale_columns", [0, 16, 32, 64, 128])
@pytest.mark.parametrize("rows, columns, layout", [(1, 1, "packed"), (3, 7, "odd"), (9, 16, "packed"), (5, 129, "padded"),
                                                   (70, 200, "odd"), (33, 1201, "packed"), (600, 1024, "packed"),
                                                   (5, 2049, "odd"), (2, 5000, "packed"), (3, 70001, "odd")])
def test_packed_rows(ctx, kind, codes, scale_columns, rows, columns, layout):
    rng = np.random.default_rng(rows * 7919 + columns)
    v = spread(rng, rows, columns, kind)
    say(f"pack {kind} {codes} {scale_columns} {rows} x {columns} {layout}")
    st, sh = strides(columns, layout)
    x, out = Rows(kind, rows, columns, st, sh, v), Rows(kind, rows, columns, st, sh)
    q = Rows("u8", rows, columns, st, sh)
    n = -(-columns // scale_columns) if scale_columns else 1
    k = Rows("f32", rows, n, n + (0 if layout == "packed" else 5), 0)
    d = gt.packed_desc(VALUES[kind], rows, columns, CODES[codes], scale_columns, st, q.stride, k.stride)
    gt.pack_rows(ctx, d, x.ptr, q.ptr, k.ptr, stream())
    gt.unpack_rows(ctx, d, q.ptr, k.ptr, out.ptr, stream())
    torch.cuda.synchronize()
    want, scales = plain.packed(v, codes, scale_columns)
    assert np.array_equal(k.get(), scales)
    same_codes(q.get(), want, codes)
    # (code times scale in fp32, then to the type: the product has 31 bits)
    product = (want.astype(np.float32) * np.repeat(scales, scale_columns or columns, axis=1)[:, :columns].astype(np.float32))
    assert np.array_equal(out.get(), rounded(product, kind))
    for r in (q, k, out):
        r.check_outside()


def test_packed_rows_are_the_library_s_own_int8(ctx):
    rng = np.random.default_rng(3)
    v = rng.normal(size=(40, 200)).astype(np.float32)
    x, q, k = Rows("f32", 40, 200, data=v), Rows("u8", 40, 200), Rows("f32", 40, 13)
    d = gt.packed_desc(gt.VALUES_FLOAT32, 40, 200, gt.CODES_INT8, 16)
    gt.pack_rows(ctx, d, x.ptr, q.ptr, k.ptr, stream())
    rows = gt.encode_rows(gt.INT8, v.astype(np.float64))
    assert np.array_equal(q.get().view(np.int8), rows.values) and np.array_equal(k.get(), rows.scales)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_packed_tiny_and_largest_values(ctx, codes):
    """Scales that are subnormal or near the largest number."""
    rng = np.random.default_rng(5)
    v = np.zeros((8, 64), np.float32)
    for r, size in enumerate([1e-45, 3e-44, 1e-40, 1e-38, 1e-30, 1e30, 3e38, 2.0 ** -60]):
        v[r] = (rng.uniform(-1, 1, 64) * size).astype(np.float32)
    x, q, k, o = Rows("f32", 8, 64, data=v), Rows("u8", 8, 64), Rows("f32", 8, 4), Rows("f32", 8, 64)
    d = gt.packed_desc(gt.VALUES_FLOAT32, 8, 64, CODES[codes], 16)
    gt.pack_rows(ctx, d, x.ptr, q.ptr, k.ptr, stream())
    want, scales = plain.packed(v, codes, 16)
    assert np.array_equal(k.get(), scales)
    same_codes(q.get(), want, codes)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("scale_columns", [0, 32])
def test_packed_blocks_that_are_not_finite(ctx, codes, scale_columns):
    rng = np.random.default_rng(6)
    v = rng.normal(size=(6, 96))
    v[1, 40], v[2, 3], v[4, 95] = np.inf, np.nan, -np.inf
    x, q, o = Rows("bf16", 6, 96, data=v), Rows("u8", 6, 96), Rows("bf16", 6, 96)
    k = Rows("f32", 6, 3 if scale_columns else 1)
    d = gt.packed_desc(gt.VALUES_BFLOAT16, 6, 96, CODES[codes], scale_columns)
    gt.pack_rows(ctx, d, x.ptr, q.ptr, k.ptr, stream())
    gt.unpack_rows(ctx, d, q.ptr, k.ptr, o.ptr, stream())
    bad = np.zeros((6, 96), bool)
    for r, c in ((1, 40), (2, 3), (4, 95)):
        if scale_columns:
            bad[r, c // 32 * 32:c // 32 * 32 + 32] = True
        else:
            bad[r] = True
    assert np.array_equal(np.isnan(o.get()), bad) and np.array_equal(q.get()[bad], np.zeros(bad.sum()))
    want, scales = plain.packed(rounded(v, "bf16"), codes, scale_columns)
    assert np.array_equal(k.get(), scales, equal_nan=True)


# --------------------------------------------------------------------------
# norm
# --------------------------------------------------------------------------

NORM_SHAPES = [(1, 1), (2, 8), (37, 100), (600, 128), (5, 129), (600, 512), (3, 1000), (530, 1000), (517, 1201), (515, 2048),
               (1, 2048), (520, 2049), (3, 4096), (2, 8000), (2, 16384), (2, 40000), (2, 70001)]


def norm_error(s, w, epsilon):
    """Of y before its rounding: half of the sum of squares' (n + 1) U, sqrt and the division
    by n and by it, two products."""
    n = s.shape[1]
    y, _ = plain.norm(s, w, epsilon)
    return y, np.abs(y) * ((n + 1) / 2 + 8) * U


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows, columns", NORM_SHAPES)
@pytest.mark.parametrize("layout, residual, weights", [("packed", True, True), ("odd", False, False), ("padded", True, False),
                                                       ("packed", False, True)])
def test_norm_forward(ctx, kind, rows, columns, layout, residual, weights):
    rng = np.random.default_rng(rows * 31 + columns)
    st, sh = strides(columns, layout)
    say(f"norm {kind} {rows} x {columns} {layout} {residual} {weights}")
    x = Rows(kind, rows, columns, st, sh, rng.normal(size=(rows, columns)) * 3)
    b = Rows(kind, rows, columns, columns + 1, 0, rng.normal(size=(rows, columns))) if residual else None
    w = Rows(kind, 1, columns, columns, sh, rng.normal(size=(1, columns)) + 1) if weights else None
    s, y = Rows(kind, rows, columns, st, sh), Rows(kind, rows, columns, columns + 2, 0)
    d = gt.norm_desc(VALUES[kind], rows, columns, 1e-5, input_stride=st, residual_stride=columns + 1, sum_stride=st,
                     output_stride=columns + 2)
    gt.norm_forward(ctx, d, x.ptr, b.ptr if b else None, w.ptr if w else None, s.ptr if residual else None, y.ptr, None, None,
                    stream())
    torch.cuda.synchronize()
    total = x.get()
    if residual:
        # the sum of two values of the type, in fp32, then to the type
        total = rounded((x.view.float() + b.view.float()).cpu().numpy(), kind)
        assert np.array_equal(s.get(), total)
        s.check_outside()
    want, error = norm_error(total, w.get() if w else None, 1e-5)
    near(y.get(), want, error, kind)
    y.check_outside()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("rows, columns, scale_columns", [(1, 2048, 128), (5, 100, 0), (530, 1000, 32), (3, 4096, 0), (600, 128, 16),
                                                          (2, 70001, 0), (2, 70001, 64), (517, 2048, 64)])
def test_norm_into_8_bits(ctx, kind, codes, rows, columns, scale_columns):
    rng = np.random.default_rng(rows + columns)
    x = Rows(kind, rows, columns, columns + 1, 1, rng.normal(size=(rows, columns)) * 3)
    w = Rows(kind, 1, columns, data=rng.normal(size=(1, columns)) + 1)
    n = -(-columns // scale_columns) if scale_columns else 1
    q, k, y = Rows("u8", rows, columns, columns + 3, 1), Rows("f32", rows, n, n + 2), Rows(kind, rows, columns)
    d = gt.norm_desc(VALUES[kind], rows, columns, 1e-6, CODES[codes], scale_columns, input_stride=columns + 1,
                     code_stride=columns + 3, scale_stride=n + 2)
    gt.norm_forward(ctx, d, x.ptr, None, w.ptr, None, y.ptr, q.ptr, k.ptr, stream())
    torch.cuda.synchronize()
    want, error = norm_error(x.get(), w.get(), 1e-6)
    near(y.get(), want, error, kind)
    most = np.repeat(plain.packed(want, codes, scale_columns)[1], scale_columns or columns, axis=1)[:, :columns]
    top = 127 if codes == "int8" else 448
    rel = float((error / np.maximum(np.abs(want), 1e-300)).max())
    assert np.all(np.abs(np.repeat(k.get(), scale_columns or columns, axis=1)[:, :columns] - most) <= most * (rel + 2 * U))
    # a code is half a step off at most: of the block's scale, or, e4m3, of the value, not below its last step
    have = q.get()
    have = have.view(np.int8).astype(np.float64) if codes == "int8" else plain.e4m3_decode(have)
    back = have * most
    step = 0.5 * most if codes == "int8" else np.maximum(np.abs(want) * 2.0 ** -4, most * 2.0 ** -10)
    assert np.all(np.abs(back - want) <= step + 4 * (error + most * top * (rel + 4 * U)))
    q.check_outside()
    k.check_outside()
    # without outputs the codes are the same
    q2, k2 = Rows("u8", rows, columns, columns + 3, 1), Rows("f32", rows, n, n + 2)
    gt.norm_forward(ctx, d, x.ptr, None, w.ptr, None, None, q2.ptr, k2.ptr, stream())
    assert bool((q.buffer == q2.buffer).all()) and bool((k.buffer == k2.buffer).all())


@pytest.mark.parametrize("columns", [100, 1201, 4096, 70001])
def test_norm_squares_beyond_fp32(ctx, columns):
    rng = np.random.default_rng(columns)
    v = rng.normal(size=(5, columns)) * np.array([1e25, 1e-25, 1e30, 0.0, 1.0])[:, None]
    x, y = Rows("f32", 5, columns, data=v), Rows("f32", 5, columns)
    for epsilon in (0.0, 1e-6):
        d = gt.norm_desc(gt.VALUES_FLOAT32, 5, columns, epsilon)
        gt.norm_forward(ctx, d, x.ptr, None, None, None, y.ptr, None, None, stream())
        with np.errstate(invalid="ignore", divide="ignore"):
            want, error = norm_error(x.get(), None, epsilon)
        got = y.get()
        rows = [0, 1, 2, 4] if epsilon == 0.0 else [0, 1, 2, 3, 4]
        near(got[rows], want[rows], error[rows], "f32")


def test_norm_in_place_and_rows_apart(ctx):
    """sums over the residuals; a row that is not finite changes no other."""
    rng = np.random.default_rng(9)
    v, r = rng.normal(size=(700, 300)), rng.normal(size=(700, 300))
    v[17, 5], v[400, 299] = np.inf, np.nan
    x, b, y = Rows("bf16", 700, 300, data=v), Rows("bf16", 700, 300, data=r), Rows("bf16", 700, 300)
    total = rounded((x.view.float() + b.view.float()).cpu().numpy(), "bf16")
    d = gt.norm_desc(gt.VALUES_BFLOAT16, 700, 300)
    gt.norm_forward(ctx, d, x.ptr, b.ptr, None, b.ptr, y.ptr, None, None, stream())
    assert np.array_equal(b.get(), total, equal_nan=True)
    rows = np.setdiff1d(np.arange(700), [17, 400])
    want, error = norm_error(total[rows], None, 1e-6)
    near(y.get()[rows], want, error, "bf16")
    assert np.isnan(y.get()[17, 5]) and np.isnan(y.get()[400]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows, columns", NORM_SHAPES + [(5000, 256)])
@pytest.mark.parametrize("layout, past, weights, gradient", [("packed", True, True, "f32"), ("odd", False, True, "same"),
                                                             ("padded", True, False, "same")])
def test_norm_gradient(ctx, kind, rows, columns, layout, past, weights, gradient):
    rng = np.random.default_rng(rows * 17 + columns)
    st, sh = strides(columns, layout)
    say(f"norm gradient {kind} {rows} x {columns} {layout} {past} {weights} {gradient}")
    s = Rows(kind, rows, columns, st, sh, rng.normal(size=(rows, columns)) * 2)
    dy = Rows(kind, rows, columns, columns + 1, 0, rng.normal(size=(rows, columns)))
    ds = Rows(kind, rows, columns, st, sh, rng.normal(size=(rows, columns))) if past else None
    w = Rows(kind, 1, columns, data=rng.normal(size=(1, columns)) + 1) if weights else None
    dx = Rows(kind, rows, columns, columns + 2, 0)
    gkind = "f32" if gradient == "f32" else kind
    dw = Rows(gkind, 1, columns)
    d = gt.norm_desc(VALUES[kind], rows, columns, 1e-5, input_stride=columns + 2, sum_stride=st, output_stride=columns + 1)
    ws = workspace(gt.norm_workspace_bytes(d))

    def call(accumulate):
        gt.norm_gradient(ctx, d, dy.ptr, s.ptr, w.ptr if w else None, ds.ptr if ds else None, dx.ptr, dw.ptr, VALUES[gkind],
                         accumulate, ws.data_ptr(), stream())
        torch.cuda.synchronize()

    call(False)
    rdx, rdw, xsize, wsize = plain.norm_gradient(dy.get(), s.get(), w.get() if w else None, ds.get() if ds else None, 1e-5)
    # the inverse size as in norm_error, the mean of n products, a few more
    near(dx.get(), rdx, xsize * (2 * columns + 24) * U, kind)
    near(dw.get()[0], rdw, wsize * (rows + columns / 2 + 16) * U, gkind)
    dx.check_outside()
    dw.check_outside()
    assert bool((ws[-64:] == 0xA5).all())
    first = dw.get()[0]
    again = dw.buffer.clone()
    call(False)
    assert bool((dw.buffer == again).all()), "the same call gives the same bits"
    call(True)
    near(dw.get()[0], first + rdw, wsize * (rows + columns / 2 + 16) * U + np.abs(first) * U, gkind)
    # without weight gradients: the same input gradients, no workspace
    dx2 = Rows(kind, rows, columns, columns + 2, 0)
    gt.norm_gradient(ctx, d, dy.ptr, s.ptr, w.ptr if w else None, ds.ptr if ds else None, dx2.ptr, None, 0, False, None,
                     stream(), 0)
    near(dx2.get(), rdx, xsize * (2 * columns + 24) * U, kind)


def test_norm_gradient_against_differences(ctx):
    rng = np.random.default_rng(4)
    s, w, dy = rng.normal(size=(3, 50)), rng.normal(size=50), rng.normal(size=(3, 50))
    hs, hdy, hw = Rows("f32", 3, 50, data=s), Rows("f32", 3, 50, data=dy), Rows("f32", 1, 50, data=w[None])
    dx, dw = Rows("f32", 3, 50), Rows("f32", 1, 50)
    d = gt.norm_desc(gt.VALUES_FLOAT32, 3, 50, 1e-3)
    ws = workspace(gt.norm_workspace_bytes(d))
    gt.norm_gradient(ctx, d, hdy.ptr, hs.ptr, hw.ptr, None, dx.ptr, dw.ptr, 0, False, ws.data_ptr(), stream())
    s, w, dy = hs.get(), hw.get()[0], hdy.get()
    f = lambda s_, w_: float((plain.norm(s_, w_, 1e-3)[0] * dy).sum())
    for r, c in ((0, 0), (1, 17), (2, 49)):
        e = np.zeros_like(s)
        e[r, c] = 1e-5  # the difference quotient is off by h^2 times a third derivative, below 1e-8 here
        assert abs((f(s + e, w) - f(s - e, w)) / 2e-5 - dx.get()[r, c]) < 1e-5
    for c in (0, 49):
        e = np.zeros_like(w)
        e[c] = 0.5
        assert abs(f(s, w + e) - f(s, w - e) - dw.get()[0, c]) < 1e-5


def test_norm_gradient_without_rows(ctx):
    d = gt.norm_desc(gt.VALUES_BFLOAT16, 0, 40)
    dw = Rows("f32", 1, 40)
    gt.norm_gradient(ctx, d, None, None, None, None, None, dw.ptr, 0, True, None, stream())
    assert np.all(dw.get() == SENTINEL)
    gt.norm_gradient(ctx, d, None, None, None, None, None, dw.ptr, 0, False, None, stream())
    assert np.all(dw.get() == 0)
    dw.check_outside()


# --------------------------------------------------------------------------
# activations
# --------------------------------------------------------------------------

def act_error(z, name):
    """Relative to act(z) and to the sizes of act' 's terms: the library's function (2^-20 each of
    two; GELU's own polynomial is good to 4e-8 and its ten roundings, 2^-20), and the rounded argument of an exponential: |z| for SiLU, twice z^2 for GELU (of
    erfc about 2 x^2 = z^2 per relative error of its argument), for its tanh form 2 |u|, four roundings."""
    if name in ("none", "relu"):
        return np.zeros_like(z)
    if name == "silu":
        return 2.0 ** -19 + np.abs(z) * U
    if name == "gelu":
        return 2.0 ** -19 + 3 * z * z * U
    return 2.0 ** -19 + 8 * np.abs(1.6 * (z + 0.044715 * z ** 3)) * U


def act_last_steps(z, name):
    """Absolutely, besides: a factor s of act(z) below 2^-126 may be 0.  act(z) is z s, and act' is s + z s
    (1 - s) d (GELU: z e / 2.5) with d = 1, for GELU's tanh form the slope of its argument."""
    d = 1.6 * (1 + 3 * 0.044715 * z * z) if name == "gelu_tanh" else 1.0
    return (np.abs(z) * d + 1) * 2.0 ** -126


def z_values(rng, rows, columns):
    """From the middle to where the tails end (e^-80 is a normal number of fp32)."""
    z = rng.normal(size=(rows, columns)) * rng.choice([0.01, 1.0, 4.0], size=(rows, columns))
    return np.where(rng.random(z.shape) < 0.02, 0.0, z)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("codes, scale_columns", [("none", 0), ("int8", 16), ("int8", 128), ("e4m3", 32), ("e4m3", 64)])
@pytest.mark.parametrize("rows, columns, layout, gate_only, limit", [
    (1, 1, "packed", False, 0.0), (33, 1201, "odd", False, 2.0), (64, 256, "packed", True, 0.0), (7, 200, "padded", True, 1.5)])
def test_activation(ctx, kind, act, codes, scale_columns, rows, columns, layout, gate_only, limit):
    rng = np.random.default_rng(rows + columns)
    say(f"activation {kind} {act} {codes} {scale_columns} {rows} x {columns} {layout} {gate_only} {limit}")
    st, sh = strides(columns, layout)
    g = Rows(kind, rows, columns, st, sh, z_values(rng, rows, columns))
    u = None if gate_only else Rows(kind, rows, columns, columns + 1, 0, rng.normal(size=(rows, columns)) * 2)
    dy = Rows(kind, rows, columns, columns + 2, 1, rng.normal(size=(rows, columns)))
    y, again = Rows(kind, rows, columns, columns + 2, 1), Rows(kind, rows, columns, columns + 2, 1)
    n = -(-columns // scale_columns) if scale_columns else 1
    kept = [(Rows("u8", rows, columns, columns + 3, 1), Rows("f32", rows, n, n + 1)) for _ in range(2)]
    dg, du = Rows(kind, rows, columns, st, sh), Rows(kind, rows, columns, columns + 1, 0)
    d = gt.activation_desc(VALUES[kind], rows, columns, ACTS[act], limit, CODES[codes], scale_columns, st, columns + 1,
                           columns + 2, columns + 3, n + 1)
    coded = codes != "none"
    p = lambda r: None if r is None else r.ptr
    gt.activation_forward(ctx, d, g.ptr, p(u), y.ptr, *([kept[0][0].ptr, kept[0][1].ptr] if coded else [None, None]),
                          *([kept[1][0].ptr, kept[1][1].ptr] if coded and u else [None, None]), stream())
    if coded:
        gt.activation_gradient(ctx, d, dy.ptr, kept[0][0].ptr, kept[0][1].ptr, kept[1][0].ptr if u else None,
                               kept[1][1].ptr if u else None, dg.ptr, du.ptr if u else None, again.ptr, stream())
    else:
        gt.activation_gradient(ctx, d, dy.ptr, g.ptr, None, p(u), None, dg.ptr, du.ptr if u else None, again.ptr, stream())
    torch.cuda.synchronize()

    def check(out, gate, up):
        a, c, da, dc, size = plain.gated(gate, up, act, limit)
        z = np.minimum(gate, limit or np.inf)
        e = act_error(z, act)
        near(out.get(), a * c, np.abs(a * c) * (e + 2 * U) + np.abs(c) * act_last_steps(z, act), kind)
        return a, c, da, dc, size, e

    check(y, g.get(), u.get() if u else None)
    gv, uv = g.get(), u.get() if u else None
    if coded:
        for (q, k), v in zip(kept, [gv, uv]):
            if v is not None:
                want, scales = plain.packed(v, codes, scale_columns)
                assert np.array_equal(k.get(), scales)
                same_codes(q.get(), want, codes)
                q.check_outside()
                k.check_outside()
        # what the gradient reads: code times scale in fp32
        gv, uv = [None if v is None else plain.unpacked(*plain.packed(v, codes, scale_columns), scale_columns)
                  .astype(np.float32).astype(np.float64) for v in (gv, uv)]
    a, c, da, dc, size, e = check(again, gv, uv)
    dyv = dy.get()
    inside = gv <= (limit or np.inf)
    near(dg.get(), dyv * c * da, np.abs(dyv * c) * inside * (size * (2 * e + 4 * U) + act_last_steps(gv, act)), kind)
    if u:
        near(du.get(), dyv * a * dc, np.abs(dyv * dc) * (np.abs(a) * (e + 2 * U) + act_last_steps(gv, act)), kind)
        du.check_outside()
    for r in (y, again, dg):
        r.check_outside()


def test_activation_gradient_against_differences(ctx):
    rng = np.random.default_rng(8)
    for act in ("silu", "gelu", "gelu_tanh"):
        g, u, dy = (Rows("f32", 4, 40, data=rng.normal(size=(4, 40)) * 2) for _ in range(3))
        dg, du = Rows("f32", 4, 40), Rows("f32", 4, 40)
        d = gt.activation_desc(0, 4, 40, ACTS[act])
        gt.activation_gradient(ctx, d, dy.ptr, g.ptr, None, u.ptr, None, dg.ptr, du.ptr, None, stream())
        h = 1e-5
        f = lambda z: plain.activation(z, act)[0]
        slope = (f(g.get() + h) - f(g.get() - h)) / (2 * h)  # off by h^2 and 1e-16 / h
        assert np.all(np.abs(dy.get() * u.get() * slope - dg.get()) <= 1e-5 * (1 + np.abs(dg.get())))
        assert np.all(np.abs(dy.get() * f(g.get()) - du.get()) <= 1e-5 * (1 + np.abs(du.get())))


@pytest.mark.parametrize("act", list(ACTS))
def test_activation_of_values_that_are_not_finite(ctx, act):
    v = np.ones((2, 64))
    v[0, 3], v[0, 9], v[1, 40] = np.nan, np.inf, -np.inf
    g, u, y, dg = Rows("f32", 2, 64, data=v), Rows("f32", 2, 64, data=np.ones((2, 64))), Rows("f32", 2, 64), Rows("f32", 2, 64)
    d = gt.activation_desc(0, 2, 64, ACTS[act])
    gt.activation_forward(ctx, d, g.ptr, u.ptr, y.ptr, stream=stream())
    gt.activation_gradient(ctx, d, u.ptr, g.ptr, None, u.ptr, None, dg.ptr, None, None, stream())
    got, grad = y.get(), dg.get()
    finite = np.isfinite(v)
    # (act' of a straight line is 1 everywhere)
    assert np.isnan(got[0, 3]) and got[0, 9] == np.inf and (act == "none" or np.isnan(grad[0, 3]))
    assert np.all(got[finite] == got[0, 0]) and np.all(grad[finite] == grad[0, 0])
    # with a limit a NaN stays one and infinities are held
    d = gt.activation_desc(0, 2, 64, ACTS[act], 3.0)
    gt.activation_forward(ctx, d, g.ptr, g.ptr, y.ptr, stream=stream())
    got = y.get()
    a = plain.activation(np.array([3.0]), act)[0][0]
    assert np.isnan(got[0, 3]) and abs(got[0, 9] - 3 * a) < 1e-5


def test_activation_in_place(ctx):
    rng = np.random.default_rng(2)
    gv, uv, dv = (rng.normal(size=(50, 96)) for _ in range(3))
    d = gt.activation_desc(gt.VALUES_BFLOAT16, 50, 96, gt.ACTIVATION_SILU)
    g, u, dy = (Rows("bf16", 50, 96, data=v) for v in (gv, uv, dv))
    outs = [Rows("bf16", 50, 96) for _ in range(3)]
    gt.activation_gradient(ctx, d, dy.ptr, g.ptr, None, u.ptr, None, *[o.ptr for o in outs], stream())
    gt.activation_gradient(ctx, d, dy.ptr, g.ptr, None, u.ptr, None, g.ptr, u.ptr, dy.ptr, stream())
    for have, want in zip((g, u, dy), outs):
        assert bool((have.view == want.view).all())


# --------------------------------------------------------------------------
# products with an epilogue
# --------------------------------------------------------------------------

SIZES = {
    "one": ([1], 0),
    "dense few": ([32], 0),
    "dense": ([300], 0),
    "empty and single": ([0, 1, 0, 0, 2, 0], 3),
    "all empty": ([0, 0, 0], 2),
    "ragged": ([5, 0, 130, 17, 64, 1, 129, 33], 1),
    "large": ([700, 0, 900, 1], 1),
    "many groups": ([1, 0, 2] * 50, 0),
}
WIDTHS = [(1, 1), (7, 5), (64, 64), (72, 136), (129, 130), (256, 512)]
PARTS = ["", "b", "f", "r", "p", "bfrp"]


def whole(rng, *shape, top=2):
    return rng.integers(-top, top + 1, size=shape).astype(np.float64)


class Product:
    def __init__(self, kind, sizes, widths, layout, parts, act, make, whole_rows=False):
        part_sizes, first = sizes
        K, N = widths
        off = offsets_of(part_sizes, 0 if whole_rows else first)
        self.off, G = off, len(part_sizes)
        R = int(off[-1]) + (0 if whole_rows else 2)
        rng = np.random.default_rng(R * 31 + K * 7 + N)
        pad = lambda w: strides(w, layout)
        self.x = Rows(kind, R, K, *pad(K), make(rng, R, K))
        ws, wsh = pad(K)
        gs = N * ws + (0 if layout == "packed" else 8 if layout == "padded" else 5)
        self.w = make(rng, G, N, K) * 0.5 ** 2
        hold = torch.full((wsh + G * gs + 8,), 77.0, dtype=self.x.buffer.dtype, device="cuda")
        self.wview = torch.as_strided(hold, (G, N, K), (gs, ws, 1), wsh)
        self.wview.copy_(torch.as_tensor(self.w).to(hold.dtype))
        self.w = self.wview.double().cpu().numpy()
        self.b = Rows(kind, G, N, N + (1 if layout == "odd" else 0), 0, make(rng, G, N)) if "b" in parts else None
        self.f = Rows(kind, R, N, *pad(N), make(rng, R, N)) if "f" in parts else None
        self.r = Rows(kind, R, N, N + 3, 1, make(rng, R, N)) if "r" in parts else None
        self.z = Rows(kind, R, N, *pad(N)) if "p" in parts else None
        self.y = Rows(kind, R, N, *pad(N))
        self.dev = None if whole_rows else torch.from_numpy(off).cuda()
        self.d = gt.grouped_desc(VALUES[kind], G, R, K, N, self.x.stride, self.y.stride, ws, gs)
        p = lambda r: None if r is None else r.ptr
        s = lambda r: 0 if r is None else r.stride
        self.e = gt.epilogue(ACTS[act], p(self.b), p(self.f), p(self.r), p(self.z), N, s(self.b) or N, s(self.f), s(self.r), s(self.z))
        self.K, self.N, self.G, self.R, self.act, self.kind = K, N, G, R, act, kind

    def call(self, ctx, out=None):
        gt.grouped_fused_forward(ctx, self.d, self.e, None if self.dev is None else self.dev.data_ptr(), self.x.ptr,
                                 self.wview.data_ptr(), (out or self.y).ptr, stream())
        torch.cuda.synchronize()

    def reference(self):
        z, size = np.zeros((self.R, self.N)), np.zeros((self.R, self.N))
        x = self.x.get()
        for g in range(self.G):
            at = slice(self.off[g], self.off[g + 1])
            z[at], size[at] = x[at] @ self.w[g].T, np.abs(x[at]) @ np.abs(self.w[g]).T
            if self.b:
                z[at], size[at] = z[at] + self.b.get()[g], size[at] + np.abs(self.b.get()[g])
        a, da, _ = plain.activation(z, self.act)
        y = a * self.f.get() if self.f else a
        return z, size, a, y + self.r.get() if self.r else y

    def untouched(self, got):
        off = self.off
        return np.all(got[:off[0]] == SENTINEL) and np.all(got[off[-1]:] == SENTINEL)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("widths", WIDTHS)
@pytest.mark.parametrize("parts, act, layout", [("", "none", "packed"), ("b", "relu", "odd"), ("bfrp", "relu", "packed"),
                                                ("fr", "none", "padded"), ("p", "relu", "packed")])
def test_fused_product_of_whole_numbers(ctx, kind, sizes, widths, parts, act, layout):
    # |z| <= 4 * 512 / 4 + 2, times 2, plus 2, in quarters: exact in fp32, one rounding to the type
    p = Product(kind, SIZES[sizes], widths, layout, parts, act, whole)
    say(f"fused {kind} {sizes} {widths} {parts} {act} {layout}")
    p.call(ctx)
    z, _, _, y = p.reference()
    for have, want in ((p.y, y), (p.z, z)):
        if have is not None:
            got = have.get()
            inside = slice(p.off[0], p.off[-1])
            assert np.array_equal(got[inside], rounded(want, kind)[inside]) and p.untouched(got)
            have.check_outside()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("sizes, widths", [("dense few", (256, 512)), ("ragged", (129, 130)), ("large", (256, 512)), ("dense", (72, 136))])
def test_fused_product_activations(ctx, kind, act, sizes, widths):
    normal = lambda rng, *shape: rng.normal(size=shape)
    p = Product(kind, SIZES[sizes], widths, "packed", "bfrp", act, normal)
    p.call(ctx)
    z, size, a, y = p.reference()
    inside = slice(p.off[0], p.off[-1])
    ez = size * (p.K + 2) * U
    f = np.abs(p.f.get())
    # |act'| is at most 1.13 (GELU; SiLU 1.1); the activation's own error at z moved by ez
    ea = 1.13 * ez + np.abs(a) * (act_error(np.abs(z) + 1, act) + 4 * U) + 1e-30
    near(p.z.get()[inside], z[inside], ez[inside], kind)
    near(p.y.get()[inside], y[inside], (ea * f + (np.abs(a) * f + np.abs(p.r.get())) * 2 * U)[inside], kind)


@pytest.mark.parametrize("kind", KINDS)
def test_fused_product_of_all_rows_and_in_place(ctx, kind):
    for sizes in ([40], [3000]):
        p = Product(kind, (sizes, 0), (64, 96), "packed", "bfr", "relu", whole, whole_rows=True)
        p.call(ctx)
        want = p.y.get()
        assert np.array_equal(want, rounded(p.reference()[3], kind))
        # onto the residual itself
        y = Rows(kind, p.R, p.N, p.N, 0, p.r.get())
        p.e.residuals, p.e.residual_stride = y.ptr, p.N
        p.call(ctx, y)
        assert np.array_equal(y.get(), want)


def test_fused_product_offsets_out_of_order_stay_inside(ctx):
    """Offsets that descend or leave the rows: nothing but the rows is written."""
    for kind in ("bf16", "f32"):
        p = Product(kind, ([60, 50, 40], 0), (64, 64), "packed", "bfrp", "relu", whole)
        p.dev.copy_(torch.tensor([120, 20, 500, -7], dtype=torch.int32))
        p.call(ctx)
        p.y.check_outside()
        p.z.check_outside()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sizes", [([1], 0), ([300], 0), ([0, 0], 3), ([5, 0, 130, 17, 64, 1, 129, 33], 1), ([4000, 3, 9000], 0),
                                   ([1, 0, 2] * 50, 0)])
@pytest.mark.parametrize("columns, layout", [(1, "packed"), (130, "odd"), (600, "padded")])
def test_bias_gradient(ctx, kind, sizes, columns, layout):
    off = offsets_of(*sizes)
    R, G = int(off[-1]) + 2, len(sizes[0])
    rng = np.random.default_rng(R + columns)
    dy = Rows(kind, R, columns, *strides(columns, layout), rng.normal(size=(R, columns)))
    say(f"bias gradient {kind} {sizes} {columns} {layout}")
    dev = torch.from_numpy(off).cuda()
    d = gt.grouped_desc(VALUES[kind], G, R, 8, columns, output_stride=dy.stride)
    ws = workspace(gt.grouped_bias_workspace_bytes(d))
    v = dy.get()
    want = np.stack([v[off[g]:off[g + 1]].sum(axis=0) for g in range(G)])
    size = np.stack([np.abs(v[off[g]:off[g + 1]]).sum(axis=0) for g in range(G)])
    count = np.diff(off)[:, None]
    for gkind in {kind, "f32"}:
        db = Rows(gkind, G, columns)
        call = lambda add: gt.grouped_bias_gradient(ctx, d, dev.data_ptr(), dy.ptr, db.ptr, VALUES[gkind], add, ws.data_ptr(), stream())
        call(False)
        first = db.get()
        near(first, want, size * (count + 1) * U, gkind)
        db.check_outside()
        call(True)
        near(db.get(), first + want, size * (count + 1) * U + np.abs(first) * U, gkind)
    assert bool((ws[-64:] == 0xA5).all())
    if G == 1 and off[0] == 0:
        whole_rows = Rows("f32", 1, columns)
        gt.grouped_bias_gradient(ctx, d, None, dy.ptr, whole_rows.ptr, 0, False, ws.data_ptr(), stream())
        near(whole_rows.get()[0], v.sum(axis=0), np.abs(v).sum(axis=0) * (R + 1) * U, "f32")


# --------------------------------------------------------------------------
# the choice of experts
# --------------------------------------------------------------------------

ROUTES = [  # tokens, experts, k, groups, chosen groups, best
    (1, 1, 1, 1, 1, 1), (3, 2, 2, 1, 1, 1), (5, 8, 8, 1, 1, 1), (17, 14, 3, 1, 1, 1), (64, 16, 2, 4, 2, 1), (65, 64, 6, 1, 1, 1),
    (128, 64, 4, 8, 3, 2), (129, 128, 8, 8, 4, 2), (300, 60, 5, 5, 2, 2), (257, 256, 8, 8, 4, 1), (1000, 128, 8, 1, 1, 1),
    (70, 300, 32, 1, 1, 1), (40, 512, 20, 64, 16, 2), (33, 1000, 17, 1, 1, 1), (20, 1024, 32, 4, 1, 2), (4097, 24, 3, 3, 3, 1),
    (64, 32, 32, 2, 2, 1), (2000, 16, 16, 1, 1, 1)]


def check_route(ctx, kind, l, biases, k, scores, groups=1, chosen_groups=1, best=1, renormalize=True, scale=1.0, layout="packed",
                gradient=True):
    T, E = l.shape
    st, sh = strides(E, layout)
    logits = Rows(kind, T, E, st, sh, l)
    l = logits.get()
    b = None if biases is None else torch.as_tensor(biases, dtype=torch.float32).cuda()
    bv = None if b is None else b.double().cpu().numpy()
    d = gt.route_desc(VALUES[kind], T, E, k, groups, chosen_groups, best, gt.SCORES_SIGMOID if scores == "sigmoid" else gt.SCORES_SOFTMAX,
                      renormalize, scale, st)
    ws = workspace(gt.route_workspace_bytes(d))
    chosen, gates = Rows("i32", T, k), Rows("f32", T, k)
    offsets, rows, places = Rows("i32", 1, E + 1), Rows("i32", 1, T * k), Rows("i32", T, k)
    gt.route_forward(ctx, d, logits.ptr, None if b is None else b.data_ptr(), chosen.ptr, gates.ptr, offsets.ptr, rows.ptr, places.ptr,
                     ws.data_ptr(), stream())
    torch.cuda.synchronize()
    want, wgates = plain.route(l, bv, k, scores, groups, chosen_groups, best, renormalize, scale)
    assert np.array_equal(chosen.get(), want)
    # each score: exp or the logistic function and its argument's rounding, of up to E summed (k with
    # renormalize); one below 2^-126 is good to 16 steps of 2^-149
    near(gates.get(), wgates, np.abs(wgates) * (2.0 ** -18 + (E + 100) * U) + scale * 2.0 ** -145, "f32")
    for have, ref in zip((offsets, rows, places), plain.lists(want, E)):
        assert np.array_equal(have.get().reshape(-1), np.asarray(ref).reshape(-1))
    for r in (chosen, gates, offsets, rows, places):
        r.check_outside()
    assert bool((ws[-64:] == 0xA5).all())
    # without the lists, the same choice and gates
    c2, g2 = Rows("i32", T, k), Rows("f32", T, k)
    gt.route_forward(ctx, d, logits.ptr, None if b is None else b.data_ptr(), c2.ptr, g2.ptr, None, None, None, None, stream())
    assert bool((c2.buffer == chosen.buffer).all()) and bool((g2.buffer == gates.buffer).all())
    if gradient:
        rng = np.random.default_rng(T)
        dg = Rows("f32", T, k, data=rng.normal(size=(T, k)))
        dl = Rows(kind, T, E, st, sh)
        gt.route_gradient(ctx, d, logits.ptr, chosen.ptr, dg.ptr, dl.ptr, stream())
        ref, size = plain.route_gradient(l, want, dg.get(), scores, renormalize, scale)
        near(dl.get(), ref, size * (2.0 ** -17 + (E + 100) * U) + 1e-36, kind)
        dl.check_outside()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", ROUTES)
@pytest.mark.parametrize("scores, biased, renormalize, layout", [("softmax", False, True, "packed"), ("softmax", True, False, "odd"),
                                                                 ("sigmoid", True, True, "packed"), ("sigmoid", False, False, "padded")])
def test_route(ctx, kind, shape, scores, biased, renormalize, layout):
    T, E, k, groups, chosen_groups, best = shape
    rng = np.random.default_rng(T * 13 + E)
    say(f"route {kind} {shape} {scores} {biased} {renormalize} {layout}")
    l = rng.normal(size=(T, E)) * 2
    check_route(ctx, kind, l, rng.normal(size=E) * 0.1 if biased else None, k, scores, groups, chosen_groups, best, renormalize, 2.5,
                layout)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_route_ties_go_to_the_lowest_index(ctx, scores, biased):
    rng = np.random.default_rng(1)
    for T, E, k, groups, chosen_groups, best in ((50, 64, 6, 1, 1, 1), (300, 128, 8, 8, 4, 2), (40, 256, 8, 8, 4, 1), (9, 600, 20, 1, 1, 1)):
        l = rng.integers(-1, 2, size=(T, E)).astype(np.float64)
        l[0] = 0.0
        l[1] = np.where(np.arange(E) % 2, 0.0, -0.0)
        b = rng.integers(0, 2, size=E) * 0.25 if biased else None
        check_route(ctx, "f32", l, b, k, scores, groups, chosen_groups, best)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("renormalize", [False, True])
def test_route_masks(ctx, scores, biased, renormalize):
    """Masked by -inf or by the type's lowest value, rows that leave fewer than k or nothing."""
    rng = np.random.default_rng(2)
    for kind, low in (("f32", -3.4028234663852886e38), ("bf16", -3.3895313892515355e38), ("f16", -65504.0)):
        for T, E, k, groups, chosen_groups, best in ((20, 16, 4, 1, 1, 1), (150, 64, 6, 8, 3, 2), (20, 600, 9, 1, 1, 1)):
            l = rng.normal(size=(T, E))
            l[rng.random((T, E)) < 0.7] = -np.inf
            l[0] = -np.inf
            l[1] = -np.inf
            l[1, 5] = 1.0
            l[2, ::3] = low
            l[3] = low
            l[4] = np.where(np.arange(E) < E // 2, low, -np.inf)
            check_route(ctx, kind, l, rng.normal(size=E) * 0.3 if biased else None, k, scores, groups, chosen_groups, best, renormalize)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_far_logits(ctx, scores):
    """Logits whose scores under- or overflow a plain quotient."""
    rng = np.random.default_rng(3)
    l = rng.normal(size=(60, 32)) * np.repeat([1.0, 30.0, 80.0], 20)[:, None] + np.repeat([0.0, -60.0, 300.0, -300.0], 15)[:, None]
    check_route(ctx, "f32", l, None, 4, scores, renormalize=True)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_of_what_is_not_finite(ctx, scores):
    """Choices stay experts of the range, each once; other tokens' are as they were."""
    rng = np.random.default_rng(4)
    for biased in (False, True):
        l = rng.normal(size=(200, 64))
        clean = Rows("f32", 200, 64, data=l)
        l[7, 3], l[9, 60], l[11] = np.nan, np.inf, np.nan
        dirty = Rows("f32", 200, 64, data=l)
        b = torch.randn(64, device="cuda") * 0.1 if biased else None
        d = gt.route_desc(0, 200, 64, 6, 8, 4, 2, gt.SCORES_SIGMOID if scores == "sigmoid" else gt.SCORES_SOFTMAX)
        got = []
        for x in (clean, dirty):
            chosen, gates, off = Rows("i32", 200, 6), Rows("f32", 200, 6), Rows("i32", 1, 65)
            ws = workspace(gt.route_workspace_bytes(d))
            gt.route_forward(ctx, d, x.ptr, None if b is None else b.data_ptr(), chosen.ptr, gates.ptr, off.ptr, None, None, ws.data_ptr(),
                             stream())
            got.append((chosen.get(), gates.get(), off.get()))
        rows = np.setdiff1d(np.arange(200), [7, 9, 11])
        for i in range(2):
            assert np.array_equal(got[0][i][rows], got[1][i][rows])
        for t in (7, 9, 11):
            c = got[1][0][t]
            assert len(set(c.tolist())) == 6 and c.min() >= 0 and c.max() < 64
        assert got[1][2][0, -1] == 1200


def test_route_without_tokens(ctx):
    d = gt.route_desc(0, 0, 40, 4)
    off = Rows("i32", 1, 41)
    gt.route_forward(ctx, d, None, None, None, None, off.ptr, None, None, None, stream())
    assert np.all(off.get() == 0)
    off.check_outside()


@pytest.mark.parametrize("tokens", [16385, 70000])
def test_route_many_tokens(ctx, tokens):
    """More workgroups than the second kernel adds up itself."""
    rng = np.random.default_rng(5)
    l = rng.normal(size=(tokens, 32))
    x = Rows("f32", tokens, 32, data=l)
    d = gt.route_desc(0, tokens, 32, 4)
    chosen, gates = Rows("i32", tokens, 4), Rows("f32", tokens, 4)
    off, rows, places = Rows("i32", 1, 33), Rows("i32", 1, 4 * tokens), Rows("i32", tokens, 4)
    ws = workspace(gt.route_workspace_bytes(d))
    gt.route_forward(ctx, d, x.ptr, None, chosen.ptr, gates.ptr, off.ptr, rows.ptr, places.ptr, ws.data_ptr(), stream())
    want = np.argsort(-x.get(), axis=1, kind="stable")[:, :4]
    assert np.array_equal(chosen.get(), want)
    for have, ref in zip((off, rows, places), plain.lists(want, 32)):
        assert np.array_equal(have.get().reshape(-1), np.asarray(ref).reshape(-1))
    assert bool((ws[-64:] == 0xA5).all())


def test_route_gradient_of_foreign_choices(ctx):
    """The same expert twice counts twice; one outside the experts takes part in nothing."""
    rng = np.random.default_rng(6)
    l = Rows("f32", 8, 20, data=rng.normal(size=(8, 20)))
    c = rng.integers(0, 20, size=(8, 5))
    c[0], c[1, 2], c[2], c[3, 1] = 7, -1, 25, c[3, 0]
    chosen, dg = Rows("i32", 8, 5, data=c), Rows("f32", 8, 5, data=rng.normal(size=(8, 5)))
    for scores in ("softmax", "sigmoid"):
        for renormalize in (False, True):
            d = gt.route_desc(0, 8, 20, 5, scores=gt.SCORES_SIGMOID if scores == "sigmoid" else gt.SCORES_SOFTMAX, renormalize=renormalize)
            dl = Rows("f32", 8, 20)
            gt.route_gradient(ctx, d, l.ptr, chosen.ptr, dg.ptr, dl.ptr, stream())
            ref, size = plain.route_gradient(l.get(), c, dg.get(), scores, renormalize, 1.0)
            near(dl.get(), ref, size * (2.0 ** -17 + 120 * U) + 1e-36, "f32")


def test_route_gradient_against_differences(ctx):
    rng = np.random.default_rng(7)
    l = Rows("f32", 3, 12, data=rng.normal(size=(3, 12)))
    for scores in ("softmax", "sigmoid"):
        for renormalize in (False, True):
            d = gt.route_desc(0, 3, 12, 4, scores=gt.SCORES_SIGMOID if scores == "sigmoid" else gt.SCORES_SOFTMAX, renormalize=renormalize,
                              scale=1.5)
            chosen, gates, dl = Rows("i32", 3, 4), Rows("f32", 3, 4), Rows("f32", 3, 12)
            dg = Rows("f32", 3, 4, data=rng.normal(size=(3, 4)))
            gt.route_forward(ctx, d, l.ptr, None, chosen.ptr, gates.ptr, stream=stream())
            gt.route_gradient(ctx, d, l.ptr, chosen.ptr, dg.ptr, dl.ptr, stream())
            h = 1e-6

            def f(v):
                s = plain.scores(v, scores)
                m = np.take_along_axis(s, chosen.get().astype(int), axis=1)
                return float((1.5 * m / (m.sum(axis=1, keepdims=True) if renormalize else 1.0) * dg.get()).sum())

            for t, e in ((0, 0), (1, 5), (2, 11), (0, int(chosen.get()[0, 0]))):
                step = np.zeros((3, 12))
                step[t, e] = h
                assert abs((f(l.get() + step) - f(l.get() - step)) / (2 * h) - dl.get()[t, e]) < 1e-5


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("widths", [(64, 2048), (136, 2001)])
@pytest.mark.parametrize("parts, act, layout", [("", "none", "packed"), ("bfrp", "relu", "packed"), ("rp", "none", "padded"),
                                                ("bf", "relu", "padded")])
def test_fused_product_of_many_rows(ctx, kind, widths, parts, act, layout):
    """The tiles of up to 256 x 256, ragged groups and columns, whole numbers."""
    p = Product(kind, ([2100, 0, 1900, 301], 3), widths, layout, parts, act, whole)
    say(f"fused many rows {kind} {widths} {parts} {act} {layout}")
    p.call(ctx)
    z, _, _, y = p.reference()
    for have, want in ((p.y, y), (p.z, z)):
        if have is not None:
            got = have.get()
            inside = slice(p.off[0], p.off[-1])
            assert np.array_equal(got[inside], rounded(want, kind)[inside]) and p.untouched(got)
            have.check_outside()

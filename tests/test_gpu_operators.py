"""The operators over plain rows on the GPU against plain 64-bit forms
(tests/plain_rows.py).

Two kinds of data.  Small whole numbers, whose products and sums fp32 holds
exactly: outputs must then equal the 64-bit result rounded once to their
type, bit for bit, whatever the order of the sums.  And normal numbers, with a
bound by arithmetic: a sum of n terms in fp32, in any order, is off by at most
n 2^-24 (1 + n 2^-24) sum |term| <= (n + 1) 2^-24 sum |term| for the lengths
here, plus half a step of the output's type relative to the value or, below
its normal numbers, half its last step (tests say so where more roundings add
up)."""
import numpy as np
import pytest
import torch

import gotransformers_amd as gt
from tests.plain_rows import HALF_LAST_STEP, HALF_STEP, VALUES, adapted, dropout_factor, grouped, offsets_of

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SENTINEL = 77.0


@pytest.fixture(scope="module")
def ctx():
    c = gt.Context(0)
    yield c
    c.close()


def say(*a):
    print(*a, flush=True)


def stream():
    return torch.cuda.current_stream().cuda_stream


class Rows:
    """A rows x width matrix inside a larger device buffer of `kind`: rows
    `stride` values apart, `shift` values behind the buffer's start, SENTINEL
    (or `fill`) everywhere else."""

    def __init__(self, kind, rows, width, stride=None, shift=0, data=None, fill=SENTINEL):
        stride = width if stride is None else stride
        self.buf = torch.full((shift + max(rows, 1) * stride + 64,), fill, dtype=TYPES[kind], device="cuda")
        self.view = self.buf[shift:shift + max(rows, 1) * stride].view(max(rows, 1), stride)[:rows, :width]
        self.stride, self.fill = stride, fill
        if data is not None:
            self.view.copy_(torch.as_tensor(np.ascontiguousarray(data)).to(TYPES[kind]))

    @property
    def ptr(self):
        return self.view.data_ptr()

    def get(self):
        return self.view.double().cpu().numpy()

    def outside_is_untouched(self):
        was = self.view.clone()
        self.view.fill_(self.fill)
        ok = bool((self.buf == self.fill).all())
        self.view.copy_(was)
        return ok


def rounded(a, kind):
    return torch.as_tensor(a).to(TYPES[kind]).double().numpy()


def whole(rng, *shape, top=2):
    return rng.integers(-top, top + 1, size=shape).astype(np.float64)


def device_offsets(offsets):
    return torch.from_numpy(np.asarray(offsets, np.int32)).cuda()


def run_grouped(ctx, kind, off, x, w, dy, layout="packed", gradient=None, rows=None):
    """All three directions; returns the output holders (y, dx, dw).  layout:
    packed; padded (16-byte multiples between rows and matrices); odd (strides
    and addresses of single values)."""
    R, K = x.shape
    G, N = w.shape[0], w.shape[1]
    pad = {"packed": 0, "padded": 16, "odd": 3}[layout]
    shift = 1 if layout == "odd" else 0
    up = lambda v: v if layout == "packed" else -(-v // 8) * 8 + pad if layout == "padded" else v + pad
    xs, ys, ws = up(K), up(N), up(K)
    gstride = N * ws + (8 if layout == "padded" else 5 if layout == "odd" else 0)
    hx = Rows(kind, R, K, xs, shift, x)
    hdy = Rows(kind, R, N, ys, shift, dy)
    y, dx = Rows(kind, R, N, ys, shift), Rows(kind, R, K, xs, shift)
    hw = torch.full((shift + G * gstride + 8,), SENTINEL, dtype=TYPES[kind], device="cuda")
    wview = torch.as_strided(hw, (G, N, K), (gstride, ws, 1), shift)
    wview.copy_(torch.as_tensor(w).to(TYPES[kind]))
    gkind = gradient or kind
    hdw = torch.full((shift + G * gstride + 8,), SENTINEL, dtype=TYPES[gkind], device="cuda")
    dwview = torch.as_strided(hdw, (G, N, K), (gstride, ws, 1), shift)
    o = device_offsets(off)
    d = gt.grouped_desc(VALUES[kind], G, R, K, N, xs, ys, ws, gstride)
    gt.grouped_forward(ctx, d, o.data_ptr(), hx.ptr, wview.data_ptr(), y.ptr, stream())
    gt.grouped_input_gradient(ctx, d, o.data_ptr(), hdy.ptr, wview.data_ptr(), dx.ptr, stream())
    gt.grouped_weight_gradient(ctx, d, o.data_ptr(), hdy.ptr, hx.ptr, dwview.data_ptr(), VALUES[gkind], False, stream())
    torch.cuda.synchronize()
    dw = dwview.double().cpu().numpy()
    dwview.fill_(SENTINEL)
    assert bool((hdw == SENTINEL).all()), "values between the gradient matrices' rows were written"
    return y, dx, dw


# sizes of the groups, first row (rows before it and behind the last belong to no group)
SIZES = {
    "one row": ([1], 0),
    "empty and single": ([0, 1, 0, 0, 2, 0], 3),
    "all empty": ([0, 0, 0], 2),
    "ragged": ([5, 0, 130, 17, 64, 1, 129, 33], 1),
    "few per group": ([4, 3, 0, 7, 2, 9, 1, 16, 17], 0),
    "long": ([700, 0, 261], 0),
    "many groups": ([1, 0, 2] * 50, 0),
}
WIDTHS = [(1, 1), (7, 5), (8, 8), (64, 64), (72, 136), (129, 130), (256, 512), (1000, 1201)]


def check_whole(ctx, kind, sizes, widths, layout, gradient=None):
    parts, first = SIZES[sizes]
    K, N = widths
    off = offsets_of(parts, first)
    R = int(off[-1]) + 2
    rng = np.random.default_rng(R * 31 + K * 7 + N)
    # |sum| <= 4 * 1201 for y and dx, 4 * 700 for dw: exact in fp32, one rounding to the type
    x, w, dy = whole(rng, R, K), whole(rng, len(parts), N, K), whole(rng, R, N)
    say(f"grouped {kind} {sizes} K={K} N={N} {layout} gradient={gradient}")
    y, dx, dw = run_grouped(ctx, kind, off, x, w, dy, layout, gradient)
    ry, rdx, rdw = grouped(off, x, w, dy)
    for got, ref in ((y, ry), (dx, rdx)):
        want = rounded(ref, kind)
        want[:off[0]], want[off[-1]:] = SENTINEL, SENTINEL
        assert np.array_equal(got.get(), want)
        assert got.outside_is_untouched()
    assert np.array_equal(dw, rounded(rdw, gradient or kind))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("widths", WIDTHS, ids=lambda w: f"{w[0]}x{w[1]}")
def test_grouped_widths(ctx, kind, widths):
    check_whole(ctx, kind, "ragged", widths, "packed")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sizes", list(SIZES))
def test_grouped_sizes(ctx, kind, sizes):
    check_whole(ctx, kind, sizes, (136, 72), "packed", gradient="f32")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", ["padded", "odd"])
@pytest.mark.parametrize("sizes", ["few per group", "long"])
def test_grouped_layouts(ctx, kind, layout, sizes):
    check_whole(ctx, kind, sizes, (200, 264), layout)
    check_whole(ctx, kind, sizes, (37, 300), layout, gradient="f32")


@pytest.mark.parametrize("kind", list(TYPES))
def test_grouped_many_rows_per_group(ctx, kind):
    """Enough rows per group for the largest tiles, ragged against them."""
    SIZES["large"] = ([1500, 513, 0, 1031], 0)
    check_whole(ctx, kind, "large", (320, 328), "packed", gradient="f32")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sizes", ["ragged", "few per group", "long"])
def test_grouped_normal_values(ctx, kind, sizes):
    parts, first = SIZES[sizes]
    K, N = 520, 392
    off = offsets_of(parts, first)
    R = int(off[-1])
    rng = np.random.default_rng(5)
    x, w, dy = (rounded(rng.normal(size=s) * f, kind) for s, f in
                (((R, K), 1.0), ((len(parts), N, K), K ** -0.5), ((R, N), 1.0)))
    say(f"grouped normal {kind} {sizes}")
    y, dx, dw = run_grouped(ctx, kind, off, x, w, dy)
    refs = grouped(off, x, w, dy)
    sizes_of = grouped(off, np.abs(x), np.abs(w), np.abs(dy))
    for got, ref, size, n in ((y.get(), refs[0], sizes_of[0], K), (dx.get(), refs[1], sizes_of[1], N),
                              (dw, refs[2], sizes_of[2], max(parts))):
        at = slice(off[0], off[-1]) if got is not dw else slice(None)
        bound = HALF_STEP[kind] * np.abs(ref) + HALF_LAST_STEP[kind] + (n + 1) * 2.0 ** -24 * size
        assert np.all(np.abs(got[at] - ref[at]) <= (bound * (1 + 2.0 ** -7))[at])


@pytest.mark.parametrize("kind", list(TYPES))
def test_grouped_sums_that_cancel_stay_in_32_bits(ctx, kind):
    """Terms of 2^10 that cancel around ones: a sum kept in the values' own
    type would lose them."""
    K, N = 256, 16
    x = np.ones((3, K))
    x[:, ::2] = 32.0
    x[:, 0] = 1.0
    w = np.ones((1, N, K))
    w[:, :, ::4] = 32.0
    w[:, :, 2::4] = -32.0
    w[:, :, 0] = 1.0
    y, _, _ = run_grouped(ctx, kind, [0, 3], x, w, np.ones((3, N)))
    assert np.array_equal(y.get(), rounded(x @ w[0].T, kind))


@pytest.mark.parametrize("kind", list(TYPES))
def test_grouped_infinities_and_nan_stay_in_their_rows(ctx, kind):
    """NaN in one row, group or column reaches what the formula says it
    reaches and nothing else; NaN between rows, behind them and in rows of no
    group reaches nothing."""
    parts = [40, 0, 150, 7]
    off = offsets_of(parts, 2)
    R, K, N = int(off[-1]) + 3, 72, 136
    rng = np.random.default_rng(6)
    x, w, dy = whole(rng, R, K), whole(rng, 4, N, K), whole(rng, R, N)
    x[:2], dy[:2], x[-3:], dy[-3:] = np.nan, np.inf, np.nan, np.nan  # no group's
    w[1] = np.nan  # of the empty group
    x[50, 3], dy[50, 4] = np.nan, np.inf
    w[3, 5, 6] = np.inf
    hx, hdy = Rows(kind, R, K, 80, 0, x, fill=float("nan")), Rows(kind, R, N, 152, 0, dy, fill=float("nan"))
    hw = torch.full((4, N, 80), float("nan"), dtype=TYPES[kind], device="cuda")
    hw[:, :, :K].copy_(torch.as_tensor(w).to(TYPES[kind]))
    y, dx = Rows(kind, R, N, 152), Rows(kind, R, K, 80)
    dw = torch.zeros((4, N, 80), dtype=torch.float32, device="cuda")
    o = device_offsets(off)
    d = gt.grouped_desc(VALUES[kind], 4, R, K, N, 80, 152, 80)
    gt.grouped_forward(ctx, d, o.data_ptr(), hx.ptr, hw.data_ptr(), y.ptr, stream())
    gt.grouped_input_gradient(ctx, d, o.data_ptr(), hdy.ptr, hw.data_ptr(), dx.ptr, stream())
    gt.grouped_weight_gradient(ctx, d, o.data_ptr(), hdy.ptr, hx.ptr, dw.data_ptr(), gt.VALUES_FLOAT32, False, stream())
    with np.errstate(invalid="ignore"):
        ry, rdx, rdw = grouped(off, x, w, dy)
    for got, ref in ((y.get(), ry), (dx.get(), rdx)):
        assert np.all(got[:2] == SENTINEL) and np.all(got[-3:] == SENTINEL)
        assert np.array_equal(got[2:-3], rounded(ref, kind)[2:-3], equal_nan=True)
    assert np.array_equal(dw[:, :, :K].double().cpu().numpy(), rdw, equal_nan=True)
    assert bool((dw[:, :, K:] == 0).all())


@pytest.mark.parametrize("kind, gradient", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("widths", [(72, 136), (37, 41)])
def test_grouped_weight_gradients_accumulate(ctx, kind, gradient, widths):
    K, N = widths
    off = offsets_of([30, 0, 100])
    rng = np.random.default_rng(7)
    x, dy, before = whole(rng, 130, K, top=1), whole(rng, 130, N, top=1), whole(rng, 3, N, K)
    dw = torch.as_tensor(before).to(TYPES[gradient]).cuda()
    hx, hdy = Rows(kind, 130, K, data=x), Rows(kind, 130, N, data=dy)
    o = device_offsets(off)
    d = gt.grouped_desc(VALUES[kind], 3, 130, K, N)
    want = before
    for _ in range(2):  # |sum| <= 2 + 2 * 100 < 256: whole numbers bf16 holds exactly
        gt.grouped_weight_gradient(ctx, d, o.data_ptr(), hdy.ptr, hx.ptr, dw.data_ptr(), VALUES[gradient], True,
                                   stream())
        want = want + grouped(off, x, np.zeros((3, N, K)), dy)[2]
    assert np.array_equal(dw.double().cpu().numpy(), want)


def test_grouped_without_rows(ctx):
    """No rows at all: nothing to write, but every weight gradient becomes zero."""
    o = device_offsets([0, 0, 0])
    d = gt.grouped_desc(gt.VALUES_BFLOAT16, 2, 0, 24, 40)
    dw = torch.full((2, 40, 24), SENTINEL, dtype=torch.bfloat16, device="cuda")
    gt.grouped_forward(ctx, d, o.data_ptr(), None, None, None, stream())
    gt.grouped_input_gradient(ctx, d, o.data_ptr(), None, None, None, stream())
    gt.grouped_weight_gradient(ctx, d, o.data_ptr(), None, None, dw.data_ptr(), gt.VALUES_BFLOAT16, True, stream())
    assert bool((dw == SENTINEL).all())
    gt.grouped_weight_gradient(ctx, d, o.data_ptr(), None, None, dw.data_ptr(), gt.VALUES_BFLOAT16, False, stream())
    assert bool((dw == 0).all())


@pytest.mark.parametrize("bad", [[0, 90, 40, 200], [-5, 3, 1 << 30, -(1 << 31)], [100, 60, 20, 0],
                                 [(1 << 31) - 1, 0, (1 << 31) - 1, 5]])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_grouped_offsets_that_descend_stay_inside_the_buffers(ctx, bad, kind):
    rng = np.random.default_rng(8)
    x, w, dy = whole(rng, 100, 72), whole(rng, 3, 40, 72), whole(rng, 100, 40)
    say("offsets", bad, kind)
    y, dx, _ = run_grouped(ctx, kind, bad, x, w, dy)
    assert y.outside_is_untouched() and dx.outside_is_untouched()


def test_grouped_rows_beyond_two_gigabytes(ctx):
    """Row offsets that pass 2^31 values: rows 2^20 values apart."""
    R, K, N, st = 2200, 64, 48, 1 << 20
    rng = np.random.default_rng(9)
    x, w, dy = whole(rng, R, K), whole(rng, 2, N, K), whole(rng, R, N)
    big = torch.empty(R * st, dtype=torch.bfloat16, device="cuda")
    view = big.view(R, st)
    hx, hy = view[:, :K], view[:, 512:512 + N]
    hdx, hdy = view[:, 1024:1024 + K], view[:, 2048:2048 + N]
    hx.copy_(torch.as_tensor(x))
    hdy.copy_(torch.as_tensor(dy))
    hw = torch.as_tensor(w).to(torch.bfloat16).cuda()
    dw = torch.empty(2, N, K, dtype=torch.float32, device="cuda")
    off = [0, 3, R]
    o = device_offsets(off)
    d = gt.grouped_desc(gt.VALUES_BFLOAT16, 2, R, K, N, st, st)
    gt.grouped_forward(ctx, d, o.data_ptr(), hx.data_ptr(), hw.data_ptr(), hy.data_ptr(), stream())
    gt.grouped_input_gradient(ctx, d, o.data_ptr(), hdy.data_ptr(), hw.data_ptr(), hdx.data_ptr(), stream())
    gt.grouped_weight_gradient(ctx, d, o.data_ptr(), hdy.data_ptr(), hx.data_ptr(), dw.data_ptr(), gt.VALUES_FLOAT32,
                               False, stream())
    ry, rdx, rdw = grouped(off, x, w, dy)
    assert np.array_equal(hy.double().cpu().numpy(), rounded(ry, "bf16"))
    assert np.array_equal(hdx.double().cpu().numpy(), rounded(rdx, "bf16"))
    assert np.array_equal(dw.double().cpu().numpy(), rdw)


# --------------------------------------------------------------------------
# adapters
# --------------------------------------------------------------------------

def run_adapted(ctx, kind, x, w, b, adapter, down, up, scales, base=None, odd=False):
    T, K = x.shape
    n, r = down.shape[0], down.shape[1]
    N = up.shape[1]
    pad, shift = (3, 1) if odd else (0, 0)
    hx, y = Rows(kind, T, K, K + pad, shift, x), Rows(kind, T, N, N + pad, shift, base)
    hw = None if w is None else Rows(kind, N, K, K + pad, shift, w)
    flat = lambda a: Rows(kind, 1, a.size, None, shift, a.reshape(1, -1))
    hb, hd, hu = None if b is None else flat(b), flat(down), flat(up)
    hs = torch.as_tensor(scales).float().cuda()
    ha = torch.as_tensor(np.asarray(adapter, np.int32)).cuda()
    d = gt.adapted_desc(VALUES[kind], T, K, N, n, r, K + pad, N + pad, K + pad)
    need = gt.adapted_workspace_bytes(d)
    ws = torch.full((need // 4 + 64,), float("nan"), dtype=torch.float32, device="cuda")
    gt.adapted_forward(ctx, d, hx.ptr, hw and hw.ptr, hb and hb.ptr, ha.data_ptr(), hd.ptr, hu.ptr, hs.data_ptr(), y.ptr,
                       ws.data_ptr(), stream())
    torch.cuda.synchronize()
    assert y.outside_is_untouched()
    assert bool(torch.isnan(ws[need // 4:]).all()), "bytes behind the workspace were written"
    return y.get()


def adapters_of(rng, pattern, T, n):
    if pattern == "one":
        return np.full(T, n - 1)
    if pattern == "each its own":
        return np.arange(T) % n
    if pattern == "runs":
        return np.repeat(rng.integers(-1, n, size=T), 13)[:T]
    if pattern == "none":
        return np.full(T, -1)
    a = rng.integers(-1, n + 1, size=T)  # n: outside the adapters, so none
    return np.where(rng.random(T) < 0.1, np.iinfo(np.int32).min, a)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rank", [1, 3, 4, 8, 13, 16, 24, 64, 130])
def test_adapted_ranks(ctx, kind, rank):
    check_adapted_whole(ctx, kind, 37, 136, 72, rank, 5, "mixed")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 33, 64, 65, 130, 300, 600])
@pytest.mark.parametrize("pattern", ["one", "each its own", "runs", "none", "mixed"])
def test_adapted_rows(ctx, kind, T, pattern):
    check_adapted_whole(ctx, kind, T, 200, 264, 8, 40, pattern)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("widths", [(1, 1), (5, 7), (64, 16), (129, 130), (1000, 1201), (2048, 96)])
@pytest.mark.parametrize("odd", [False, True])
def test_adapted_widths(ctx, kind, widths, odd):
    for T in (3, 150):
        check_adapted_whole(ctx, kind, T, widths[0], widths[1], 16, 3, "mixed", odd=odd)


def check_adapted_whole(ctx, kind, T, K, N, rank, n, pattern, odd=False):
    """Whole numbers, with and without the shared product and the biases.
    |Down x| <= 2 K and |y| <= 4 K + 2 + rank * 2 K: Down's and Up's entries in
    {-1, 0, 1} with three in four zero keep every partial sum far below 2^24."""
    rng = np.random.default_rng(T * 101 + K + N + rank)
    sparse = lambda *s: whole(rng, *s, top=1) * (rng.random(s) < 0.25)
    x, w, b = whole(rng, T, K, top=1), whole(rng, N, K), whole(rng, N)
    down, up = sparse(n, rank, K), sparse(n, N, rank)
    scales = 2.0 ** rng.integers(-1, 2, size=n)
    base = whole(rng, T, N, top=9)
    adapter = adapters_of(rng, pattern, T, n)
    say(f"adapted {kind} T={T} K={K} N={N} rank={rank} adapters={n} {pattern} odd={odd}")
    for ww, bb in ((w, b), (w, None), (None, None), (None, b)):
        start = base if ww is None else None
        got = run_adapted(ctx, kind, x, ww, bb, adapter, down, up, scales, base=start, odd=odd)
        ref, _ = adapted(x, ww, bb, adapter, down, up, scales, base=start)
        assert np.array_equal(got, rounded(ref, kind)), (ww is None, bb is None)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("T, K, N, rank, n", [(1024, 72, 264, 16, 5), (8200, 72, 264, 16, 5), (16390, 72, 40, 8, 1),
                                              (2100, 64, 520, 64, 1023), (5470, 136, 40, 24, 17),
                                              (3300, 200, 300, 40, 100)])
@pytest.mark.parametrize("pattern", ["one", "each its own", "runs", "none", "mixed"])
def test_adapted_many_rows(ctx, kind, T, K, N, rank, n, pattern):
    """Many rows, below and above where they are sorted by adapter, in every
    order of them."""
    check_adapted_whole(ctx, kind, T, K, N, rank, n, pattern)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("K, N, rank, n, odd", [(64, 48, 72, 3, False), (64, 48, 36, 3, False), (68, 48, 40, 3, False),
                                                (64, 48, 48, 1024, False), (64, 48, 64, 3, True)])
def test_adapted_many_rows_that_cannot_be_sorted(ctx, kind, K, N, rank, n, odd):
    """Ranks, widths, counts of adapters and strides the sorted form does not take."""
    check_adapted_whole(ctx, kind, (1 << 17) // rank + 3, K, N, rank, n, "mixed", odd=odd)


def test_adapted_scales_of_a_row_do_not_touch_another(ctx):
    """fp16 parts of u are scaled by row: rows with u near 2^40 and 2^-20 side by
    side, of one adapter, each exact to its own size."""
    for T, rank in ((70, 8), (300, 8), (2200, 64)):
        K, N = 64, 72
        rng = np.random.default_rng(T)
        x = np.zeros((T, K))
        x[:, 0] = np.where(np.arange(T) % 2 == 0, 2.0 ** 10, 2.0 ** -10)
        w, b = np.zeros((N, K)), whole(rng, N)
        w[:, 0] = 2.0 ** -10
        down, up = np.zeros((1, rank, K)), np.zeros((1, N, rank))
        down[0, :, 0] = 2.0 ** 12
        up[0, :, 0] = 2.0 ** -20 * whole(rng, N)
        got = run_adapted(ctx, "f16", x, w, b, np.zeros(T, int), down, up, [1.0])
        ref, _ = adapted(x, w, b, np.zeros(T, int), down, up, [1.0])
        assert np.array_equal(got, rounded(ref, "f16"))
        got = run_adapted(ctx, "f16", x, w, b, np.zeros(T, int), down, up, [2.0 ** 18])
        ref, _ = adapted(x, w, b, np.zeros(T, int), down, up, [2.0 ** 18])
        # Up's values are fp16 subnormals here.  The matrix cores align a sum to
        # its products' exponents before normalising, a subnormal factor's being
        # that of 2^-14: a sum with |u| = 2^20 keeps what is above 2^20 2^-14 2^-24
        # per product (two parts of one rank), whatever the product's value
        bound = HALF_STEP["f16"] * np.abs(ref) + 2 * 2.0 ** (20 - 14 - 24)
        assert np.all(np.abs(got - ref)[1::2] <= bound[1::2])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("T, rank", [(1, 16), (48, 16), (300, 32), (4200, 32)])
def test_adapted_normal_values(ctx, kind, T, rank):
    K, N, n = 520, 392, 7
    rng = np.random.default_rng(11)
    make = lambda *s, f=1.0: rounded(rng.normal(size=s) * f, kind)
    x, w, b = make(T, K), make(N, K, f=K ** -0.5), make(N)
    down, up = make(n, rank, K, f=K ** -0.5), make(n, N, rank, f=rank ** -0.5)
    scales = np.float32(rng.uniform(0.5, 2, size=n)).astype(np.float64)
    adapter = adapters_of(rng, "mixed", T, n)
    got = run_adapted(ctx, kind, x, w, b, adapter, down, up, scales)
    ref, size = adapted(x, w, b, adapter, down, up, scales)
    # K terms of the shared sum; K, the scale and rank terms of the adapter's; bias and the two parts' sum;
    # bf16: u in two parts loses 2^-16 of it (the rest of 8 bits cut off, rounded to 8), fp16 2^-22
    bound = HALF_STEP[kind] * np.abs(ref) + HALF_LAST_STEP[kind] + (K + rank + 4) * 2.0 ** -24 * size
    bound += {"bf16": 2.0 ** -16, "f16": 2.0 ** -22, "f32": 0.0}[kind] * size
    assert np.all(np.abs(got - ref) <= bound * (1 + 2.0 ** -7))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("T, rank", [(20, 8), (140, 8), (300, 8), (2100, 64)])
def test_adapted_nan_stays_with_its_request(ctx, kind, T, rank):
    """A request whose row or adapter holds NaN or infinity leaves the other
    requests' rows as they are without it."""
    rng = np.random.default_rng(12)
    K, N, n = 136, 72, 6
    sparse = lambda *s: whole(rng, *s, top=1) * (rng.random(s) < 0.25)
    x, w = whole(rng, T, K, top=1), whole(rng, N, K)
    down, up, scales = sparse(n, rank, K), sparse(n, N, rank), np.ones(n)
    adapter = np.arange(T) % 5 - 1  # -1 .. 3; adapters 4 and 5 are no row's
    clean = run_adapted(ctx, kind, x, w, None, adapter, down, up, scales)
    down[2], up[3], down[4], up[5] = np.nan, np.inf, np.nan, np.nan
    x[7] = np.nan  # adapter 1
    got = run_adapted(ctx, kind, x, w, None, adapter, down, up, scales)
    touched = (adapter == 2) | (adapter == 3) | (np.arange(T) == 7)
    assert np.array_equal(got[~touched], clean[~touched])
    assert np.all(~np.isfinite(got[adapter == 2])) and np.all(np.isnan(got[7]))


def test_adapted_rows_without_adapter_keep_their_bits(ctx):
    """Added to an existing product, rows without an adapter are not written:
    a negative zero and a NaN's bits stay."""
    base = np.full((6, 24), -0.0)
    y = torch.as_tensor(base).to(torch.float16).cuda()
    y[3] = float("nan")
    before = y.view(torch.int16).clone()
    x = torch.ones(6, 16, dtype=torch.float16, device="cuda")
    down, up = torch.ones(1, 4, 16, dtype=torch.float16, device="cuda"), torch.ones(1, 24, 4, dtype=torch.float16, device="cuda")
    s = torch.ones(1, device="cuda")
    a = torch.tensor([-1, -1, 0, -1, -1, 1], dtype=torch.int32, device="cuda")
    d = gt.adapted_desc(gt.VALUES_FLOAT16, 6, 16, 24, 1, 4)
    ws = torch.empty(gt.adapted_workspace_bytes(d), dtype=torch.uint8, device="cuda")
    gt.adapted_forward(ctx, d, x.data_ptr(), None, None, a.data_ptr(), down.data_ptr(), up.data_ptr(), s.data_ptr(),
                       y.data_ptr(), ws.data_ptr(), stream())
    after = y.view(torch.int16)
    keep = torch.tensor([0, 1, 3, 4, 5], device="cuda")
    assert torch.equal(after[keep], before[keep])
    assert bool((y[2] == 64).all())


def test_adapted_keeps_the_ranks_products_in_fp32(ctx):
    """Down x = 1 + 2^-12 in every rank: rounded to bf16 it would be 1, and Up =
    2^12 - ... would then give 0 instead of 1 per rank."""
    K, N = 16, 32
    x = np.zeros((1, K))
    x[0, 0], x[0, 1] = 1.0, 2.0 ** -12
    down = np.zeros((1, 2, K))
    down[0, :, 0], down[0, 0, 1] = 1.0, 1.0  # u = (1 + 2^-12, 1)
    up = np.zeros((1, N, 2))
    up[0, :, 0], up[0, :, 1] = 4096.0, -4096.0  # y = 4096 * 2^-12 = 1
    for kind in ("bf16", "f16"):
        got = run_adapted(ctx, kind, x, np.zeros((N, K)), None, [0], down, up, [1.0])
        assert np.array_equal(got, np.ones((1, N)))


# --------------------------------------------------------------------------
# dropout
# --------------------------------------------------------------------------

@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows, columns", [(1, 1), (3, 7), (5, 8), (17, 9), (64, 256), (33, 1201)])
@pytest.mark.parametrize("rate", [0.0, 0.1, 0.5, 0.99999])
def test_dropout_forward_and_backward(ctx, kind, rows, columns, rate):
    rng = np.random.default_rng(rows * columns)
    x, dy, base = (rounded(rng.normal(size=(rows, columns)), kind) for _ in range(3))
    x[0, 0] = np.inf
    seed, offset = 0x123456789ABCDEF, 0xFEDCBA9876543210
    f, keep = dropout_factor(rows, columns, rate, seed, offset)
    say(f"dropout {kind} {rows}x{columns} rate={rate} kept {keep.mean():.3f}")
    for pad, shift in ((0, 0), (3, 1)):
        hx, hdy = Rows(kind, rows, columns, columns + pad, shift, x), Rows(kind, rows, columns, columns + pad, shift, dy)
        hb = Rows(kind, rows, columns, columns + 8, 0, base)
        y, yb, dx = (Rows(kind, rows, columns, columns + pad, shift) for _ in range(3))
        d = gt.dropout_desc(VALUES[kind], rows, columns, columns + pad, columns + 8, columns + pad)
        gt.dropout(ctx, d, hx.ptr, None, y.ptr, rate, seed, offset, stream())
        gt.dropout(ctx, d, hx.ptr, hb.ptr, yb.ptr, rate, seed, offset, stream())
        gt.dropout(ctx, d, hdy.ptr, None, dx.ptr, rate, seed, offset, stream())
        # the scale rounded to fp32, the product to fp32, the sum to fp32, the result to the type
        for got, v, b in ((y, x, 0.0), (yb, x, base), (dx, dy, 0.0)):
            with np.errstate(invalid="ignore"):
                term = np.where(keep, v * f, 0.0)
                ref = b + term
            g = got.get()
            assert np.array_equal(np.isfinite(g), np.isfinite(rounded(ref, kind)))
            at = np.isfinite(g)
            size = np.abs(term[at]) + np.abs(np.broadcast_to(b, term.shape)[at])
            bound = HALF_STEP[kind] * np.abs(ref[at]) + 3 * 2.0 ** -24 * size
            bound = bound * (1 + 2.0 ** -7) + HALF_LAST_STEP[kind]
            assert np.all(np.abs(g[at] - ref[at]) <= bound)
            if b is not base:
                assert np.all(g[~keep] == 0.0)
            assert got.outside_is_untouched()


def test_dropout_in_place_and_other_counters(ctx):
    rng = np.random.default_rng(3)
    x = rounded(rng.normal(size=(40, 77)), "f32")
    d = gt.dropout_desc(gt.VALUES_FLOAT32, 40, 77)
    masks = []
    for seed, offset in ((1, 0), (1, 1), (2, 0), (1 << 63, 0), (1, 1 << 40)):
        h = Rows("f32", 40, 77, data=np.ones((40, 77)))
        gt.dropout(ctx, d, h.ptr, None, h.ptr, 0.5, seed, offset, stream())
        f, keep = dropout_factor(40, 77, 0.5, seed, offset)
        assert np.array_equal(h.get(), f)
        masks.append(keep)
    for i in range(len(masks)):
        for j in range(i):  # independent halves agree in about half the places
            assert 0.4 < (masks[i] == masks[j]).mean() < 0.6
    h = Rows("f32", 40, 77, data=x)
    v = Rows("f32", 40, 77, data=np.ones((40, 77)))
    gt.dropout(ctx, d, v.ptr, h.ptr, h.ptr, 0.5, 1, 0, stream())
    assert np.array_equal(h.get(), (x + dropout_factor(40, 77, 0.5, 1, 0)[0]).astype(np.float32))


# --------------------------------------------------------------------------
# together, on streams and in graphs
# --------------------------------------------------------------------------

def layer_step(ctx, kind, off, x, w, dy, rate, counter):
    """dropout -> experts -> gradients, device tensors in and out."""
    R, K = x.shape
    G, N = w.shape[:2]
    t, v = TYPES[kind], VALUES[kind]
    xd, y, dxd, dx = (torch.empty_like(a) for a in (x, dy, x, x))
    dw = torch.empty(G, N, K, dtype=torch.float32, device="cuda")
    dd, gd = gt.dropout_desc(v, R, K), gt.grouped_desc(v, G, R, K, N)

    def step():
        s = stream()
        gt.dropout(ctx, dd, x.data_ptr(), None, xd.data_ptr(), rate, 99, counter, s)
        gt.grouped_forward(ctx, gd, off.data_ptr(), xd.data_ptr(), w.data_ptr(), y.data_ptr(), s)
        gt.grouped_weight_gradient(ctx, gd, off.data_ptr(), dy.data_ptr(), xd.data_ptr(), dw.data_ptr(),
                                   gt.VALUES_FLOAT32, False, s)
        gt.grouped_input_gradient(ctx, gd, off.data_ptr(), dy.data_ptr(), w.data_ptr(), dxd.data_ptr(), s)
        gt.dropout(ctx, dd, dxd.data_ptr(), None, dx.data_ptr(), rate, 99, counter, s)

    return step, (y, dw, dx)


def test_experts_train_on_a_layers_routing(ctx):
    """The routing of a layer (its expert offsets and rows) drives the grouped
    products of experts in training precision behind a dropout; the loss
    sum(dy * y)'s gradients against differences of the whole run."""
    from tests.moe_fixtures import INT8, make_moe
    spec = make_moe(gt.encode_rows, d=32, h=48, E=5, k=2, S=0, precision=INT8, seed=3)
    rng = np.random.default_rng(4)
    T, K, N = 23, 32, 48
    m = gt.MixtureOfExperts.from_spec(ctx, spec)
    try:
        r = m.route_from_logits(rng.normal(size=(T, 5)))
    finally:
        m.destroy()
    off = device_offsets(r.offsets)
    tokens = rng.normal(size=(T, K))
    x = torch.as_tensor(tokens[r.rows]).float().cuda()
    w = torch.as_tensor(rng.normal(size=(5, N, K)) * K ** -0.5).float().cuda()
    dy = torch.as_tensor(rng.normal(size=(2 * T, N))).float().cuda()
    step, (y, dw, dx) = layer_step(ctx, "f32", off, x, w, dy, 0.3, 5)
    step()
    gx, gw = dx.double().cpu().numpy(), dw.double().cpu().numpy()

    def loss():
        step()
        return float((y.double() * dy.double()).sum())

    # the loss is linear in x and in w: a difference over 2 h is the gradient
    # up to the rounding of y, at most (K + 2) 2^-24 relative to the terms' sum
    size = float((x.abs().double().sum()) * w.abs().max() * dy.abs().max() * N)
    bound = 2 * (K + 2) * 2.0 ** -24 * size
    for t, g, index in ((x, gx, (0, 0)), (x, gx, (7, 31)), (x, gx, (45, 3)), (w, gw, (0, 0, 0)), (w, gw, (3, 40, 17)),
                        (w, gw, (4, 47, 31))):
        was = float(t[index])
        t[index] = was + 4.0
        high = loss()
        t[index] = was - 4.0
        low = loss()
        t[index] = was
        assert abs((high - low) / 8.0 - g[index]) <= bound
    f, _ = dropout_factor(2 * T, K, 0.3, 99, 5)
    xd = x.double().cpu().numpy() * f
    ry, rdx, rdw = grouped(r.offsets, xd, w.double().cpu().numpy(), dy.double().cpu().numpy())
    loss()
    assert np.max(np.abs(y.double().cpu().numpy() - ry)) <= 1e-5 * np.max(np.abs(ry))
    assert np.max(np.abs(gw - rdw)) <= 1e-5 * np.max(np.abs(rdw))
    assert np.max(np.abs(gx - rdx * f)) <= 1e-5 * np.max(np.abs(rdx * f))


@pytest.mark.parametrize("kind", list(TYPES))
def test_operators_in_a_replayed_graph(ctx, kind):
    """A whole step and an adapted projection captured once and replayed with
    other data between eager calls; timing enabled stays out of the graph."""
    rng = np.random.default_rng(14)
    off = device_offsets(offsets_of([70, 0, 9, 200]))
    make = lambda *s: torch.as_tensor(whole(rng, *s)).to(TYPES[kind]).cuda()
    x, w, dy = make(279, 72), make(4, 136, 72), make(279, 136)
    step, outs = layer_step(ctx, kind, off, x, w, dy, 0.5, 3)
    ad = torch.as_tensor(rng.integers(-1, 3, size=279).astype(np.int32)).cuda()
    down, up, sc = make(3, 8, 72), make(3, 136, 8), torch.ones(3, device="cuda")
    ws = torch.empty(gt.adapted_workspace_bytes(gt.adapted_desc(VALUES[kind], 279, 72, 136, 3, 8)), dtype=torch.uint8,
                     device="cuda")
    z = torch.empty(279, 136, dtype=TYPES[kind], device="cuda")

    def both():
        step()
        gt.adapted_forward(ctx, gt.adapted_desc(VALUES[kind], 279, 72, 136, 3, 8), x.data_ptr(), w.data_ptr(), None,
                           ad.data_ptr(), down.data_ptr(), up.data_ptr(), sc.data_ptr(), z.data_ptr(), ws.data_ptr(),
                           stream())

    both()
    torch.cuda.synchronize()
    before = gt.device_allocations()
    ctx.timing(True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        both()
    ctx.timing(False)
    for i in range(4):
        for t in (x, w, dy):
            t.copy_(make(*t.shape))
        both()
        torch.cuda.synchronize()
        want = [o.clone() for o in (*outs, z)]
        for o in (*outs, z):
            o.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip((*outs, z), want):
            assert torch.equal(a, b)
    assert gt.device_allocations() == before


def test_operators_on_two_streams_at_once(ctx):
    rng = np.random.default_rng(15)
    jobs = []
    for i in range(2):
        off = device_offsets(offsets_of([300, 40, 0, 500]))
        make = lambda *s: torch.as_tensor(whole(rng, *s)).bfloat16().cuda()
        jobs.append(layer_step(ctx, "bf16", off, make(840, 256), make(4, 320, 256), make(840, 320), 0.25, i))
    want = []
    for step, outs in jobs:
        step()
        torch.cuda.synchronize()
        want.append([o.clone() for o in outs])
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(5):
        for s, (step, _) in zip(streams, jobs):
            with torch.cuda.stream(s):
                step()
    torch.cuda.synchronize()
    for w, (_, outs) in zip(want, jobs):
        for a, b in zip(w, outs):
            assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("G, K, N", [(3, 136, 72), (40, 520, 264)])
def test_grouped_weight_gradients_accumulate_with_one_rounding(ctx, kind, G, K, N):
    """A 16-bit gradient that is added to: the sum of both in fp32, rounded once.
    Whole numbers up to 4 * 300 + 4000 < 2^24 are exact in fp32; in the type
    neither the new sum nor the result is, so a second rounding would show."""
    rng = np.random.default_rng(21)
    off = offsets_of([300, 0, 41] + [7] * (G - 3))
    R = int(off[-1])
    x, dy = whole(rng, R, K), whole(rng, R, N)
    before = rounded(rng.integers(-4000, 4001, size=(G, N, K)), kind)
    say(f"accumulate {kind} {G} of {K} x {N}")
    dw = torch.as_tensor(before).to(TYPES[kind]).cuda()
    hx, hdy, o = Rows(kind, R, K, data=x), Rows(kind, R, N, data=dy), device_offsets(off)
    gt.grouped_weight_gradient(ctx, gt.grouped_desc(VALUES[kind], G, R, K, N), o.data_ptr(), hdy.ptr, hx.ptr,
                               dw.data_ptr(), VALUES[kind], True, stream())
    want = rounded(before + grouped(off, x, np.zeros((G, N, K)), dy)[2], kind)
    assert np.array_equal(dw.double().cpu().numpy(), want)


@pytest.mark.parametrize("bad", [[0, 4096] * 10 + [0], [4096] * 20 + [0], [-1, 1 << 30] * 10 + [-(1 << 31)],
                                 [0] * 19 + [(1 << 31) - 1, 5]])
def test_many_rows_offsets_that_descend_stay_inside_the_buffers(ctx, bad):
    rng = np.random.default_rng(22)
    G, R, K, N = 20, 4096, 72, 2048
    x, w, dy = whole(rng, R, K), whole(rng, G, N, K), whole(rng, R, N)
    say("offsets", bad)
    y, dx, _ = run_grouped(ctx, "bf16", bad, x, w, dy)
    assert y.outside_is_untouched() and dx.outside_is_untouched()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("stride, shift", [(2059, 1), (2064, 4), (2056, 0)])
def test_many_rows_to_outputs_of_any_alignment(ctx, kind, stride, shift):
    """Aligned operands, outputs whose rows are not: the large tiles of every
    direction and of sorted adapters, with a last column tile of eight."""
    rng = np.random.default_rng(27)
    G, K, N = 8, 520, 2056
    off = offsets_of([900, 0, 1300, 77, 500, 0, 400, 511])
    R = int(off[-1])
    x, w, dy = whole(rng, R, K, top=1), whole(rng, G, N, K, top=1), whole(rng, R, N, top=1)
    say(f"any alignment {kind} stride={stride} shift={shift}")
    ry, rdx, rdw = grouped(off, x, w, dy)
    hx, hdy, o = Rows(kind, R, K, data=x), Rows(kind, R, N, data=dy), device_offsets(off)
    hw = torch.as_tensor(w).to(TYPES[kind]).cuda()
    narrow = stride - N + K
    y, dx = Rows(kind, R, N, stride, shift), Rows(kind, R, K, narrow, shift)
    dw = Rows(kind, G * N, K, narrow, shift)
    v = VALUES[kind]
    gt.grouped_forward(ctx, gt.grouped_desc(v, G, R, K, N, K, stride), o.data_ptr(), hx.ptr, hw.data_ptr(), y.ptr, stream())
    gt.grouped_input_gradient(ctx, gt.grouped_desc(v, G, R, K, N, narrow, N), o.data_ptr(), hdy.ptr, hw.data_ptr(), dx.ptr,
                              stream())
    gt.grouped_weight_gradient(ctx, gt.grouped_desc(v, G, R, K, N, K, N, narrow, N * narrow), o.data_ptr(), hdy.ptr,
                               hx.ptr, dw.ptr, v, False, stream())
    for got, ref in ((y, ry), (dx, rdx), (dw, rdw.reshape(G * N, K))):
        assert np.array_equal(got.get(), rounded(ref, kind)) and got.outside_is_untouched()
    n, rank = 5, 64
    down = whole(rng, n, rank, K, top=1) * (rng.random((n, rank, K)) < 0.25)
    up = whole(rng, n, N, rank, top=1) * (rng.random((n, N, rank)) < 0.25)
    adapter = adapters_of(rng, "mixed", R, n)
    ref, _ = adapted(x, w[0], None, adapter, down, up, np.ones(n))
    dev = lambda a: torch.as_tensor(a).to(TYPES[kind]).cuda()
    hd, hu, hs = dev(down), dev(up), torch.ones(n, device="cuda")
    ha = torch.as_tensor(adapter.astype(np.int32)).cuda()
    d = gt.adapted_desc(v, R, K, N, n, rank, K, stride)
    ws = torch.empty(gt.adapted_workspace_bytes(d), dtype=torch.uint8, device="cuda")
    z = Rows(kind, R, N, stride, shift)
    gt.adapted_forward(ctx, d, hx.ptr, hw.data_ptr(), None, ha.data_ptr(), hd.data_ptr(), hu.data_ptr(), hs.data_ptr(),
                       z.ptr, ws.data_ptr(), stream())
    # |u| <= 520, |y| <= 520 + 64 * 520 < 2^24 and below fp16's 65504: exact in fp32, one rounding
    assert np.array_equal(z.get(), rounded(ref, kind)) and z.outside_is_untouched()


def test_adapted_rows_beyond_two_gigabytes(ctx):
    """Row offsets that pass 2^31 values: rows 2^20 values apart."""
    R, K, N, st, n, rank = 2200, 64, 48, 1 << 20, 5, 64
    rng = np.random.default_rng(23)
    x, w = whole(rng, R, K, top=1), whole(rng, N, K)
    down, up = whole(rng, n, rank, K, top=1), whole(rng, n, N, rank, top=1) * (rng.random((n, N, rank)) < 0.25)
    adapter = adapters_of(rng, "mixed", R, n)
    ref, _ = adapted(x, w, None, adapter, down, up, np.ones(n))
    view = torch.empty(R * st, dtype=torch.bfloat16, device="cuda").view(R, st)
    hx, hy = view[:, :K], view[:, 512:512 + N]
    hx.copy_(torch.as_tensor(x))
    dev = lambda v: torch.as_tensor(v).bfloat16().cuda()
    hw, hd, hu, hs = dev(w), dev(down), dev(up), torch.ones(n, device="cuda")
    ha = torch.as_tensor(adapter.astype(np.int32)).cuda()
    d = gt.adapted_desc(gt.VALUES_BFLOAT16, R, K, N, n, rank, st, st)
    ws = torch.empty(gt.adapted_workspace_bytes(d), dtype=torch.uint8, device="cuda")
    gt.adapted_forward(ctx, d, hx.data_ptr(), hw.data_ptr(), None, ha.data_ptr(), hd.data_ptr(), hu.data_ptr(),
                       hs.data_ptr(), hy.data_ptr(), ws.data_ptr(), stream())
    # |u| <= 64, |y| < 2^24: exact in fp32, one rounding
    assert np.array_equal(hy.double().cpu().numpy(), rounded(ref, "bf16"))


def many_rows(kind, seed):
    """The operators' forms for many rows: a training step and an adapted
    projection with its rows sorted, each with its own buffers."""
    rng = np.random.default_rng(seed)
    off = device_offsets(offsets_of([900, 0, 1300, 77, 2500, 0, 400, 1100]))
    make = lambda *s: torch.as_tensor(rng.normal(size=s)).to(TYPES[kind]).cuda()
    R, G, K, N, n, rank = 6277, 8, 520, 2056, 9, 32
    x, w, dy = make(R, K), make(G, N, K), make(R, N)
    down, up, sc = make(n, rank, K), make(n, N, rank), torch.ones(n, device="cuda")
    ad = torch.as_tensor(rng.integers(-1, n, size=R).astype(np.int32)).cuda()
    d = gt.adapted_desc(VALUES[kind], R, K, N, n, rank)
    ws = torch.empty(gt.adapted_workspace_bytes(d), dtype=torch.uint8, device="cuda")
    z = torch.empty_like(dy)

    def make_step(ctx):
        step, outs = layer_step(ctx, kind, off, x, w, dy, 0.25, seed)

        def both():
            step()
            gt.adapted_forward(ctx, d, x.data_ptr(), w[0].data_ptr(), None, ad.data_ptr(), down.data_ptr(),
                               up.data_ptr(), sc.data_ptr(), z.data_ptr(), ws.data_ptr(), stream())

        return both, (*outs, z)

    return make_step, (x, w, dy, ad)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_many_rows_do_not_change_between_runs(ctx, kind):
    """Mixed rows of an adapter are sorted in any order; their sums are the same."""
    make_step, _ = many_rows(kind, 24)
    step, outs = make_step(ctx)
    step()
    first = [o.clone() for o in outs]
    for _ in range(5):
        for o in outs:
            o.fill_(float("nan"))
        step()
        for a, b in zip(first, outs):
            assert torch.equal(a, b)


def test_many_rows_in_a_replayed_graph(ctx):
    make_step, data = many_rows("bf16", 25)
    step, outs = make_step(ctx)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for i in range(3):
        for t in data[:3]:
            t.copy_(torch.randn_like(t.float()))
        data[3].copy_(torch.randint(-1, 9, data[3].shape, device="cuda", dtype=torch.int32))
        step()
        torch.cuda.synchronize()
        want = [o.clone() for o in outs]
        for o in outs:
            o.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_many_rows_on_two_streams_at_once(ctx):
    jobs = [many_rows("bf16", 26 + i)[0](ctx) for i in range(2)]
    want = []
    for step, outs in jobs:
        step()
        torch.cuda.synchronize()
        want.append([o.clone() for o in outs])
        for o in outs:
            o.fill_(float("nan"))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        for s, (step, _) in zip(streams, jobs):
            with torch.cuda.stream(s):
                step()
    torch.cuda.synchronize()
    for w, (_, outs) in zip(want, jobs):
        for a, b in zip(w, outs):
            assert torch.equal(a, b)


def test_results_do_not_change_between_runs(ctx):
    """Sums have one order: normal numbers give the same bits every time."""
    rng = np.random.default_rng(16)
    off = device_offsets(offsets_of([300, 40, 0, 500]))
    for kind in TYPES:
        make = lambda *s: torch.as_tensor(rng.normal(size=s)).to(TYPES[kind]).cuda()
        step, outs = layer_step(ctx, kind, off, make(840, 250), make(4, 322, 250), make(840, 322), 0.25, 7)
        step()
        first = [o.clone() for o in outs]
        for _ in range(3):
            step()
            for a, b in zip(first, outs):
                assert torch.equal(a, b)


def test_operators_refuse_a_closed_context():
    c = gt.Context(0)
    handle = c.handle
    gt.library().gtmoe_close(handle)
    d = gt.dropout_desc(gt.VALUES_FLOAT32, 1, 1)
    with pytest.raises(gt.InvalidArgument, match="context is closed"):
        gt.dropout(c, d, 1 << 40, None, 1 << 41, 0.5, 0, 0)
    c.close()


def test_operators_answer_an_injected_failure(ctx):
    x = torch.ones(8, device="cuda")
    d = gt.dropout_desc(gt.VALUES_FLOAT32, 1, 8)
    gt.inject_failure("gtmoe_dropout", gt.ERR_DEVICE)
    with pytest.raises(gt.GtmoeError, match="injected failure in gtmoe_dropout"):
        gt.dropout(ctx, d, x.data_ptr(), None, x.data_ptr(), 0.5, 0, 0, stream())
    gt.dropout(ctx, d, x.data_ptr(), None, x.data_ptr(), 0.0, 0, 0, stream())
    assert bool((x == 1).all())


def test_operators_are_timed_by_name(ctx):
    x = torch.ones(64, 64, device="cuda")
    y = torch.empty(64, 64, device="cuda")
    d = gt.dropout_desc(gt.VALUES_FLOAT32, 64, 64)
    ctx.timing_reset()
    ctx.timing(True)
    gt.dropout(ctx, d, x.data_ptr(), None, y.data_ptr(), 0.5, 0, 0, stream())
    times = ctx.timing_read()
    ctx.timing(False)
    ctx.timing_reset()
    assert times["dropout"][1] == 1 and times["dropout"][0] > 0


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("stride, shift", [(520, 0), (524, 4), (523, 1)])
def test_many_tiles_of_weight_gradients_accumulate_in_fp32(ctx, kind, stride, shift):
    """Micro-batches summed in fp32 matrices of any alignment, an empty group
    among them: whole numbers up to 2 * 4 * 300 + 50, exact in fp32."""
    rng = np.random.default_rng(31)
    G, K, N = 40, 520, 264
    off = offsets_of([300, 0, 41] + [7] * (G - 3))
    R = int(off[-1])
    x, dy, before = whole(rng, R, K), whole(rng, R, N), whole(rng, G, N, K, top=50)
    say(f"accumulate fp32 {kind} stride={stride} shift={shift}")
    dw = Rows("f32", G * N, K, stride, shift, before.reshape(G * N, K))
    hx, hdy, o = Rows(kind, R, K, data=x), Rows(kind, R, N, data=dy), device_offsets(off)
    d = gt.grouped_desc(VALUES[kind], G, R, K, N, K, N, stride, N * stride)
    want = before
    for _ in range(2):
        gt.grouped_weight_gradient(ctx, d, o.data_ptr(), hdy.ptr, hx.ptr, dw.ptr, gt.VALUES_FLOAT32, True, stream())
        want = want + grouped(off, x, np.zeros((G, N, K)), dy)[2]
    assert np.array_equal(dw.get(), want.reshape(G * N, K)) and dw.outside_is_untouched()
    gt.grouped_weight_gradient(ctx, d, o.data_ptr(), hdy.ptr, hx.ptr, dw.ptr, gt.VALUES_FLOAT32, False, stream())
    assert np.array_equal(dw.get(), ((want - before) / 2).reshape(G * N, K)) and dw.outside_is_untouched()


# rows and ranks: few rows; tiles with the rows in order; rows sorted by adapter
FORMS = [(20, 8), (300, 8), (300, 24), (2100, 64), (8200, 16), (5470, 24)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("T, rank", FORMS)
@pytest.mark.parametrize("pattern", ["one", "runs", "each its own"])
def test_adapted_holds_the_ranks_products_in_fp32_in_every_form(ctx, kind, T, rank, pattern):
    """Down x is 1 + 2^-9 + 2^-18 in one rank and 1 + 2^-9 in another, whose Up
    values cancel up to their last bits: 2^10 2^-18 is left, and nothing where
    Down x is held in 16 bits."""
    K, N, n = 16, 40, 7
    rng = np.random.default_rng(T + rank)
    x = np.zeros((T, K))
    x[:, 0], x[:, 1], x[:, 2] = 1.0, 2.0 ** -9, 2.0 ** -9
    down, up = np.zeros((n, rank, K)), np.zeros((n, N, rank))
    for a in range(n):
        i, j = rng.choice(rank, 2, replace=False)
        down[a, [i, j], 0], down[a, [i, j], 1], down[a, i, 2] = 1.0, 1.0, 2.0 ** -9
        up[a, :, i] = 2.0 ** 10 * rng.choice([-1.0, 1.0], N)
        up[a, :, j] = -up[a, :, i]
    adapter = adapters_of(rng, pattern, T, n)
    say(f"fp32 ranks {kind} T={T} rank={rank} {pattern}")
    for w, base in ((np.zeros((N, K)), None), (None, np.zeros((T, N)))):
        got = run_adapted(ctx, kind, x, w, None, adapter, down, up, np.ones(n), base=base)
        ref, _ = adapted(x, w, None, adapter, down, up, np.ones(n), base=base)
        assert set(np.unique(np.abs(ref))) <= {0.0, 2.0 ** -8}
        assert np.array_equal(got, ref)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("T, rank", FORMS)
@pytest.mark.parametrize("pattern", ["one", "runs", "each its own"])
def test_adapted_ranks_of_unlike_sizes(ctx, kind, T, rank, pattern):
    """Ranks whose products with the row are up to 2^24 apart, Up's values as far
    apart the other way: every rank weighs the same in the output."""
    K, N, n = 64, 72, 7
    rng = np.random.default_rng(T * 3 + rank)
    make = lambda *s, f=1.0: rounded(rng.normal(size=s) * f, kind)
    x, w, b = make(T, K), make(N, K), make(N)
    size_of = 2.0 ** (12 - 24 * rng.permutation(rank) / max(rank - 1, 1)).round()
    down, up = make(n, rank, K, f=size_of[:, None]), make(n, N, rank, f=1 / size_of)
    scales = np.float32(rng.uniform(0.5, 2, size=n)).astype(np.float64)
    adapter = adapters_of(rng, pattern, T, n)
    say(f"unlike ranks {kind} T={T} rank={rank} {pattern}")
    for ww, base in ((w, None), (None, make(T, N))):
        got = run_adapted(ctx, kind, x, ww, b, adapter, down, up, scales, base=base)
        ref, size = adapted(x, ww, b, adapter, down, up, scales, base=base)
        # K terms of the shared sum; K, the scale and rank terms of the adapter's; bias and the two parts' sum
        bound = HALF_STEP[kind] * np.abs(ref) + HALF_LAST_STEP[kind] + (K + rank + 4) * 2.0 ** -24 * size
        assert np.all(np.abs(got - ref) <= bound * (1 + 2.0 ** -7))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("T, rank", [(20, 8), (140, 8), (300, 24), (2100, 64), (8200, 16)])
def test_adapted_infinities_of_a_row_stay_in_it(ctx, kind, T, rank):
    """A row with an infinity, or whose Down product overflows fp32, is not finite;
    the rows beside it, of the same adapter or another, are as without it."""
    rng = np.random.default_rng(33)
    K, N, n = 72, 40, 4
    sparse = lambda *s: whole(rng, *s, top=1) * (rng.random(s) < 0.25)
    x, w = whole(rng, T, K, top=1), whole(rng, N, K)
    down, up, scales = sparse(n, rank, K), sparse(n, N, rank), np.ones(n)
    down[:, :, 5] = up[:, :, 0] = 1.0
    scales[3] = 2.0 ** 125
    x[:, 5] = 0.0
    adapter = np.where(np.arange(T) % 4 == 3, -1, np.arange(T) % 3)
    base = whole(rng, T, N)
    say(f"infinities {kind} T={T} rank={rank}")
    for ww, start in ((w, None), (None, base)):
        clean = run_adapted(ctx, kind, x, ww, None, adapter, down, up, scales, base=start)
        bad, a = x.copy(), adapter.copy()
        bad[4, 5], bad[9, 5] = np.inf, -np.inf
        a[10], bad[10, 5] = 3, 4096.0  # 2^125 4096
        got = run_adapted(ctx, kind, bad, ww, None, a, down, up, scales, base=start)
        keep = ~np.isin(np.arange(T), [4, 9, 10])
        assert np.array_equal(got[keep], clean[keep])
        assert not np.any(np.isfinite(got[[4, 9, 10]]))

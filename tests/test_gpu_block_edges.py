"""The operators of a block in plain rows where rows, sizes and numbers end: against the plain
64-bit forms of tests/plain_block.py, bounds as in tests/test_gpu_block_rows.py.  U is fp32's largest
relative rounding error."""
import numpy as np
import pytest
import torch

import gotransformers_amd as gt
from tests import plain_block as plain
from tests.device_rows import Rows, rounded, say, stream
from tests.plain_rows import HALF_LAST_STEP, HALF_STEP, VALUES
from tests.test_gpu_block_rows import Product, whole

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
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


# --------------------------------------------------------------------------
# norm
# --------------------------------------------------------------------------

# rows that leave threads of the last workgroup without one: by one workgroup and by many
SHAPES = [(5, 100), (300, 100), (5, 300), (1001, 300), (521, 1000), (3, 1000), (5, 2048), (3, 20000)]


def gradient_of_norm(ctx, kind, s, dy, w, epsilon, ds=None, onto=False):
    """(s, dy, w, ds as they are on the device, dx, dw in fp32) of one call; onto: dx in ds' place."""
    rows, columns = s.shape
    s, dy, w = Rows(kind, rows, columns, data=s), Rows(kind, rows, columns, data=dy), Rows(kind, 1, columns, data=w[None])
    ds = None if ds is None else Rows(kind, rows, columns, data=ds)
    past = None if ds is None else ds.get()
    dx, dw = ds if onto else Rows(kind, rows, columns), Rows("f32", 1, columns)
    d = gt.norm_desc(VALUES[kind], rows, columns, epsilon)
    ws = workspace(gt.norm_workspace_bytes(d))
    gt.norm_gradient(ctx, d, dy.ptr, s.ptr, w.ptr, None if ds is None else ds.ptr, dx.ptr, dw.ptr, gt.VALUES_FLOAT32, False,
                     ws.data_ptr(), stream())
    torch.cuda.synchronize()
    assert bool((ws[-64:] == 0xA5).all())
    dx.check_outside()
    dw.check_outside()
    return s.get(), dy.get(), w.get()[0], past, dx.get(), dw.get()[0]


def check_gradient_of_norm(ctx, kind, s, dy, w, epsilon, ds=None):
    s, dy, w, ds, dx, dw = gradient_of_norm(ctx, kind, s, dy, w, epsilon, ds)
    rows, columns = s.shape
    rdx, rdw, xsize, wsize = plain.norm_gradient(dy, s, w, ds, epsilon)
    near(dx, rdx, xsize * (2 * columns + 24) * U, kind)
    near(dw, rdw, wsize * (rows + columns / 2 + 16) * U, "f32")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows, columns", SHAPES)
@pytest.mark.parametrize("epsilon", [0.0, 1e-80])
def test_norm_gradient_without_epsilon(ctx, kind, rows, columns, epsilon):
    say(f"norm gradient {kind} {rows} x {columns} epsilon {epsilon}")
    rng = np.random.default_rng(rows + columns)
    make = lambda: rng.normal(size=(rows, columns))
    check_gradient_of_norm(ctx, kind, make() * 2, make(), make()[0] + 1, epsilon, make())


@pytest.mark.parametrize("rows, columns", SHAPES)
@pytest.mark.parametrize("epsilon", [0.0, 1e-6])
def test_norm_gradient_of_squares_beyond_fp32(ctx, rows, columns, epsilon):
    rng = np.random.default_rng(rows + columns)
    make = lambda: rng.normal(size=(rows, columns))
    size = np.resize([1e25, 1.0, 1e-20, 1e30, 1e-25], rows)[:, None]
    check_gradient_of_norm(ctx, "f32", make() * size, make(), make()[0] + 1, epsilon)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows, columns", SHAPES)
def test_norm_gradient_onto_the_sums_gradients(ctx, kind, rows, columns):
    rng = np.random.default_rng(rows * 3 + columns)
    s, dy, ds = (rng.normal(size=(rows, columns)) for _ in range(3))
    w = rng.normal(size=columns)
    apart = gradient_of_norm(ctx, kind, s, dy, w, 1e-6, ds)
    onto = gradient_of_norm(ctx, kind, s, dy, w, 1e-6, ds, True)
    assert np.array_equal(apart[4], onto[4]) and np.array_equal(apart[5], onto[5])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows, columns", SHAPES)
def test_norm_of_rows_next_to_the_ends_of_fp32(ctx, kind, rows, columns):
    """Without epsilon 1 / sqrt(mean(s^2)) of rows of subnormal numbers is beyond fp32, of the largest
    subnormal: the quotient and the weights' gradients are of the size of one all the same."""
    rng = np.random.default_rng(rows + 5 * columns)
    say(f"norm at the ends {kind} {rows} x {columns}")
    top = 3.4e38 if kind == "f32" else 3.3e38
    size = np.resize([1e-40, 2e38, 1e-38, 3e-37, top], rows)[:, None]
    v = rng.uniform(-1, 1, size=(rows, columns)) * size
    v[0, 1::2] = 0.0
    x, y, w = Rows(kind, rows, columns, data=v), Rows(kind, rows, columns), rng.normal(size=columns) + 1
    hw = Rows(kind, 1, columns, data=w[None])
    d = gt.norm_desc(VALUES[kind], rows, columns, 0.0)
    gt.norm_forward(ctx, d, x.ptr, None, hw.ptr, None, y.ptr, None, None, stream())
    want, _ = plain.norm(x.get(), hw.get()[0], 0.0)
    # the inverse from 64 bits and two products; a product with the power of two may leave subnormal bits, half a
    # step of 2^-149 beside s r of the row's size 1
    near(y.get(), want, (4 * np.abs(want) + np.abs(hw.get())) * U, kind)
    # output gradients so small that the input gradients are numbers of fp32, and no smaller: their products
    # with s r, of the size of one, stay normal numbers
    dy = rng.normal(size=(rows, columns)) * np.where(size < 1e-30, 1e-10, 0.01)
    check_gradient_of_norm(ctx, kind, v, dy, w, 0.0)


@pytest.mark.parametrize("columns", [100, 2048, 20000])
def test_norm_of_the_smallest_numbers(ctx, columns):
    """A row of 2^-149, the next with zeros in it; codes of their quotients."""
    v = np.zeros((3, columns))
    v[0], v[1, ::3], v[2] = 2.0 ** -149, -2.0 ** -149, 1.0
    x, y, q, k = Rows("f32", 3, columns, data=v), Rows("f32", 3, columns), Rows("u8", 3, columns), Rows("f32", 3, 1)
    d = gt.norm_desc(gt.VALUES_FLOAT32, 3, columns, 0.0, gt.CODES_INT8, 0)
    gt.norm_forward(ctx, d, x.ptr, None, None, None, y.ptr, q.ptr, k.ptr, stream())
    want, _ = plain.norm(x.get(), None, 0.0)
    near(y.get(), want, 4 * np.abs(want) * U, "f32")
    assert np.array_equal(q.get().view(np.int8), np.sign(v) * 127)


# --------------------------------------------------------------------------
# activations
# --------------------------------------------------------------------------

ACTS = {"none": gt.ACTIVATION_NONE, "relu": gt.ACTIVATION_RELU, "silu": gt.ACTIVATION_SILU, "gelu": gt.ACTIVATION_GELU,
        "gelu_tanh": gt.ACTIVATION_GELU_TANH}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", list(ACTS))
def test_activation_of_the_largest_gates(ctx, kind, act):
    """Where act(z) is z or 0, and act' 1 or 0, all but exactly: up to the type's largest number."""
    top = float(torch.finfo({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[kind]).max)
    z = np.array([1e3, 1e4, 65504.0] + ([] if kind == "f16" else [1e10, 1.8e19, 1e20, 1e30]) + [top])
    z = np.concatenate([z, -z])[None]
    n = z.shape[1]
    g, u, dy = Rows(kind, 1, n, data=z), Rows(kind, 1, n, data=np.full((1, n), 0.5)), Rows(kind, 1, n, data=np.full((1, n), 0.25))
    y, dg, du = (Rows(kind, 1, n) for _ in range(3))
    d = gt.activation_desc(VALUES[kind], 1, n, ACTS[act])
    gt.activation_forward(ctx, d, g.ptr, u.ptr, y.ptr, stream=stream())
    z = g.get()
    on = np.ones_like(z) if act == "none" else (z > 0).astype(float)
    assert np.array_equal(y.get(), z * on / 2)
    gt.activation_gradient(ctx, d, dy.ptr, g.ptr, None, u.ptr, None, dg.ptr, du.ptr, y.ptr, stream())
    assert np.array_equal(y.get(), z * on / 2) and np.array_equal(dg.get(), on / 8) and np.array_equal(du.get(), z * on / 4)


def curve(ctx, kind, act, z):
    """(act, act') at z by the operators."""
    n = z.size
    g, one = Rows(kind, 1, n, data=z[None]), Rows(kind, 1, n, data=np.ones((1, n)))
    y, again, dg = Rows(kind, 1, n), Rows(kind, 1, n), Rows(kind, 1, n)
    d = gt.activation_desc(VALUES[kind], 1, n, ACTS[act])
    gt.activation_forward(ctx, d, g.ptr, None, y.ptr, stream=stream())
    gt.activation_gradient(ctx, d, one.ptr, g.ptr, None, None, None, dg.ptr, None, again.ptr, stream())
    assert bool((again.buffer == y.buffer).all())
    return g.get()[0], y.get()[0], dg.get()[0]


# where act(z) is 2^-150: half of the smallest number
TAILS = {"silu": -108.6, "gelu": -14.3, "gelu_tanh": -10.9}


@pytest.mark.parametrize("act", list(TAILS))
def test_activation_of_fp32_rows(ctx, act):
    """Bounds, in units of 2^-24 of the value, or for the slope of its terms: SiLU's and the tanh form's
    power of two 2.2 (a unit of the hardware's, the argument's fraction), the reciprocal 3.2, two products: 8.
    GELU's power 2.2, its t 2.6, the polynomial's fit 1.1 and roundings 4, three products: 14.  Slopes take three
    more roundings of each term, the tanh form's four of the argument's slope."""
    rng = np.random.default_rng(1)
    z = np.concatenate([np.linspace(TAILS[act], 20, 20001), rng.normal(size=20000) * 3, rng.normal(size=200) * 1e-30])
    z, y, slope = curve(ctx, "f32", act, z)
    want, d, size = plain.activation(z, act)
    near(y, want, 16 * U * np.abs(want), "f32")
    near(slope, d, 24 * U * size + 2.0 ** -148, "f32")
    near_by = (z > -8) & (z < 8) & (np.abs(z) > 1e-3)
    rms = lambda e: float(np.sqrt(np.mean(e * e)))
    say(f"{act} rms relative error {rms((y / want - 1)[near_by]):.2e}")


@pytest.mark.parametrize("act", list(TAILS))
def test_activation_of_bf16_rows_to_the_smallest_numbers(ctx, act):
    """2^-14 is 1024 units of 2^-24: of |z|, of z^2 / 2 (GELU) or of five times the argument (the tanh form), up
    to 109, at most 550, and 40 for the functions and products."""
    z = np.linspace(TAILS[act], 4, 4001)
    z, y, slope = curve(ctx, "bf16", act, z)
    want, d, size = plain.activation(z, act)
    assert np.abs(want[z < 0]).min() < 2.0 ** -133
    near(y, want, 2.0 ** -14 * np.abs(want) + 2.0 ** -149, "bf16")
    near(slope, d, 2.0 ** -14 * size + 2.0 ** -148, "bf16")


# --------------------------------------------------------------------------
# the choice of experts
# --------------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens, experts, k, biased", [(300, 64, 6, False), (40, 128, 8, True), (33, 24, 3, False), (20, 700, 20, True)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_route_gates_and_gradients_are_rounded_once(ctx, kind, tokens, experts, k, biased, scores, renormalize):
    """Scores, their sums and the gradients are taken in 64 bits (the exponential to 1e-14, 1024 terms): 1e-12 of
    the terms, and one rounding; a 16-bit gradient is rounded to fp32 first.  Small scores stay as exact."""
    rng = np.random.default_rng(tokens + experts)
    say(f"gates {kind} {tokens} {experts} {k} {biased} {scores} {renormalize}")
    far = np.repeat([1.0, 20.0, 60.0], -(-tokens // 3))[:tokens, None]
    l, dg = rng.normal(size=(tokens, experts)) * far, rng.normal(size=(tokens, k))
    l, dg = Rows(kind, tokens, experts, data=l), Rows("f32", tokens, k, data=dg)
    b = torch.as_tensor(rng.normal(size=experts) * 0.1, dtype=torch.float32).cuda() if biased else None
    chosen, gates, dl = Rows("i32", tokens, k), Rows("f32", tokens, k), Rows(kind, tokens, experts)
    d = gt.route_desc(VALUES[kind], tokens, experts, k, scores=gt.SCORES_SIGMOID if scores == "sigmoid" else gt.SCORES_SOFTMAX,
                      renormalize=renormalize, scale=0.1)
    gt.route_forward(ctx, d, l.ptr, None if b is None else b.data_ptr(), chosen.ptr, gates.ptr, stream=stream())
    want, wgates = plain.route(l.get(), None if b is None else b.double().cpu().numpy(), k, scores, renormalize=renormalize, scale=0.1)
    assert np.array_equal(chosen.get(), want)
    near(gates.get(), wgates, 1e-12 * np.abs(wgates), "f32")
    gt.route_gradient(ctx, d, l.ptr, chosen.ptr, dg.ptr, dl.ptr, stream())
    ref, size = plain.route_gradient(l.get(), want, dg.get(), scores, renormalize, 0.1)
    near(dl.get(), ref, 1e-12 * size + (0.0 if kind == "f32" else np.abs(ref) * U + 2.0 ** -150), kind)


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("renormalize", [False, True])
def test_route_gates_of_what_is_not_finite(ctx, biased, renormalize):
    """Of a softmax: a sum that NaN or +infinity is in leaves no gate finite, other tokens' gates stay."""
    rng = np.random.default_rng(3)
    l = rng.normal(size=(40, 32))
    l[3, 5], l[8, 0], l[9] = np.nan, np.inf, np.nan
    l = Rows("f32", 40, 32, data=l)
    b = torch.zeros(32, device="cuda") if biased else None
    chosen, gates = Rows("i32", 40, 4), Rows("f32", 40, 4)
    d = gt.route_desc(0, 40, 32, 4, renormalize=renormalize)
    gt.route_forward(ctx, d, l.ptr, None if b is None else b.data_ptr(), chosen.ptr, gates.ptr, stream=stream())
    got = gates.get()
    sums = [9] if renormalize else [3, 8, 9]
    if 0 in chosen.get()[8]:
        sums.append(8)
    assert not np.isfinite(got[sums]).any()
    assert np.isfinite(got[np.setdiff1d(np.arange(40), [3, 8, 9])]).all()


# --------------------------------------------------------------------------
# bias gradients
# --------------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sizes, columns", [([300], 130), ([32], 2048), ([9000, 0, 3, 4000], 70), ([1, 700] * 40, 33)])
def test_bias_gradients_are_rounded_once(ctx, kind, sizes, columns):
    """Sums in 64 bits: below 2^-40 of the terms, 2^14 at most, and one rounding, also where terms of 1e4 cancel."""
    off = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    R, G = int(off[-1]), len(sizes)
    rng = np.random.default_rng(R)
    v = rng.normal(size=(R, columns)) + 1e4 * (-1.0) ** np.arange(R)[:, None]
    dy, db = Rows(kind, R, columns, data=v), Rows("f32", G, columns)
    d = gt.grouped_desc(VALUES[kind], G, R, 8, columns)
    dev, ws = torch.from_numpy(off).cuda(), workspace(gt.grouped_bias_workspace_bytes(d))
    # (the workspace as a buffer, whose size is checked)
    with pytest.raises(gt.InvalidArgument, match="the workspace has 16 bytes"):
        gt.grouped_bias_gradient(ctx, d, dev.data_ptr(), dy.ptr, db.ptr, gt.VALUES_FLOAT32, False, ws[:16], stream())
    gt.grouped_bias_gradient(ctx, d, dev.data_ptr(), dy.ptr, db.ptr, gt.VALUES_FLOAT32, False, ws, stream())
    v = dy.get()
    want = np.stack([v[off[g]:off[g + 1]].sum(axis=0) for g in range(G)])
    size = np.stack([np.abs(v[off[g]:off[g + 1]]).sum(axis=0) for g in range(G)])
    near(db.get(), want, size * 2.0 ** -40, "f32")
    assert bool((ws[-64:] == 0xA5).all())


# --------------------------------------------------------------------------
# products with an epilogue
# --------------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("groups, rows", [(65, 13), (130, 5), (300, 45), (300, 46), (200, 200)])
@pytest.mark.parametrize("widths", [(72, 136), (129, 130)])
@pytest.mark.parametrize("layout", ["packed", "odd"])
def test_fused_product_of_few_rows_in_many_groups(ctx, kind, groups, rows, widths, layout):
    """Whole numbers, exact in fp32; the 64th group, the next and the last are among those with rows.  Three
    rows more are of no group: 48 of all are the few rows' kernel's, 49 the tiles'."""
    rng = np.random.default_rng(groups + rows)
    sizes = np.bincount(np.concatenate([[63, 64, groups - 1], rng.integers(0, groups, size=rows - 3)]), minlength=groups)
    p = Product(kind, (list(sizes), 1), widths, layout, "bfrp", "relu", whole)
    say(f"few rows {kind} {groups} {rows} {widths} {layout}")
    p.call(ctx)
    z, _, _, y = p.reference()
    inside = slice(p.off[0], p.off[-1])
    for have, want in ((p.y, y), (p.z, z)):
        got = have.get()
        assert np.array_equal(got[inside], rounded(want, kind)[inside]) and p.untouched(got)
        have.check_outside()

"""The operators of a block in plain rows where rows, sizes and numbers end: against the plain
64-bit forms of tests/plain_block.py, bounds as in tests/test_gpu_block_rows.py.  U is fp32's largest
relative rounding error."""
import numpy as np
import pytest
import torch

import gotransformers_amd as gt
from tests import plain_block as plain
from tests.device_rows import Rows, say, stream
from tests.plain_rows import HALF_LAST_STEP, HALF_STEP, VALUES

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

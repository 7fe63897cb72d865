"""Dropout on the adapters' inputs in the training path, against the oracle
with the same masks (made by the plain generator of tests/plain_rows.py), and
the oracle's own gradients with masks against finite differences (CPU).  Bars
as in test_gpu_lora.py."""
import numpy as np
import pytest

import gotransformers_amd as gt
from oracle import lora
from tests.moe_fixtures import FLOAT32, FP4, INT8, make_moe
from tests.plain_rows import dropout_factor

FWD_TOL, GRAD_TOL = 1e-4, 2e-4
OFFSET = {"gate": 0, "up": 1, "down": 2, "router": 3}


def masks(rate, seed, call, rows):
    """The factors of forward number `call`, as oracle.lora.forward takes them."""
    def dropout(which, positions, columns):
        return dropout_factor(rows, columns, rate, seed, 4 * call + OFFSET[which])[0][positions]
    return dropout


@pytest.mark.parametrize("hashed", [False, True])
def test_oracle_gradients_with_dropout(hashed):
    spec = make_moe(gt.encode_rows, d=5, h=6, E=3, k=2, S=1, precision=FLOAT32, seed=2, use_hash=hashed)
    rng = np.random.default_rng(3)
    adapters = lora.make_adapters(spec, 2, 4.0, rng)
    T = 4
    x = rng.normal(size=(T, 5))
    ids = np.arange(T) if hashed else None
    dropout = masks(0.4, 11, 2, T * 3)
    assert lora.gradient_check(spec, adapters, x, ids, dropout=dropout) == []
    a, _ = lora.forward(spec, adapters, x, ids)
    b, _ = lora.forward(spec, adapters, x, ids, dropout=dropout)
    assert not np.allclose(a, b)


def rel(a, b):
    return float(np.max(np.abs(a - b)) / max(float(np.max(np.abs(b))), 1e-30))


CASES = {
    # name: (d, h, E, k, S, precision, clamp, hash, T, rank)
    "ragged int8 shared": (37, 53, 5, 2, 1, INT8, 0.0, False, 29, 4),
    "fp4 clamped": (64, 96, 6, 3, 2, FP4, 0.3, False, 17, 5),
    "hash routing": (32, 48, 6, 2, 1, FP4, 0.0, True, 11, 4),
    "many positions": (256, 128, 4, 2, 1, INT8, 0.0, False, 300, 16),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CASES))
def test_training_with_adapter_dropout(name):
    d, h, E, k, S, prec, clamp, hashed, T, rank = CASES[name]
    print(f"adapter dropout {name}", flush=True)
    spec = make_moe(gt.encode_rows, d=d, h=h, E=E, k=k, S=S, precision=prec, seed=5, clamp=clamp,
                    use_hash=hashed)
    rng = np.random.default_rng(6)
    adapters = lora.make_adapters(spec, rank, 2.0 * rank, rng, up_scale=0.2)
    ids = rng.integers(0, 1000, T) if hashed else None
    xs, gs = rng.normal(size=(2, T, d)), rng.uniform(-1, 1, (2, T, d))
    rate, seed = 0.3, 0xABCDEF0123456789
    with gt.Context(0) as ctx:
        m = gt.MixtureOfExperts.from_spec(ctx, spec)
        try:
            m.add_adapters(rank, 2.0 * rank)
            for (kind, i, which), ad in adapters.items():
                m.set_adapter(kind, i, which, ad.down, ad.up)
            plain = m.forward(xs[0], ids)
            m.set_adapter_dropout(rate, seed)
            grads = lora.zero_grads(spec, adapters)
            for call in range(2):  # gradients add up over micro-batches, each with its own masks
                y = m.forward(xs[call], ids)
                r = m.last_routing()
                # what is set between a forward and its backward counts for the next forward
                m.set_adapter_dropout(0.0) if call == 1 else None
                dx = m.backward(gs[call])
                ref_y, st = lora.forward(spec, adapters, xs[call], ids, chosen=None if hashed else r.chosen,
                                         dropout=masks(rate, seed, call, T * (S + k)))
                ref_dx = lora.backward(spec, adapters, st, gs[call], grads)
                assert rel(y, ref_y) <= FWD_TOL
                assert rel(dx, ref_dx) <= GRAD_TOL
                assert call or rel(y, plain) > 10 * FWD_TOL
            for (kind, i, which), (dn, up) in grads.items():
                if kind == "router" and hashed:
                    continue
                got = m.adapter_gradients(kind, i, which)
                assert rel(got[0], dn) <= GRAD_TOL or np.max(np.abs(dn)) == 0 == np.max(np.abs(got[0]))
                assert rel(got[1], up) <= GRAD_TOL or np.max(np.abs(up)) == 0 == np.max(np.abs(got[1]))
            # off: as before the dropout, bit for bit; the same seed again: the same masks again
            assert np.array_equal(m.forward(xs[0], ids), plain)
            m.set_adapter_dropout(rate, seed)
            again = m.forward(xs[0], ids)
            m.set_adapter_dropout(rate, seed)
            assert np.array_equal(m.forward(xs[0], ids), again)
            assert not np.array_equal(m.forward(xs[0], ids), again)  # the next call's masks
            m.remove_adapters()
            m.add_adapters(rank, 2.0 * rank)
            for (kind, i, which), ad in adapters.items():
                m.set_adapter(kind, i, which, ad.down, ad.up)
            assert np.array_equal(m.forward(xs[0], ids), plain)
        finally:
            m.destroy()


@pytest.mark.gpu
def test_adapter_dropout_refusals():
    spec = make_moe(gt.encode_rows, d=16, h=16, E=2, k=1, S=0, precision=INT8, seed=1)
    with gt.Context(0) as ctx:
        m = gt.MixtureOfExperts.from_spec(ctx, spec)
        try:
            with pytest.raises(gt.GtmoeError, match="no low-rank adapters"):
                m.set_adapter_dropout(0.1)
            m.add_adapters(2, 4.0)
            for rate in (-0.1, 1.0, float("nan")):
                with pytest.raises(gt.InvalidArgument, match="rate must be"):
                    m.set_adapter_dropout(rate)
        finally:
            m.destroy()


@pytest.mark.gpu
def test_failed_forward_leaves_nothing_for_the_backward():
    """A forward that runs out of memory -- where the masked inputs are
    allocated, the training buffers or the forward's own -- leaves no state of
    the forward before it behind: the backward answers that there is none.  The
    next forward takes the masks the failed one would have taken."""
    d, h, S, k, T, rank = 40, 56, 1, 2, 9, 4
    spec = make_moe(gt.encode_rows, d=d, h=h, E=4, k=k, S=S, precision=INT8, seed=9)
    rng = np.random.default_rng(10)
    adapters = lora.make_adapters(spec, rank, 2.0 * rank, rng, up_scale=0.2)
    x, g = rng.normal(size=(T, d)), rng.uniform(-1, 1, (T, d))
    big = rng.normal(size=(300, d))
    rate, seed = 0.4, 1234567
    with gt.Context(0) as ctx:
        m = gt.MixtureOfExperts.from_spec(ctx, spec)
        try:
            m.add_adapters(rank, 2.0 * rank)
            for (kind, i, which), ad in adapters.items():
                m.set_adapter(kind, i, which, ad.down, ad.up)

            def check(call):
                """A forward and its backward with the masks of forward number `call`."""
                m.zero_adapter_gradients()
                y, r = m.forward(x), m.last_routing()
                dx = m.backward(g)
                grads = lora.zero_grads(spec, adapters)
                ref_y, st = lora.forward(spec, adapters, x, chosen=r.chosen, dropout=masks(rate, seed, call, T * (S + k)))
                ref_dx = lora.backward(spec, adapters, st, g, grads)
                assert rel(y, ref_y) <= FWD_TOL and rel(dx, ref_dx) <= GRAD_TOL
                got, ref = m.adapter_gradients("shared", 0, "down"), grads[("shared", 0, "down")]
                assert rel(got[0], ref[0]) <= GRAD_TOL and rel(got[1], ref[1]) <= GRAD_TOL

            def fails(rows):
                print(f"adapter dropout: a forward of {rows.shape[0]} rows without memory", flush=True)
                gt.inject_failure("hipMalloc", gt.ERR_OUT_OF_MEMORY)
                with pytest.raises(gt.GtmoeError, match="out of memory"):
                    m.forward(rows)
                for tokens in (x, big):
                    with pytest.raises(gt.GtmoeError, match="call Forward before Backward") as info:
                        m.backward(np.zeros_like(tokens))
                    assert info.value.code == gt.ERR_NOT_READY

            m.forward(x)  # without dropout: its allocations are all but the masked inputs'
            m.set_adapter_dropout(rate, seed)
            fails(x)
            fails(x)
            check(0)
            check(1)
            fails(big)  # the forward's workspace
            m.remove_adapters()
            m.forward(big)  # the workspace has room now
            m.add_adapters(rank, 2.0 * rank)
            for (kind, i, which), ad in adapters.items():
                m.set_adapter(kind, i, which, ad.down, ad.up)
            m.set_adapter_dropout(rate, seed)
            check(0)
            fails(big)  # the training buffers
            check(1)
            # a call that is refused before it starts changes nothing
            y = m.forward(x)
            with pytest.raises(gt.InvalidArgument):
                m.backward(np.zeros((T + 1, d)))
            assert y.shape == m.backward(g).shape
        finally:
            m.destroy()

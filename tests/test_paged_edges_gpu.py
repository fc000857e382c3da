"""Paged operators where single rules meet: idle sequences beside busy ones, weights that hang far below a row's largest, ends of the ranges."""
import ctypes as C

import numpy as np
import pytest

import _paged as P
import test_logits_rules_gpu as L
from _support import load_package

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    f = load_package().ffi
    f.require_device()
    return f


@pytest.mark.parametrize("cache,qt", [("f16", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16")])
def test_sequences_without_positions_between_others(g, cache, qt):
    """A captured step's idle slots: one row and no position.  Many lists to a CTA, every second one empty; the same bits every time."""
    specs = [(1, 0 if b % 2 else 1 + b % 64) for b in range(512)]
    bt = P.Batch(specs, 16, 8, 64, 16, cache, seed=41)
    bt.upload()
    q = P.random_queries(bt, qt)
    q64 = P.to_f64(q, qt)
    want, mag = P.attention64(bt, q64)
    first = P.run_attention(bt, q, qt)
    assert (np.abs(P.to_f64(first, qt) - want) <= P.attention_tolerance(bt, q64, want, mag, qt)).all()
    assert (P.to_f64(first, qt)[1::2] == 0).all()
    for _ in range(20):
        assert np.array_equal(P.run_attention(bt, q, qt).view(P.itype(qt)), first.view(P.itype(qt)))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,V,hist", [(6, 500, 0), (3, 40000, 0), (20, 50257, 0), (6, 2000, 40)])
def test_zeros_of_both_signs_are_one_value(g, t, M, V, hist):
    """The first of a row's largest values where these are -0 and +0, in lanes of one warp and far apart; the same as the plain arg-max."""
    c = L.Case(M, V, hist=hist, penalties=("repetition",), t=t, seed=51)
    x = -1.0 - np.abs(c.rng.normal(0, 4, (M, V)))
    first = np.zeros(M, int)
    for m in range(M):
        at = np.sort(c.rng.choice(V, 4, replace=False)) if m % 2 else np.array([5, 77, 90, 120]) + 7 * m
        x[m, at] = [-0.0, 0.0, -0.0, 0.0]
        first[m] = at[0]
    c.logits[:, :V] = P.to_type(x, t)
    got, nxt = L.run(g, c)
    assert np.array_equal(nxt, first)
    if t == "f32":
        rows, one = P.device(got), g.DeviceBuffer(4)
        for m in range(M):
            g.check(g.cuda().greta_cuda_argmax(None, rows.ptr + m * c.ld * 4, V, one.ptr))
            assert one.download(np.int32)[0] == first[m]

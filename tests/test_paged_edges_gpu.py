"""Paged operators where single rules meet: idle sequences beside busy ones, weights that hang far below a row's largest, ends of the ranges."""
import ctypes as C

import numpy as np
import pytest

import _paged as P
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

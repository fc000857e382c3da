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


def check_sink(cache, qt, rows, nats, n=4097, H=8, G=2, window=0):
    """A first key of no value whose score is `nats` above all others', alike in a head: what a row's outputs are made of hangs far below its largest weight, and a weight's
    rounding does not average out."""
    d, page = 64, 32
    bt = P.Batch([(rows, n)], H, G, d, page, cache, seed=rows)
    k = np.zeros((n, G, d))
    k[:, :, 0] = 20 - nats
    k[0, :, 0] = 20
    v = bt.rng.normal(2, 1, (n, G, d))
    v[0] = 0
    p = np.arange(n)
    bt.k[bt.table[0, p // page], :, p % page] = P.to_type(k, cache).view(np.uint16)
    bt.v[bt.table[0, p // page], :, p % page] = P.to_type(v, cache).view(np.uint16)
    bt.upload()
    q64 = np.zeros((rows, H, d))
    q64[:, :, 0] = 8 - np.arange(H) / 8  # exact, as its products with the keys are
    got = P.to_f64(P.run_attention(bt, P.to_type(q64, qt), qt, scale=0.125), qt)
    want, mag = P.attention64(bt, q64, scale=0.125)
    # In powers of two: scores up to X are rounded as they are scaled, and their largest, by the scale's 2^-23 of their distance D and in the subtraction.  Exponential and split: 2^-22 each.
    X, D, one = 20 * 1.4427, nats * 1.4427, 2.0 ** -24
    weight = np.log(2) * one * (3 * D + 2 * X) + 2.0 ** -21
    # Sums: a tile of 64 keys to the next, of weights and of outputs; within one four products of every term and eight sums.
    sums = (2 * n / 64 + 32) * one
    least = 2.0 ** -40 if cache == "f16" else 0.0  # of the largest weight: where fp16's steps end
    if qt != "f32":  # probabilities of 16 bits, at least 2^7 times as large as the weight against the row's largest
        weight, least = weight + P.HALF[qt], 2.0 ** -32 if cache == "f16" else 0.0
    seen = np.abs(P.to_f64(P.to_type(v, cache), cache)).sum(0).max()
    tol = mag * (2 * weight + sums) + least * seen + np.abs(want) * P.HALF[qt]  # the sum of weights is above 1
    worst = float((np.abs(got - want) / tol).max())
    assert worst <= 1, worst


@pytest.mark.parametrize("nats", [8, 10, 12, 14, 18])
@pytest.mark.parametrize("cache,qt,rows", [("f16", "f32", 1), ("bf16", "f32", 1), ("f16", "f32", 5), ("bf16", "f32", 5), ("f16", "f32", 200), ("f16", "f16", 1), ("bf16", "bf16", 1)])
def test_outputs_that_hang_on_small_weights(g, cache, qt, rows, nats):
    check_sink(cache, qt, rows, nats)


@pytest.mark.parametrize("nats", [8, 10, 12, 14, 18])
@pytest.mark.parametrize("cache,rows", [("f16", 5), ("f16", 200), ("bf16", 200), ("f16", 700)])
def test_outputs_of_portions_that_hang_on_small_weights(g, cache, rows, nats):
    check_sink(cache, cache, rows, nats)


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("specs,H,G", [([(1, 4096)] * 4, 16, 2), ([(1, 20011)], 5, 1), ([(40, 4096)], 4, 2)])
def test_fp32_calls_over_long_lists_keep_fp32_precision(g, cache, specs, H, G):
    """By the root of the mean square.  Weights of one 16-bit value would leave 1e-4 and more; sums kept in the tensor core's accumulators 4e-6."""
    bt = P.Batch(specs, H, G, 128, 64, cache, seed=43)
    bt.upload()
    q = P.random_queries(bt, "f32")
    want, _ = P.attention64(bt, q.astype(np.float64))
    got = P.run_attention(bt, q, "f32").astype(np.float64)
    assert np.sqrt(((got - want) ** 2).mean() / (want ** 2).mean()) <= 2e-6


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("far", [6, 10, 14])
@pytest.mark.parametrize("rows", [1, 5])
def test_small_elements_beside_a_large_one(g, cache, far, rows):
    """fp32 queries whose largest element meets keys of zero there: scores are made of an element that is 2^-far of it, as exactly as if it stood alone."""
    n, H, G, d, page = 500, 4, 2, 64, 32
    bt = P.Batch([(rows, n)], H, G, d, page, cache, seed=61)
    k = np.zeros((n, G, d))
    k[:, :, 1] = np.round(bt.rng.uniform(-64, 64, (n, G)))  # exact in both types
    p = np.arange(n)
    bt.k[bt.table[0, p // page], :, p % page] = P.to_type(k, cache).view(np.uint16)
    bt.upload()
    q = np.zeros((rows, H, d), np.float32)
    q[:, :, 1] = bt.rng.uniform(1, 2, (rows, H))
    q[:, :, 0] = 2.0 ** far
    got = P.run_attention(bt, q, "f32", scale=0.125).astype(np.float64)
    want, mag = P.attention64(bt, q.astype(np.float64), scale=0.125)
    # Scores up to 16: the element by 2^-22 in its terms, two sums, the scale's 2^-23 and one rounding more; of a score and of the largest one.  Exponential and split 2^-22 each, sums of eight tiles.
    weight = 2 * 16 * (2.0 ** -22 + 4 * 2.0 ** -23) + 2.0 ** -21
    assert (np.abs(got - want) <= mag * (2 * weight + 48 * 2.0 ** -24) + 1e-9).all()


def test_rows_of_several_tensors_in_one_buffer(g):
    """Queries, keys, values, rotated queries and outputs as columns of one buffer, and logits beside what is made of them."""
    lib, T, H, G, d, V = g.cuda(), 6, 4, 2, 64, 40
    bt = P.Batch([(4, 4), (2, 2)], H, G, d, 16, "f16", seed=71)
    bt.upload()
    widths = dict(q=H * d, k=G * d, v=G * d, turned=H * d, o=H * d, logits=V, out=V)
    at, ld = {}, 0
    for name, n in widths.items():
        at[name], ld = ld, ld + n
    rng = np.random.default_rng(72)
    x = rng.normal(0, 1, (T, ld)).astype(np.float32)
    buf = P.device(x)
    p = lambda name: buf.ptr + 4 * at[name]
    c, r = bt.structs()
    rot = g.Rotation(dims=d, interleaved=0, base=10000.0, freq=None, amplitude=1.0)
    ws = g.DeviceBuffer(lib.greta_cuda_paged_attn_workspace_bytes(d), zero=True)
    g.check(lib.greta_cuda_paged_append(None, C.byref(c), C.byref(r), C.byref(rot), 0, p("q"), ld, p("k"), ld, p("v"), ld, H, p("turned"), 0, ld))
    g.check(lib.greta_cuda_paged_append(None, C.byref(c), C.byref(r), C.byref(rot), 0, p("q"), ld, p("k"), ld, p("v"), ld, H, p("q"), 0, ld))  # in place between the others
    g.check(lib.greta_cuda_paged_attn(None, C.byref(c), C.byref(r), p("turned"), 0, ld, p("o"), ld, H, 0.125, 0, ws.ptr, ws.nbytes))
    g.check(lib.greta_cuda_logits_adjust(None, C.byref(g.LogitsRules()), 0, p("logits"), ld, p("out"), ld, T, V, None))
    y = buf.download(np.float32).reshape(T, ld)
    col = lambda a, name: a[:, at[name]:at[name] + widths[name]]
    for name in ("k", "v", "logits"):
        assert np.array_equal(col(y, name), col(x, name))
    assert np.array_equal(col(y, "out"), col(x, "logits")) and np.array_equal(col(y, "q"), col(y, "turned"))
    for pool, name in ((bt.dk, "k"), (bt.dv, "v")):
        setattr(bt, name, pool.download(np.uint16).reshape(bt.k.shape))
    q64 = col(y, "turned").reshape(T, H, d).astype(np.float64)
    want, mag = P.attention64(bt, q64)
    assert (np.abs(col(y, "o").reshape(T, H, d) - want) <= P.attention_tolerance(bt, q64, want, mag, "f32")).all()


@pytest.mark.parametrize("cache,qt,rows", [("f16", "f32", 1), ("bf16", "bf16", 1), ("f16", "f32", 40), ("f16", "f16", 40)])
@pytest.mark.parametrize("spoilt", [False, True])
def test_positions_up_to_the_end_of_the_range(g, cache, qt, rows, spoilt):
    """A table for 2^31 - 8 positions, all in use, and a window over the last of them; NaN in hidden values of the last page where `spoilt`."""
    page, d, H, G, window = 8, 64, 4, 2, 100
    ld, near = 2 ** 28 - 1, 1024  # the last 1024 positions have pages of their own
    bt = P.Batch([(rows, near)], H, G, d, page, cache, seed=81)
    if spoilt:  # of the last position, which the last row alone sees
        bt.v[bt.table[0, -1], :, page - 1, 5] = P.NAN16
    bt.upload()
    q = P.random_queries(bt, qt)
    q64 = P.to_f64(q, qt)
    if spoilt:
        clean = bt.v.copy()
        bt.v[bt.table[0, -1], :, page - 1, 5] = 0
        want, mag = P.attention64(bt, q64, window)
        tol, bt.v = P.attention_tolerance(bt, q64, want, mag, qt), clean
    else:
        want, mag = P.attention64(bt, q64, window)
        tol = P.attention_tolerance(bt, q64, want, mag, qt)
    table = g.DeviceBuffer(4 * ld)
    table.fill(0xFF)
    table.upload(bt.table[0, :near // page], offset=4 * (ld - near // page))
    bt.dt, bt.dl = table, P.device(np.array([ld * page], np.uint32))
    bt.table = np.broadcast_to(np.int32(-1), (1, ld))
    got = P.to_f64(P.run_attention(bt, q, qt, window), qt)
    right = np.abs(got - want) <= tol
    if spoilt:
        assert not np.isfinite(got[-1, :, 5]).any()
        right[-1, :, 5] = True
    assert right.all()


@pytest.mark.parametrize("cache,qt,batch", [("bf16", "f32", 15), ("bf16", "f32", 17), ("f16", "f32", 111), ("f16", "f32", 112), ("f16", "f16", 378), ("bf16", "bf16", 379)])
def test_batches_around_what_two_ctas_leave_room_for(g, cache, qt, batch):
    P.check_attention([(1, 1 + b * 7 % 200) for b in range(batch)], 4, 2, 128, 64, cache, qt, seed=91)


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("size", [1e-34, 1e31, 3e36])
def test_fp32_queries_near_the_ends_of_their_range(g, size, cache):
    bt = P.Batch([(1, 200), (30, 90)], 4, 2, 64, 16, cache, seed=3)
    bt.upload()
    q = P.random_queries(bt, "f32", size)
    scale = float(np.float32(0.125 / size))
    got = P.run_attention(bt, q, "f32", scale=scale)
    want, mag = P.attention64(bt, q.astype(np.float64), scale=scale)
    assert (np.abs(got - want) <= P.attention_tolerance(bt, q.astype(np.float64), want, mag, "f32", scale=scale)).all()


@pytest.mark.parametrize("dims", [64, 6])
def test_appends_of_two_sequences_to_a_page_they_share(g, dims):
    """Equal rows stay whole; of unequal ones every element is the one's or the other's."""
    lib, T, G, d = g.cuda(), 16, 2, 64
    bt = P.Batch([(8, 8), (8, 8)], 2, G, d, 8, "f16", seed=95)
    bt.table[1] = bt.table[0]
    bt.upload()
    rng = np.random.default_rng(96)
    c, r = bt.structs()
    rot = g.Rotation(dims=dims, interleaved=0, base=10000.0, freq=None, amplitude=1.0)

    def call(k, v):
        dk, dv = P.device(k), P.device(v)
        g.check(lib.greta_cuda_paged_append(None, C.byref(c), C.byref(r), C.byref(rot), 0, None, 0, dk.ptr, G * d, dv.ptr, G * d, 0, None, 0, 0))
        g.check(lib.greta_cuda_device_synchronize())
        return [b.download(np.uint16).reshape(bt.k.shape)[bt.table[0, 0]] for b in (bt.dk, bt.dv)]

    one, two = (rng.normal(0, 1, (2, 8, G, d)).astype(np.float32) for _ in range(2))
    alone = [call(*(np.concatenate([a, a]) for a in x)) for x in (one, two)]
    assert np.array_equal(alone[0][1], one[1].transpose(1, 0, 2).astype(np.float16).view(np.uint16))
    both = call(*(np.concatenate([a, b]) for a, b in zip(one, two)))
    for got, x, y in zip(both, *alone):
        assert ((got == x) | (got == y)).all()


@pytest.mark.parametrize("cache,qt", [("f16", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("rows,window", [(1, 0), (40, 0), (140, 0), (140, 100)])
def test_infinities_that_a_row_sees_beside_hidden_ones(g, cache, qt, rows, window):
    """An infinity stays one (of its sign) in the rows that see it, whatever the same element of hidden keys is; with one of the other sign, or NaN, it is NaN."""
    n = 300
    bt = P.Batch([(rows, n)], 4, 2, 64, 32, cache, seed=97)
    inf = np.uint16(0x7C00 if cache == "f16" else 0x7F80)
    spoil = [(20, 9, inf), (n - 30, 3, inf), (n - 10, 3, P.NAN16), (n - 25, 17, inf | 0x8000), (n - 5, 17, inf), (n - 28, 40, inf | 0x8000), (n - 1, 40, inf | 0x8000)]
    for j, e, _ in spoil:
        bt.v[bt.table[0, j // 32], :, j % 32, e] = 0
    q = P.random_queries(bt, qt)
    q64 = P.to_f64(q, qt)
    want, mag = P.attention64(bt, q64, window)
    tol = P.attention_tolerance(bt, q64, want, mag, qt)
    pos = np.arange(n - rows, n)
    for j, e, x in spoil:
        bt.v[bt.table[0, j // 32], :, j % 32, e] = x
        sees = (pos >= j) & ((pos < j + window) if window else True)
        with np.errstate(invalid="ignore"):
            want[sees, :, e] += np.nan if x == P.NAN16 else -np.inf if x >> 15 else np.inf
    bt.upload()
    got = P.to_f64(P.run_attention(bt, q, qt, window), qt)
    odd = ~np.isfinite(want)
    assert odd.any() and np.array_equal(got[odd], want[odd], equal_nan=True)
    assert (np.abs(got[~odd] - want[~odd]) <= tol[~odd]).all()


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("specs,H,G", [([(1, 577)] * 8, 32, 32), ([(1, 4096)] * 4, 64, 8), ([(20, 577)], 32, 4)])
def test_scores_of_fp32_calls_are_rounded_sums(g, cache, specs, H, G):
    """By the root of the mean square 2^-21 of the outputs: about twice what 32-bit arithmetic in any order leaves.  Scores summed up in the tensor core alone, which cuts off: 5.6e-7 and more."""
    bt = P.Batch(specs, H, G, 128, 16, cache, seed=99)
    bt.upload()
    q = P.random_queries(bt, "f32")
    want, _ = P.attention64(bt, q.astype(np.float64))
    got = P.run_attention(bt, q, "f32").astype(np.float64)
    err = np.sqrt(((got - want) ** 2).mean() / (want ** 2).mean())
    assert err <= 2.0 ** -21, err

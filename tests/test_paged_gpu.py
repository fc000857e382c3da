"""Paged append and paged attention against 64 bits: ragged batches, odd sizes, masks, pages and strides."""
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


TYPES = [("f16", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16")]


# ---------------------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("cache,qt", TYPES)
@pytest.mark.parametrize("specs,H,G,d,page", [
    ([(1, 1)], 1, 1, 8, 8),
    ([(1, 64), (1, 65), (1, 63), (1, 1)], 8, 2, 64, 16),
    ([(1, 300), (0, 40), (1, 7), (1, 1999)], 32, 4, 128, 32),
    ([(1, 513)], 16, 1, 128, 128),
    ([(1, 777), (1, 90)], 6, 2, 96, 64),
    ([(1, 2500)], 7, 1, 80, 256),
    ([(1, 120)] * 33, 4, 4, 40, 8),
])
def test_single_tokens(g, cache, qt, specs, H, G, d, page):
    P.check_attention(specs, H, G, d, page, cache, qt, seed=len(specs) + d)


@pytest.mark.parametrize("cache,qt", TYPES)
@pytest.mark.parametrize("specs,H,G,d,page,window", [
    ([(5, 500), (5, 5), (5, 68)], 8, 2, 64, 16, 0),
    ([(33, 33)], 4, 4, 128, 32, 0),
    ([(17, 200), (1, 300), (40, 100), (3, 3)], 8, 1, 128, 16, 0),
    ([(130, 260), (64, 64)], 6, 2, 72, 64, 0),
    ([(9, 700), (1, 700)], 4, 2, 64, 32, 100),
    ([(70, 150), (2, 640)], 3, 1, 128, 128, 1),
    ([(200, 333)], 5, 1, 48, 256, 64),
    ([(300, 700), (1, 2000), (129, 129), (128, 256)], 8, 2, 128, 64, 0),
    ([(257, 1000)], 2, 1, 64, 128, 300),
])
def test_portions(g, cache, qt, specs, H, G, d, page, window):
    P.check_attention(specs, H, G, d, page, cache, qt, window=window, seed=H + d)


@pytest.mark.parametrize("cache,qt", TYPES)
@pytest.mark.parametrize("rows", [1, 40])
def test_lengths_of_zero_and_rows_without_positions(g, cache, qt, rows):
    """No keys at all, fewer positions than rows, no rows: zeros where there is nothing to see, the rest as always."""
    P.check_attention([(rows, 0), (0, 0), (rows, rows), (rows, max(rows - 3, 1)), (0, 100)], 4, 2, 64, 16, cache, qt)


@pytest.mark.parametrize("cache,qt", TYPES)
@pytest.mark.parametrize("rows", [1, 50])
def test_strides_and_rows_behind_the_last_sequence(g, cache, qt, rows):
    P.check_attention([(rows, 130), (1, 77)], 4, 2, 64, 32, cache, qt, pad=24, spare_rows=9)


@pytest.mark.parametrize("cache,qt", [("f16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("rows,gain", [(1, 30.0), (50, 30.0), (150, 8.0)])
def test_large_scores(g, cache, qt, rows, gain):
    """Weights between 0 and 1 that hang on single keys; maxima that grow from tile to tile."""
    P.check_attention([(rows, 700), (rows, rows)], 4, 2, 64, 32, cache, qt, gain=gain)


@pytest.mark.parametrize("size", [1e-4, 3e4])
@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_fp32_queries_of_any_size(g, size, cache):
    bt = P.Batch([(1, 200), (30, 90)], 4, 2, 64, 16, cache, seed=3)
    bt.upload()
    q = P.random_queries(bt, "f32", size)
    scale = 0.125 / size
    got = P.run_attention(bt, q, "f32", scale=scale)
    want, mag = P.attention64(bt, q.astype(np.float64), scale=scale)
    assert (np.abs(got - want) <= P.attention_tolerance(bt, q.astype(np.float64), want, mag, "f32", scale=scale)).all()


@pytest.mark.parametrize("cache,qt", TYPES)
def test_a_long_list_split_over_the_gpu(g, cache, qt):
    """One KV head: its tiles fall to every CTA and are joined; the same bits every time, workspace used again."""
    bt = P.Batch([(1, 20011)], 5, 1, 128, 64, cache, seed=4)
    bt.upload()
    q = P.random_queries(bt, qt)
    ws = g.DeviceBuffer(g.cuda().greta_cuda_paged_attn_workspace_bytes(bt.d), zero=True)
    first = P.run_attention(bt, q, qt, workspace=ws)
    q64 = P.to_f64(q, qt)
    want, mag = P.attention64(bt, q64)
    assert (np.abs(P.to_f64(first, qt) - want) <= P.attention_tolerance(bt, q64, want, mag, qt)).all()
    for _ in range(3):
        assert np.array_equal(P.run_attention(bt, q, qt, workspace=ws).view(P.itype(qt)), first.view(P.itype(qt)))
    assert (ws.download(np.uint32, 65536 // 4) == 0).all()


@pytest.mark.parametrize("cache,qt", TYPES)
@pytest.mark.parametrize("rows,window", [(1, 0), (40, 0), (140, 0), (40, 33), (140, 100)])
def test_values_of_hidden_keys_that_are_no_finite_numbers(g, cache, qt, rows, window):
    """Infinities and NaN in single value columns of positions that some rows see: the others are as with zeros there, to the tolerance of either."""
    n = 300
    bt = P.Batch([(rows, n)], 4, 2, 64, 32, cache, seed=5)
    bad = [(n - 1, 3), (n - 20, 40), (n - 41, 7), (10, 63)]
    clean = bt.v.copy()
    for j, e in bad:
        clean[bt.table[0, j // 32], :, j % 32, e] = 0
    dirty = clean.copy()
    for i, (j, e) in enumerate(bad):
        dirty[bt.table[0, j // 32], i % 2, j % 32, e] = 0x7FFF if i % 2 else (0x7C00 if cache == "f16" else 0xFF80)
    q = P.random_queries(bt, qt)
    bt.v = clean
    want, mag = P.attention64(bt, P.to_f64(q, qt), window)
    tol = P.attention_tolerance(bt, P.to_f64(q, qt), want, mag, qt)
    bt.v = dirty
    bt.upload()
    got = P.to_f64(P.run_attention(bt, q, qt, window), qt)
    pos = np.arange(n - rows, n)
    spoilt = np.zeros((rows, 4, 64), bool)
    for i, (j, e) in enumerate(bad):
        sees = (pos >= j) & ((pos < j + window) if window else True)
        spoilt[sees, (i % 2) * 2:(i % 2) * 2 + 2, e] = True
    assert not np.isfinite(got[spoilt]).any()
    assert (np.abs(got - want)[~spoilt] <= tol[~spoilt]).all()


@pytest.mark.parametrize("cache,qt", TYPES)
@pytest.mark.parametrize("rows", [1, 90])
def test_keys_of_hidden_positions_may_be_anything(g, cache, qt, rows):
    """Keys behind the rows of earlier ones: NaN in the last position's key spoils the last row alone."""
    n = 260
    bt = P.Batch([(rows, n)], 2, 1, 64, 16, cache, seed=6)
    q = P.random_queries(bt, qt)
    want, mag = P.attention64(bt, P.to_f64(q, qt))
    tol = P.attention_tolerance(bt, P.to_f64(q, qt), want, mag, qt)
    bt.k[bt.table[0, (n - 1) // 16], 0, (n - 1) % 16] = P.NAN16
    bt.upload()
    got = P.to_f64(P.run_attention(bt, q, qt), qt)
    assert not np.isfinite(got[-1]).any()
    assert (np.abs(got - want) <= tol)[:-1].all()


@pytest.mark.parametrize("cache,qt", [("f16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("rows", [1, 60])
def test_pages_that_are_none(g, cache, qt, rows):
    """Entries outside the pool: keys and values of zero."""
    bt = P.Batch([(rows, 200), (rows, 150)], 4, 2, 64, 32, cache, seed=7)
    bt.upload()
    q = P.random_queries(bt, qt)
    holes = [(0, 1, -1), (0, 3, bt.pages), (1, 0, 2 ** 31 - 1), (1, 4, -2 ** 31)]
    for b, i, bad in holes:
        good = bt.table[b, i]
        bt.k[good], bt.v[good] = 0, 0
    q64 = P.to_f64(q, qt)
    want, mag = P.attention64(bt, q64)
    tol = P.attention_tolerance(bt, q64, want, mag, qt)
    for b, i, bad in holes:
        bt.table[b, i] = bad
    bt.dt = P.device(bt.table)
    got = P.to_f64(P.run_attention(bt, q, qt), qt)
    assert (np.abs(got - want) <= tol).all()


def test_lengths_past_the_table_and_starts_past_the_tokens(g):
    """Device data that promise more than the buffers hold are taken as their ends."""
    bt = P.Batch([(2, 64), (3, 96)], 2, 1, 64, 32, "f16", seed=8)
    bt.upload()
    q = P.random_queries(bt, "f16")
    want = P.run_attention(bt, q, "f16")
    bt.ds = P.device(np.array([0, 2, 900], np.uint32))
    bt.dl = P.device(np.array([64, 2 ** 32 - 1], np.uint32))
    bt2 = P.run_attention(bt, q, "f16")
    assert np.array_equal(want.view(np.uint16), bt2.view(np.uint16))


@pytest.mark.parametrize("qt,rows", [("f32", 1), ("f16", 1), ("f16", 100)])
def test_captured_steps_read_lengths_when_they_run(g, qt, rows):
    """A captured call replayed after the lengths and the table have changed on the device; two graphs that share a workspace."""
    lib = g.cuda()
    bt = P.Batch([(rows, 400), (rows, 520)], 4, 2, 64, 32, "f16", seed=9)
    bt.upload()
    q = P.random_queries(bt, qt)
    ws = g.DeviceBuffer(lib.greta_cuda_paged_attn_workspace_bytes(64), zero=True)
    long = P.run_attention(bt, q, qt, workspace=ws)
    bt.lens = [rows, 333]
    bt.specs = list(zip(bt.rows, bt.lens))
    q64 = P.to_f64(q, qt)
    want, mag = P.attention64(bt, q64)
    tol = P.attention_tolerance(bt, q64, want, mag, qt)
    stream = C.c_void_p()
    g.check(lib.greta_cuda_stream_create(C.byref(stream)))
    dq, outs, graphs = P.device(q), [], []
    c, r = bt.structs()
    for _ in range(2):
        o = g.DeviceBuffer(q.nbytes)
        graph, ex = C.c_void_p(), C.c_void_p()
        g.check(lib.greta_cuda_graph_capture_begin(stream))
        g.check(lib.greta_cuda_paged_attn(stream, C.byref(c), C.byref(r), dq.ptr, P.FMT[qt], 256, o.ptr, 256, 4, 0.125, 0, ws.ptr, ws.nbytes))
        g.check(lib.greta_cuda_graph_capture_end(stream, C.byref(graph)))
        g.check(lib.greta_cuda_graph_instantiate(graph, C.byref(ex)))
        outs.append(o)
        graphs.append((graph, ex))
    for _, ex in graphs:
        g.check(lib.greta_cuda_graph_launch(ex, stream))
    g.check(lib.greta_cuda_stream_synchronize(stream))
    for o in outs:
        assert np.array_equal(o.download(P.itype(qt)), long.reshape(-1).view(P.itype(qt)))
    bt.dl.upload(np.array(bt.lens, np.uint32))
    for _, ex in graphs:
        g.check(lib.greta_cuda_graph_launch(ex, stream))
    g.check(lib.greta_cuda_stream_synchronize(stream))
    for o in outs:
        got = P.to_f64(o.download(q.dtype).reshape(q.shape), qt)
        assert (np.abs(got - want) <= tol).all()
    for graph, ex in graphs:
        lib.greta_cuda_graph_exec_destroy(ex)
        lib.greta_cuda_graph_destroy(graph)
    lib.greta_cuda_stream_destroy(stream)


def test_two_streams_with_a_workspace_each(g):
    lib = g.cuda()
    bt = P.Batch([(1, 3000)] * 4, 16, 2, 128, 64, "bf16", seed=10)
    bt.upload()
    q = P.random_queries(bt, "bf16")
    want = P.run_attention(bt, q, "bf16")
    c, r = bt.structs()
    dq, streams, outs, ws = P.device(q), [], [], []
    for _ in range(2):
        s = C.c_void_p()
        g.check(lib.greta_cuda_stream_create(C.byref(s)))
        streams.append(s)
        outs.append(g.DeviceBuffer(q.nbytes))
        ws.append(g.DeviceBuffer(lib.greta_cuda_paged_attn_workspace_bytes(128), zero=True))
    for _ in range(10):
        for s, o, w in zip(streams, outs, ws):
            g.check(lib.greta_cuda_paged_attn(s, C.byref(c), C.byref(r), dq.ptr, P.FMT["bf16"], 2048, o.ptr, 2048, 16, 128 ** -0.5, 0, w.ptr, w.nbytes))
    g.check(lib.greta_cuda_device_synchronize())
    for o in outs:
        assert np.array_equal(o.download(np.uint16), want.reshape(-1))
    for s in streams:
        lib.greta_cuda_stream_destroy(s)


# ---------------------------------------------------------------------------------------------------------------- append
def append(g, bt, t, qt, dims, base=10000.0, freq=None, interleaved=False, amplitude=1.0, pad=0, with_q=True, in_place=False, stream=None):
    """Random new rows through the call -> q, k, v as given and what came of them: q_out, k pool, v pool."""
    lib, rng = g.cuda(), np.random.default_rng(17)
    H, G, d, T = bt.H, bt.G, bt.d, bt.tokens
    x = [P.to_type(rng.normal(0, 1, (T, n, d)), t) for n in (H, G, G)]
    lds = [H * d + pad, G * d + pad, G * d + 2 * pad]
    bufs = []
    for a, ld in zip(x, lds):
        y = np.zeros((T, ld), a.dtype)
        y[:, :a[0].size] = a.reshape(T, -1)
        bufs.append(P.device(y))
    ld_out = lds[0] if in_place else H * d + 3 * pad
    out = bufs[0] if in_place else g.DeviceBuffer(T * ld_out * (4 if qt == "f32" else 2))
    if not in_place:
        out.fill(0x5A)
    c, r = bt.structs()
    f = np.ascontiguousarray(freq, np.float64) if freq is not None else None
    rot = g.Rotation(dims=dims, interleaved=int(interleaved), base=base, freq=f.ctypes.data if f is not None else None, amplitude=amplitude)
    g.check(lib.greta_cuda_paged_append(stream, C.byref(c), C.byref(r), C.byref(rot), P.FMT[t], bufs[0].ptr if with_q else None, lds[0], bufs[1].ptr, lds[1],
                                        bufs[2].ptr, lds[2], H, out.ptr if with_q else None, P.FMT[qt], ld_out))
    g.check(lib.greta_cuda_device_synchronize())
    q = out.download(np.float32 if qt == "f32" else np.float16 if qt == "f16" else np.uint16, T * ld_out).reshape(T, ld_out)
    return x, q, bt.dk.download(np.uint16).reshape(bt.k.shape), bt.dv.download(np.uint16).reshape(bt.v.shape)


def check_append(g, specs, H, G, d, page, cache, t, qt, dims, base=10000.0, freq=None, interleaved=False, amplitude=1.0, pad=0, spare_rows=0, in_place=False):
    bt = P.Batch(specs, H, G, d, page, cache, seed=H + d, spare_rows=spare_rows)
    bt.upload()
    (q, k, v), got_q, got_k, got_v = append(g, bt, t, qt, dims, base, freq, interleaved, amplitude, pad, in_place=in_place)
    q, k, v = (P.to_f64(a, t) for a in (q, k, v))
    pos = np.concatenate([np.arange(n - r, n) for r, n in specs]).astype(int)
    turn = lambda x: P.rotated64(x[:bt.used], pos, dims, base, freq, interleaved, amplitude)

    def tolerance(x, want, out):
        """Sine and cosine: 2^-23 of the angle's 24 bits (half a turn), 2 units in the last place of the function, the amplitude's rounding: 2^-21.5 in all; products
        and their sum: 2^-23.  Of both elements of a pair; then half a step of the type."""
        size = np.abs(x[:bt.used]).max(-1, keepdims=True) * 2 * max(amplitude, 1.0)
        return size * 2.0 ** -21 + np.abs(want) * P.HALF[out] + (2.0 ** -25 if out == "f16" else 0)

    sane = pos >= 0
    want = turn(q)
    if not in_place:
        assert (np.ascontiguousarray(got_q[:bt.used][~sane]).view(np.uint8) == 0x5A).all() and (np.ascontiguousarray(got_q[bt.used:]).view(np.uint8) == 0x5A).all()
    y = P.to_f64(got_q, qt)[:bt.used, :H * d].reshape(-1, H, d)
    assert (np.abs(y - want) <= tolerance(q, want, qt))[sane].all()
    # the cache: written rows as they should be, every other bit as it was
    touched = np.zeros((bt.pages, page), bool)
    wk, wv = turn(k), v[:bt.used]
    tk = tolerance(k, wk, cache)
    seq = np.repeat(np.arange(len(specs)), [r for r, _ in specs])
    as64 = lambda a: P.to_f64(a.view(np.float16) if cache == "f16" else a, cache)
    for i in range(bt.used):
        if pos[i] < 0:
            continue
        pg, row = bt.table[seq[i], pos[i] // page], pos[i] % page
        touched[pg, row] = True
        assert (np.abs(as64(got_k[pg, :, row]) - wk[i]) <= tk[i]).all()
        assert np.array_equal(got_v[pg, :, row], P.to_type(wv[i], cache).view(np.uint16))
    for a, was in ((got_k, bt.k), (got_v, bt.v)):
        assert np.array_equal(a.transpose(0, 2, 1, 3)[~touched], was.transpose(0, 2, 1, 3)[~touched])


@pytest.mark.parametrize("t,qt,cache", [("f32", "f32", "f16"), ("f32", "f16", "f16"), ("f16", "f16", "f16"), ("bf16", "bf16", "bf16"), ("f32", "bf16", "bf16"), ("bf16", "f32", "f16")])
@pytest.mark.parametrize("specs,H,G,d,page,dims,interleaved", [
    ([(1, 1)], 1, 1, 8, 8, 8, False),
    ([(1, 500), (0, 30), (3, 77), (70, 70)], 8, 2, 64, 16, 64, False),
    ([(5, 40), (1, 9)], 6, 3, 96, 32, 32, True),
    ([(2, 100)], 7, 1, 80, 64, 80, True),
    ([(2, 100)], 3, 1, 128, 64, 6, False),
    ([(4, 20), (5, 3)], 4, 4, 128, 256, 0, False),
    ([(9, 9)], 4, 2, 40, 16, 36, True),
])
def test_append(g, t, qt, cache, specs, H, G, d, page, dims, interleaved):
    check_append(g, specs, H, G, d, page, cache, t, qt, dims, interleaved=interleaved)


def test_append_many_sequences(g):
    """More sequences than a CTA has threads, empty ones among them."""
    check_append(g, [(b % 3, b % 3 + b % 7) for b in range(1024)], 2, 1, 64, 8, "f16", "f32", "f32", 64)


@pytest.mark.parametrize("base,pos", [(10000.0, 131071), (500000.0, 1048575), (10000.0, 16777215)])
def test_append_at_far_positions(g, base, pos):
    bt = P.Batch([(3, 3)], 2, 1, 64, 256, "bf16", seed=11)
    n = pos + 1
    bt.lens, bt.specs = [n], [(3, n)]
    bt.table = np.full((1, -(-n // 256)), -1, np.int32)
    bt.table[0, -1], bt.table[0, -2] = 1, 2
    bt.k = bt.v = np.full((bt.pages, 1, 256, 64), P.NAN16, np.uint16)
    bt.upload()
    (q, k, _), got, _, _ = append(g, bt, "f32", "f32", 64, base)
    want = P.rotated64(q.astype(np.float64), np.arange(pos - 2, pos + 1), 64, base)
    assert (np.abs(got.reshape(want.shape) - want) <= 2 * np.abs(q).max(-1, keepdims=True) * 2.0 ** -21).all()


def test_append_with_given_frequencies_and_amplitude(g):
    freq = np.array([3.5, 1.0, -0.7, 0.0, 1e-3, 7.0, 12.566, 1e-7])
    check_append(g, [(6, 5000), (2, 2)], 4, 2, 64, 128, "f16", "f32", "f32", 16, freq=freq, amplitude=1.4)


def test_append_strides_in_place_and_spare_rows(g):
    check_append(g, [(3, 30), (2, 2)], 4, 2, 64, 16, "f16", "f32", "f32", 64, pad=16, spare_rows=5)
    check_append(g, [(3, 30), (2, 2)], 4, 2, 64, 16, "bf16", "bf16", "bf16", 64, pad=8, spare_rows=2, in_place=True)


def test_append_without_queries_and_to_pages_that_are_none(g):
    bt = P.Batch([(40, 80)], 2, 1, 64, 16, "f16", seed=12)
    bt.table[0, 3], bt.table[0, 4] = bt.pages, -5
    bt.upload()
    (q, k, v), _, got_k, got_v = append(g, bt, "f16", "f16", 64, with_q=False)
    live = [(bt.table[0, p // 16], p % 16, i) for i, p in enumerate(range(40, 80)) if 0 <= bt.table[0, p // 16] < bt.pages]
    assert len(live) == 8
    touched = np.zeros((bt.pages, 16), bool)
    for pg, row, i in live:
        touched[pg, row] = True
        assert np.array_equal(got_v[pg, :, row], v[i].view(np.uint16))
    assert np.array_equal(got_v.transpose(0, 2, 1, 3)[~touched], bt.v.transpose(0, 2, 1, 3)[~touched])
    assert np.array_equal(got_k.transpose(0, 2, 1, 3)[~touched], bt.k.transpose(0, 2, 1, 3)[~touched])


def test_pools_past_32_bits(g):
    """Pages whose elements lie behind 2^32: append writes them, attention reads them."""
    lib, page, d = g.cuda(), 256, 128
    pages = 2 ** 32 // (page * d) + 40
    bt = P.Batch([(20, 20), (1, 1)], 2, 1, d, page, "f16", seed=13)
    bt.specs, bt.rows, bt.lens = [(600, 600), (1, 1)], [600, 1], [600, 1]
    bt.start, bt.used, bt.tokens, bt.pages = np.array([0, 600, 601], np.uint32), 601, 601, pages
    bt.table = np.array([[pages - 1, pages - 30, pages - 2], [pages - 7, 0, 0]], np.int32)
    bt.dk, bt.dv = (g.DeviceBuffer(pages * page * d * 2) for _ in range(2))
    bt.dt, bt.ds, bt.dl = P.device(bt.table), P.device(bt.start), P.device(np.array(bt.lens, np.uint32))
    rng = np.random.default_rng(3)
    q, k, v = (P.to_type(rng.normal(0, 1, (601, n, d)), "f16") for n in (2, 1, 1))
    c, r = bt.structs()
    rot = g.Rotation(dims=0, interleaved=0, base=1.0, freq=None, amplitude=1.0)
    dk, dv = P.device(k), P.device(v)
    g.check(lib.greta_cuda_paged_append(None, C.byref(c), C.byref(r), C.byref(rot), 1, None, 0, dk.ptr, d, dv.ptr, d, 2, None, 1, 0))
    got = P.to_f64(P.run_attention(bt, q, "f16"), "f16")
    small = P.Batch([(600, 600), (1, 1)], 2, 1, d, page, "f16", seed=13)
    for b, at in ((0, 0), (1, 600)):
        p = np.arange(small.lens[b])
        small.k[small.table[b, p // page], :, p % page] = k[at:at + len(p)].view(np.uint16)
        small.v[small.table[b, p // page], :, p % page] = v[at:at + len(p)].view(np.uint16)
    q64 = P.to_f64(q, "f16")
    want, mag = P.attention64(small, q64)
    assert (np.abs(got - want) <= P.attention_tolerance(small, q64, want, mag, "f16")).all()

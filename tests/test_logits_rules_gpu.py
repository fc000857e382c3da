"""Rules on logits and the arg-max behind them against 64 bits."""
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


class Case:
    def __init__(self, M, V, hist=0, cap=None, prompt=True, penalties=("repetition", "frequency", "presence"), biases=0, mask=False, t="f32", pad=0, seed=0, low=0):
        rng = self.rng = np.random.default_rng(seed)
        self.M, self.V, self.t, self.ld = M, V, t, V + pad
        x = np.zeros((M, self.ld), np.float32)
        x[:, :V] = rng.normal(0, 4, (M, V))
        self.logits = P.to_type(x, t)
        self.cap = cap or max(hist, 1)
        self.ids = None
        if hist:
            self.ids = rng.integers(-low, min(V, 3 * hist) + low, (M, self.cap)).astype(np.int32)
            self.n = rng.integers(1, hist + 1, M).astype(np.uint32)
            self.prompt = (self.n // 2).astype(np.uint32) if prompt else None
        self.pen = {n: (rng.uniform(0, 2, M) + (0.5 if n == "repetition" else 0)).astype(np.float32) for n in penalties} if hist else {}
        self.start = None
        if biases:
            count = rng.integers(0, biases + 1, M)
            self.start = np.concatenate([[0], np.cumsum(count)]).astype(np.uint32)
            self.bias_ids = rng.integers(-low, V + low, int(self.start[-1]) or 1).astype(np.int32)
            self.bias = rng.normal(0, 5, self.bias_ids.size).astype(np.float32)
        self.mask = rng.integers(0, 2 ** 32, (M, (V + 31) // 32 + 1), dtype=np.uint32) if mask else None

    def rules(self, g):
        self.keep = k = {}
        if self.ids is not None:
            k["ids"], k["n_ids"] = P.device(self.ids), P.device(self.n)
            if self.prompt is not None:
                k["n_prompt"] = P.device(self.prompt)
        for n, a in self.pen.items():
            k[n] = P.device(a)
        if self.start is not None:
            k["bias_ids"], k["bias"], k["bias_start"] = P.device(self.bias_ids), P.device(self.bias), P.device(self.start)
        if self.mask is not None:
            k["allowed"] = P.device(self.mask)
        return g.LogitsRules(ld_ids=self.cap, ld_allowed=self.mask.shape[1] if self.mask is not None else 0, **{n: b.ptr for n, b in k.items()})

    def want(self, m):
        b = None
        if self.start is not None:
            i = slice(int(self.start[m]), int(self.start[m + 1]))
            b = list(zip(self.bias_ids[i].tolist(), self.bias[i].tolist()))
        pen = {n: float(a[m]) for n, a in self.pen.items()}
        return P.rules64(P.to_f64(self.logits[m, :self.V], self.t), self.V, ids=self.ids[m] if self.ids is not None else None, n_ids=int(self.n[m]) if self.ids is not None else 0,
                         n_prompt=int(self.prompt[m]) if self.ids is not None and self.prompt is not None else 0, biases=b, allowed=self.mask[m] if self.mask is not None else None, **pen)


def run(g, c, in_place=False, out=True, advance=False, pos=None):
    lib, r = g.cuda(), c.rules(g)
    x = P.device(c.logits)
    y = x if in_place else g.DeviceBuffer(c.logits.nbytes)
    if not in_place:
        y.fill(0x5A)
    nxt = P.device(np.full(c.M + 1, -7, np.int32))
    args = [None, C.byref(r), P.FMT[c.t], x.ptr, c.ld, y.ptr if out else None, c.ld, c.M, c.V, nxt.ptr]
    if advance:
        g.check(lib.greta_cuda_logits_adjust_advance(*args, pos))
    else:
        g.check(lib.greta_cuda_logits_adjust(*args))
    g.check(lib.greta_cuda_device_synchronize())
    n = nxt.download(np.int32)
    assert n[-1] == -7
    return y.download(c.logits.dtype).reshape(c.M, c.ld), n[:-1]


def check(g, c, in_place=False):
    got, nxt = run(g, c, in_place)
    if c.ld > c.V and not in_place:
        assert (np.ascontiguousarray(got[:, c.V:]).view(np.uint8) == 0x5A).all()
    y = P.to_f64(got, c.t)[:, :c.V]
    for m in range(c.M):
        want = c.want(m)
        hidden = np.isneginf(want)
        assert np.isneginf(y[m, hidden]).all()
        # five roundings of values not above the sum of sizes, then half a step of the type
        size = np.abs(P.to_f64(c.logits[m, :c.V], c.t)) * 3 + 2 * np.abs(np.where(hidden, 0, want)) + 2 * c.cap + 25
        tol = 5 * 2.0 ** -24 * size + np.abs(np.where(hidden, 0, want)) * P.HALF[c.t]
        assert (np.abs(y[m][~hidden] - want[~hidden]) <= tol[~hidden]).all()
        assert nxt[m] == (int(y[m].argmax()) if not hidden.all() else 0)  # the first maximum of the row as it is written


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kw", [
    dict(M=1, V=1), dict(M=1, V=1, hist=3, mask=True), dict(M=3, V=33, hist=5, biases=4, mask=True), dict(M=2, V=4096, hist=700), dict(M=2, V=4097, hist=50, mask=True),
    dict(M=5, V=32000, hist=900, biases=30), dict(M=2, V=50257, hist=3000, biases=100, mask=True), dict(M=2, V=128256, hist=5000, mask=True),
    dict(M=1, V=250002, hist=2000, biases=500, mask=True), dict(M=40, V=1000, hist=64, biases=5, mask=True), dict(M=3, V=9000, biases=64), dict(M=3, V=20000, mask=True)])
def test_rules(g, t, kw):
    check(g, Case(t=t, seed=kw["V"], **kw))


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("kw", [dict(hist=300, biases=100, mask=True), dict(hist=30000, biases=20000, mask=True), dict(hist=20000), dict(biases=20000), dict(mask=True)])
def test_rules_of_many_rows(g, t, kw):
    """Several chunks a CTA: ids and biases of a slice kept, and more of them than are kept."""
    check(g, Case(M=20, V=50257, t=t, seed=9, **kw))


@pytest.mark.parametrize("pen", [(), ("repetition",), ("frequency",), ("presence", "frequency")])
@pytest.mark.parametrize("prompt", [True, False])
def test_single_rules(g, pen, prompt):
    check(g, Case(3, 5000, hist=400, penalties=pen, prompt=prompt))


@pytest.mark.parametrize("t,pad", [("f32", 8), ("f32", 1), ("bf16", 3), ("f16", 8)])
def test_rows_apart_and_in_place(g, t, pad):
    check(g, Case(3, 4999, hist=100, biases=10, mask=True, t=t, pad=pad))
    check(g, Case(3, 4999, hist=100, biases=10, mask=True, t=t, pad=pad), in_place=True)


def test_ids_outside_the_vocabulary(g):
    check(g, Case(4, 300, hist=200, biases=50, low=60))


def test_counts_longer_than_the_list(g):
    c = Case(2, 1000, hist=30, seed=1)
    c.n[:] = 4000000000  # taken as the list's length
    d = Case(2, 1000, hist=30, seed=1)
    d.n[:] = c.cap
    c.prompt = d.prompt = None
    a, b = run(g, c), run(g, d)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_rows_that_the_mask_leaves_empty_and_values_that_are_no_numbers(g):
    c = Case(4, 9000, mask=True)
    c.mask[0] = 0
    c.mask[1:] = 0xFFFFFFFF
    c.logits[1, 77] = np.nan          # never the maximum
    c.logits[2, 0] = np.nan           # but in the first place
    c.logits[3, :] = -np.inf
    got, nxt = run(g, c)
    assert np.isneginf(got[0]).all() and nxt[0] == 0
    assert nxt[1] == int(np.nanargmax(c.logits[1])) and np.isnan(got[1, 77])
    assert nxt[2] == 0 and nxt[3] == 0


def test_masked_values_may_be_anything(g):
    c = Case(1, 500, mask=True)
    bits = (c.mask[0][np.arange(500) // 32] >> (np.arange(500) % 32).astype(np.uint32)) & 1
    c.logits[0, bits == 0] = np.resize([np.nan, np.inf, 3e38], int((bits == 0).sum()))
    got, nxt = run(g, c)
    assert np.isneginf(got[0, bits == 0]).all()
    assert nxt[0] == int(np.where(bits == 1, c.logits[0], -np.inf).argmax())


def test_only_the_choice(g):
    c = Case(3, 40000, hist=300, mask=True)
    got, a = run(g, c)
    _, b = run(g, c, out=False)
    assert np.array_equal(a, b)


def test_ties_go_to_the_lowest_id(g):
    c = Case(2, 20000, mask=True, t="bf16")
    c.logits[:] = P.to_type(np.float32(1.5), "bf16")
    _, nxt = run(g, c)
    bits = (c.mask[:, np.arange(20000) // 32] >> (np.arange(20000) % 32).astype(np.uint32)) & 1
    assert np.array_equal(nxt, bits.argmax(1))


def test_steps_that_feed_themselves(g):
    """Captured once and replayed: every chosen id joins the text and is penalised in the next step, until the list is full."""
    lib, M, V, cap, steps = g.cuda(), 3, 6000, 12, 12
    c = Case(M, V, hist=4, cap=cap, seed=5)
    c.pen = {"frequency": np.full(M, 1.5, np.float32), "repetition": np.full(M, 1.1, np.float32)}
    r, x, nxt = c.rules(g), P.device(c.logits), g.DeviceBuffer(4 * M)
    pos = P.device(np.array([5, 6, 7], np.uint32))
    s, graph, ex = C.c_void_p(), C.c_void_p(), C.c_void_p()
    g.check(lib.greta_cuda_stream_create(C.byref(s)))
    g.check(lib.greta_cuda_graph_capture_begin(s))
    g.check(lib.greta_cuda_logits_adjust_advance(s, C.byref(r), 0, x.ptr, V, None, 0, M, V, nxt.ptr, pos.ptr))
    g.check(lib.greta_cuda_graph_capture_end(s, C.byref(graph)))
    g.check(lib.greta_cuda_graph_instantiate(graph, C.byref(ex)))
    for _ in range(steps):
        g.check(lib.greta_cuda_graph_launch(ex, s))
    g.check(lib.greta_cuda_stream_synchronize(s))
    got, n = c.keep["ids"].download(np.int32).reshape(M, cap), c.keep["n_ids"].download(np.uint32)
    for m in range(M):
        ids, k = c.ids[m].copy(), int(c.n[m])
        for _ in range(steps):
            y = P.rules64(c.logits[m], V, ids=ids, n_ids=k, n_prompt=int(c.prompt[m]), repetition=np.float32(1.1), frequency=1.5).astype(np.float32)
            if k < cap:
                ids[k] = int(y.argmax())
                k += 1
        assert np.array_equal(got[m], ids) and n[m] == k == cap
    assert np.array_equal(pos.download(np.uint32), np.array([5, 6, 7]) + steps)
    lib.greta_cuda_graph_exec_destroy(ex)
    lib.greta_cuda_graph_destroy(graph)
    lib.greta_cuda_stream_destroy(s)

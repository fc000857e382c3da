"""Ragged batches over a paged cache for the tests: buffers on the device, and the operators in 64 bits."""
import ctypes as C
import math

import numpy as np

from _support import load_package

FMT = {"f32": 0, "f16": 1, "bf16": 2}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative to the value
NAN16 = 0x7FFF  # a NaN in both 16-bit types


def to_type(x, t):
    """float -> the type's array (bf16 as its 16 bits), round to nearest even."""
    if t == "f32":
        return np.asarray(x, np.float32)
    if t == "f16":
        return np.asarray(x, np.float32).astype(np.float16)
    u = np.ascontiguousarray(np.asarray(x, np.float32)).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def to_f64(a, t):
    if t == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def itype(t):
    return np.float32 if t == "f32" else np.uint16


def device(a):
    g = load_package().ffi
    return g.DeviceBuffer.from_numpy(np.ascontiguousarray(a))


class Batch:
    """specs: (rows, len) of each sequence.  The pools are NaN but for the positions that sequences hold; pages are scattered."""

    def __init__(self, specs, H, G, d, page, cache="f16", seed=0, spare_rows=0, extra_pages=3, gap=0):
        rng = self.rng = np.random.default_rng(seed)
        self.specs, self.H, self.G, self.d, self.page, self.cache = specs, H, G, d, page, cache
        self.rows, self.lens = [s[0] for s in specs], [s[1] for s in specs]
        self.start = np.concatenate([[0], np.cumsum(self.rows)]).astype(np.uint32)
        self.used = int(self.start[-1])
        self.tokens = self.used + spare_rows
        need = [-(-n // page) for n in self.lens]
        self.pages = sum(need) + extra_pages
        self.table = np.full((len(specs), max(max(need), 1) + gap), -1, np.int32)
        order, at = rng.permutation(self.pages).astype(np.int32), 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (self.pages, G, page, d)
        live = np.zeros((self.pages, page), bool)
        for b, n in enumerate(self.lens):
            p = np.arange(n)
            live[self.table[b, p // page], p % page] = True
        keep = live[:, None, :, None]
        nan = np.array(NAN16, np.uint16)
        self.k, self.v = (np.where(keep, to_type(rng.normal(0, 1, shape), cache).view(np.uint16), nan) for _ in range(2))

    def dense(self, pool, b):
        """[len][G][d] in float64."""
        p = np.arange(self.lens[b])
        x = pool[self.table[b, p // self.page], :, p % self.page]
        return to_f64(x.view(np.float16) if self.cache == "f16" else x, self.cache)

    def upload(self):
        self.dk, self.dv, self.dt = device(self.k), device(self.v), device(self.table)
        self.ds, self.dl = device(self.start), device(np.array(self.lens, np.uint32))

    def structs(self, max_rows=None):
        f = load_package().ffi
        c = f.PagedCache(fmt=FMT[self.cache], k=self.dk.ptr, v=self.dv.ptr, pages=self.pages, kv_heads=self.G, page=self.page, dim=self.d, table=self.dt.ptr,
                         ld_table=self.table.shape[1])
        r = f.Ragged(batch=len(self.specs), tokens=self.tokens, max_rows=max(self.rows) if max_rows is None else max_rows, start=self.ds.ptr, len=self.dl.ptr)
        return c, r


def attention64(bt, q, window=0, scale=None):
    """q [tokens][H][d] float64 -> outputs, and sum_j p_j |v_j| of each (what a relative error of the weights is multiplied by)."""
    scale = bt.d ** -0.5 if scale is None else scale
    out, mag = np.zeros((bt.tokens, bt.H, bt.d)), np.zeros((bt.tokens, bt.H, bt.d))
    grp = bt.H // bt.G
    for b, (r, n) in enumerate(bt.specs):
        if n == 0 or r == 0:
            continue
        k, v = bt.dense(bt.k, b), bt.dense(bt.v, b)
        pos, key = np.arange(n - r, n)[:, None], np.arange(n)[None]
        seen = key <= pos
        if window:
            seen &= key > pos - window
        at = int(bt.start[b])
        for h in range(bt.H):
            s = np.where(seen, q[at:at + r, h] @ k[:, h // grp].T * scale, -np.inf)
            m = s.max(1, keepdims=True)
            w = np.exp(s - np.where(np.isfinite(m), m, 0.0))
            l = w.sum(1, keepdims=True)
            w = np.divide(w, l, out=np.zeros_like(w), where=l > 0)
            out[at:at + r, h] = w @ v[:, h // grp]
            mag[at:at + r, h] = w @ np.abs(v[:, h // grp])
    return out, mag


def attention_tolerance(bt, q, want, mag, qt, scale=None):
    """Of each output.  Scores: fp32 queries keep 22 bits of a row's largest element (two fp16 values, three bf16 values more), products are summed in fp32 (at
    most 24 sums a score, 2^-23 each of the largest partial sum); a score off by x moves its weight by x, and all of them the sum.  Weights: 2^-22 of the
    exponential, the rounding of the probabilities to the cache's type (fp32 calls: 2^-22).  Sums over keys: 2^-23 of the partial sum per 16 keys and term.  Output: half a step."""
    scale = bt.d ** -0.5 if scale is None else scale
    n = max(bt.lens)
    kmax = max(float(np.abs(bt.dense(bt.k, b)).sum(2).max()) if bt.lens[b] else 0.0 for b in range(len(bt.specs)))
    qmax = np.abs(q).max(2, keepdims=True)
    score = scale * qmax * kmax * ((2.0 ** -22 if qt == "f32" else 0.0) + 24 * 2.0 ** -23 / 8)  # partial sums are below an eighth of the sum of sizes at random signs
    weight = 2.0 ** -22 + (2.0 ** -22 if qt == "f32" else HALF[bt.cache])
    sums = (n / 16 * 3 + 8) * 2.0 ** -23
    return mag * (2 * score + weight + sums) + np.abs(want) * HALF[qt] + 1e-30


def run_attention(bt, q, qt, window=0, scale=None, max_rows=None, pad=0, stream=None, workspace=None):
    """q in its type [tokens][H][d] -> o in its type; rows `pad` elements further apart than they are long; o starts as a pattern."""
    g = load_package().ffi
    ld = bt.H * bt.d + pad
    qd = np.zeros((bt.tokens, ld), q.dtype)
    qd[:, :bt.H * bt.d] = q.reshape(bt.tokens, -1)
    dq, do = device(qd), g.DeviceBuffer(max(qd.nbytes, 16))
    do.fill(0x5A)
    ws = workspace or g.DeviceBuffer(g.cuda().greta_cuda_paged_attn_workspace_bytes(bt.d), zero=True)
    c, r = bt.structs(max_rows)
    scale = bt.d ** -0.5 if scale is None else scale
    g.check(g.cuda().greta_cuda_paged_attn(stream, C.byref(c), C.byref(r), dq.ptr, FMT[qt], ld, do.ptr, ld, bt.H, scale, window, ws.ptr, ws.nbytes), "paged_attn")
    code = C.c_int(-1)
    g.check(g.cuda().greta_cuda_gemm_segments_status(stream, C.byref(code)))
    g.check(g.cuda().greta_cuda_device_synchronize())
    assert code.value == 0
    o = do.download(q.dtype, bt.tokens * ld).reshape(bt.tokens, ld)
    assert (o[bt.used:].view(np.uint8) == 0x5A).all() and (np.ascontiguousarray(o[:, bt.H * bt.d:]).view(np.uint8) == 0x5A).all()
    return np.ascontiguousarray(o[:, :bt.H * bt.d]).reshape(bt.tokens, bt.H, bt.d)


def random_queries(bt, qt, gain=1.0, seed=1):
    rng = np.random.default_rng(seed)
    return to_type(rng.normal(0, gain, (bt.tokens, bt.H, bt.d)) * rng.uniform(0.3, 1, (bt.tokens, 1, 1)), qt)


def check_attention(specs, H, G, d, page, cache, qt, window=0, gain=1.0, pad=0, spare_rows=0, seed=0, max_rows=None):
    bt = Batch(specs, H, G, d, page, cache, seed=seed, spare_rows=spare_rows)
    bt.upload()
    q = random_queries(bt, qt, gain, seed + 1)
    got = to_f64(run_attention(bt, q, qt, window, pad=pad, max_rows=max_rows), qt)[:bt.used]
    q64 = to_f64(q, qt)
    want, mag = attention64(bt, q64, window)
    tol = attention_tolerance(bt, q64, want, mag, qt)[:bt.used]
    err = np.abs(got - want[:bt.used])
    assert np.isfinite(got).all()
    worst = float((err / tol).max()) if bt.used else 0.0
    assert worst <= 1, (worst, np.unravel_index((err / tol).argmax(), err.shape))
    return worst


def rotated64(x, pos, dims, base=None, freq=None, interleaved=False, amplitude=1.0):
    """x [T][heads][d] float64; angles in extended precision."""
    half = dims // 2
    f = np.asarray(freq, np.longdouble) if freq is not None else np.longdouble(base) ** (-2 * np.arange(half, dtype=np.longdouble) / max(dims, 1))
    turn = 2 * np.longdouble("3.14159265358979323846264338327950288")
    a = np.mod(np.asarray(pos, np.longdouble)[:, None] * (f / turn)[None], 1) * turn
    c, s = (np.cos(a) * amplitude).astype(np.float64)[:, None], (np.sin(a) * amplitude).astype(np.float64)[:, None]
    y = x.copy()
    i, j = (slice(0, dims, 2), slice(1, dims, 2)) if interleaved else (slice(0, half), slice(half, dims))
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    return y


def rules64(logits, V, ids=None, n_ids=None, n_prompt=None, repetition=None, frequency=None, presence=None, biases=None, allowed=None):
    """One row in float64; biases: list of (id, value)."""
    x = logits.astype(np.float64).copy()
    if ids is not None:
        ids = ids[:n_ids]
        ok = (ids >= 0) & (ids < V)
        seen = np.unique(ids[ok])
        if repetition is not None:
            x[seen] = np.where(x[seen] > 0, x[seen] / np.float64(repetition), x[seen] * np.float64(repetition))
        said = ids[n_prompt or 0:]
        count = np.bincount(said[(said >= 0) & (said < V)], minlength=V)
        x -= (frequency or 0.0) * count + (presence or 0.0) * (count > 0)
    for t, v in dict(biases or []).items():
        if 0 <= t < V:
            x[t] += v
    if allowed is not None:
        bit = (allowed[np.arange(V) // 32] >> (np.arange(V) % 32).astype(np.uint32)) & 1
        x[bit == 0] = -math.inf
    return x

"""Append, attention and rules on logits as a serving loop runs them, and calls at the borders of their forms."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

import _paged as P
import test_paged_gpu as T
from _support import load_package

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    f = load_package().ffi
    f.require_device()
    return f


@pytest.mark.parametrize("cache,qt,window", [("f16", "f32", 0), ("f16", "f16", 20), ("bf16", "f32", 20), ("bf16", "bf16", 0)])
def test_prompts_then_captured_steps(g, cache, qt, window):
    """Heads of an id's embedding are its queries, keys and values, and the outputs of a row are its logits: portions of prompts (of no row and of one among them),
    then a captured step that is replayed: the chosen ids are the next step's tokens, lengths and texts grow on the device."""
    lib, B, H, G, d, page, steps = g.cuda(), 4, 4, 2, 64, 16, 9
    V, C3, dims, base = H * d, (H + 2 * G) * d, 64, 10000.0
    rng = np.random.default_rng(21)
    prompt = [38, 0, 1, 17]  # rows of the portions; one more token of each is the first step's
    cap = max(prompt) + 1 + steps
    emb = rng.normal(0, 1, (V, C3)).astype(np.float32)
    ids = np.full((B, cap), -1, np.int32)
    for b, n in enumerate(prompt):
        ids[b, :n + 1] = rng.integers(0, V, n + 1)
    pages_each = -(-cap // page)
    bt = P.Batch([(n, n) for n in prompt], H, G, d, page, cache, seed=22, gap=0)
    bt.pages = B * pages_each
    bt.table = rng.permutation(bt.pages).astype(np.int32).reshape(B, pages_each)
    bt.k = bt.v = np.full((bt.pages, G, page, d), P.NAN16, np.uint16)
    bt.upload()
    c, r = bt.structs()
    rot = g.Rotation(dims=dims, interleaved=0, base=base, freq=None, amplitude=1.0)
    ws = g.DeviceBuffer(lib.greta_cuda_paged_attn_workspace_bytes(d), zero=True)
    demb, item = P.device(emb), 4 if qt == "f32" else 2
    s, graph, ex = C.c_void_p(), C.c_void_p(), C.c_void_p()
    g.check(lib.greta_cuda_stream_create(C.byref(s)))

    def layer(c, r, tokens, x, q, o):
        g.check(lib.greta_cuda_embedding(s, tokens, demb.ptr, 0, x.ptr, r.tokens, C3, V))
        g.check(lib.greta_cuda_paged_append(s, C.byref(c), C.byref(r), C.byref(rot), 0, x.ptr, C3, x.ptr + V * 4, C3, x.ptr + (V + G * d) * 4, C3, H, q.ptr, P.FMT[qt], V))
        g.check(lib.greta_cuda_paged_attn(s, C.byref(c), C.byref(r), q.ptr, P.FMT[qt], V, o.ptr, V, H, d ** -0.5, window, ws.ptr, ws.nbytes))

    first = np.concatenate([ids[b, :n] for b, n in enumerate(prompt)])
    buffers = lambda n: (g.DeviceBuffer(n * C3 * 4), g.DeviceBuffer(n * V * item), g.DeviceBuffer(n * V * item))
    dfirst, prompts, step = P.device(first), buffers(len(first)), buffers(B)
    layer(c, r, dfirst.ptr, *prompts)
    # the steps: one row a sequence, its position and the text's end go up by one each time
    start, length = P.device(np.arange(B + 1, dtype=np.uint32)), P.device(np.array(prompt, np.uint32) + 1)
    r1 = g.Ragged(batch=B, tokens=B, max_rows=1, start=start.ptr, len=length.ptr)
    text, n_ids, n_prompt = P.device(ids), P.device(np.array(prompt, np.uint32) + 1), P.device(np.array(prompt, np.uint32) + 1)
    rep, freq = np.array([1.25, 1.0, 1.5, 1.125], np.float32), np.array([0.5, 0.25, 0.0, 1.0], np.float32)
    allowed = rng.integers(0, 2 ** 32, (B, V // 32), dtype=np.uint32)
    keep = [P.device(a) for a in (rep, freq, allowed)]
    rules = g.LogitsRules(ids=text.ptr, ld_ids=cap, n_ids=n_ids.ptr, n_prompt=n_prompt.ptr, repetition=keep[0].ptr, frequency=keep[1].ptr, allowed=keep[2].ptr, ld_allowed=V // 32)
    token = P.device(np.array([ids[b, n] for b, n in enumerate(prompt)], np.int32))
    g.check(lib.greta_cuda_graph_capture_begin(s))
    layer(c, r1, token.ptr, *step)
    g.check(lib.greta_cuda_logits_adjust_advance(s, C.byref(rules), P.FMT[qt], step[2].ptr, V, None, 0, B, V, token.ptr, length.ptr))
    g.check(lib.greta_cuda_graph_capture_end(s, C.byref(graph)))
    g.check(lib.greta_cuda_graph_instantiate(graph, C.byref(ex)))
    outs = []
    for _ in range(steps):
        g.check(lib.greta_cuda_graph_launch(ex, s))
        g.check(lib.greta_cuda_stream_synchronize(s))
        outs.append(P.to_f64(step[2].download(P.to_type([0.0], qt).dtype).reshape(B, V), qt))
    got_ids = text.download(np.int32).reshape(B, cap)
    code = C.c_int(-1)
    g.check(lib.greta_cuda_gemm_segments_status(s, C.byref(code)))
    assert code.value == 0
    assert np.array_equal(length.download(np.uint32), np.array(prompt) + 1 + steps) and np.array_equal(n_ids.download(np.uint32), np.array(prompt) + 1 + steps)
    got_first = P.to_f64(prompts[2].download(P.to_type([0.0], qt).dtype).reshape(-1, V), qt)
    at = 0
    for b, n in enumerate(prompt):
        L = n + steps
        assert np.array_equal(got_ids[b, :n + 1], ids[b, :n + 1]) and (got_ids[b, L + 1:] == -1).all()
        x = emb[got_ids[b, :L]].astype(np.float64)
        pos = np.arange(L)
        q, k = (P.rotated64(y.reshape(L, -1, d), pos, dims, base) for y in (x[:, :V], x[:, V:V + G * d]))
        v = x[:, V + G * d:].reshape(L, G, d)
        rows = np.concatenate([got_first[at:at + n], [o[b] for o in outs]]).reshape(L, H, d)
        at += n
        for h in range(H):
            sc = q[:, h] @ k[:, h // 2].T * d ** -0.5
            seen = (pos[None] <= pos[:, None]) & ((pos[None] > pos[:, None] - window) if window else True)
            w = np.exp(np.where(seen, sc, -np.inf) - np.where(seen, sc, -np.inf).max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            want, mag = w @ v[:, h // 2], w @ np.abs(v[:, h // 2])
            # Each factor of a product of a score is off by its rounding (queries by their type's, keys by the cache's) and by 2^-20 of its size for the turn's sine and cosine
            # (of the pair: of both elements, at most sqrt(2) of the larger), sums of 64 products by 64 steps of 2^-23; so is a score, and a weight by exp of twice that (its sum too).
            near = np.where(seen, np.abs(q[:, h]) @ np.abs(k[:, h // 2]).T, 0).max(1, keepdims=True)
            turned = np.where(seen, np.abs(q[:, h]).max(1, keepdims=True) * np.abs(k[:, h // 2]).sum(1)[None] + np.abs(q[:, h]).sum(1, keepdims=True) * np.abs(k[:, h // 2]).max(1)[None], 0)
            off = d ** -0.5 * (near * (P.HALF[cache] + P.HALF[qt] + 64 * 2.0 ** -23) + turned.max(1, keepdims=True) * 2 * 2.0 ** -20)
            tol = mag * (np.expm1(2 * off) + P.HALF[cache] * (2 if qt != "f32" else 1) + 2.0 ** -21 + L * 2.0 ** -23) + np.abs(want) * P.HALF[qt]
            assert (np.abs(rows[:, h] - want) <= tol).all()
        # the choices: of the logits as they came, to which the rules are applied in 32 bits
        for i in range(steps):
            y = P.rules64(outs[i][b], V, ids=got_ids[b], n_ids=n + 1 + i, n_prompt=n + 1, repetition=rep[b], frequency=float(freq[b]), allowed=allowed[b])
            if qt != "f32":
                y = P.to_f64(P.to_type(y.astype(np.float32), qt), qt)
            best = got_ids[b, n + 1 + i]
            # of both: one rounding of each of three rules of values below 16, and where rounding to 16 bits falls the other way, one step
            assert y[best] >= y.max() - 6 * 2.0 ** -24 * 16 - (4 * P.HALF[qt] * max(abs(y.max()), abs(y[best])) if qt != "f32" else 0)
    lib.greta_cuda_graph_exec_destroy(ex)
    lib.greta_cuda_graph_destroy(graph)
    lib.greta_cuda_stream_destroy(s)


@pytest.mark.parametrize("cache,qt", [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("specs,H,G,d,page,window", [
    ([(300, 5000)], 4, 1, 128, 64, 0),            # few long blocks: shared and joined
    ([(1, 6000), (40, 3000), (2, 5)], 8, 1, 64, 16, 0),
    ([(130, 170)] * 40, 8, 4, 64, 32, 0),         # many blocks alike: drawn one by one
    ([(70, 90)] * 50 + [(0, 4), (9, 900)], 6, 6, 40, 8, 64),
    ([(3, 200), (1, 130)], 128, 1, 64, 64, 0),    # 128 heads over one, and more than a tile has rows
    ([(3, 200), (1, 130)], 130, 1, 64, 64, 0),
    ([(2, 257)], 192, 1, 128, 128, 100),
])
def test_blocks_drawn_and_shared(g, cache, qt, specs, H, G, d, page, window):
    P.check_attention(specs, H, G, d, page, cache, qt, window, seed=31)


@pytest.mark.parametrize("qt,most", [("f32", 1), ("f16", 1), ("f16", 7), ("f16", 64)])
def test_rows_past_the_bound_are_not_looked_at(g, qt, most):
    """Sequences of more rows than max_rows: the first ones have their outputs, the others stay as they were."""
    bt = P.Batch([(90, 200), (3, 40), (70, 70)], 4, 2, 64, 16, "f16", seed=33)
    bt.upload()
    q = P.random_queries(bt, qt)
    q64 = P.to_f64(q, qt)
    got = P.run_attention(bt, q, qt, max_rows=most)
    want, mag = P.attention64(bt, q64)
    tol = P.attention_tolerance(bt, q64, want, mag, qt)
    inside = np.concatenate([np.arange(r) < most for r in bt.rows])
    assert (np.abs(P.to_f64(got, qt) - want) <= tol)[inside].all()
    assert (np.ascontiguousarray(got[~inside]).view(np.uint8) == 0x5A).all()


def test_tables_with_room_for_more_than_32_bits_of_tiles(g):
    """Short sequences behind a table for 2^31 positions: the call is as good as any."""
    bt = P.Batch([(700, 900), (1300, 1500)], 8, 2, 64, 256, "f16", seed=34)
    bt.table = np.ascontiguousarray(bt.table[:1])
    ld = 2 ** 31 // 256 - 1
    bt.specs, bt.rows, bt.lens = [(700, 900)], [700], [900]
    bt.start, bt.used, bt.tokens = np.array([0, 700], np.uint32), 700, 2000
    wide = np.full((1, ld), -1, np.int32)
    wide[:, :bt.table.shape[1]] = bt.table
    bt.table = wide
    bt.upload()
    q = P.random_queries(bt, "f16")
    q64 = P.to_f64(q, "f16")
    got = P.to_f64(P.run_attention(bt, q, "f16"), "f16")
    want, mag = P.attention64(bt, q64)
    tol = P.attention_tolerance(bt, q64, want, mag, "f16")
    assert (np.abs(got - want) <= tol)[:700].all()


def test_prompts_said_to_be_longer_than_the_text(g):
    """n_prompt behind n_ids: nothing has been said yet, the repetition penalty stays."""
    rng, V = np.random.default_rng(35), 500
    x = rng.normal(0, 3, (2, V)).astype(np.float32)
    ids = rng.integers(0, V, (2, 20)).astype(np.int32)
    n, prompt = np.array([12, 0], np.uint32), np.array([40, 3], np.uint32)
    pen = [np.array([1.5, 1.5], np.float32), np.array([2.0, 2.0], np.float32)]
    keep = [P.device(a) for a in (x, ids, n, prompt, *pen)]
    out, nxt = g.DeviceBuffer(x.nbytes), g.DeviceBuffer(8)
    rules = g.LogitsRules(ids=keep[1].ptr, ld_ids=20, n_ids=keep[2].ptr, n_prompt=keep[3].ptr, repetition=keep[4].ptr, frequency=keep[5].ptr)
    g.check(g.cuda().greta_cuda_logits_adjust(None, C.byref(rules), 0, keep[0].ptr, V, out.ptr, V, 2, V, nxt.ptr))
    got = out.download(np.float32).reshape(2, V)
    for m in range(2):
        want = P.rules64(x[m], V, ids=ids[m], n_ids=int(n[m]), n_prompt=int(n[m]), repetition=np.float32(1.5), frequency=2.0)
        assert (np.abs(got[m] - want) <= 2.0 ** -23 * np.abs(want)).all()
        assert nxt.download(np.int32)[m] == got[m].argmax()


@pytest.mark.parametrize("t,cache", [("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("d,dims,interleaved", [(8, 0, False), (16, 16, False), (16, 16, True), (16, 0, False), (24, 16, False), (32, 32, False)])
def test_append_of_small_heads(g, t, cache, d, dims, interleaved):
    """Heads of one unit and of a few."""
    T.check_append(g, [(3, 20), (1, 9), (40, 40)], 6, 3, d, 8, cache, t, t, dims, interleaved=interleaved)


@pytest.mark.parametrize("qt,most", [("f32", 2), ("f16", 2), ("f16", 40)])
def test_attention_of_many_sequences(g, qt, most):
    """As many sequences as a call takes, empty ones among them."""
    P.check_attention([(b % (most + 1), b % (most + 1) + b % 37) for b in range(1024)], 4, 2, 64, 16, "f16", qt, seed=36)


def test_first_calls_of_a_process_are_captured(g):
    """Attributes, occupancies and the error word are asked for while a stream is being captured."""
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, os.path.join(here, "_fresh_capture.py")], cwd=here, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stdout + r.stderr

"""Refusals of the operators on paged caches and of the rules on logits: arguments are checked before anything is launched."""
import ctypes as C

import pytest

from _support import load_package


@pytest.fixture(scope="module")
def f():
    p = load_package()
    p.build()
    return p.ffi


def _args(f):
    buf = (C.c_uint8 * 4096)()
    p = (C.addressof(buf) + 15) & ~15
    cache = dict(fmt=1, k=p, v=p, pages=4, kv_heads=2, page=16, dim=64, table=p, ld_table=4)
    rows = dict(batch=2, tokens=3, max_rows=0, start=p, len=p)
    return buf, p, cache, rows


CACHE = [dict(fmt=0), dict(fmt=8), dict(k=None), dict(v=None), dict(table=None), dict(dim=0), dict(dim=4), dict(dim=60), dict(dim=136), dict(page=0), dict(page=4), dict(page=24),
         dict(page=512), dict(pages=0), dict(kv_heads=0), dict(pages=1 << 28, page=256), dict(ld_table=0), dict(ld_table=1 << 28), "k+8", "v+2"]
ROWS = [dict(batch=0), dict(batch=1025), dict(start=None), dict(len=None), dict(tokens=1 << 24)]


def _spoil(d, bad):
    if isinstance(bad, str):
        name, by = bad.split("+")
        return dict(d, **{name: d[name] + int(by)})
    return dict(d, **bad)


def _append(f, cache, rows, p, rot=None, fmt=0, q="p", ld_q=256, k="p", ld_k=128, v="p", ld_v=128, heads=4, q_out="p+", q_fmt=0, ld_out=256):
    at = lambda x: {"p": p, "p+": p + 16, "p+8": p + 8, None: None}[x]
    r = f.Rotation(**dict(dict(dims=64, interleaved=0, base=10000.0, freq=None, amplitude=1.0), **(rot or {})))
    return f.cuda().greta_cuda_paged_append(None, C.byref(f.PagedCache(**cache)), C.byref(f.Ragged(**rows)), C.byref(r), fmt, at(q), ld_q, at(k), ld_k, at(v), ld_v, heads,
                                            at(q_out), q_fmt, ld_out)


def _attn(f, cache, rows, p, q="p", q_fmt=0, ld_q=256, o="p+", ld_o=256, heads=4, scale=0.125, window=0, ws="p", ws_bytes=1 << 40):
    at = lambda x: {"p": p, "p+": p + 16, "p+8": p + 8, None: None}[x]
    return f.cuda().greta_cuda_paged_attn(None, C.byref(f.PagedCache(**cache)), C.byref(f.Ragged(**rows)), at(q), q_fmt, ld_q, at(o), ld_o, heads, scale, window, at(ws), ws_bytes)


@pytest.mark.parametrize("bad", CACHE)
def test_caches_that_are_refused(f, bad):
    buf, p, cache, rows = _args(f)
    cache = _spoil(cache, bad)
    assert _append(f, cache, rows, p) == 4 and b"paged_append" in f.cuda().greta_cuda_last_error()
    assert _attn(f, cache, rows, p) == 4 and b"paged_attn" in f.cuda().greta_cuda_last_error()


@pytest.mark.parametrize("bad", ROWS)
def test_batches_that_are_refused(f, bad):
    buf, p, cache, rows = _args(f)
    rows = _spoil(rows, bad)
    assert _append(f, cache, rows, p) == 4 and _attn(f, cache, rows, p) == 4


@pytest.mark.parametrize("bad", [dict(fmt=8), dict(q_fmt=8), dict(rot=dict(dims=66)), dict(rot=dict(dims=3)), dict(rot=dict(base=0.0)), dict(rot=dict(base=-1.0)), dict(k=None), dict(v=None),
                                 dict(q=None), dict(q_out=None), dict(heads=0), dict(ld_q=252), dict(ld_k=124), dict(ld_v=124), dict(ld_out=252), dict(ld_q=258),
                                 dict(q="p+8"), dict(k="p+8"), dict(v="p+8"), dict(q_out="p+8"), dict(q_out="p", q_fmt=1), dict(q_out="p", ld_out=260)])
def test_appends_that_are_refused(f, bad):
    buf, p, cache, rows = _args(f)
    assert _append(f, cache, rows, p, **bad) == 4


def test_frequencies_that_are_no_numbers(f):
    buf, p, cache, rows = _args(f)
    freq = (C.c_double * 32)(*[1.0] * 31, float("nan"))
    assert _append(f, cache, rows, p, rot=dict(freq=C.addressof(freq))) == 4


@pytest.mark.parametrize("bad", [dict(q_fmt=2), dict(q_fmt=8), dict(q=None), dict(o=None), dict(ws=None), dict(heads=0), dict(heads=5), dict(ld_q=252), dict(ld_o=252),
                                 dict(ld_q=258), dict(q="p+8"), dict(o="p+8"), dict(o="p"), dict(window=1 << 31), dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(ws_bytes=1 << 16), dict(ws="p+8")])
def test_attentions_that_are_refused(f, bad):
    buf, p, cache, rows = _args(f)
    assert _attn(f, cache, rows, p, **bad) == 4


def test_nothing_to_do(f):
    buf, p, cache, rows = _args(f)
    rows["tokens"] = 0
    assert _append(f, cache, rows, p) == 0 and _attn(f, cache, rows, p) == 0


def _adjust(f, p, rules=None, advance=False, fmt=0, logits="p", ld=100, out="p+", ld_out=100, M=2, V=100, nxt="p"):
    at = lambda x: {"p": p, "p+": p + 16, "p+1": p + 1, None: None}[x]
    r = C.byref(f.LogitsRules(**(rules or {})))
    lib = f.cuda()
    if advance:
        return lib.greta_cuda_logits_adjust_advance(None, r, fmt, at(logits), ld, at(out), ld_out, M, V, at(nxt), None)
    return lib.greta_cuda_logits_adjust(None, r, fmt, at(logits), ld, at(out), ld_out, M, V, at(nxt))


def test_rules_that_are_refused(f):
    buf, p, _, _ = _args(f)
    for bad in (dict(fmt=8), dict(logits=None), dict(out=None, nxt=None), dict(V=0), dict(ld=99), dict(ld_out=99), dict(out="p", ld_out=104), dict(M=65536), dict(logits="p+1"),
                dict(rules=dict(ids=p, ld_ids=4)), dict(rules=dict(ids=p, n_ids=p)), dict(rules=dict(bias_ids=p, bias=p)), dict(rules=dict(bias_ids=p, bias_start=p)),
                dict(rules=dict(allowed=p, ld_allowed=3)), dict(advance=True), dict(advance=True, nxt=None, rules=dict(ids=p, ld_ids=4, n_ids=p))):
        assert _adjust(f, p, **bad) == 4, bad
    assert _adjust(f, p, M=0) == 0

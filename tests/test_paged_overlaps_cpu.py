"""Outputs that lie over inputs in a way that no kernel allows for are refused; rows of two tensors between each other are none such."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from _support import ROOT, load_package


@pytest.fixture(scope="module")
def f():
    p = load_package()
    p.build()
    return p.ffi


@pytest.fixture(scope="module")
def rows_meet(tmp_path_factory):
    """The host check of the kernels' sources by itself."""
    text = open(os.path.join(ROOT, "gretacore-v3_b200", "csrc", "greta_common.cuh")).read()
    at = text.index("inline bool rows_meet(")
    d = tmp_path_factory.mktemp("meet")
    src, so = str(d / "meet.cpp"), str(d / "meet.so")
    open(src, "w").write("#include <stdint.h>\n#include <stddef.h>\n#include <algorithm>\n" + text[at:text.index("\n}\n", at) + 3] +
                         'extern "C" int meet(uint64_t a, size_t pa, size_t wa, uint64_t b, size_t pb, size_t wb, size_t n) { return rows_meet((void *)a, pa, wa, (void *)b, pb, wb, n); }\n')
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-o", so, src], check=True)
    fn = C.CDLL(so).meet
    fn.argtypes = [C.c_uint64, C.c_size_t, C.c_size_t, C.c_uint64, C.c_size_t, C.c_size_t, C.c_size_t]
    return fn


def test_rows_that_meet(rows_meet):
    rng = np.random.default_rng(1)
    met = 0
    for _ in range(20000):
        n = int(rng.integers(0, 6))
        wa, wb = (int(x) for x in rng.integers(1, 9, 2))
        pa = wa + int(rng.integers(0, 12))
        pb = pa if rng.random() < 0.5 and pa >= wb else wb + int(rng.integers(0, 12))
        a, b = 1000, 1000 + int(rng.integers(-90, 90))
        used = np.zeros(3000, bool)
        for i in range(n):
            used[a + i * pa:a + i * pa + wa] = True
        want = any(used[b + i * pb:b + i * pb + wb].any() for i in range(n))
        assert bool(rows_meet(a, pa, wa, b, pb, wb, n)) == want, (a, pa, wa, b, pb, wb, n)
        met += want
    assert 2000 < met < 18000


def test_far_and_long_rows(rows_meet):
    assert not rows_meet(1 << 40, 1 << 34, 64, (1 << 40) + 64, 1 << 34, 64, 1 << 24)
    assert rows_meet(1 << 40, 1 << 34, 65, (1 << 40) + 64, 1 << 34, 64, 1 << 24)
    assert not rows_meet(1 << 62, 64, 64, 1 << 20, 64, 64, 1 << 24) and not rows_meet(1 << 20, 64, 64, 1 << 62, 64, 64, 1 << 24)


def _buf():
    buf = (C.c_uint8 * 65536)()
    return buf, (C.addressof(buf) + 1023) & ~1023


@pytest.mark.parametrize("off,ld_q,ld_o", [(16, 256, 256), (0, 256, 512), (1024 - 16, 256, 512), (2 * 2048 + 1008, 512, 512), (-1008, 256, 256), (2048, 256, 256)])
def test_outputs_of_attention_over_its_queries(f, off, ld_q, ld_o):
    """Three rows of 1024 bytes."""
    buf, p = _buf()
    p += 8192
    cache = f.PagedCache(fmt=1, k=p, v=p, pages=4, kv_heads=2, page=16, dim=64, table=p, ld_table=4)
    rows = f.Ragged(batch=2, tokens=3, max_rows=0, start=p, len=p)
    assert f.cuda().greta_cuda_paged_attn(None, C.byref(cache), C.byref(rows), p, 0, ld_q, p + off, ld_o, 4, 0.125, 0, p, 1 << 40) == 4
    assert (b"overlaps" if off else b"in place") in f.cuda().greta_cuda_last_error()


@pytest.mark.parametrize("q,k,v,out", [(0, 16384, 20480, 16), (0, 16384, 20480, 2048 + 1008), (0, 16384, 20480, 16384 - 16), (0, 16384, 20480, 20480 + 2048), (0, 512, 4096, 0)])
def test_rotated_queries_over_what_is_read(f, q, k, v, out):
    buf, p = _buf()
    p += 4096
    cache = f.PagedCache(fmt=1, k=p, v=p, pages=4, kv_heads=2, page=16, dim=64, table=p, ld_table=4)
    rows = f.Ragged(batch=2, tokens=3, max_rows=0, start=p, len=p)
    rot = f.Rotation(dims=64, interleaved=0, base=10000.0, freq=None, amplitude=1.0)
    assert f.cuda().greta_cuda_paged_append(None, C.byref(cache), C.byref(rows), C.byref(rot), 0, p + q, 256, p + k, 256, p + v, 256, 4, p + out, 0, 256) == 4
    assert b"overlaps" in f.cuda().greta_cuda_last_error()


@pytest.mark.parametrize("off,ld,ld_out", [(4, 100, 100), (396, 100, 200), (-396, 100, 100), (400, 100, 100), (796, 200, 200)])
def test_adjusted_logits_over_the_logits(f, off, ld, ld_out):
    """Two rows of 100."""
    buf, p = _buf()
    p += 4096
    assert f.cuda().greta_cuda_logits_adjust(None, C.byref(f.LogitsRules()), 0, p, ld, p + off, ld_out, 2, 100, None) == 4
    assert b"overlaps" in f.cuda().greta_cuda_last_error()


@pytest.mark.parametrize("scale", [3e38, 2.4e38])
def test_scales_that_leave_the_range_in_powers_of_two(f, scale):
    buf, p = _buf()
    cache = f.PagedCache(fmt=1, k=p, v=p, pages=4, kv_heads=2, page=16, dim=64, table=p, ld_table=4)
    rows = f.Ragged(batch=2, tokens=3, max_rows=0, start=p, len=p)
    assert f.cuda().greta_cuda_paged_attn(None, C.byref(cache), C.byref(rows), p, 0, 256, p + 4096, 256, 4, scale, 0, p, 1 << 40) == 4
    assert b"scale" in f.cuda().greta_cuda_last_error()

"""A process whose first calls of the paged operators are captured; what the replay gives is compared with the calls as they are."""
import ctypes as C

import numpy as np

import _paged as P
from _support import load_package

g = load_package().ffi
lib = g.cuda()
for rows, qt in ((1, "f32"), (40, "f16")):
    bt = P.Batch([(rows, 200), (rows, 90)], 4, 2, 64, 16, "f16", seed=1)
    bt.upload()
    q = P.random_queries(bt, qt)
    ws = g.DeviceBuffer(lib.greta_cuda_paged_attn_workspace_bytes(64), zero=True)
    c, r = bt.structs()
    dq, o, nxt = P.device(q), g.DeviceBuffer(q.nbytes), g.DeviceBuffer(4 * bt.tokens)
    rules = g.LogitsRules()
    s, graph, ex = C.c_void_p(), C.c_void_p(), C.c_void_p()
    g.check(lib.greta_cuda_stream_create(C.byref(s)))
    g.check(lib.greta_cuda_graph_capture_begin(s))
    g.check(lib.greta_cuda_paged_attn(s, C.byref(c), C.byref(r), dq.ptr, P.FMT[qt], 256, o.ptr, 256, 4, 0.125, 0, ws.ptr, ws.nbytes))
    g.check(lib.greta_cuda_logits_adjust(s, C.byref(rules), P.FMT[qt], o.ptr, 256, None, 0, bt.tokens, 256, nxt.ptr))
    g.check(lib.greta_cuda_graph_capture_end(s, C.byref(graph)))
    g.check(lib.greta_cuda_graph_instantiate(graph, C.byref(ex)))
    g.check(lib.greta_cuda_graph_launch(ex, s))
    g.check(lib.greta_cuda_stream_synchronize(s))
    got = o.download(P.itype(qt))
    want = P.run_attention(bt, q, qt)
    assert np.array_equal(got, want.reshape(-1).view(P.itype(qt)))
    assert np.array_equal(nxt.download(np.int32), P.to_f64(want.reshape(bt.tokens, 256), qt).argmax(1))
print("same")

"""Operators of a serving step over a paged cache, measured through the C interface.

  append   new tokens of a ragged batch: queries and keys rotated to their positions, keys and values written into their pages
           (greta_cuda_paged_append)
  attend   those tokens against all keys of their sequences, from one token a sequence to whole prompts (greta_cuda_paged_attn)
  adjust   penalties for repeated tokens, biases and the grammar's mask on logits, and the arg-max of what is left
           (greta_cuda_logits_adjust)

Sequence b holds rows start[b] .. start[b + 1] - 1 of the token buffers and len[b] positions with them; position p lies in page
table[b][p / page] at row p % page, pages are [kv_heads][page][dim].
"""
import ctypes
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one sequence of the 7B shape, a token behind a 512-token prompt: latency
        dict(name="attend_decode_7b", op="attend", batch=1, rows="1", lens="577:577", heads=32, kv_heads=32, dim=128, page=16, window=0, q="f32", cache="f16"),
        # 16 sequences of the 70B shape decoding in step around 4096 positions: the whole cache once
        dict(name="attend_decode_70b_b16", op="attend", batch=16, rows="1", lens="3841:4352", heads=64, kv_heads=8, dim=128, page=32, window=0, q="f32",
             cache="f16"),
        # a busy server: 96 sequences of all ages
        dict(name="attend_decode_ragged_b96", op="attend", batch=96, rows="1", lens="1:8192", heads=32, kv_heads=8, dim=128, page=64, window=0, q="bf16",
             cache="bf16"),
        # five drafted tokens a sequence verified at once, sliding window, heads of 64
        dict(name="attend_verify_b8", op="attend", batch=8, rows="5", lens="900:2500", heads=32, kv_heads=4, dim=64, page=16, window=1024, q="f16", cache="f16"),
        # a portion of a long document: 512 new tokens behind 15872 cached ones
        dict(name="attend_chunk_16k", op="attend", batch=1, rows="512", lens="16384:16384", heads=64, kv_heads=8, dim=128, page=64, window=0, q="bf16",
             cache="bf16"),
        # a whole prompt of the 7B shape
        dict(name="attend_prompt_2048", op="attend", batch=1, rows="2048", lens="2048:2048", heads=32, kv_heads=32, dim=128, page=128, window=0, q="f16",
             cache="f16"),
        # a step that mixes three prompts' portions with 21 decoding sequences
        dict(name="attend_mixed_b24", op="attend", batch=24, rows="700,1024,333,1", lens="1025:6000", heads=64, kv_heads=8, dim=128, page=32, window=0,
             q="bf16", cache="bf16"),
        # the new rows of a decode step of the 70B shape: latency
        dict(name="append_decode_70b_b16", op="append", batch=16, rows="1", lens="3841:4352", heads=64, kv_heads=8, dim=128, page=32, fmt="f32", q="f32",
             cache="f16", base=500000.0, rot=128, interleaved=False),
        # a prompt of the 7B shape: fp32 projections, fp16 queries for the attention behind
        dict(name="append_prompt_2048", op="append", batch=1, rows="2048", lens="2048:2048", heads=32, kv_heads=32, dim=128, page=128, fmt="f32", q="f16",
             cache="f16", base=10000.0, rot=128, interleaved=False),
        # 16384 tokens of eight prompts, some at far positions
        dict(name="append_long_16k", op="append", batch=8, rows="2048", lens="2048:131072", heads=64, kv_heads=8, dim=128, page=64, fmt="bf16", q="bf16",
             cache="bf16", base=500000.0, rot=128, interleaved=False),
        # the choice of one sequence's next token, 7B vocabulary, everything it wrote penalised
        dict(name="adjust_one", op="adjust", batch=1, vocab=32000, history=700, biases=20, mask=False, fmt="f32"),
        # 64 sequences under grammars, 70B vocabulary, long histories
        dict(name="adjust_grammar_b64", op="adjust", batch=64, vocab=128256, history=4096, biases=300, mask=True, fmt="f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "adjust"])
    if op == "adjust":
        vocab = rng.choice([32000, 50257, 128256, _log(rng, 1000, 150000)])
        return dict(op=op, batch=_log(rng, 1, 64), vocab=vocab, history=_log(rng, 1, 4096), biases=rng.choice([0, _log(rng, 1, 300)]), mask=rng.random() < 0.5,
                    fmt=rng.choice(["f32", "f32", "f16", "bf16"]))
    kv_heads = rng.choice([1, 2, 4, 8])
    shape = dict(heads=kv_heads * rng.choice([1, 2, 3, 4, 7, 8]), kv_heads=kv_heads, dim=rng.choice([64, 80, 96, 128, 128, 128]), page=rng.choice([16, 32, 64, 128]),
                 cache=rng.choice(["f16", "bf16"]))
    decode = rng.random() < 0.5
    if op == "append":
        rows = 1 if decode else _log(rng, 2, 2048)
        batch = _log(rng, 1, 96) if decode else _log(rng, 1, 8)
        return dict(op=op, batch=batch, rows=str(rows), lens=f"{rows}:{max(rows, _log(rng, 64, 131072))}", fmt=rng.choice(["f32", shape["cache"]]),
                    q=rng.choice(["f32", shape["cache"]]), base=rng.choice([10000.0, 500000.0]), rot=rng.choice([shape["dim"], 32]),
                    interleaved=rng.random() < 0.3, **shape)
    window = rng.choice([0, 0, 0, _log(rng, 64, 2048)])
    if decode:
        rows, most = rng.choice([1, 1, 1, 2, 4, 5]), _log(rng, 16, 8192)
        return dict(op=op, batch=_log(rng, 1, 96), rows=str(rows), lens=f"{min(max(rows, rng.choice([1, most // 2])), most)}:{most}", window=window,
                    q=rng.choice(["f32", shape["cache"]]), **shape)
    rows = _log(rng, 6, 1024)
    most = max(rows, _log(rng, 64, 12000))
    batch = max(1, min(_log(rng, 1, 24), 2048 // rows))
    return dict(op=op, batch=batch, rows=rng.choice([str(rows), f"{rows},1", f"{rows},{max(1, rows // 3)},2"]), lens=f"{rows}:{most}", window=window,
                q=shape["cache"], **shape)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed, device=DEV):
    return torch.Generator(device=device).manual_seed(seed * 7919 + 17)


def _layout(case, seed):
    """Rows and lengths of each sequence: lengths spread over their range (over its logarithm), never below the rows."""
    kinds = [int(r) for r in case["rows"].split(",")]
    B = case["batch"]
    rows = [kinds[min(b, len(kinds) - 1)] for b in range(B)]
    lo, hi = (int(x) for x in case["lens"].split(":"))
    u = torch.rand(B, generator=_gen(seed, "cpu"), dtype=torch.float64).tolist()
    return rows, [max(r, min(hi, round(math.exp(math.log(lo) + x * (math.log(hi + 1) - math.log(lo)))))) for r, x in zip(rows, u)]


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "adjust":
        return _prepare_adjust(case, g, seed)
    rows, lens = _layout(case, seed)
    B, G, d, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    tokens, H = sum(rows), case["heads"]
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    # pages that are read or written, scattered over the pool; the others of a table are never touched
    first = [(n - r) // page if case["op"] == "append" else 0 for r, n in zip(rows, lens)]
    need = [(n - 1) // page + 1 - f for n, f in zip(lens, first)]
    pages = (sum((r + page - 2) // page + 1 for r in rows) if case["op"] == "append" else sum(need)) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(B, max((n - 1) // page + 1 for n in lens), dtype=torch.int32, device=DEV)
    at = 0
    for b in range(B):
        table[b, first[b]:first[b] + need[b]] = order[at:at + need[b]]
        at += need[b]
    ct = TYPES[case["cache"]]
    s = dict(case=case, rows=rows, lens=lens, start=start, table=table, pages=pages, tokens=tokens,
             d_start=torch.tensor(start, dtype=torch.int32, device=DEV), d_len=torch.tensor(lens, dtype=torch.int32, device=DEV))

    def normal(t, *shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32 if t == torch.float32 else torch.float16).to(t)

    s["k_cache"], s["v_cache"] = normal(ct, pages, G, page, d), normal(ct, pages, G, page, d)
    if case["op"] == "attend":
        s["q"] = normal(TYPES[case["q"]], tokens, H, d) * (0.5 + torch.rand(tokens, 1, 1, generator=g, device=DEV)).to(TYPES[case["q"]])
        s["o"] = torch.empty_like(s["q"])
    else:
        t = TYPES[case["fmt"]]
        s["q"], s["k"], s["v"] = normal(t, tokens, H, d), normal(t, tokens, G, d), normal(t, tokens, G, d)
        s["q_out"] = torch.empty(tokens, H, d, dtype=TYPES[case["q"]], device=DEV)
    if own:
        _handles(s)
    return s


def _prepare_adjust(case, g, seed):
    M, V, n = case["batch"], case["vocab"], case["history"]
    t = TYPES[case["fmt"]]
    u = torch.rand(M, generator=_gen(seed, "cpu"), dtype=torch.float64).tolist()
    n_ids = [max(1, round(n * (0.25 + 0.75 * x))) for x in u]
    n_prompt = [k // 3 for k in n_ids]
    # a text repeats its frequent words: squared uniform ids
    ids = (torch.rand(M, n, generator=g, device=DEV) ** 2 * V).to(torch.int32).clamp_(max=V - 1)
    logits = torch.randn(M, V, generator=g, device=DEV) * 3
    bump = torch.rand(M, n, generator=g, device=DEV) * 8  # what was said before is likely again
    logits.scatter_reduce_(1, ids.long(), bump, "amax")
    s = dict(case=case, ids=ids, n_ids=n_ids, n_prompt=n_prompt, logits=logits.to(t), out=torch.empty(M, V, dtype=t, device=DEV),
             next=torch.empty(M, dtype=torch.int32, device=DEV), d_n=torch.tensor(n_ids, dtype=torch.int32, device=DEV),
             d_prompt=torch.tensor(n_prompt, dtype=torch.int32, device=DEV),
             repetition=1.0 + 0.3 * torch.rand(M, generator=g, device=DEV), frequency=0.5 * torch.rand(M, generator=g, device=DEV),
             presence=0.5 * torch.rand(M, generator=g, device=DEV), bias_ids=None, allowed=None)
    if case["biases"]:
        k = case["biases"]
        rank = torch.rand(M, min(V, 8 * k + 64), generator=g, device=DEV).argsort(1)[:, :k]
        s["bias_ids"] = (rank * (V // rank.shape[1] // 9 + 1) % V).to(torch.int32).contiguous()
        s["bias"] = torch.randn(M, k, generator=g, device=DEV) * 4
        s["bias_start"] = torch.arange(0, M * k + 1, k, dtype=torch.int32, device=DEV)
    if case["mask"]:
        words = (V + 31) // 32
        s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (M, words), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    if own:
        _handles(s)
    return s


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _seq_rows(s, b):
    """Page and row in it of every position of sequence b."""
    p = torch.arange(s["lens"][b], device=DEV)
    page = s["case"]["page"]
    return s["table"][b].long()[p // page], p % page


def _plain_attend(s):
    c = s["case"]
    H, G, d = c["heads"], c["kv_heads"], c["dim"]
    group, scale = H // G, 1.0 / math.sqrt(d)
    out = torch.empty(s["tokens"], H, d, dtype=TYPES[c["q"]], device=DEV)
    for b in range(c["batch"]):
        r, n = s["rows"][b], s["lens"][b]
        pg, at = _seq_rows(s, b)
        k, v = s["k_cache"][pg, :, at].float(), s["v_cache"][pg, :, at].float()  # [n][G][d]
        q = s["q"][s["start"][b]:s["start"][b] + r].float()
        mine, keys = torch.arange(n - r, n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
        hidden = keys > mine
        if c["window"]:
            hidden = hidden | (keys + c["window"] <= mine)
        hidden = hidden[:, None].expand(r, group, n).reshape(r * group, n)
        o = torch.empty(r, H, d, device=DEV)
        for h in range(G):
            x = (q[:, h * group:(h + 1) * group].reshape(r * group, d) @ k[:, h].T) * scale
            x.masked_fill_(hidden, -math.inf)
            x = torch.exp(x - x.amax(1, keepdim=True))
            o[:, h * group:(h + 1) * group] = ((x @ v[:, h]) / x.sum(1, keepdim=True)).view(r, group, d)
        out[s["start"][b]:s["start"][b] + r] = o
    return out


def _positions(s):
    return torch.cat([torch.arange(n - r, n, device=DEV) for r, n in zip(s["rows"], s["lens"])])


def _plain_append(s):
    c = s["case"]
    rot, half = c["rot"], c["rot"] // 2
    freq = c["base"] ** (-torch.arange(half, device=DEV, dtype=torch.float64) * 2 / rot)
    angle = _positions(s).double()[:, None] * freq
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turn(x):
        x = x.float()
        a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if c["interleaved"] else (x[..., :half], x[..., half:rot])
        a, b = a * cos - b * sin, b * cos + a * sin
        y = torch.stack([a, b], -1).flatten(-2) if c["interleaved"] else torch.cat([a, b], -1)
        return torch.cat([y, x[..., rot:]], -1)

    s["q_out"].copy_(turn(s["q"]))
    k, at = turn(s["k"]).to(TYPES[c["cache"]]), 0
    for b in range(c["batch"]):
        r, n = s["rows"][b], s["lens"][b]
        p = torch.arange(n - r, n, device=DEV)
        pg, row = s["table"][b].long()[p // c["page"]], p % c["page"]
        s["k_cache"][pg, :, row] = k[at:at + r]
        s["v_cache"][pg, :, row] = s["v"][at:at + r].to(TYPES[c["cache"]])
        at += r
    return s["q_out"], s["k_cache"], s["v_cache"]


def _bits(words, V):
    return ((words[:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1).flatten(1)[:, :V].bool()


def _plain_adjust(s):
    c = s["case"]
    M, V = c["batch"], c["vocab"]
    ids = s["ids"].long()
    at = torch.arange(ids.shape[1], device=DEV)[None]
    there = at < s["d_n"][:, None]
    seen = torch.zeros(M, V, device=DEV).scatter_add_(1, ids, there.float()) > 0
    count = torch.zeros(M, V, device=DEV).scatter_add_(1, ids, (there & (at >= s["d_prompt"][:, None])).float())
    x, r = s["logits"].float(), s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count
    x = x - torch.where(count > 0, s["presence"][:, None], 0.0)
    if s["bias_ids"] is not None:
        x = x + torch.zeros(M, V, device=DEV).scatter_(1, s["bias_ids"].long(), s["bias"])
    if s["allowed"] is not None:
        x = x.masked_fill(~_bits(s["allowed"], V), -math.inf)
    x = x.to(TYPES[c["fmt"]])
    return x, _first_max(x)


def _first_max(x):
    where = torch.where(x == x.amax(1, keepdim=True), torch.arange(x.shape[1], device=DEV)[None], x.shape[1])
    return where.amin(1).to(torch.int32)


# ---------------------------------------------------------------------------------------------------------------- this library
def _handles(s):
    """Descriptions of the call, as a program keeps them beside its buffers."""
    from __graft_entry__ import load_package
    f = load_package().ffi
    c = s["case"]
    fmt = {"f32": f.FMT_F32, "f16": f.FMT_F16, "bf16": f.FMT_BF16}
    s["lib"], s["check"] = f.cuda(), f.check
    ptr = lambda t: None if t is None else t.data_ptr()
    if c["op"] == "adjust":
        b, M = s["bias_ids"], c["batch"]
        s["rules"] = f.LogitsRules(ids=ptr(s["ids"]), ld_ids=s["ids"].shape[1], n_ids=ptr(s["d_n"]), n_prompt=ptr(s["d_prompt"]), repetition=ptr(s["repetition"]),
                                   frequency=ptr(s["frequency"]), presence=ptr(s["presence"]), bias_ids=ptr(b), bias=ptr(s["bias"]) if b is not None else None,
                                   bias_start=ptr(s["bias_start"]) if b is not None else None, allowed=ptr(s["allowed"]),
                                   ld_allowed=s["allowed"].shape[1] if s["allowed"] is not None else 0)
        s["fmt"] = fmt[c["fmt"]]
        return
    s["cache"] = f.PagedCache(fmt=fmt[c["cache"]], k=ptr(s["k_cache"]), v=ptr(s["v_cache"]), pages=s["pages"], kv_heads=c["kv_heads"], page=c["page"],
                              dim=c["dim"], table=ptr(s["table"]), ld_table=s["table"].shape[1])
    s["ragged"] = f.Ragged(batch=c["batch"], tokens=s["tokens"], max_rows=max(s["rows"]), start=ptr(s["d_start"]), len=ptr(s["d_len"]))
    s["q_fmt"] = fmt[c["q"]]
    if c["op"] == "attend":
        n = s["lib"].greta_cuda_paged_attn_workspace_bytes(c["dim"])
        s["workspace"], s["workspace_bytes"] = torch.zeros(n, dtype=torch.uint8, device=DEV), n
    else:
        s["in_fmt"] = fmt[c["fmt"]]
        s["rotation"] = f.Rotation(dims=c["rot"], interleaved=int(c["interleaved"]), base=c["base"], freq=None, amplitude=1.0)


def _own_attend(s):
    c, ld = s["case"], s["case"]["heads"] * s["case"]["dim"]
    s["check"](s["lib"].greta_cuda_paged_attn(torch.cuda.current_stream().cuda_stream, ctypes.byref(s["cache"]), ctypes.byref(s["ragged"]), s["q"].data_ptr(),
                                              s["q_fmt"], ld, s["o"].data_ptr(), ld, c["heads"], 1.0 / math.sqrt(c["dim"]), c["window"],
                                              s["workspace"].data_ptr(), s["workspace_bytes"]), "paged_attn")
    return s["o"]


def _own_append(s):
    c = s["case"]
    ld, ld_kv = c["heads"] * c["dim"], c["kv_heads"] * c["dim"]
    s["check"](s["lib"].greta_cuda_paged_append(torch.cuda.current_stream().cuda_stream, ctypes.byref(s["cache"]), ctypes.byref(s["ragged"]),
                                                ctypes.byref(s["rotation"]), s["in_fmt"], s["q"].data_ptr(), ld, s["k"].data_ptr(), ld_kv, s["v"].data_ptr(),
                                                ld_kv, c["heads"], s["q_out"].data_ptr(), s["q_fmt"], ld), "paged_append")
    return s["q_out"], s["k_cache"], s["v_cache"]


def _own_adjust(s):
    M, V = s["case"]["batch"], s["case"]["vocab"]
    s["check"](s["lib"].greta_cuda_logits_adjust(torch.cuda.current_stream().cuda_stream, ctypes.byref(s["rules"]), s["fmt"], s["logits"].data_ptr(), V,
                                                 s["out"].data_ptr(), V, M, V, s["next"].data_ptr()), "logits_adjust")
    return s["out"], s["next"]


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"attend": _plain_attend, "append": _plain_append, "adjust": _plain_adjust}[op](state)
    if "lib" not in state:
        _handles(state)
    return {"attend": _own_attend, "append": _own_append, "adjust": _own_adjust}[op](state)


# ---------------------------------------------------------------------------------------------------------------- what a pass needs
def _pairs(r, n, window):
    """Query-key pairs of r rows at the end of n positions, and the keys that any of them sees."""
    seen = sum(min(p + 1, window) if window else p + 1 for p in range(n - r, n))
    return seen, min(n, r - 1 + window) if window else n


def work(case):
    if case["op"] == "adjust":
        M, V = case["batch"], case["vocab"]
        n = 2 * M * V * SIZE[case["fmt"]] + M * (4 * case["history"] * 5 // 8 + 8 * case["biases"]) + (M * V // 8 if case["mask"] else 0)
        return {"bytes": n, "flops": 4 * M * V}
    rows, lens = _layout(case, 0)
    H, G, d, T = case["heads"], case["kv_heads"], case["dim"], sum(rows)
    if case["op"] == "append":
        return {"bytes": T * d * ((H + 2 * G) * SIZE[case["fmt"]] + H * SIZE[case["q"]] + 2 * G * SIZE[case["cache"]]), "flops": 3 * T * (H + G) * case["rot"]}
    pairs, keys = (sum(x) for x in zip(*(_pairs(r, n, case["window"]) for r, n in zip(rows, lens))))
    return {"bytes": 2 * T * H * d * SIZE[case["q"]] + 2 * keys * G * d * SIZE[case["cache"]], "flops": 4 * pairs * H * d}


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """From the definitions, head by head (or row by row), in float64."""
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    f64 = torch.float64
    if case["op"] == "adjust":
        return _exact_adjust(s, f64)
    H, G, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    starts = s["start"]
    if case["op"] == "attend":
        out = torch.zeros(s["tokens"], H, d, dtype=f64, device=DEV)
        for b in range(case["batch"]):
            n, r = s["lens"][b], s["rows"][b]
            held = s["table"][b, :(n + page - 1) // page].long()
            for g in range(G):
                k = s["k_cache"][held, g].reshape(-1, d)[:n].to(f64)
                v = s["v_cache"][held, g].reshape(-1, d)[:n].to(f64)
                for h in range(g * (H // G), (g + 1) * (H // G)):
                    score = torch.einsum("rd,nd->rn", s["q"][starts[b]:starts[b + 1], h].to(f64), k) * d ** -0.5
                    far = (torch.arange(r, device=DEV) + n - r)[:, None] - torch.arange(n, device=DEV)
                    seen = far >= 0
                    if case["window"]:
                        seen &= far < case["window"]
                    score = torch.where(seen, score, torch.full_like(score, -math.inf))
                    out[starts[b]:starts[b + 1], h] = torch.softmax(score, -1) @ v
        return out
    rot, base = case["rot"], case["base"]
    where = [(b, s["lens"][b] - s["rows"][b] + i) for b in range(case["batch"]) for i in range(s["rows"][b])]
    p = torch.tensor([x[1] for x in where], dtype=f64, device=DEV)
    pair = torch.arange(rot // 2, device=DEV)
    z = torch.polar(torch.ones(1, dtype=f64, device=DEV), torch.outer(p, torch.exp(-2.0 * pair.to(f64) / rot * math.log(base))))[:, None]
    first, second = (2 * pair, 2 * pair + 1) if case["interleaved"] else (pair, pair + rot // 2)

    def turned(x):
        y = x.to(f64)
        w = torch.complex(y[..., first], y[..., second]) * z
        y[..., first], y[..., second] = w.real, w.imag
        return y

    q, k = turned(s["q"].clone()), turned(s["k"].clone())
    kc, vc = s["k_cache"].to(f64), s["v_cache"].to(f64)
    slot = s["table"].long()[torch.tensor([x[0] for x in where], device=DEV), (p.long() // page)]
    kc[slot, :, p.long() % page], vc[slot, :, p.long() % page] = k, s["v"].to(f64)
    return q, kc, vc


def _exact_adjust(s, f64):
    case, out = s["case"], []
    V = case["vocab"]
    for m in range(case["batch"]):
        ids = s["ids"][m, :s["n_ids"][m]].long()
        x = s["logits"][m].to(f64)
        said = torch.bincount(ids[s["n_prompt"][m]:], minlength=V).to(f64)
        r = s["repetition"][m].to(f64)
        for_seen = torch.maximum(x / r, torch.zeros((), dtype=f64, device=DEV)) + torch.minimum(x * r, torch.zeros((), dtype=f64, device=DEV))
        x = torch.where(torch.bincount(ids, minlength=V) > 0, for_seen, x)
        x = x - said * s["frequency"][m].to(f64) - (said > 0).to(f64) * s["presence"][m].to(f64)
        if s["bias_ids"] is not None:
            x[s["bias_ids"][m].long()] += s["bias"][m].to(f64)
        if s["allowed"] is not None:
            j = torch.arange(V, device=DEV)
            x[(s["allowed"][m].long()[j // 32] >> (j % 32)) % 2 == 0] = -math.inf
        out.append(x)
    x = torch.stack(out)
    return x, _first_max(x.to(TYPES[case["fmt"]]))

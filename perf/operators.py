"""Cases for the serving operators around the 8-bit paged KV cache: rotary
positions, the append that rotates and quantizes new tokens into the cache,
attention over the cache, and the page operations (fork, extend, free,
compact).  `run` computes a case either with the framework (`own`) or in
plain torch operations in 32 bits; `exact` gives the definition in 64 bits.

Sizes: 16 query / 2 KV heads of 128 and 36 layers are the 3B-class model of
the benchmark, 40 / 8 heads of 128 the 14B/32B-class one, heads of 64 the
other head size that the decode attention serves.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 16          # tokens that share one scale
QMAX = {"int8": 127.0, "e4m3": 448.0}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases -------------------------------------------------------------

def listed():
    return [
        # one token of the 3B-class model: the smallest rotation there is, all latency
        dict(name="rotary_token_f32", op="rotary", dtype="f32", layout="interleaved", tokens=1, heads=16, dim=128,
             rot=128, inverse=False, spare=0),
        # a prompt of the 14B-class model, q inside the fused projection's rows, half of each head rotated
        dict(name="rotary_prompt_bf16", op="rotary", dtype="bf16", layout="half", tokens=8191, heads=40, dim=128,
             rot=64, inverse=False, spare=2048),
        # a decode step of 48 sequences: k and v of one token each into partly filled blocks, q rotated beside
        dict(name="append_step_f32_int8", op="append", dtype="f32", fmt="int8", layout="interleaved", batch=48,
             heads=40, kv_heads=8, dim=128, rot=128, page=64, new_min=1, new_max=1, len_min=20, len_max=4000, mix=1),
        # ragged prompts written at once
        dict(name="append_prompts_bf16_e4m3", op="append", dtype="bf16", fmt="e4m3", layout="half", batch=7,
             heads=40, kv_heads=8, dim=128, rot=128, page=128, new_min=300, new_max=4097, len_min=300, len_max=6000,
             mix=2),
        # the 3B-class decode step at its benchmarked context of 1,024 tokens
        dict(name="attend_token_f32_int8", op="attend", dtype="f32", fmt="int8", batch=1, heads=16, kv_heads=2,
             dim=128, page=64, new_min=1, new_max=1, len_min=1024, len_max=1024, window=0, mix=3),
        # a serving batch of the 14B-class model with ragged contexts
        dict(name="attend_batch_bf16_e4m3", op="attend", dtype="bf16", fmt="e4m3", batch=32, heads=40, kv_heads=8,
             dim=128, page=64, new_min=1, new_max=1, len_min=500, len_max=9000, window=0, mix=4),
        # one very long context: the cache is read once, by all of the card
        dict(name="attend_long_f32_int8", op="attend", dtype="f32", fmt="int8", batch=1, heads=40, kv_heads=8,
             dim=128, page=128, new_min=1, new_max=1, len_min=200001, len_max=200001, window=0, mix=5),
        # several proposed tokens a sequence verified at once, heads of 64, a sliding window
        dict(name="attend_verify_f16_int8", op="attend", dtype="f16", fmt="int8", batch=9, heads=8, kv_heads=8,
             dim=64, page=16, new_min=3, new_max=5, len_min=40, len_max=3001, window=1000, mix=6),
        # chunks of prompts of the 3B-class model with part of the context already cached
        dict(name="attend_chunk_f32_int8", op="attend", dtype="f32", fmt="int8", batch=3, heads=16, kv_heads=2,
             dim=128, page=64, new_min=333, new_max=1024, len_min=1000, len_max=2500, window=0, mix=7),
        # a long prompt's chunk of the 14B-class model: matrix products bound it
        dict(name="attend_prompt_bf16_e4m3", op="attend", dtype="bf16", fmt="e4m3", batch=1, heads=40, kv_heads=8,
             dim=128, page=128, new_min=4096, new_max=4096, len_min=8192, len_max=8192, window=0, mix=8),
        # parallel sampling on the 3B-class model: 60 children drop their old branch, fork anew, grow by a token
        dict(name="pages_fork_int8", op="fork", fmt="int8", layers=36, kv_heads=2, dim=128, page=64, parents=4,
             children=60, len_min=100, len_max=900, mix=9),
        # a pool with holes after many sequences left: the used pages move down
        dict(name="pages_compact_e4m3", op="compact", fmt="e4m3", layers=36, kv_heads=2, dim=128, page=32, parents=24,
             children=0, len_min=100, len_max=900, mix=10),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "attend", "prompt", "fork", "compact"])
    dtype, fmt = rng.choice(list(DTYPES)), rng.choice(list(QMAX))
    heads, kv_heads, dim = rng.choice([(16, 2, 128), (40, 8, 128), (8, 8, 64), (12, 3, 64), (7, 1, 128), (6, 6, 128)])
    page, layout, mix = rng.choice([16, 32, 64, 128]), rng.choice(["interleaved", "half"]), rng.randrange(1 << 20)
    if op == "rotary":
        return dict(op=op, dtype=dtype, layout=layout, tokens=_log(rng, 1, 8191), heads=heads, dim=dim,
                    rot=rng.choice([dim, dim // 2, dim - 2, 2 * rng.randint(1, dim // 2)]), inverse=rng.random() < 0.3,
                    spare=rng.choice([0, 8, 129]))
    if op == "append":
        batch = _log(rng, 1, 48)
        most = _log(rng, 1, max(1, 20000 // batch))
        return dict(op=op, dtype=dtype, fmt=fmt, layout=layout, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim,
                    rot=rng.choice([dim, dim // 2]), page=page, new_min=rng.randint(1, most), new_max=most,
                    len_min=rng.randint(1, most), len_max=most + _log(rng, 1, 3000), mix=mix)
    if op == "attend":
        batch = _log(rng, 1, 32)
        most = _log(rng, 1, max(2, 200000 // batch))
        new = rng.choice([1, 1, 1, rng.randint(2, 8)])
        return dict(op="attend", dtype=dtype, fmt=fmt, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                    new_min=1, new_max=min(new, most), len_min=rng.randint(1, most), len_max=most,
                    window=rng.choice([0, 0, 0, rng.randint(1, 2000)]), mix=mix)
    if op == "prompt":
        batch = rng.randint(1, 4)
        most = _log(rng, 17, 4096 // batch)
        return dict(op="attend", dtype=dtype, fmt=fmt, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                    new_min=rng.randint(1, most), new_max=most, len_min=rng.randint(1, most),
                    len_max=most + _log(rng, 1, 4096), window=rng.choice([0, 0, 0, rng.randint(1, 2000)]), mix=mix)
    return dict(op=op, fmt=fmt, layers=rng.choice([3, 24, 36]), kv_heads=kv_heads, dim=dim, page=page,
                parents=rng.randint(2, 20), children=rng.randint(1, 60) if op == "fork" else 0,
                len_min=rng.randint(1, 200), len_max=rng.randint(201, 900), mix=mix)


def _plan(case):
    """Lengths (new tokens included) and new tokens of each sequence."""
    rng = random.Random(case["mix"])
    lens, news = [], []
    for b in range(case["batch"]):
        n = case["new_max"] if b == 0 else rng.randint(case["new_min"], case["new_max"])
        length = case["len_max"] if b == 0 else _log(rng, case["len_min"], case["len_max"])
        lens.append(max(length, n))
        news.append(n)
    return lens, news


def _page_plan(case):
    rng = random.Random(case["mix"])
    parents = [_log(rng, case["len_min"], case["len_max"]) for _ in range(case["parents"])]
    return parents, [rng.randrange(case["parents"]) for _ in range(case["children"])]


# ---- the inputs ------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _tables(rot, positions):
    """cos and sin [positions][rot/2], base 1e6, each rounded once from 64 bits."""
    freq = 1e6 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _pool(case, layers, pages, g):
    """Keys and values of earlier tokens, quantized: some channels of the keys are several times the others."""
    kvh, page, dim = case["kv_heads"], case["page"], case["dim"]
    out = {}
    for name in ("k", "v"):
        shape = (layers * pages * kvh * (page // BLOCK), BLOCK, dim)
        wide = 1.0 + 3.0 * (torch.rand(dim, device="cuda", generator=g) < 0.05) if name == "k" else 1.0
        codes = torch.empty(shape, dtype=torch.uint8, device="cuda")
        scale = torch.empty(shape[0], device="cuda")
        for at in range(0, shape[0], 1 << 16):
            x = torch.randn((min(1 << 16, shape[0] - at), BLOCK, dim), device="cuda", generator=g) * wide
            s = _pow2(x.abs().amax(dim=(1, 2)), case["fmt"])
            scale[at:at + x.shape[0]] = s
            codes[at:at + x.shape[0]] = _encode(x / s[:, None, None], case["fmt"])
        out[name] = codes.view(layers, pages, kvh, page, dim)
        out[name + "_scale"] = scale.view(layers, pages, kvh, page // BLOCK)
    return out


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "rotary":
        T, H, D = case["tokens"], case["heads"], case["dim"]
        rows = torch.randn(T, H * D + case["spare"], device="cuda", generator=g).to(DTYPES[case["dtype"]])
        cos, sin = _tables(case["rot"], 16384)
        pos = torch.randint(0, 16384 - T, (1,), device="cuda", generator=g) + torch.arange(T, device="cuda")
        return dict(case=case, x=rows[:, :H * D].view(T, H, D), cos=cos, sin=sin, pos=pos.int())
    if case["op"] in ("fork", "compact"):
        return _prepare_pages(case, g)
    lens, news = _plan(case)
    B, H, KVH, D, P = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    dt = DTYPES[case["dtype"]]
    T = sum(news)
    cap = max(-(-n // P) for n in lens) + 1
    need = [-(-n // P) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, device="cuda", generator=g).int()
    table = torch.full((B, cap), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    st = dict(case=case, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
              cu=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_new=max(news), max_len=max(lens),
              q=torch.randn(T, H, D, device="cuda", generator=g).to(dt), **_pool(case, 1, pages, g))
    if case["op"] == "append":
        # the projections' output: q, k and v of a token in one row
        kv = torch.randn(T, 2 * KVH * D, device="cuda", generator=g).to(dt)
        st["new_k"], st["new_v"] = kv[:, :KVH * D].view(T, KVH, D), kv[:, KVH * D:].view(T, KVH, D)
        st["cos"], st["sin"] = _tables(case["rot"], max(lens))
        # the rows read back: every valid token of each block that the call writes to
        seq, pos = [], []
        for b, (n, m) in enumerate(zip(lens, news)):
            first = (n - m) // BLOCK * BLOCK
            seq.append(torch.full((n - first,), b, dtype=torch.int32, device="cuda"))
            pos.append(torch.arange(first, n, dtype=torch.int32, device="cuda"))
        st["seq"], st["pos"] = torch.cat(seq), torch.cat(pos)
    if own:
        from vibrant_b200 import kv8
        st["cache"] = kv8.Cache(1, pages, P, KVH, D, case["fmt"], buffers=(st["k"], st["v"], st["k_scale"],
                                                                            st["v_scale"]))
        st["batch"] = kv8.Batch(table, st["lens"], cu_tokens=st["cu"], tokens=T, max_tokens=max(news),
                                max_len=max(lens))
    return st


def _prepare_pages(case, g):
    P = case["page"]
    parents, kids = _page_plan(case)
    lens = parents + [0] * len(kids)
    need = [-(-n // P) for n in lens]
    if case["op"] == "fork":
        # the children hold an older branch of one page; a tenth of the pool is left over
        lens = parents + [max(1, P // 2)] * len(kids)
        need = [-(-n // P) for n in lens]
        pages = sum(need) + 2 * len(kids) + 8
    else:
        pages = 2 * sum(need)  # half of the pool is holes
    cap = max(need) + 2
    order = torch.randperm(pages, device="cuda", generator=g).int()
    table = torch.full((len(lens), cap), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    refs[order[:at].long()] = 1
    # one buffer of bookkeeping: the table, the lengths, the references
    book = torch.cat([table.reshape(-1), torch.tensor(lens, dtype=torch.int32, device="cuda"), refs])
    st = dict(case=case, book=book, start=book.clone(), rows=len(lens), cap=cap, pages=pages)
    _split_book(st)
    shape = (case["layers"], pages, case["kv_heads"], P, case["dim"])
    for name in ("k", "v"):
        codes = torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=g)
        st[name] = codes & 0xFE if case["fmt"] == "e4m3" else codes  # e4m3: without the two NaN codes
        st[name + "_scale"] = torch.exp2(torch.randint(-9, 3, shape[:3] + (P // BLOCK,), device="cuda",
                                                       generator=g).float())
    st["src"] = torch.tensor(kids, dtype=torch.int32, device="cuda")
    st["dst"] = torch.arange(len(parents), len(lens), dtype=torch.int32, device="cuda")
    st["one"] = torch.ones(len(kids), dtype=torch.int32, device="cuda")
    if own:
        from vibrant_b200 import kv8
        st["cache"] = kv8.Cache(case["layers"], pages, P, case["kv_heads"], case["dim"], case["fmt"],
                                buffers=(st["k"], st["v"], st["k_scale"], st["v_scale"]))
        st["seqs"] = kv8.Sequences(st["cache"], len(lens), cap, buffers=(st["table"], st["lens"], st["refs"]))
    return st


def _split_book(st):
    n = st["rows"] * st["cap"]
    st["table"] = st["book"][:n].view(st["rows"], st["cap"])
    st["lens"] = st["book"][n:n + st["rows"]]
    st["refs"] = st["book"][n + st["rows"]:]


# ---- one pass --------------------------------------------------------------

def run(st):
    case = st["case"]
    return {"rotary": _run_rotary, "append": _run_append, "attend": _run_attend, "fork": _run_fork,
            "compact": _run_compact}[case["op"]](st, case)


def _run_rotary(st, case):
    if own:
        from vibrant_b200 import tensor as vt
        return vt.rotary(st["x"], st["cos"], st["sin"], st["pos"], layout=case["layout"], inverse=case["inverse"])
    return _rotate(st["x"], st["cos"], st["sin"], st["pos"], case["layout"], case["inverse"]).to(st["x"].dtype)


def _run_append(st, case):
    if own:
        q = st["cache"].append(0, st["batch"], st["new_k"], st["new_v"], q=st["q"], cos=st["cos"], sin=st["sin"],
                               layout=case["layout"])
        k, v = st["cache"].read(0, st["batch"], st["seq"], st["pos"])
        return {"q": q, "k": k, "v": v}
    T = st["q"].shape[0]
    pos = torch.arange(T, device="cuda")
    seq = torch.searchsorted(st["cu"][1:].long(), pos, right=True)
    pos = pos - st["cu"].long()[seq + 1] + st["lens"].long()[seq]
    q = _rotate(st["q"], st["cos"], st["sin"], pos, case["layout"], False).to(st["q"].dtype)
    k = _rotate(st["new_k"], st["cos"], st["sin"], pos, case["layout"], False)
    _append(st, case, "k", k)
    _append(st, case, "v", st["new_v"].float())
    return {"q": q, "k": _read(st, case, "k"), "v": _read(st, case, "v")}


def _run_attend(st, case):
    if own:
        return st["cache"].attend(0, st["batch"], st["q"], window=case["window"])
    H, KVH, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    G, B, N = H // KVH, case["batch"], st["max_new"]
    used = -(-st["max_len"] // P)
    page = st["table"][:, :used].long().clamp(min=0)
    lens, cu = st["lens"].long(), st["cu"].long()
    new = cu[1:] - cu[:-1]

    def rows(name):  # [B, KVH, used * P, D]
        x = _decode(st[name][0][page], case["fmt"])
        x = x.view(B, used, KVH, P // BLOCK, BLOCK, D) * st[name + "_scale"][0][page][..., None, None]
        return x.permute(0, 2, 1, 3, 4, 5).reshape(B, KVH, used * P, D)

    i = torch.arange(N, device="cuda")
    at = (cu[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)
    q = st["q"].float()[at].view(B, N, KVH, G, D).permute(0, 2, 3, 1, 4).reshape(B, KVH, G * N, D)
    s = q @ rows("k").transpose(2, 3)
    s *= 1.0 / math.sqrt(D)
    j = torch.arange(used * P, device="cuda")
    p = (lens - new)[:, None] + i  # [B, N]: the positions of the queries
    seen = (j <= p[..., None]) & (j < lens[:, None, None])
    if case["window"]:
        seen &= j > p[..., None] - case["window"]
    s = s.view(B, KVH, G, N, used * P).masked_fill_(~seen[:, None, None], -math.inf)
    s -= s.amax(dim=-1, keepdim=True)
    s = s.exp_()
    s /= s.sum(dim=-1, keepdim=True)
    o = s.view(B, KVH, G * N, used * P) @ rows("v")
    o = o.view(B, KVH, G, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, H, D)
    t = torch.arange(st["q"].shape[0], device="cuda")
    seq = torch.searchsorted(cu[1:], t, right=True)
    return o[seq, t - cu[seq]].to(st["q"].dtype)


def _state(st):
    kind = torch.float8_e4m3fn if st["case"]["fmt"] == "e4m3" else torch.int8
    return [st["k"].view(kind), st["v"].view(kind), st["k_scale"], st["v_scale"], st["table"], st["lens"], st["refs"]]


def _run_fork(st, case):
    if own:
        s = st["seqs"]
        s.free(st["dst"])
        s.fork(st["src"], st["dst"])
        s.extend(st["dst"], st["one"])
        return _state(st)
    P, table, lens, refs = case["page"], st["table"], st["lens"], st["refs"]
    col = torch.arange(st["cap"], device="cuda")
    src, dst = st["src"].long(), st["dst"].long()
    # free: the children's pages lose a reference
    held = table[dst]
    there = held >= 0
    refs.index_add_(0, held.clamp(min=0).reshape(-1).long(), -there.reshape(-1).int())
    # fork: whole pages are shared, the part-filled last one goes into a free page (the lowest first)
    n = lens[src]
    full, part = n // P, n % P > 0
    row = torch.where(col < full[:, None], table[src], -1)
    refs.index_add_(0, row.clamp(min=0).reshape(-1).long(), (row >= 0).reshape(-1).int())
    free = torch.argsort(refs > 0, stable=True)
    new = free[(part.cumsum(0) - part.int())]
    old = table[src].gather(1, full[:, None].long().clamp(max=st["cap"] - 1))[:, 0]
    row = torch.where((col == full[:, None]) & part[:, None], new[:, None].int(), row)
    refs.index_add_(0, new, part.int())
    # a child without such a page moves nothing: its parent's first page onto itself
    old, new = torch.where(part, old, table[src, 0]).long(), torch.where(part, new, table[src, 0].long())
    for name in ("k", "v", "k_scale", "v_scale"):
        st[name][:, new] = st[name][:, old]
    # extend by one token: a child whose pages are full takes a free page
    more = (n % P == 0)
    free = torch.argsort(refs > 0, stable=True)
    new = free[(more.cumsum(0) - more.int())]
    row = torch.where((col == full[:, None]) & more[:, None], new[:, None].int(), row)
    refs.index_add_(0, new, more.int())
    table[dst] = row
    lens[dst] = n + 1
    return _state(st)


def _run_compact(st, case):
    # the same holes in every pass: the bookkeeping as it stood (the pages that moved still hold their contents)
    st["book"].copy_(st["start"])
    if own:
        st["seqs"].compact()
        return _state(st)
    table, refs = st["table"], st["refs"]
    page = torch.arange(st["pages"], device="cuda")
    used = refs > 0
    count = used.sum()
    # the k-th used page above the count goes to the k-th free page below it
    holes = (~used & (page < count)).nonzero()[:, 0]
    movers = (used & (page >= count)).nonzero()[:, 0]
    for name in ("k", "v", "k_scale", "v_scale"):
        st[name][:, holes] = st[name][:, movers]
    to = page.int().index_copy(0, movers, holes.int())
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    refs[holes] = refs[movers]
    refs[movers] = 0
    return _state(st)


# ---- the plain forms' parts ------------------------------------------------

def _rotate(x, cos, sin, pos, layout, inverse):
    x = x.float()
    half = cos.shape[1]
    c, s = cos[pos.long()][:, None], sin[pos.long()][:, None]
    if inverse:
        s = -s
    if layout == "half":
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * c - b * s, a * s + b * c, x[..., 2 * half:]], dim=-1)
    a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
    turned = torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1)


def _pow2(a, fmt):
    """The least power of two s in [2^-64, 2^63] with a <= qmax * s."""
    top = 6 if fmt == "int8" else 8
    e = torch.frexp(a.clamp(min=1e-30))[1] - 1 - top
    s = torch.exp2(e.float())
    s = torch.where(a > QMAX[fmt] * s, s * 2, s)
    return s.clamp(2.0 ** -64, 2.0 ** 63)


def _encode(x, fmt):
    if fmt == "int8":
        return x.round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _decode(codes, fmt):
    return codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float()


def _append(st, case, name, x):
    """Writes x [T, KVH, D] as the last tokens of the sequences; a block's
    scale covers its new tokens and is never below the one it had."""
    P, KVH, D, fmt = case["page"], case["kv_heads"], case["dim"], case["fmt"]
    lens, cu = st["lens"].long(), st["cu"].long()
    first = lens - (cu[1:] - cu[:-1])
    many = st["max_new"] // BLOCK + 2
    block = (first // BLOCK)[:, None] + torch.arange(many, device="cuda")  # [B, many]
    pos = block[..., None] * BLOCK + torch.arange(BLOCK, device="cuda")    # [B, many, 16]
    is_new = (pos >= first[:, None, None]) & (pos < lens[:, None, None])
    is_old = (pos < first[:, None, None]) & is_new.any(-1, keepdim=True)
    at = (cu[:-1, None, None] + pos - first[:, None, None]).clamp(0, x.shape[0] - 1)
    new = x[at].permute(0, 1, 3, 2, 4)  # [B, many, KVH, 16, D]
    page = st["table"].long().gather(1, (block * BLOCK // P).clamp(max=st["table"].shape[1] - 1)).clamp(min=0)
    inside = block % (P // BLOCK)
    codes = st[name].view(-1, KVH, P // BLOCK, BLOCK, D)
    scale = st[name + "_scale"].view(-1, KVH, P // BLOCK)
    head = torch.arange(KVH, device="cuda")
    where = (page[..., None], head, inside[..., None])
    s_new = _pow2((new.abs() * is_new[:, :, None, :, None]).amax(dim=(3, 4)), fmt)
    s_old = scale[where]
    s = torch.where(is_old.any(-1)[..., None], torch.maximum(s_old, s_new), s_new)
    old = codes[where]
    kept = _encode(_decode(old, fmt) * (s_old / s)[..., None, None], fmt)
    fresh = _encode(new * (1.0 / s)[..., None, None], fmt)
    out = torch.where(is_new[:, :, None, :, None], fresh, torch.where(is_old[:, :, None, :, None], kept, old))
    touched = is_new.any(-1)
    where = tuple(w.expand(s.shape)[touched] for w in where)
    codes[where] = out[touched]
    scale[where] = s[touched]


def _read(st, case, name):
    P = case["page"]
    seq, pos = st["seq"].long(), st["pos"].long()
    page = st["table"].long()[seq, pos // P]
    inside = pos % P
    return _decode(st[name][0][page, :, inside], case["fmt"]) * st[name + "_scale"][0][page, :, inside // BLOCK][..., None]


# ---- the definition in 64 bits ---------------------------------------------

def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None  # nothing is computed: pages move
    st = prepare(case, seed)
    if case["op"] == "rotary":
        return _turn64(st["x"], st, st["pos"].long(), case["layout"], -1.0 if case["inverse"] else 1.0)
    lens, cu = st["lens"].tolist(), st["cu"].tolist()
    return _exact_append(case, st, lens, cu) if case["op"] == "append" else _exact_attend(case, st, lens, cu)


def _turn64(x, st, pos, layout, sign):
    """Each pair as a complex number times cos + i sin."""
    x = x.double().clone()
    turn = torch.complex(st["cos"].double(), sign * st["sin"].double())[pos][:, None]
    half = turn.shape[-1]
    if layout == "half":
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
        x[..., :half], x[..., half:2 * half] = z.real, z.imag
    else:
        z = torch.complex(x[..., :2 * half:2], x[..., 1:2 * half:2]) * turn
        x[..., :2 * half:2], x[..., 1:2 * half:2] = z.real, z.imag
    return x


def _values64(case, st, name, b, n):
    """[KVH, n, D]: the cached rows of sequence b."""
    P = case["page"]
    page = st["table"][b, :-(-n // P)].long()
    codes = st[name][0][page]
    codes = codes.view(torch.int8).double() if case["fmt"] == "int8" else codes.view(torch.float8_e4m3fn).double()
    codes = codes * st[name + "_scale"][0][page].double().repeat_interleave(BLOCK, dim=2)[..., None]
    return codes.transpose(0, 1).reshape(case["kv_heads"], -1, case["dim"])[:, :n]


def _code64(y, fmt):
    """y rounded to the format, ties to even, saturating."""
    if fmt == "int8":
        return torch.round(y).clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(y / step) * step).clamp(-448, 448)


def _exact_append(case, st, lens, cu):
    T = st["q"].shape[0]
    pos = torch.cat([torch.arange(n - (e - a), n, device="cuda") for n, a, e in zip(lens, cu, cu[1:])])
    fresh = {"k": _turn64(st["new_k"], st, pos, case["layout"], 1.0), "v": st["new_v"].double()}
    out = {"q": _turn64(st["q"], st, pos, case["layout"], 1.0), "k": [], "v": []}
    assert out["q"].shape[0] == T
    top = QMAX[case["fmt"]]
    for name in ("k", "v"):
        for b, n in enumerate(lens):
            first = n - (cu[b + 1] - cu[b])
            low = first // BLOCK * BLOCK
            rows = torch.cat([_values64(case, st, name, b, first)[:, low:].transpose(0, 1),
                              fresh[name][cu[b]:cu[b + 1]]])  # [n - low, KVH, D]
            grown = torch.cat([rows, rows.new_zeros((-rows.shape[0] % BLOCK,) + rows.shape[1:])])
            grown = grown.view(-1, BLOCK, *rows.shape[1:])
            newer = (torch.arange(low, low + grown.shape[0] * BLOCK, device="cuda") >= first).view(-1, BLOCK)
            a = (grown.abs() * newer[..., None, None]).amax(dim=(1, 3))  # [blocks, KVH]
            s = torch.exp2(torch.ceil(torch.log2(a / top))).clamp(2.0 ** -64, 2.0 ** 63)
            if low < first:
                page = int(st["table"][b, low // case["page"]])
                s[0] = torch.maximum(s[0], st[name + "_scale"][0, page, :, low % case["page"] // BLOCK].double())
            s = s[:, None, :, None]
            out[name].append((_code64(grown / s, case["fmt"]) * s).flatten(0, 1)[:n - low])
        out[name] = torch.cat(out[name])
    return out


def _exact_attend(case, st, lens, cu):
    H, KVH, D = case["heads"], case["kv_heads"], case["dim"]
    G = H // KVH
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        m = cu[b + 1] - cu[b]
        k, v = _values64(case, st, "k", b, n), _values64(case, st, "v", b, n)
        p = torch.arange(n - m, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")
        hidden = (j > p) if not case["window"] else (j > p) | (j <= p - case["window"])
        for h in range(H):
            s = (st["q"][cu[b]:cu[b + 1], h].double() @ k[h // G].T) / math.sqrt(D)
            out[cu[b]:cu[b + 1], h] = torch.softmax(s.masked_fill(hidden, -math.inf), dim=-1) @ v[h // G]
    return out


# ---- what a pass cannot do without -----------------------------------------

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}.get(case.get("dtype"), 0)
    if case["op"] == "rotary":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * size + case["tokens"] * (4 * case["rot"] + 4), "flops": 3 * n}
    D, KVH = case["dim"], case["kv_heads"]
    row = 2 * KVH * (D + 4 / BLOCK)  # a cached token's codes and scales, K and V
    if case["op"] in ("fork", "compact"):
        parents, kids = _page_plan(case)
        P = case["page"]
        if case["op"] == "fork":
            moved = sum(parents[i] % P > 0 for i in kids)
        else:
            moved = sum(-(-n // P) for n in parents) / 2  # half of the used pages lie above, on average
        return {"bytes": 2 * moved * case["layers"] * P * row, "flops": 0}
    lens, news = _plan(case)
    T, H = sum(news), case["heads"]
    if case["op"] == "append":
        touched = sum(n - (n - m) // BLOCK * BLOCK for n, m in zip(lens, news))
        old = touched - T
        # q in and out, k and v in, the codes out, the older codes of the first blocks in; then the rows read back
        return {"bytes": T * (2 * H + 2 * KVH) * D * size + touched * row + old * row + touched * (row + 8 * KVH * D)
                + T * case["rot"] * 4, "flops": 3 * T * (H + KVH) * D}
    pairs, read = 0, 0
    for n, m in zip(lens, news):
        w = case["window"] or n
        pairs += sum(min(p + 1, w) for p in range(n - m, n))
        read += min(n, m - 1 + w)
    return {"bytes": 2 * T * H * D * size + read * row, "flops": 4 * D * H * pairs}

"""The 8-bit paged KV cache: append (codes and scales bit for bit against a
float32 restatement), read-back, and attention against float64."""
import numpy as np
import pytest

import kv8_helpers as kh

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


def _cache(pool, layers=1, layer=0):
    """A device cache whose `layer` holds the host pool; other layers are poison."""
    import torch
    from vibrant_b200 import kv8
    pages, kvh, page, dim = pool.shape
    c = kv8.Cache(layers, pages, page, kvh, dim, pool.fmt)
    for t, a in ((c.k, pool.k), (c.v, pool.v), (c.k_scale, pool.ks), (c.v_scale, pool.vs)):
        t.fill_(127 if t.dtype == torch.uint8 else float("nan"))
        t[layer].copy_(torch.from_numpy(a))
    return c


def _batch(table, lens, cu, slots=None, max_len=None):
    import torch
    from vibrant_b200 import kv8
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()  # noqa: E731
    news = np.diff(cu)
    return kv8.Batch(dev(table), dev(lens), cu_tokens=dev(cu), slots=None if slots is None else dev(slots),
                     tokens=int(cu[-1]), max_tokens=max(1, int(news.max())), max_len=max_len)


def _same_pool(c, layer, pool):
    for t, a in ((c.k, pool.k), (c.v, pool.v), (c.k_scale, pool.ks), (c.v_scale, pool.vs)):
        got = t[layer].cpu().numpy()
        assert np.array_equal(got.view(np.uint8), a.view(np.uint8)), np.argwhere(got != a)[:4]


# (lengths with the new tokens, new tokens) of each sequence
APPENDS = [([1], [1]), ([17], [1]), ([16], [1]), ([16, 33, 0, 100], [16, 17, 0, 1]), ([70, 5, 48], [70, 3, 15]),
           ([130], [40])]


def _append(fmt, dtype, D, KVH, page, layout, rot, lens, news, pages=24):
    import torch
    from vibrant_b200 import tensor as vt, vkq
    rng = np.random.default_rng(sum(lens) + D + KVH)
    H = 2 * KVH + KVH
    pool = kh.Pool(pages, KVH, page, D, fmt, rng)
    table = kh.table_for(rng, lens, page, pages)
    cu = np.concatenate([[0], np.cumsum(news)])
    T = int(cu[-1])
    c = _cache(pool, layers=2, layer=1)
    dt = getattr(torch, DT[dtype])
    # k, v and q in the rows of one projection; some blocks' values far larger or smaller than others'
    rows = torch.from_numpy((rng.standard_normal((T, (H + 2 * KVH) * D)) *
                             2.0 ** rng.integers(-12, 6, (T, 1))).astype(np.float32)).cuda().to(dt)
    q, k, v = (t.unflatten(1, (-1, D)) for t in rows.split([H * D, KVH * D, KVH * D], dim=1))
    batch = _batch(table, lens, cu)
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, news)])
    cos = sin = None
    if layout:
        cos, sin = vt.rotary_tables(rot, 1e4, max(lens))
        got_q = c.append(1, batch, k, v, q=q, cos=cos, sin=sin, layout=layout)
        turn = lambda x: kh.rotate(x.float().cpu().numpy(), cos.cpu().numpy(), sin.cpu().numpy(), pos, layout)  # noqa: E731
        assert torch.equal(got_q.cpu(), torch.from_numpy(turn(q)).to(dt))
    else:
        assert c.append(1, batch, k, v) is None
        turn = lambda x: x.float().cpu().numpy()  # noqa: E731
    nk, nv = turn(k), v.float().cpu().numpy()
    for b in range(len(lens)):
        pool.append("k", table[b], lens[b] - news[b], nk[cu[b]:cu[b + 1]])
        pool.append("v", table[b], lens[b] - news[b], nv[cu[b]:cu[b + 1]])
    _same_pool(c, 1, pool)
    assert bool((c.k[0] == 127).all()) and bool(torch.isnan(c.v_scale[0]).all())
    assert vkq.device_status(0) == vkq.OK
    # rows read back
    seq = np.repeat(np.arange(len(lens)), lens).astype(np.int32)
    at = np.concatenate([np.arange(n) for n in lens]).astype(np.int32)
    rk, rv = c.read(1, batch, torch.from_numpy(seq).cuda(), torch.from_numpy(at).cuda())
    for which, r in (("k", rk), ("v", rv)):
        want = np.concatenate([pool.rows(which, table[b], n).transpose(1, 0, 2) for b, n in enumerate(lens)])
        assert np.array_equal(r.cpu().numpy().astype(np.float64), want)
    assert vkq.device_status(0) == vkq.OK


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,D,KVH,page,layout,rot", [
    ("f32", 128, 2, 64, "interleaved", 128), ("bf16", 128, 1, 16, "half", 128), ("f16", 64, 3, 32, "half", 30),
    ("f32", 64, 1, 128, "half", 64), ("bf16", 64, 2, 48, "interleaved", 32), ("f32", 128, 2, 16, None, 0)])
@pytest.mark.parametrize("lens,news", APPENDS, ids=str)
def test_append_matches_float32(fmt, dtype, D, KVH, page, layout, rot, lens, news):
    _append(fmt, dtype, D, KVH, page, layout, rot, lens, news)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,D,KVH,page,layout,rot", [
    ("f32", 128, 2, 64, "interleaved", 64), ("bf16", 128, 3, 64, "half", 128), ("f16", 64, 1, 128, None, 0)])
def test_append_of_long_prompts(fmt, dtype, D, KVH, page, layout, rot):
    """Enough tokens that a CTA takes all heads of its block; ragged ends, a single token among them."""
    _append(fmt, dtype, D, KVH, page, layout, rot, [5003, 40, 0, 3100], [4990, 1, 0, 3100], pages=136)


@pytest.mark.parametrize("fmt,bound", [("int8", 1.0), ("e4m3", None)])
def test_append_token_by_token(fmt, bound):
    """A block filled by 16 calls whose values grow: what the repeated
    roundings add up to stays within one step of the last scale (half a step
    each, the scales at least doubling), and equals the restatement."""
    import torch
    rng = np.random.default_rng(4)
    pool = kh.Pool(3, 1, 16, 64, fmt, rng)
    c = _cache(pool)
    x = (rng.standard_normal((16, 1, 64)) * (1.4 ** np.arange(16))[:, None, None]).astype(np.float32)
    for t in range(16):
        batch = _batch([[2]], [t + 1], [0, 1])
        row = torch.from_numpy(x[t:t + 1]).cuda()
        c.append(0, batch, row, row)
        pool.append("k", [2], t, x[t:t + 1])
        pool.append("v", [2], t, x[t:t + 1])
    _same_pool(c, 0, pool)
    got = pool.rows("k", [2], 16)[0]
    if bound is not None:
        assert float(np.abs(got - x[:, 0]).max()) <= bound * float(pool.ks[2, 0, 0])


def test_append_values_outside_the_numbers():
    """NaN is stored as 0, infinities saturate, neither sets a block's scale;
    tiny and huge blocks keep their scale within [2^-64, 2^63]."""
    import torch
    rng = np.random.default_rng(5)
    for fmt in ("int8", "e4m3"):
        pool = kh.Pool(4, 2, 16, 64, fmt, rng)
        c = _cache(pool)
        x = rng.standard_normal((40, 2, 64)).astype(np.float32)
        x[3, 0, 5], x[4, 0, 6], x[5, 1, 7] = np.nan, np.inf, -np.inf
        x[16:32, 0] = 0.0
        x[16:32, 1] = np.nan
        x[32:, 0] *= np.float32(1e-30)
        x[32:, 1] *= np.float32(1e30)
        t = torch.from_numpy(x).cuda()
        c.append(0, _batch([[3, 1, 0]], [40], [0, 40]), t, t)
        pool.append("k", [3, 1, 0], 0, x)
        pool.append("v", [3, 1, 0], 0, x)
        _same_pool(c, 0, pool)
        assert np.isfinite(pool.rows("k", [3, 1, 0], 40)).all()


def test_append_bad_sequences():
    """A length or page out of bounds: nothing of it is written, the others are, the status says so."""
    import torch
    from vibrant_b200 import vkq
    rng = np.random.default_rng(6)
    pool = kh.Pool(4, 1, 16, 64, "int8", rng)
    x = rng.standard_normal((4, 1, 64)).astype(np.float32)
    t = torch.from_numpy(x).cuda()
    # sequence 0 is longer than the table, 1 has a page out of range, 2 more new tokens than its length, 3 is good
    table = [[0, 1], [9, -1], [2, -1], [3, -1]]
    lens = [33, 1, 0, 5]
    c = _cache(pool)
    c.append(0, _batch(table, lens, [0, 1, 2, 3, 4]), t, t)
    assert vkq.device_status(0) == vkq.ERR_INVALID_ARGUMENT
    pool.append("k", [3], 4, x[3:])
    pool.append("v", [3], 4, x[3:])
    _same_pool(c, 0, pool)
    # offsets that leave the tokens, and a slot that leaves the rows
    c.append(0, _batch(table, lens, [0, 1, 2, 3, 4], slots=[3, 4, -1, 7]), t[:4], t[:4])
    assert vkq.device_status(0) == vkq.ERR_INVALID_ARGUMENT
    pool.append("k", [3], 4, x[:1])
    pool.append("v", [3], 4, x[:1])
    _same_pool(c, 0, pool)
    seq = torch.tensor([3, 3, 4, 1, -1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([0, 5, 0, 0, 0], dtype=torch.int32, device="cuda")
    k, v = c.read(0, _batch(table, lens, [0, 1, 2, 3, 4]), seq, pos, dtype=torch.bfloat16)
    assert vkq.device_status(0) == vkq.ERR_INVALID_ARGUMENT
    assert bool(torch.isfinite(k[0]).all()) and bool(torch.isnan(k[1:]).all()) and bool(torch.isnan(v[1:]).all())


def _attend(dtype, fmt, H, KVH, D, page, lens, news, causal=True, window=0, scale=None, seed=0, qscale=1.0,
            slots=None, max_len=None, spare=0):
    import torch
    from vibrant_b200 import vkq
    rng = np.random.default_rng(seed + sum(lens) + H + D)
    need = sum(-(-n // page) for n in lens)
    pool = kh.Pool(need + 2, KVH, page, D, fmt, rng)
    table = kh.table_for(rng, lens, page, need + 2)
    cu = np.concatenate([[0], np.cumsum(news)])
    T = int(cu[-1])
    rows = torch.from_numpy((rng.standard_normal((T, H * D + spare)) * qscale).astype(np.float32)).cuda()
    rows = rows.to(getattr(torch, DT[dtype]))
    q = rows[:, spare:].unflatten(1, (H, D))
    c = _cache(pool, layers=2, layer=1)
    # codes past the lengths are never used: int8 -128 and e4m3 NaN there
    bad = np.uint8(0x80 if fmt == "int8" else 0x7F)
    k, v = c.k.cpu().numpy(), c.v.cpu().numpy()
    for b, n in enumerate(lens):
        if n % page:
            k[1, table[b, n // page], :, n % page:] = bad
            v[1, table[b, n // page], :, n % page:] = bad
    c.k.copy_(torch.from_numpy(k))
    c.v.copy_(torch.from_numpy(v))
    batch = _batch(table, lens, cu, max_len=max_len)
    got = c.attend(1, batch, q, causal=causal, window=window, scale=scale)
    assert vkq.device_status(0) == vkq.OK
    sc = float(np.float32(D ** -0.5 if scale is None else scale))
    out, bound, size = kh.attention(q.float().cpu().numpy(), pool, table, lens, cu, sc, causal, window)
    got64 = got.float().cpu().numpy().astype(np.float64)
    err = np.abs(got64 - out) - kh.attention_tolerance(dtype, out, bound, size)
    assert float(err.max()) <= 0.0, (float(err.max()), np.unravel_index(err.argmax(), err.shape))
    again = c.attend(1, batch, q, causal=causal, window=window, scale=scale)
    assert torch.equal(got, again)  # the same bits whatever the timing, and a workspace left ready
    return got64, out


HEADS = [(16, 2, 128), (5, 1, 128), (6, 6, 64), (24, 8, 64), (33, 1, 64)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("H,KVH,D", HEADS, ids=str)
@pytest.mark.parametrize("page,lens", [(16, [1]), (64, [1, 2, 15, 16, 17, 31, 32, 33, 64, 65]), (128, [1000, 7]),
                                       (32, [5000])], ids=str)
def test_decode_matches_float64(dtype, fmt, H, KVH, D, page, lens):
    _attend(dtype, fmt, H, KVH, D, page, lens, [1] * len(lens))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("H,KVH,D", HEADS, ids=str)
@pytest.mark.parametrize("page,lens,news,window", [
    (16, [5, 3, 40], [5, 1, 3], 0), (64, [300, 129, 64], [7, 129, 0], 0), (64, [300, 129, 64], [7, 129, 1], 33),
    (32, [700], [257], 1), (128, [513, 100], [512, 100], 100), (64, [1024], [384], 0)], ids=str)
def test_chunks_match_float64(dtype, fmt, H, KVH, D, page, lens, news, window):
    _attend(dtype, fmt, H, KVH, D, page, lens, news, window=window)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("lens,news", [([90], [90]), ([200, 33], [3, 33]), ([700], [1])], ids=str)
def test_without_causal(dtype, lens, news):
    _attend(dtype, "int8", 8, 2, 64, 32, lens, news, causal=False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("news", [1, 200])
def test_peaked_and_flat_scores(dtype, news):
    """Scores hundreds apart and scores all alike."""
    _attend(dtype, "int8", 8, 2, 128, 64, [400], [news], qscale=40.0)
    _attend(dtype, "e4m3", 8, 2, 128, 64, [400], [news], qscale=1e-6)
    _attend(dtype, "int8", 8, 2, 64, 64, [400], [news], scale=1e-3 if dtype == "f16" else 1e-9, qscale=1e3)


def test_rows_that_see_nothing():
    """More new tokens than the length: the tokens before position 0 give zeros."""
    for dtype in ("f32", "bf16"):
        got, out = _attend(dtype, "int8", 8, 2, 64, 16, [3, 0], [5, 2])
        assert (got[:2] == 0).all() and (got[5:] == 0).all() and (out[2] != 0).any()
        got, _ = _attend(dtype, "e4m3", 8, 2, 128, 16, [3, 200], [150, 200])
        assert (got[:147] == 0).all() and (got[147] != 0).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_and_unaligned_rows(dtype):
    for spare in (1, 8, 64):
        _attend(dtype, "int8", 6, 2, 64, 32, [100, 40], [1, 1], spare=spare)
        _attend(dtype, "int8", 6, 2, 64, 32, [300, 140], [150, 140], spare=spare)


@pytest.fixture(params=[1 << 15, 1 << 18], ids=lambda n: f"bound{n}")
def wide(request, monkeypatch):
    """Tables whose bound on the lengths is large: many rows then take the 128-row
    tiles, in several ranges of keys, whatever the lengths are."""
    plain = _batch

    def batch(table, lens, cu, slots=None, max_len=None):
        pages = np.full((table.shape[0], request.param // 16), -1, np.int32)
        pages[:, :table.shape[1]] = table
        return plain(pages, lens, cu, slots, request.param)

    monkeypatch.setitem(globals(), "_batch", batch)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("H,KVH,D", HEADS, ids=str)
@pytest.mark.parametrize("page,lens,news,window", [
    (64, [300, 129, 64], [7, 129, 0], 0), (64, [300, 129, 64], [7, 129, 1], 33), (32, [700], [257], 1),
    (128, [513, 100], [512, 100], 100), (16, [3000, 1], [40, 1], 0)], ids=str)
def test_many_rows_match_float64(wide, dtype, fmt, H, KVH, D, page, lens, news, window):
    _attend(dtype, fmt, H, KVH, D, page, lens, news, window=window)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_many_rows_without_causal(wide, dtype):
    _attend(dtype, "int8", 8, 2, 64, 32, [90], [90], causal=False)
    _attend(dtype, "e4m3", 8, 2, 128, 64, [2500, 33], [40, 33], causal=False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_many_rows_peaked_and_flat(wide, dtype):
    test_peaked_and_flat_scores(dtype, 200)


def test_many_rows_that_see_nothing(wide):
    for dtype in ("f32", "bf16"):
        got, _ = _attend(dtype, "e4m3", 8, 2, 128, 16, [3, 200], [150, 200])
        assert (got[:147] == 0).all() and (got[147] != 0).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows_strided_and_unaligned(wide, dtype):
    for spare in (1, 8, 64):
        _attend(dtype, "int8", 6, 2, 64, 32, [300, 140], [150, 140], spare=spare)
        _attend(dtype, "int8", 6, 2, 128, 32, [1300, 140], [150, 140], spare=spare)


def test_many_rows_non_finite_query(wide):
    test_non_finite_query_stays_in_its_row()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows_bad_pages(wide, dtype):
    """A page out of bounds gives NaN for the rows that see it; other sequences are right."""
    import torch
    from vibrant_b200 import vkq
    rng = np.random.default_rng(12)
    pool = kh.Pool(200, 1, 16, 64, "int8", rng)
    lens, news = [1300, 1300], 100
    table = kh.table_for(rng, lens, 16, 200)
    c = _cache(pool)
    q = torch.randn(2 * news, 2, 64, device="cuda").to(getattr(torch, DT[dtype]))
    cu = np.array([0, news, 2 * news])
    for at, page in ((4, 200), (60, -1)):
        wrong = table.copy()
        wrong[1, at] = page
        got = c.attend(0, _batch(wrong, lens, cu), q).float().cpu().numpy()
        assert vkq.device_status(0) == vkq.ERR_INVALID_ARGUMENT
        assert np.isnan(got[news:]).all()
        out, bound, size = kh.attention(q.float().cpu().numpy()[:news], pool, table[:1], lens[:1], cu[:2], float(np.float32(0.125)))
        assert float((np.abs(got[:news] - out) - kh.attention_tolerance(dtype, out, bound, size)).max()) <= 0
    assert vkq.device_status(0) == vkq.OK


def test_many_rows_bad_offsets(wide):
    """Token offsets and lengths out of bounds: reported, NaN where the rows are known."""
    import torch
    from vibrant_b200 import vkq
    rng = np.random.default_rng(13)
    pool = kh.Pool(40, 1, 16, 64, "int8", rng)
    lens = [130, 130]
    table = kh.table_for(rng, lens, 16, 40)
    c = _cache(pool)
    q = torch.randn(200, 2, 64, device="cuda")
    want = c.attend(0, _batch(table, lens, [0, 100, 200]), q)
    assert vkq.device_status(0) == vkq.OK
    for cu in ([0, 100, 205], [0, 100, 90], [-1, 100, 200]):
        b = _batch(table, lens, [0, 100, 200])
        b.tensors[3].copy_(torch.tensor(cu, dtype=torch.int32))
        got = c.attend(0, b, q)
        assert vkq.device_status(0) == vkq.ERR_INVALID_ARGUMENT
        good = slice(0, 100) if cu[0] == 0 else slice(100, 200)
        assert torch.equal(got[good], want[good])
    got = c.attend(0, _batch(table, [-1, 130], [0, 100, 200]), q)
    assert vkq.device_status(0) == vkq.ERR_INVALID_ARGUMENT
    assert bool(torch.isnan(got[:100]).all()) and torch.equal(got[100:], want[100:])
    assert vkq.device_status(0) == vkq.OK


def test_slots_and_output_strides():
    import torch
    from vibrant_b200 import kv8
    rng = np.random.default_rng(8)
    pool = kh.Pool(12, 2, 16, 64, "int8", rng)
    lens = [40, 0, 25, 90]
    table = kh.table_for(rng, lens, 16, 12)
    c = _cache(pool)
    q = torch.randn(2, 4, 64, device="cuda")
    wide = torch.full((2, 6, 64), float("nan"), device="cuda")
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()  # noqa: E731
    b = kv8.Batch(dev(table), dev(lens), slots=dev([3, 0]))  # one token each
    got = c.attend(0, b, q, out=wide[:, 1:5])
    out, bound, size = kh.attention(q.cpu().numpy(), pool, table[[3, 0]], [90, 40], [0, 1, 2], float(np.float32(0.125)))
    assert float((np.abs(got.cpu().numpy() - out) - kh.attention_tolerance("f32", out, bound, size)).max()) <= 0
    assert bool(torch.isnan(wide[:, 0]).all()) and bool(torch.isnan(wide[:, 5]).all())


@pytest.mark.parametrize("news", [1, 100])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_bad_sequences(dtype, news):
    """A length or page out of bounds gives NaN for its rows, the others are right, the status says so."""
    import torch
    from vibrant_b200 import vkq
    rng = np.random.default_rng(9)
    dt = getattr(torch, DT[dtype])
    pool = kh.Pool(40, 1, 16, 64, "int8", rng)
    lens = [130, 130, 130]
    table = kh.table_for(rng, lens, 16, 40)
    table[1, 4] = 40
    c = _cache(pool)
    cu = np.array([0, news, 2 * news, 3 * news])
    q = torch.randn(3 * news, 2, 64, device="cuda").to(dt)
    shown = np.array(lens)
    shown[2] = 16 * table.shape[1] + 1
    got = c.attend(0, _batch(table, shown, cu), q).float().cpu().numpy()
    assert vkq.device_status(0) == vkq.ERR_INVALID_ARGUMENT
    # a causal row whose keys end before the bad page may still be right: the last rows of sequence 1 are not
    assert np.isnan(got[2 * news - 1]).all() and np.isnan(got[2 * news:]).all()
    out, bound, size = kh.attention(q.float().cpu().numpy()[:news], pool, table[:1], lens[:1], cu[:2], float(np.float32(0.125)))
    assert float((np.abs(got[:news] - out) - kh.attention_tolerance(dtype, out, bound, size)).max()) <= 0
    # token offsets out of bounds: no row of theirs is known
    c.attend(0, _batch(table, lens, [0, news, 3 * news + 5, 3 * news]), q)
    assert vkq.device_status(0) == vkq.ERR_INVALID_ARGUMENT
    assert vkq.device_status(0) == vkq.OK


def test_non_finite_query_stays_in_its_row():
    import torch
    for dtype in ("f32", "bf16"):
        for news in (1, 120):
            rng = np.random.default_rng(10)
            pool = kh.Pool(20, 1, 16, 64, "e4m3", rng)
            table = kh.table_for(rng, [150], 16, 20)
            c = _cache(pool)
            q = torch.randn(news, 4, 64, device="cuda").to(getattr(torch, DT[dtype]))
            batch = _batch(table, [150], [0, news])
            want = c.attend(0, batch, q)
            q[0, 1, 3], q[0, 2, 3] = float("nan"), float("inf")
            got = c.attend(0, batch, q)
            assert bool(torch.isnan(got[0, 1]).all()) and bool(torch.isnan(got[0, 2]).all())
            assert torch.equal(got[0, [0, 3]], want[0, [0, 3]]) and torch.equal(got[1:], want[1:])


def test_other_stream_and_graph():
    """On a stream of its own, and replayed in a CUDA graph while the lengths grow on the device."""
    import torch
    rng = np.random.default_rng(11)
    pool = kh.Pool(40, 2, 16, 128, "int8", rng)
    table = kh.table_for(rng, [500], 16, 40)
    c = _cache(pool)
    lens = torch.tensor([100], dtype=torch.int32, device="cuda")
    from vibrant_b200 import kv8
    b = kv8.Batch(torch.from_numpy(table).cuda(), lens, max_len=500)
    q = torch.randn(1, 8, 128, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = c.attend(0, b, q)
    s.synchronize()
    ref = lambda n: kh.attention(q.cpu().numpy(), pool, table, [n], [0, 1], float(np.float32(128 ** -0.5)))  # noqa: E731
    o, bound, size = ref(100)
    assert float((np.abs(out.cpu().numpy() - o) - kh.attention_tolerance("f32", o, bound, size)).max()) <= 0
    ws = torch.zeros(c.workspace_bytes(b, q.dtype, 8), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.attend(0, b, q, out=out, ws=ws)
    for n in (1, 100, 333, 500):
        lens.fill_(n)
        graph.replay()
        o, bound, size = ref(n)
        assert float((np.abs(out.cpu().numpy() - o) - kh.attention_tolerance("f32", o, bound, size)).max()) <= 0


def test_refusals():
    import torch
    from vibrant_b200 import kv8, vkq
    c = kv8.Cache(1, 8, 16, 2, 64)
    table = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")
    b = kv8.Batch(table, lens)
    x = torch.zeros(2, 2, 64, device="cuda")
    q = torch.zeros(2, 4, 64, device="cuda")
    cos = torch.ones(64, 32, device="cuda")
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")

    def attn(cache=None, batch=None, **kw):
        a = dict(dtype=vkq.F32, q=q.data_ptr(), qs=256, o=q.data_ptr(), os=256, heads=4, scale=0.1, ws=ws.data_ptr(),
                 wb=ws.numel(), causal=True, window=0, layer=0)
        a.update(kw)
        vkq.kv8_attention(cache or c.struct, a["layer"], batch or b.bounds(16), a["dtype"], a["q"], a["qs"], a["o"],
                          a["os"], a["heads"], a["scale"], a["ws"], a["wb"], a["causal"], a["window"], device=0)

    def changed(struct, **kw):
        s = type(struct).from_buffer_copy(struct)
        for k, v in kw.items():
            setattr(s, k, v)
        return s

    I, U, M, W = vkq.ERR_INVALID_ARGUMENT, vkq.ERR_UNSUPPORTED, vkq.ERR_MISALIGNED, vkq.ERR_WORKSPACE
    bb = b.bounds(16)
    for kw, status in [(dict(dtype=3), U), (dict(heads=3), I), (dict(heads=0), I), (dict(scale=0.0), I),
                       (dict(scale=float("nan")), I), (dict(window=-1), I), (dict(window=5, causal=False), I),
                       (dict(ws=None), W), (dict(wb=100), W), (dict(q=None), I), (dict(q=q.data_ptr() + 2), M),
                       (dict(qs=255), I), (dict(layer=1), I), (dict(layer=-1), I),
                       (dict(cache=changed(c.struct, format=2)), U), (dict(cache=changed(c.struct, head_dim=96)), U),
                       (dict(cache=changed(c.struct, page_size=24)), I), (dict(cache=changed(c.struct, k=None)), I),
                       (dict(cache=changed(c.struct, k=c.k.data_ptr() + 4)), M),
                       (dict(cache=changed(c.struct, num_pages=0)), I),
                       (dict(batch=changed(bb, batch=3)), I), (dict(batch=changed(bb, max_len=65)), I),
                       (dict(batch=changed(bb, tokens=1)), I), (dict(batch=changed(bb, table=None)), I),
                       (dict(batch=changed(bb, max_tokens=0)), I), (dict(batch=changed(bb, batch=70000)), I)]:
        with pytest.raises(vkq.VkqError) as e:
            attn(**kw)
        assert e.value.status == status, kw
    attn(batch=changed(bb, tokens=0, cu_tokens=lens.data_ptr()))  # nothing to do
    for kw, status in [(dict(rot=63), I), (dict(rot=66), I), (dict(layout=5), I), (dict(seq=0), I),
                       (dict(sin=None), I), (dict(ks=127), I), (dict(k=None), I), (dict(heads=3), I),
                       (dict(qo=None), I), (dict(qos=512), I)]:
        a = dict(k=x.data_ptr(), ks=128, rot=64, layout=0, seq=64, sin=cos.data_ptr(), heads=4, qo=q.data_ptr(), qos=256)
        a.update(kw)
        with pytest.raises(vkq.VkqError) as e:
            vkq.kv8_append(c.struct, 0, bb, vkq.F32, a["k"], a["ks"], x.data_ptr(), 128, q.data_ptr(), 256, a["qo"],
                           a["qos"], a["heads"], cos.data_ptr(), a["sin"], a["seq"], a["rot"], a["layout"], device=0)
        assert e.value.status == status, kw
    one = lens.data_ptr()
    for args, status in [((None, one, 1, 0, x.data_ptr(), None), I), ((one, one, 0, 0, x.data_ptr(), None), I),
                         ((one, one, 1, 0, None, None), I), ((one, one, 1, 7, x.data_ptr(), None), U),
                         ((one, one, 1, 0, x.data_ptr() + 4, None), M)]:
        with pytest.raises(vkq.VkqError) as e:
            vkq.kv8_read(c.struct, 0, bb, *args, device=0)
        assert e.value.status == status, args
    for bad in (lambda: c.attend(0, b, q[:1]), lambda: c.attend(0, b, q.double()), lambda: c.append(0, b, x, x.half()),
                lambda: c.append(0, b, x, x, q=q), lambda: kv8.Cache(1, 8, 20, 2, 64),
                lambda: kv8.Cache(1, 8, 16, 2, 64, "int4"), lambda: kv8.Batch(table.long(), lens),
                lambda: c.attend(0, b, q.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            bad()
    assert vkq.device_status(0) == vkq.OK

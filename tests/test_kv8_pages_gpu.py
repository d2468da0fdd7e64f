"""The page operations of the 8-bit KV cache against a plain restatement of
their rules (a page is free when no row holds it, the lowest numbers first)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Model:
    """The rules in plain Python; pool [layers, pages, 4 arrays]."""

    def __init__(self, rows, cap, pages, page, pool):
        self.table = np.full((rows, cap), -1, np.int32)
        self.lens = np.zeros(rows, np.int32)
        self.refs = np.zeros(pages, np.int32)
        self.page, self.cap, self.pool = page, cap, pool

    def _take(self, k):
        free = np.flatnonzero(self.refs == 0)[:k]
        self.refs[free] = 1
        return free

    def extend(self, slots, add):
        done, seen, owed = [], set(), 0
        start = int((self.refs == 0).sum())
        for r, a in zip(slots, add):
            ok = 0 <= r < len(self.lens) and r not in seen and a >= 0 and self.lens[r] + a <= self.cap * self.page
            if ok:
                have = -(-int(self.lens[r]) // self.page)
                need = -(-int(self.lens[r] + a) // self.page) - have
                ok = need == 0 or owed + need <= start
                owed += need
                if ok:
                    self.table[r, have:have + need] = self._take(need)
                    self.lens[r] += a
            seen.add(r)
            done.append(int(ok))
        return done

    def fork(self, src, dst):
        before, done, seen, owed = self.lens.copy(), [], set(), 0
        start = int((self.refs == 0).sum())
        for s, d in zip(src, dst):
            ok = 0 <= d < len(before) and 0 <= s < len(before) and s != d and d not in seen and before[d] == 0
            if ok:
                n = int(before[s])
                full, part = n // self.page, int(n % self.page > 0)
                ok = not part or owed + 1 <= start
                owed += part
                if ok:
                    if part:
                        new = self._take(1)[0]
                        for x in self.pool:
                            x[:, new] = x[:, self.table[s, full]]
                        self.table[d, full] = new
                    self.table[d, :full] = self.table[s, :full]
                    np.add.at(self.refs, self.table[s, :full], 1)
                    self.lens[d] = n
            seen.add(d)
            done.append(int(ok))
        return done

    def free(self, slots):
        done, seen = [], set()
        for r in slots:
            ok = 0 <= r < len(self.lens) and r not in seen
            if ok:
                n = -(-int(self.lens[r]) // self.page)
                np.subtract.at(self.refs, self.table[r, :n], 1)
                self.table[r, :n] = -1
                self.lens[r] = 0
            seen.add(r)
            done.append(int(ok))
        return done

    def compact(self):
        u = int((self.refs > 0).sum())
        holes = np.flatnonzero(self.refs[:u] == 0)
        movers = u + np.flatnonzero(self.refs[u:] > 0)
        to = np.arange(len(self.refs), dtype=np.int32)
        to[movers] = holes
        for x in self.pool:
            x[:, holes] = x[:, movers]
        self.refs[holes], self.refs[movers] = self.refs[movers], 0
        self.table = np.where(self.table >= 0, to[self.table], -1).astype(np.int32)
        return u


def _make(layers, pages, page, kvh, dim, rows, cap, seed=0):
    import torch
    from vibrant_b200 import kv8
    c = kv8.Cache(layers, pages, page, kvh, dim)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c.k.random_(0, 256, generator=g)
    c.v.random_(0, 256, generator=g)
    c.k_scale.uniform_(generator=g)
    c.v_scale.uniform_(generator=g)
    m = Model(rows, cap, pages, page, [t.cpu().numpy() for t in (c.k, c.v, c.k_scale, c.v_scale)])
    return c, kv8.Sequences(c, rows, cap), m


def _dev(a):
    import torch
    return torch.tensor(list(a), dtype=torch.int32, device="cuda")


def _check(c, s, m):
    assert np.array_equal(s.table.cpu().numpy(), m.table)
    assert np.array_equal(s.lens.cpu().numpy(), m.lens)
    assert np.array_equal(s.refs.cpu().numpy(), m.refs)
    for t, x in zip((c.k, c.v, c.k_scale, c.v_scale), m.pool):
        assert np.array_equal(t.cpu().numpy(), x)


def _do(s, m, what, *lists):
    import torch
    done = torch.full((len(lists[0]),), -1, dtype=torch.int32, device="cuda")
    getattr(s, what)(*(_dev(x) for x in lists), done=done)
    want = getattr(m, what)(*lists)
    assert done.tolist() == want, what
    return want


@pytest.mark.parametrize("layers,pages,page,kvh,dim", [(1, 40, 16, 1, 64), (3, 200, 32, 2, 128), (2, 1030, 64, 3, 64)])
def test_random_histories(layers, pages, page, kvh, dim):
    """Growing, forking, emptying and compacting in random order, down to an empty pool."""
    from vibrant_b200 import vkq
    import torch
    rows, cap = 24, 9
    c, s, m = _make(layers, pages, page, kvh, dim, rows, cap, seed=pages)
    rng = np.random.default_rng(pages)
    for step in range(40):
        live, empty = np.flatnonzero(m.lens > 0), np.flatnonzero(m.lens == 0)
        op = rng.integers(0, 4)
        if op == 0 or not len(live):
            pick = rng.permutation(rows)[:rng.integers(1, rows)]
            room = cap * page - m.lens[pick]
            _do(s, m, "extend", pick.tolist(), [int(rng.integers(0, min(r, 3 * page) + 1)) for r in room])
        elif op == 1 and len(empty):
            dst = rng.permutation(empty)[:rng.integers(1, len(empty) + 1)]
            _do(s, m, "fork", rng.choice(live, len(dst)).tolist(), dst.tolist())
        elif op == 2:
            _do(s, m, "free", rng.permutation(live)[:rng.integers(1, len(live) + 1)].tolist())
        else:
            used = torch.zeros(1, dtype=torch.int32, device="cuda")
            s.compact(used)
            assert int(used) == m.compact()
        if step % 8 == 7:
            _check(c, s, m)
    _do(s, m, "free", list(range(rows)))
    _check(c, s, m)
    assert not m.refs.any()
    assert vkq.device_status(0) == vkq.OK


def test_pool_runs_out():
    """Rows in the order listed: those whose pages are past the last free one stay as they were."""
    from vibrant_b200 import vkq
    c, s, m = _make(1, 10, 16, 1, 64, 8, 6)
    assert _do(s, m, "extend", [0, 1, 2, 3], [33, 80, 64, 16]) == [1, 1, 0, 0]
    _check(c, s, m)
    assert _do(s, m, "extend", [2, 1, 0], [40, 0, 15]) == [0, 1, 1]  # 2 wants three pages of two; the others none
    assert _do(s, m, "fork", [0, 1, 0], [4, 5, 6]) == [1, 1, 1]      # both part-filled pages of row 0's copies? row 0 is full
    _check(c, s, m)
    assert _do(s, m, "extend", [2], [17]) == [1]
    assert _do(s, m, "fork", [2], [7]) == [0]                        # its part-filled page finds no free one
    _check(c, s, m)
    assert vkq.device_status(0) == vkq.OK


def test_invalid_rows():
    """Rows out of range, listed twice, or not empty: left out and reported; the others are served."""
    from vibrant_b200 import vkq
    c, s, m = _make(2, 30, 16, 1, 64, 6, 4)
    assert _do(s, m, "extend", [0, 0, 6, -1, 1, 2], [20, 5, 5, 5, 65, 30]) == [1, 0, 0, 0, 0, 1]
    assert vkq.device_status(0) == vkq.ERR_INVALID_ARGUMENT
    assert _do(s, m, "fork", [0, 0, 2, 9, 3], [3, 3, 0, 4, 3]) == [1, 0, 0, 0, 0]
    assert vkq.device_status(0) == vkq.ERR_INVALID_ARGUMENT
    assert _do(s, m, "fork", [5, 0], [4, 5]) == [1, 1]  # row 5 was empty when the call began
    assert vkq.device_status(0) == vkq.OK
    assert _do(s, m, "free", [0, 7, 0, 3]) == [1, 0, 0, 1]
    assert vkq.device_status(0) == vkq.ERR_INVALID_ARGUMENT
    _check(c, s, m)
    assert _do(s, m, "extend", [1], [-1]) == [0]
    assert vkq.device_status(0) == vkq.ERR_INVALID_ARGUMENT


def test_copy_pages():
    import torch
    from vibrant_b200 import vkq
    c, s, m = _make(3, 20, 48, 3, 64, 2, 2)
    c.copy_pages(_dev([3, 7, 3]), _dev([0, 19, 11]))
    for x in m.pool:
        x[:, 0], x[:, 19], x[:, 11] = x[:, 3].copy(), x[:, 7].copy(), x[:, 3].copy()
    _check(c, s, m)
    assert vkq.device_status(0) == vkq.OK
    c.copy_pages(_dev([3, 20, 5]), _dev([-1, 2, 6]))
    for x in m.pool:
        x[:, 6] = x[:, 5].copy()
    _check(c, s, m)
    assert vkq.device_status(0) == vkq.ERR_INVALID_ARGUMENT
    assert torch.cuda.is_available()


def test_forked_sequences_attend_alike_and_part():
    """A fork reads what its parent reads; after both grow, neither sees the other's token."""
    import torch
    from vibrant_b200 import kv8
    c = kv8.Cache(1, 12, 16, 1, 64)
    s = kv8.Sequences(c, 3, 4)
    x = torch.randn(21, 1, 64, device="cuda")
    s.extend(_dev([0]), _dev([21]))
    c.append(0, s.batch(_dev([0]), tokens=21, cu_tokens=_dev([0, 21]), max_tokens=21), x, x)
    s.fork(_dev([0, 0]), _dev([1, 2]))
    q = torch.randn(1, 2, 64, device="cuda").expand(3, 2, 64).contiguous()
    rows = _dev([0, 1, 2])
    o = c.attend(0, s.batch(rows), q)
    assert torch.equal(o[0], o[1]) and torch.equal(o[0], o[2])
    s.extend(rows, _dev([1, 1, 1]))
    y = torch.randn(3, 1, 64, device="cuda")
    c.append(0, s.batch(rows), y, y)
    o = c.attend(0, s.batch(rows), q)
    assert not torch.equal(o[0], o[1]) and not torch.equal(o[1], o[2])
    k, _ = c.read(0, s.batch(rows), rows, _dev([21, 21, 21]))
    step = c.k_scale[0, s.table[rows.long(), 1].long(), 0, 0][:, None, None]
    assert bool(((k - y).abs() <= 0.5 * step).all())


def test_page_refusals():
    import torch
    from vibrant_b200 import kv8, vkq
    c = kv8.Cache(1, 8, 16, 1, 64)
    s = kv8.Sequences(c, 4, 4)
    a, ws = _dev([0, 1]).data_ptr(), s._ws
    I, M, W = vkq.ERR_INVALID_ARGUMENT, vkq.ERR_MISALIGNED, vkq.ERR_WORKSPACE
    big = vkq.Kv8SeqsStruct.from_buffer_copy(s.struct)
    big.max_pages = 1 << 27
    null = vkq.Kv8SeqsStruct.from_buffer_copy(s.struct)
    null.refs = None
    for seqs, slots, n, w, wb, status in [(s.struct, None, 1, ws.data_ptr(), ws.numel(), I),
                                          (s.struct, a, 0, ws.data_ptr(), ws.numel(), I),
                                          (s.struct, a, 5, ws.data_ptr(), ws.numel(), I),
                                          (s.struct, a + 2, 1, ws.data_ptr(), ws.numel(), I),
                                          (s.struct, a, 1, None, 0, W), (s.struct, a, 1, ws.data_ptr(), 8, W),
                                          (s.struct, a, 1, ws.data_ptr() + 4, ws.numel(), W),
                                          (big, a, 1, ws.data_ptr(), ws.numel(), I),
                                          (null, a, 1, ws.data_ptr(), ws.numel(), I)]:
        for call in (lambda: vkq.kv8_extend(c.struct, seqs, slots, a, n, None, w, wb, device=0),
                     lambda: vkq.kv8_fork(c.struct, seqs, a, slots, n, None, w, wb, device=0),
                     lambda: vkq.kv8_free(c.struct, seqs, slots, n, None, w, wb, device=0)):
            with pytest.raises(vkq.VkqError) as e:
                call()
            assert e.value.status == status
    with pytest.raises(vkq.VkqError) as e:
        vkq.kv8_compact(c.struct, s.struct, a + 2, ws.data_ptr(), ws.numel(), device=0)
    assert e.value.status == M
    for src, dst, n in [(None, a, 1), (a, a, 0), (a, a, 9)]:
        with pytest.raises(vkq.VkqError) as e:
            vkq.kv8_copy_pages(c.struct, src, dst, n, device=0)
        assert e.value.status == I
    for bad in (lambda: s.extend(_dev([0]).long(), _dev([1])), lambda: s.extend(_dev([0, 1]), _dev([1])),
                lambda: s.fork(_dev([0]), _dev([1, 2])), lambda: kv8.Sequences(c, 4, 4, buffers=(s.table, s.lens, s.lens))):
        with pytest.raises(ValueError):
            bad()
    s.extend(_dev([]), _dev([]))
    assert vkq.device_status(0) == vkq.OK
    assert torch.cuda.is_available()

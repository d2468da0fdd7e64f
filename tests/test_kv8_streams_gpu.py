"""The 8-bit KV cache under CUDA graphs and on streams that are not the current one."""
import numpy as np
import pytest

import kv8_helpers as kh

pytestmark = pytest.mark.gpu


def _cache(pool):
    import torch
    from vibrant_b200 import kv8
    pages, kvh, page, dim = pool.shape
    bufs = tuple(torch.from_numpy(a[None]).cuda() for a in (pool.k, pool.v, pool.ks, pool.vs))
    return kv8.Cache(1, pages, page, kvh, dim, pool.fmt, buffers=bufs)


def _ints(a):
    import torch
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def test_graphs_captured_with_the_caches_own_workspace():
    """Two captured sizes, the smaller first; calls that need more workspace and
    other tensors after each; then the graphs replayed, the smaller one last."""
    import torch
    from vibrant_b200 import kv8, vkq
    rng = np.random.default_rng(21)
    lens = [3000] * 16
    pool = kh.Pool(16 * 188, 2, 16, 64, "int8", rng)
    table = kh.table_for(rng, lens, 16, 16 * 188, spare=0)
    c = _cache(pool)
    rows, len_t = torch.from_numpy(table).cuda(), _ints(lens)
    stream = torch.cuda.Stream()
    graphs = []
    for n in (1, 4):  # sequences of the captured step
        b = kv8.Batch(rows, len_t, slots=_ints(list(range(n))), max_len=3008)
        q = torch.randn(n, 8, 64, device="cuda")
        out = torch.empty_like(q)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            c.attend(0, b, q, out=out)  # brings the workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            c.attend(0, b, q, out=out)
        torch.cuda.synchronize()
        want = c.attend(0, b, q)
        # a chunk whose ranges of keys take more, and tensors that may get what was freed
        many = kv8.Batch(rows, len_t, cu_tokens=_ints([0, 200]), slots=_ints([0]), tokens=200, max_tokens=200, max_len=3008)
        before = c._ws[stream.cuda_stream].numel()
        with torch.cuda.stream(stream):
            c.attend(0, many, torch.randn(200, 8, 64, device="cuda"))
            assert n > 1 or c._ws[stream.cuda_stream].numel() > before
            junk = [torch.full((size,), 0x5A, dtype=torch.uint8, device="cuda") for size in (1 << 20, before) * 4]
        torch.cuda.synchronize()
        junk += [torch.full((size,), 0x5A, dtype=torch.uint8, device="cuda") for size in (1 << 20, before) * 4]
        graphs.append((graph, q, out, want, junk))
    for graph, q, out, want, _ in reversed(graphs):
        out.fill_(float("nan"))
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    for *_, junk in graphs:
        assert all(bool((t == 0x5A).all()) for t in junk)
    assert vkq.device_status(0) == vkq.OK


def _calls():
    """Calls that bring a result [64, 8, 64] of float32 (or several), on a stream that they are given."""
    import torch
    from vibrant_b200 import kv8, synth, tensor as vt, vkq
    rng = np.random.default_rng(22)
    lens = [90] * 64
    pool = kh.Pool(64 * 6, 8, 16, 64, "int8", rng)
    table = kh.table_for(rng, lens, 16, 64 * 6, spare=0)
    c = _cache(pool)
    b = kv8.Batch(torch.from_numpy(table).cuda(), _ints(lens))
    cos, sin = vt.rotary_tables(64, 1e4, 2048)
    x = torch.randn(64, 8, 64, device="cuda")
    pos = torch.arange(64, dtype=torch.int32, device="cuda")
    w = vt.QuantWeight(vkq.Q6_K, 256, 512, synth.weights(vkq.Q6_K, 256, 512, 3))
    w4 = vt.QuantWeight(vkq.Q4_K, 256, 512, synth.weights(vkq.Q4_K, 256, 512, 4))
    rows = torch.randn(64, 256, device="cuda")
    loose = torch.randn(256, 64, device="cuda").t()  # not contiguous
    return {"rotary": lambda s: (vt.rotary(x, cos, sin, pos, stream=s),),
            "rotary_tables": lambda s: vt.rotary_tables(32, 1e4, 2048, stream=s),
            "append": lambda s: (c.append(0, b, x, x, q=x, cos=cos, sin=sin, stream=s),),
            "read": lambda s: c.read(0, b, pos, pos, stream=s),
            "attend": lambda s: (c.attend(0, b, x, stream=s),),
            "matmul": lambda s: (vt.matmul(rows, w, stream=s),),
            "matmul of a view": lambda s: (vt.matmul(loose, w, stream=s),),
            "linear_fused": lambda s: tuple(vt.linear_fused(rows[:1].expand(4, 256), [w4], stream=s)),
            "dequantize": lambda s: (vt.dequantize(w, stream=s),),
            "dequant_transpose": lambda s: (vt.dequant_transpose(w, stream=s),)}


@pytest.mark.parametrize("name", ["rotary", "rotary_tables", "append", "read", "attend", "matmul", "matmul of a view",
                                  "linear_fused", "dequantize", "dequant_transpose"])
def test_results_on_another_stream(name):
    """A result written on `stream` takes no memory that the current stream
    still reads, and, dropped, is not written again before the current stream
    has read it."""
    import torch
    from vibrant_b200 import vkq
    call = _calls()[name]
    want = [t.clone() for t in call(None)]
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    call(other)  # workspaces and kernels are there
    torch.cuda.synchronize()
    held = [torch.full_like(t, 7.0) for t in want]
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)  # the current stream is some 50 ms behind
    seen = [t.clone() for t in held]
    del held
    got = call(other)  # runs at once
    other.synchronize()
    torch.cuda.synchronize()
    assert all(bool((t == 7.0).all()) for t in seen)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # read late on the current stream, dropped, and the same memory asked for on the other one
    torch.cuda._sleep(100_000_000)
    late = [t.clone() for t in got]
    shapes = [(t.shape, t.dtype) for t in got]
    del got
    with torch.cuda.stream(other):
        junk = [torch.full(s, 9.0, dtype=d, device="cuda") for s, d in shapes * 4]
    other.synchronize()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(late, want)) and len(junk) == 4 * len(want)
    assert vkq.device_status(0) == vkq.OK


def test_captured_product_after_its_workspace_grew():
    """A product split along K, captured with the cached workspace; then one that needs more."""
    import torch
    from vibrant_b200 import synth, tensor as vt, vkq
    w = vt.QuantWeight(vkq.Q6_K, 2048, 512, synth.weights(vkq.Q6_K, 2048, 512, 3))
    x = torch.randn(2, 2048, device="cuda")
    side = torch.cuda.Stream()
    vt._WS.pop((0, 0), None)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = vt.matmul(x, w)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = vt.matmul(x, w)
    cached = vt._WS.get((0, 0))
    if cached is not None:
        size = cached.numel()
        del cached
        vt.workspace(4 * size, 0)
        junk = [torch.full((size,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(8)]
        with torch.cuda.stream(side):
            junk += [torch.full((size,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(8)]
        torch.cuda.synchronize()
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    if cached_size := vt.workspace_bytes(vkq.Q6_K, 2, 2048, 512, 0):
        assert cached_size <= size and all(bool((t == 0x5A).all()) for t in junk)

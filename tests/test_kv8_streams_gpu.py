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

"""CPU checks of what the 8-bit KV cache's binding keeps and refuses."""
import contextlib
import weakref

import pytest


@pytest.fixture
def bare(monkeypatch):
    """A cache without pool or GPU, whose workspaces are host tensors; capturing[0] says whether a capture runs."""
    import torch
    from vibrant_b200 import kv8
    capturing = [False]
    monkeypatch.setattr(kv8, "stream_of", lambda device, stream: 7)
    monkeypatch.setattr(torch.cuda, "stream", lambda stream: contextlib.nullcontext())
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: None)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: capturing[0])
    c = kv8.Cache.__new__(kv8.Cache)
    c.device, c._ws, c._captured = torch.device("cpu"), {}, []
    return c, capturing


def test_workspace_of_a_captured_graph_is_kept(bare):
    """A graph holds the address of the workspace that its capture was given:
    a later call that needs more must not free it."""
    c, capturing = bare
    c._workspace(100, None)
    capturing[0] = True
    seen = weakref.ref(c._workspace(100, None))
    again = c._workspace(200, None)
    assert again is seen()
    del again
    capturing[0] = False
    more = c._workspace(1 << 22, None)
    assert more.numel() >= 1 << 22 and int(more.count_nonzero()) == 0
    assert seen() is not None and seen() is not more


def test_workspace_no_capture_has_seen_is_replaced(bare):
    c, _ = bare
    seen = weakref.ref(c._workspace(100, None))
    c._workspace(1 << 22, None)
    assert seen() is None


def test_workspace_does_not_grow_in_a_capture(bare):
    c, capturing = bare
    c._workspace(100, None)
    capturing[0] = True
    with pytest.raises(RuntimeError):
        c._workspace(1 << 22, None)


def test_batch_or_workspace_of_another_device(bare, monkeypatch):
    """Their addresses would mean nothing there: refused before any launch."""
    import torch
    from vibrant_b200 import kv8, vkq
    calls = []
    for name in ("kv8_append", "kv8_read", "kv8_attention"):
        monkeypatch.setattr(vkq, name, lambda *a, **k: calls.append(a))
    monkeypatch.setattr(vkq, "kv8_attention_workspace_bytes", lambda *a, **k: calls.append(a) or 64)
    c, _ = bare
    c.page_size, c.kv_heads, c.head_dim, c.struct, c._need = 16, 1, 64, None, {}
    here, there = (kv8.Batch(torch.zeros(2, 4, dtype=torch.int32, device=d), torch.ones(2, dtype=torch.int32, device=d))
                   for d in ("cpu", "meta"))
    x = torch.zeros(2, 1, 64)
    at = torch.zeros(2, dtype=torch.int32)
    for call in (lambda b: c.append(0, b, x, x), lambda b: c.read(0, b, at, at), lambda b: c.attend(0, b, x),
                 lambda b: c.attend(0, b, x, ws=torch.zeros(64)), lambda b: c.workspace_bytes(b, torch.float32, 1)):
        with pytest.raises(ValueError):
            call(there)
        assert not calls
        call(here)
        assert calls
        calls.clear()
        c._need.clear()
    for ws in (torch.zeros(64, device="meta"), torch.zeros(64, 2)[:, 0]):
        with pytest.raises(ValueError):
            c.attend(0, here, x, ws=ws)
    assert not calls
    c.attend(0, here, x, ws=torch.zeros(64))  # float32: 256 bytes
    assert 256 in calls[0]


def test_one_batch_with_caches_of_two_page_sizes():
    """The bound on the lengths is the table's for each cache, not the first one's."""
    import torch
    from vibrant_b200 import kv8
    table, lens = torch.zeros(2, 10, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    b = kv8.Batch(table, lens)
    assert [b.bounds(page).max_len for page in (16, 64, 32)] == [160, 640, 320]
    b = kv8.Batch(table, lens, max_len=100)
    assert [b.bounds(page).max_len for page in (16, 64)] == [100, 100]
    assert kv8.Batch(table, lens, max_len=0).bounds(16).max_len == 0


def test_workspace_of_the_products(monkeypatch):
    """The same for the workspace of the matrix products, which a captured step
    uses beside the cache's; one made in a capture is the graph's alone."""
    import torch
    from vibrant_b200 import tensor as vt
    capturing, zeros = [False], torch.zeros
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(torch, "zeros", lambda n, dtype, device: zeros(n, dtype=dtype))
    monkeypatch.setattr(vt, "_WS", {})
    monkeypatch.setattr(vt, "_WS_CAPTURED", [], raising=False)
    free = weakref.ref(vt.workspace(100, 0))
    vt.workspace(3 << 20, 0)
    assert free() is None
    capturing[0] = True
    seen = weakref.ref(vt.workspace(100, 0))
    own = vt.workspace(4 << 20, 0)
    capturing[0] = False
    assert vt.workspace(100, 0) is seen() and own is not seen()
    more = vt.workspace(5 << 20, 0)
    assert seen() is not None and vt.workspace(4 << 20, 0) is more

"""Page operations where a row holds more than 2^20 pages."""
import pytest

pytestmark = pytest.mark.gpu


def test_rows_that_grow_by_more_than_a_million_pages():
    """Rows of one call never get the same page, however much the one before grows."""
    import torch
    from vibrant_b200 import kv8, vkq
    big, pages = (1 << 20) + 5, (1 << 20) + 40
    c = kv8.Cache(1, pages, 16, 1, 64)
    s = kv8.Sequences(c, 4, big)
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    done = torch.full((4,), -1, dtype=torch.int32, device="cuda")
    s.extend(dev([2, 0, 3, 1]), dev([16 * big, 16 * 7, 16 * 29, 16]), done=done)
    assert done.tolist() == [1, 1, 0, 0]  # row 3's pages end past the pool's, and with them row 1's
    want = torch.arange(big, dtype=torch.int32, device="cuda")
    assert torch.equal(s.table[2], want)
    assert torch.equal(s.table[0, :7], big + want[:7]) and bool((s.table[0, 7:] == -1).all())
    assert bool((s.table[3] == -1).all()) and bool((s.table[1] == -1).all())
    assert s.lens.tolist() == [16 * 7, 0, 16 * big, 0]
    assert torch.equal(s.refs, (torch.arange(pages, device="cuda") < big + 7).int())
    # the pages given back go to the next call's rows in order
    s.free(dev([2]))
    s.extend(dev([1, 2]), dev([16 * big, 16]), done=done[:2])
    assert done[:2].tolist() == [1, 1] and vkq.device_status(0) == vkq.OK
    assert torch.equal(s.table[1], want) and int(s.table[2, 0]) == big + 7

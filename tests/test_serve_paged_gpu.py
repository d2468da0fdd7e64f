"""The example that serves forks of one prompt from the paged cache."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(__file__), "..", "examples"))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_serves_forks(fmt):
    import torch
    import serve_paged
    model = serve_paged.Decoder()
    kw = dict(prompt=333, chunk=200, forks=5, steps=10, fmt=fmt, page=16, model=model)
    chosen, logits, cache, seqs = serve_paged.serve(**kw)
    # where the pages lie changes nothing
    again, logits2, _, loose = serve_paged.serve(compact=False, **kw)
    assert torch.equal(chosen, again) and torch.equal(logits, logits2) and bool(torch.isfinite(logits).all())
    # forks 0, 2 and 4 went on to the end, 1 and 3 for half of it
    assert bool((chosen[0::2] >= 0).all()) and bool((chosen[1::2, :5] >= 0).all()) and bool((chosen[1::2, 5:] == -1).all())
    assert seqs.lens.tolist() == [0, 343, 0, 343, 0, 343]
    # the prompt's whole pages are shared by three, each has its own last two (333 = 20 * 16 + 13, 343 = 21 * 16 + 7)
    refs = sorted(seqs.refs.tolist(), reverse=True)
    assert refs[:26] == [3] * 20 + [1] * 6 and not any(refs[26:])
    # packed: the pages in use come first; otherwise the same number of them
    assert bool((seqs.refs[:26] > 0).all()) and sorted(loose.refs.tolist(), reverse=True) == refs

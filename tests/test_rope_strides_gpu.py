"""vkq_rotary refuses outputs in which two heads share values, and no others."""
import itertools
import random

import pytest

pytestmark = pytest.mark.gpu


def _meet(T, H, a, b, D):
    at = [t * a + h * b for t in range(T) for h in range(H)]
    return any(abs(x - y) < D for x, y in itertools.combinations(at, 2))


def test_outputs_whose_heads_meet_are_refused():
    import torch
    from vibrant_b200 import tensor as vt, vkq
    D = 8
    rng = random.Random(31)
    shapes = [(2, 3, 8, 8), (2, 3, 16, 8), (3, 2, 8, 16), (2, 2, 24, 16), (1, 3, 0, 8), (3, 1, 8, 0), (3, 3, 24, 8),
              (3, 3, 8, 24), (2, 5, 20, 8), (5, 2, 8, 23), (40, 3, 9, 352), (3, 40, 352, 9)]
    shapes += [(rng.randint(1, 6), rng.randint(1, 6), rng.randint(8, 60), rng.randint(8, 60)) for _ in range(300)]
    cos, sin = vt.rotary_tables(D, 1e4, 16)
    served = refused = 0
    for T, H, a, b in shapes:
        x = torch.randn(T, H, D, device="cuda")
        pos = torch.arange(T, dtype=torch.int32, device="cuda") % 16
        buf = torch.full((T * a + H * b + D,), 5.0, device="cuda")
        out = buf.as_strided((T, H, D), (a, b, 1))
        if _meet(T, H, a, b, D):
            with pytest.raises(vkq.VkqError) as e:
                vt.rotary(x, cos, sin, pos, out=out)
            assert e.value.status == vkq.ERR_INVALID_ARGUMENT and bool((buf == 5.0).all())
            refused += 1
        else:
            vt.rotary(x, cos, sin, pos, out=out)
            assert torch.equal(out, vt.rotary(x, cos, sin, pos)) and int((buf == 5.0).sum()) == buf.numel() - x.numel()
            served += 1
    assert served > 50 and refused > 50
    assert vkq.device_status(0) == vkq.OK

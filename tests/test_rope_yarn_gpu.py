"""vkq_rotary_tables_f32 with VKQ_ROPE_SCALE_YARN where the ramp ends past the
last pair: frequencies worked out here from the published definition (Peng et
al., "YaRN: Efficient Context Window Extension of Large Language Models",
sections 3.2 and 3.4): pair i makes r_i = orig_len / (2 pi base^(2i / rot))
turns within orig_len; the pairs between the ones that make beta_fast and
beta_slow turns (rounded outward to whole pairs, within 0 .. rot - 1) go over
from the plain frequency to the interpolated one linearly in i."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _pair_of_turns(turns, rot, base, orig):
    """The (real) pair number that makes so many turns within orig_len."""
    return math.log(orig / (2 * math.pi * turns), base) * rot / 2


def _frequencies(rot, base, factor, orig, fast, slow):
    first = max(math.floor(_pair_of_turns(fast, rot, base, orig)), 0)
    last = min(math.ceil(_pair_of_turns(slow, rot, base, orig)), rot - 1)
    out = []
    for i in range(rot // 2):
        plain = base ** (-2.0 * i / rot)
        if i <= first:
            w = 0.0
        elif i >= last:
            w = 1.0
        else:
            w = (i - first) / (last - first)
        out.append((1 - w) * plain + w * plain / factor)
    return np.array(out)


@pytest.mark.parametrize("rot,base,factor,orig", [
    (128, 1e4, 4.0, 131072),   # the ramp: pairs 45 .. 70 of 64
    (64, 1e4, 8.0, 65536), (64, 1e4, 8.0, 1 << 20), (6, 500.0, 16.0, 4096), (2, 100.0, 2.0, 1 << 20),
    (128, 1e4, 16.0, 1 << 40),  # all pairs turn more than beta_fast times: none is interpolated
    (128, 1e6, 4.0, 32768), (128, 5e5, 8.0, 8192), (96, 1e4, 4.0, 4096)])  # ends within the pairs
def test_yarn_tables_follow_the_definition(rot, base, factor, orig):
    """Half a unit of float32, what angles up to 40,000 radians in float64
    leave (2^-37), and 2^-35 for a ramp worked out in another order."""
    from vibrant_b200 import tensor as vt
    n = 40000
    cos, sin = vt.rotary_tables(rot, base, n, scaling="yarn", factor=factor, orig_len=orig, attn_factor=1.0)
    angle = np.arange(n, dtype=np.float64)[:, None] * _frequencies(rot, base, factor, orig, 32.0, 1.0)
    assert float(np.abs(cos.cpu().numpy() - np.cos(angle)).max()) <= 2.0 ** -24 + 2.0 ** -34
    assert float(np.abs(sin.cpu().numpy() - np.sin(angle)).max()) <= 2.0 ** -24 + 2.0 ** -34

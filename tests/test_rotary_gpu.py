"""vkq_rotary and vkq_rotary_tables_f32: bit for bit against float32 numpy
(each product and sum rounded on its own, the result rounded once), the tables
against float64, the inverse as gradient, and refusals."""
import math

import numpy as np
import pytest

import kv8_helpers as kh

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


def _setup(dtype, T, H, D, rot, spare, seed, max_seq=300):
    import torch
    from vibrant_b200 import tensor as vt
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows = torch.randn(T, H * D + spare, device="cuda", generator=g).to(getattr(torch, DT[dtype]))
    x = rows[:, spare:].unflatten(1, (H, D)) if spare else rows.view(T, H, D)
    pos = torch.randint(0, max_seq, (T,), device="cuda", generator=g, dtype=torch.int32)
    cos, sin = vt.rotary_tables(rot, 10000.0, max_seq)
    return x, cos, sin, pos


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,H,D,rot,spare", [
    (1, 16, 128, 128, 0), (7, 5, 128, 64, 0), (3, 40, 128, 128, 2048), (5, 3, 64, 64, 1),  # spare 1: unaligned rows
    (2, 2, 64, 62, 0), (4, 1, 80, 16, 8), (3, 2, 10, 6, 0), (2, 3, 2, 2, 0), (300, 9, 128, 96, 0),
], ids=lambda v: str(v))
def test_rotary_matches_float32(dtype, layout, T, H, D, rot, spare):
    import torch
    from vibrant_b200 import tensor as vt, vkq
    x, cos, sin, pos = _setup(dtype, T, H, D, rot, spare, seed=T + D + rot)
    want = torch.from_numpy(kh.rotate(x.float().cpu().numpy(), cos.cpu().numpy(), sin.cpu().numpy(),
                                      pos.cpu().numpy(), layout)).to(x.dtype)
    keep = x.clone()
    got = vt.rotary(x, cos, sin, pos, layout=layout)
    assert torch.equal(got.cpu(), want)
    assert torch.equal(x, keep)
    back = vt.rotary(x, cos, sin, pos, layout=layout, inverse=True).cpu()
    want_back = torch.from_numpy(kh.rotate(x.float().cpu().numpy(), cos.cpu().numpy(), sin.cpu().numpy(),
                                           pos.cpu().numpy(), layout, inverse=True)).to(x.dtype)
    assert torch.equal(back, want_back)
    vt.rotary(x, cos, sin, pos, layout=layout, out=x)  # in place, at the rows' strides
    assert torch.equal(x.cpu(), want)
    assert vkq.device_status(0) == vkq.OK


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rotary_heads_before_tokens(layout):
    """A [heads, tokens, D] buffer seen as [tokens, heads, D]."""
    import torch
    from vibrant_b200 import tensor as vt
    x, cos, sin, pos = _setup("f32", 9, 4, 64, 32, 0, seed=5)
    want = vt.rotary(x, cos, sin, pos, layout=layout)
    turned = x.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty(4, 9, 64, device="cuda").transpose(0, 1)
    assert torch.equal(vt.rotary(turned, cos, sin, pos, layout=layout, out=out), want)


def test_rotary_inverse_is_the_gradient():
    """<g, R x> = <R^T g, x>: the inverse is the transpose, and undoes the rotation."""
    import torch
    from vibrant_b200 import tensor as vt
    x, cos, sin, pos = _setup("f32", 11, 3, 64, 48, 0, seed=6)
    g = torch.randn_like(x)
    lhs = (g.double() * vt.rotary(x, cos, sin, pos, layout="half").double()).sum()
    rhs = (vt.rotary(g, cos, sin, pos, layout="half", inverse=True).double() * x.double()).sum()
    bound = (g.double().abs() * x.double().abs()).sum() * 2
    assert abs(float(lhs - rhs)) <= 4 * 2.0 ** -24 * float(bound)  # four float32 roundings a product
    back = vt.rotary(vt.rotary(x, cos, sin, pos), cos, sin, pos, inverse=True)
    pairs = (x.double().unflatten(2, (-1, 2)) ** 2).sum(-1).sqrt()[..., None].expand(-1, -1, -1, 2).flatten(2)
    assert bool(((back.double() - x.double()).abs() <= 8 * 2.0 ** -24 * pairs).all())


def test_rotary_bad_position():
    """A token outside the tables stays unwritten, the others are served, the status says so."""
    import torch
    from vibrant_b200 import tensor as vt, vkq
    for D, rot in ((64, 64), (64, 30)):
        x, cos, sin, pos = _setup("f32", 4, 2, D, rot, 0, seed=7, max_seq=50)
        pos[1], pos[3] = 50, -1
        out = torch.full_like(x, float("nan"))
        vt.rotary(x, cos, sin, pos, out=out)
        assert vkq.device_status(0) == vkq.ERR_INVALID_ARGUMENT
        assert torch.isnan(out[1]).all() and torch.isnan(out[3]).all()
        assert torch.isfinite(out[0]).all() and torch.isfinite(out[2]).all()
        assert vkq.device_status(0) == vkq.OK


def _frequencies(rot, base, scaling, factor, orig, fast, slow):
    i = np.arange(rot // 2, dtype=np.float64)
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    t = base ** (-2 * i / rot)
    if scaling == "linear":
        return t / factor
    if scaling != "yarn":
        return t
    d = lambda b: rot * math.log(orig / (2 * math.pi * b)) / (2 * math.log(base))  # noqa: E731
    lo = min(max(math.floor(d(fast)), 0), rot // 2 - 1)
    hi = min(max(math.ceil(d(slow)), 0), rot // 2 - 1)
    w = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
    return t / factor * w + t * (1 - w)


@pytest.mark.parametrize("scaling,factor,orig,attn", [("none", 1.0, 0, 0.0), ("linear", 4.0, 0, 0.0),
                                                      ("ntk", 8.0, 0, 0.0), ("yarn", 16.0, 4096, 0.0),
                                                      ("yarn", 2.0, 32768, 1.0)])
@pytest.mark.parametrize("rot,base", [(128, 1e6), (64, 10000.0), (6, 500.0)])
def test_rotary_tables(rot, base, scaling, factor, orig, attn):
    """Each entry rounded once: half a unit of float32, and what an angle of
    up to 40,000 radians in float64 leaves (2^-37)."""
    import torch
    from vibrant_b200 import tensor as vt
    n = 40000
    cos, sin = vt.rotary_tables(rot, base, n, scaling=scaling, factor=factor, orig_len=orig, attn_factor=attn)
    angle = np.arange(n, dtype=np.float64)[:, None] * _frequencies(rot, base, scaling, factor, orig, 32.0, 1.0)
    m = 1.0
    if scaling == "yarn":
        m = attn or 0.1 * math.log(factor) + 1
    assert float(np.abs(cos.cpu().numpy() - np.cos(angle) * m).max()) <= m * (2.0 ** -24 + 2.0 ** -36)
    assert float(np.abs(sin.cpu().numpy() - np.sin(angle) * m).max()) <= m * (2.0 ** -24 + 2.0 ** -36)
    assert torch.cuda.is_available()


def test_rotary_refusals():
    import torch
    from vibrant_b200 import tensor as vt, vkq
    buf = torch.zeros(1 << 12, device="cuda")
    p = buf.data_ptr()

    def call(**kw):
        a = dict(dtype=vkq.F32, x=p, xs=(128, 64), out=p, os=(128, 64), T=2, H=2, D=64, rot=64, seq=4, layout=0)
        a.update(kw)
        vkq.rotary(a["dtype"], a["x"], a["xs"], a["out"], a["os"], p, p, p, a["T"], a["H"], a["D"], a["rot"], a["seq"],
                   a["layout"], device=0)

    for bad, status in [(dict(dtype=12), vkq.ERR_UNSUPPORTED), (dict(x=None), vkq.ERR_INVALID_ARGUMENT),
                        (dict(rot=63), vkq.ERR_INVALID_ARGUMENT), (dict(rot=66), vkq.ERR_INVALID_ARGUMENT),
                        (dict(T=0), vkq.ERR_INVALID_ARGUMENT), (dict(H=-1), vkq.ERR_INVALID_ARGUMENT),
                        (dict(seq=0), vkq.ERR_INVALID_ARGUMENT), (dict(layout=2), vkq.ERR_INVALID_ARGUMENT),
                        (dict(xs=(-1, 64)), vkq.ERR_INVALID_ARGUMENT), (dict(os=(128, 63)), vkq.ERR_INVALID_ARGUMENT),
                        (dict(x=p + 2), vkq.ERR_MISALIGNED)]:
        with pytest.raises(vkq.VkqError) as e:
            call(**bad)
        assert e.value.status == status, bad
    for bad, status in [(dict(base=1.0), vkq.ERR_INVALID_ARGUMENT), (dict(rot=5), vkq.ERR_INVALID_ARGUMENT),
                        (dict(scaling=1, factor=0.5), vkq.ERR_INVALID_ARGUMENT), (dict(scaling=4), vkq.ERR_UNSUPPORTED),
                        (dict(scaling=3, factor=2.0), vkq.ERR_INVALID_ARGUMENT),  # no original length
                        (dict(scaling=2, factor=2.0, rot=2), vkq.ERR_INVALID_ARGUMENT)]:
        a = dict(rot=64, base=1e4, scaling=0, factor=1.0)
        a.update(bad)
        with pytest.raises(vkq.VkqError) as e:
            vkq.rotary_tables_f32(p, p, 8, a["rot"], a["base"], a["scaling"], a["factor"], device=0)
        assert e.value.status == status, bad
    x = torch.zeros(3, 2, 64, device="cuda")
    cos = torch.zeros(5, 32, device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    for args in [(x.double(), cos, cos, pos), (x[0], cos, cos, pos), (x, cos, cos[:, :16], pos),
                 (x, cos, cos, pos.long()), (x, cos, cos, pos[:2]), (x.transpose(1, 2), cos, cos, pos)]:
        with pytest.raises(ValueError):
            vt.rotary(*args)
    assert vt.rotary(x[:0], cos, cos, pos[:0]).shape == (0, 2, 64)
    assert vkq.device_status(0) == vkq.OK

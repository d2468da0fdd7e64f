"""Attention of prompt chunks over contexts of 200,000 and a million cached
tokens, where values of one sign show what the sums lose."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,tokens,n", [("float16", 4096, 200000), ("bfloat16", 8192, 1 << 20),
                                            ("float32", 512, 200000)])
def test_sums_of_one_sign_over_long_contexts(dtype, tokens, n):
    """Scores of a few tenths and V codes 64 .. 127: every output is a mean of
    n values of one sign.  What the sums lose is the mean of the relative
    errors over 40 heads of 128 dimensions, in which the outputs' rounding
    averages out (half a unit is 2^-11 or 2^-8 of a value, a 5,120th of its
    variance below 2^-16 or 2^-13): at most a quarter of half a unit for
    float16, an eighth for bfloat16, 2^-18 for float32 (2^-20 of the scores'
    terms and float32 sums).  Each output is within half a unit (float32: none)
    and 2^-11 (float32: 1e-5) of the value."""
    import torch
    from vibrant_b200 import kv8, vkq
    H, D, page = 40, 128, 64
    pages = -(-n // page)
    g = torch.Generator(device="cuda").manual_seed(n)
    c = kv8.Cache(1, pages, page, 1, D)
    c.v.random_(64, 128, generator=g)
    c.k.random_(0, 256, generator=g)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    order = torch.randperm(pages, generator=g, device="cuda")
    b = kv8.Batch(order.int().view(1, -1), ints([n]), cu_tokens=ints([0, tokens]), tokens=tokens, max_tokens=tokens, max_len=n)
    q = torch.randn(tokens, H, D, generator=g, device="cuda").to(getattr(torch, dtype))
    scale = 1 / (74 * 128 ** 0.5)
    got = c.attend(0, b, q, scale=scale)[-1].double()  # the last token sees the whole context
    assert vkq.device_status(0) == vkq.OK
    k, v = (t[0, order, 0].view(torch.int8).flatten(0, 1)[:n].double() for t in (c.k, c.v))
    want = torch.softmax(q[-1].double() @ k.T * float(torch.tensor(scale, dtype=torch.float32)), dim=1) @ v
    rel = (got - want) / want
    bias, half, rest = {"float16": (2.0 ** -13, 2.0 ** -11, 2.0 ** -11), "bfloat16": (2.0 ** -11, 2.0 ** -8, 2.0 ** -11),
                        "float32": (2.0 ** -18, 0.0, 1e-5)}[dtype]
    assert abs(float(rel.mean())) <= bias, float(rel.mean())
    assert float(rel.abs().max()) <= half + rest


@pytest.mark.parametrize("dtype,tokens,n,window", [
    ("float16", 900, 40000, 0), ("float16", 70, 40000, 0), ("float16", 900, 50000, 33000), ("float16", 4096, 120000, 0),
    ("bfloat16", 900, 150000, 0), ("float32", 300, 40000, 0)])
def test_rising_and_falling_scores_over_long_contexts(dtype, tokens, n, window):
    """Scores that rise (even heads) or fall (odd ones) by 60 over the context, V
    of both signs: the running maximum moves all the way, or not at all.  Some
    rows against float64 and the bound that the header states."""
    import torch
    from vibrant_b200 import kv8, vkq
    H, D, page = 40, 128, 64
    pages = -(-n // page)
    g = torch.Generator(device="cuda").manual_seed(n + tokens)
    c = kv8.Cache(1, pages, page, 1, D)
    c.v.random_(0, 256, generator=g)
    c.v[c.v == 128] = 1  # -128 is no code
    codes = torch.randint(-40, 41, (pages * page, D), generator=g, device="cuda")
    codes[:, 0] = torch.arange(pages * page, device="cuda") * 120 // (pages * page)
    order = torch.randperm(pages, generator=g, device="cuda")
    c.k[0, order, 0] = codes.to(torch.int8).view(torch.uint8).view(pages, page, D)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    b = kv8.Batch(order.int().view(1, -1), ints([n]), cu_tokens=ints([0, tokens]), tokens=tokens, max_tokens=tokens, max_len=n)
    q = torch.randn(tokens, H, D, generator=g, device="cuda")
    q[:, 0::2, 0], q[:, 1::2, 0] = 500.0, -500.0
    q = q.to(getattr(torch, dtype))
    scale = 1e-3
    got = c.attend(0, b, q, scale=scale, window=window)
    assert torch.equal(got, c.attend(0, b, q, scale=scale, window=window)) and vkq.device_status(0) == vkq.OK
    k, v = codes[:n].double(), c.v[0, order, 0].view(torch.int8).flatten(0, 1)[:n].double()
    scale = float(torch.tensor(scale, dtype=torch.float32))
    for row in (0, tokens // 2, tokens - 1):
        at = n - tokens + row
        lo = max(at - window + 1, 0) if window else 0
        kk, vv, qq = k[lo:at + 1], v[lo:at + 1], q[row].double()
        p = torch.softmax(qq @ kk.T * scale, dim=1)
        out, mass = p @ vv, p @ vv.abs()
        size = (qq.abs() @ kk.abs().T * scale).amax(dim=1, keepdim=True)
        floor = p.amax(dim=1, keepdim=True) * vv.abs().sum(dim=0)
        tol = (1e-5 + 2.0 ** -20 * size) * mass
        if dtype == "float32":
            tol += 2.0 ** -39 * floor
        else:
            tol += 2.0 ** -31 * floor + 2.0 ** -10 * mass + (2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -11) * 1.001 * out.abs()
        assert bool(((got[row].double() - out).abs() <= tol).all())

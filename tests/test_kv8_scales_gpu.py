"""Attention over blocks whose V scales lie far apart, with dimensions in which
the blocks of the large scale hold zeros, against float64 and the bounds that
the header states for calls of few and of many rows."""
import numpy as np
import pytest

import kv8_helpers as kh

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


def _reference(q, pool, row, n, scale):
    """float64 output of the last q.shape[0] tokens of a sequence of n (causal), sum_j p_j |v_j|, both forms of F
    (max p s sum |c|, max p sum |v|) and each row's largest sum of score terms."""
    T, H, D = q.shape
    g = H // pool.shape[1]
    k, v = pool.rows("k", row, n), pool.rows("v", row, n)
    s = np.repeat(pool.vs[row[:-(-n // pool.page)]].transpose(1, 0, 2).reshape(pool.shape[1], -1), kh.BLOCK, axis=1)[:, :n]
    s = s.astype(np.float64)
    seen = np.arange(n)[None] <= np.arange(n - T, n)[:, None]
    out, mass, many, few, size = (np.zeros((T, H, D)) for _ in range(5))
    for h in range(H):
        kk, vv, ss, qq = k[h // g], v[h // g], s[h // g], q[:, h].astype(np.float64)
        x = np.where(seen, qq @ kk.T * scale, -np.inf)
        p = np.exp(x - x.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        out[:, h], mass[:, h] = p @ vv, p @ np.abs(vv)
        many[:, h] = (p * ss).max(axis=1, keepdims=True) * (seen @ np.abs(vv / ss[:, None]))
        few[:, h] = p.max(axis=1, keepdims=True) * (seen @ np.abs(vv))
        size[:, h] = np.where(seen, np.abs(qq) @ np.abs(kk).T * scale, 0.0).max(axis=1, keepdims=True)
    return out, mass, many, few, size


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("apart", [8, 20, 40, 60])
@pytest.mark.parametrize("H,KVH,D", [(8, 2, 64), (20, 2, 128)], ids=str)
@pytest.mark.parametrize("news,many", [(1, False), (3, False), (70, True)])
def test_scales_far_apart(dtype, fmt, apart, H, KVH, D, news, many):
    import torch
    from vibrant_b200 import kv8, vkq
    n, page, pages = 700, 32, 24
    rng = np.random.default_rng(apart + D + news)
    pool = kh.Pool(pages, KVH, page, D, fmt, rng)
    large = rng.random(pool.vs.shape) < 0.3
    pool.vs = np.where(large, 2.0 ** (apart - 30), 2.0 ** -30).astype(np.float32)
    blocks = pool.v.reshape(pages, KVH, page // kh.BLOCK, kh.BLOCK, D)
    blocks[large, :, :D // 2] = 0  # a view: half of the dimensions see the small scales alone
    row = rng.permutation(pages)[:-(-n // page)].astype(np.int32)
    c = kv8.Cache(1, pages, page, KVH, D, fmt,
                  buffers=tuple(torch.from_numpy(a[None]).cuda() for a in (pool.k, pool.v, pool.ks, pool.vs)))
    q = torch.from_numpy(rng.standard_normal((news, H, D)).astype(np.float32)).cuda().to(getattr(torch, DT[dtype]))
    width = (1 << 18) // page if many else len(row)  # a large bound on the length: the kernel of many rows
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, :len(row)] = torch.from_numpy(row)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = kv8.Batch(table, ints([n]), cu_tokens=ints([0, news]), tokens=news, max_tokens=news)
    got = c.attend(0, batch, q).double().cpu().numpy()
    assert vkq.device_status(0) == vkq.OK
    out, mass, f_many, f_few, size = _reference(q.float().cpu().numpy(), pool, row, n, float(np.float32(D ** -0.5)))
    floor = (2.0 ** -39 if dtype == "f32" else 2.0 ** -31) * f_many if many else 2.0 ** -39 * f_few
    tol = 1.01 * floor + (1e-5 + 2.0 ** -20 * size) * mass
    if dtype != "f32":
        unit, tiny = (2.0 ** -8, 0.0) if dtype == "bf16" else (2.0 ** -11, 2.0 ** -25)
        tol += unit * 1.001 * np.abs(out) + 2.0 ** -10 * mass + tiny
    err = np.where(np.isinf(got), 0.0, np.abs(got - out) - tol)
    beyond = np.isinf(got)  # a float16 output past its range, and only there
    assert not beyond.any() or dtype == "f16"
    assert (np.sign(got[beyond]) * out[beyond] + tol[beyond] >= 65520).all()
    assert float(err.max()) <= 0.0, (float(err.max()), np.unravel_index(err.argmax(), err.shape))

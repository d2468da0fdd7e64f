"""Calls on the 8-bit KV cache whose arguments no launch could hold, or that lie
on another device or in another cache than they are used with."""
import pytest

pytestmark = pytest.mark.gpu


def _small(dtype="float16"):
    import torch
    from vibrant_b200 import kv8
    c = kv8.Cache(1, 8, 16, 2, 64)
    table = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")
    return c, kv8.Batch(table, lens), torch.zeros(2, 4, 64, device="cuda", dtype=getattr(torch, dtype))


def _changed(struct, **kw):
    s = type(struct).from_buffer_copy(struct)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("dtype,batch,kv_heads,heads,max_tokens,max_len", [
    ("F16", 65535, 32, 32, 1 << 20, 1 << 20),   # 2^33 tiles
    ("BF16", 65535, 64, 64, 1 << 18, 1 << 20),  # 2^32 tiles
    ("F32", 65535, 32, 32, 1 << 20, 64),        # 2^34 tiles of one range
    ("F32", 65535, 512, 512, 16384, 64),        # 2^32 tiles
])
def test_attention_refuses_what_no_grid_holds(dtype, batch, kv_heads, heads, max_tokens, max_len):
    import torch
    from vibrant_b200 import vkq
    c, b, q = _small()
    cache = _changed(c.struct, kv_heads=kv_heads)
    p = b.tensors[1].data_ptr()
    wide = _changed(b.bounds(16), rows=65535, batch=batch, cu_tokens=p, max_pages=1 << 20, tokens=1 << 20,
                    max_tokens=max_tokens, max_len=max_len)
    code = getattr(vkq, dtype)
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    for call in (lambda: vkq.kv8_attention_workspace_bytes(cache, wide, code, heads, device=0),
                 lambda: vkq.kv8_attention(cache, 0, wide, code, q.data_ptr(), heads * 64, q.data_ptr(), heads * 64, heads,
                                           0.125, ws.data_ptr(), ws.numel(), device=0)):
        with pytest.raises(vkq.VkqError) as e:
            call()
        assert e.value.status == vkq.ERR_UNSUPPORTED
    assert vkq.device_status(0) == vkq.OK


def test_attention_serves_wide_bounds():
    """Bounds far above what is there, short of the limit: the same products in another kernel."""
    import torch
    from vibrant_b200 import kv8, vkq
    c, b, q = _small("float32")
    b.tensors[0][1] += 4  # pages of its own
    table, lens = b.tensors[:2]
    x = torch.randn(2, 2, 64, device="cuda")
    c.append(0, b, x, x)
    seq, pos = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([0, 1], [0, 0]))
    v = c.read(0, b, seq, pos)[1].repeat_interleave(2, dim=1)  # one key: the output is its v
    wide = kv8.Batch(table, lens, max_tokens=1 << 20)  # 2 sequences and KV heads: 65,536 tiles
    for batch in (b, wide):
        got = c.attend(0, batch, q.normal_())
        assert bool(((got - v).abs() <= 1e-5 * v.abs()).all())
    assert vkq.device_status(0) == vkq.OK


def test_batch_and_workspace_of_the_host_are_refused():
    import torch
    from vibrant_b200 import kv8, vkq
    c, b, q = _small("float32")
    host = kv8.Batch(b.tensors[0].cpu(), b.tensors[1].cpu())
    x = q[:, :2].contiguous()
    for bad in (lambda: c.append(0, host, x, x), lambda: c.attend(0, host, q), lambda: c.read(0, host, *b.tensors[1:2] * 2),
                lambda: c.attend(0, b, q, ws=torch.zeros(1 << 20, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            bad()
    assert vkq.device_status(0) == vkq.OK

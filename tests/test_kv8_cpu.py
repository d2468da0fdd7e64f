"""CPU checks of the 8-bit KV cache's bindings and of the tests' restatements."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import kv8_helpers as kh

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("c_name,py_name", [("vkq_kv8_cache", "Kv8CacheStruct"), ("vkq_kv8_batch", "Kv8BatchStruct"),
                                            ("vkq_kv8_seqs", "Kv8SeqsStruct")])
def test_structs_match_the_header(tmp_path, c_name, py_name):
    """Sizes and offsets of the ctypes structs are those a C compiler gives the header's."""
    from vibrant_b200 import vkq
    cls = getattr(vkq, py_name)
    names = [f[0] for f in cls._fields_]
    body = "".join(f'printf("%zu ", offsetof({c_name}, {n}));' for n in names)
    src = tmp_path / "s.c"
    src.write_text(f'#include <stdio.h>\n#include <vkq.h>\nint main(void){{{body}printf("%zu", sizeof({c_name}));}}')
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(cls, n).offset for n in names] + [ctypes.sizeof(cls)]


def test_entry_points_fail_without_a_gpu():
    import torch
    from vibrant_b200 import vkq
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(vkq.VkqError):
        vkq.kv8_copy_pages(vkq.Kv8CacheStruct(), None, None, 1, device=0)


def test_workspace_query_needs_no_gpu():
    from vibrant_b200 import vkq
    c, s = vkq.Kv8CacheStruct(num_pages=100), vkq.Kv8SeqsStruct(rows=7)
    assert vkq.kv8_pages_workspace_bytes(c, s) >= 4 * (100 * 2 + 7)
    with pytest.raises(vkq.VkqError):
        vkq.kv8_pages_workspace_bytes(vkq.Kv8CacheStruct(), s)


def test_restated_codes():
    import torch
    x = np.concatenate([np.linspace(-500, 500, 4001), np.linspace(-0.05, 0.05, 4001)]).astype(np.float32)
    want = torch.from_numpy(np.clip(x, -448, 448)).to(torch.float8_e4m3fn)
    assert np.array_equal(kh.encode(x, "e4m3"), want.view(torch.uint8).numpy())
    assert np.array_equal(kh.decode(kh.encode(x, "e4m3"), "e4m3"), want.float().numpy())
    codes = np.arange(256, dtype=np.uint8)
    vals = kh.decode(codes, "e4m3")
    keep = ~np.isnan(vals)
    assert np.array_equal(kh.encode(vals[keep], "e4m3"), codes[keep])
    assert kh.encode(np.float32([0.5, 1.5, -2.5, 200, np.nan]), "int8").view(np.int8).tolist() == [0, 2, -2, 127, 0]
    assert kh.scale_for(127, "int8") == 1 and kh.scale_for(127.1, "int8") == 2 and kh.scale_for(0, "int8") == 2.0 ** -64
    assert kh.scale_for(448, "e4m3") == 1 and kh.scale_for(449, "e4m3") == 2

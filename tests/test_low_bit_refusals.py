"""CPU tests of what the low-bit calls refuse: prefix files whose rows or sizes
cannot be right, and pools of an unknown type."""
import struct

import numpy as np
import pytest

from test_prefix_file import fnv1a64


def q4_file(path, body, n_tokens, heads=2, dim=16, layers=1, dtype=2):
    path.write_bytes(struct.pack("<8s8I q f I Q", b"S1KVPFX\0", 1, 64, layers, heads, dim, 16, dtype, 0, n_tokens, 1e6, 0,
                                 fnv1a64(body)) + body)
    return path


def q4_body(rows, dim=16, s=0x3F80, m=0x3F80):
    row = bytes(range(dim // 2)) + struct.pack("<HH", s, m)
    return row * rows


@pytest.mark.parametrize("s,m,ok", [(0x3F80, 0xBF80, True), (0, 0, True), (0x7F7F, 0xFF7F, True), (0x7FC0, 0x7FC0, True),
                                    (0xBF80, 0x3F80, False), (0x7F80, 0, False), (0x3F80, 0x7F80, False),
                                    (0x3F80, 0xFF80, False), (0x7FC0, 0, False), (0x3F80, 0x7FC0, False),
                                    (0x8000, 0x3F80, False), (0x7FC1, 0x7FC0, False)])
def test_rows_that_append_does_not_write(s1kv, tmp_path, s, m, ok):
    body = q4_body(11) + q4_body(1, s=s, m=m)
    path = q4_file(tmp_path / "a", body, 3)
    if ok:
        assert s1kv.prefix_file_info(path)["n_tokens"] == 3
        return
    with pytest.raises(s1kv.S1KVError) as e:
        s1kv.prefix_file_info(path)
    assert e.value.status == s1kv.EINVAL and "row 11" in str(e.value)


@pytest.mark.parametrize("n,heads,dim,layers,dtype", [(1 << 62, 1, 8, 1, 2), (1 << 62, 2, 4, 4, 0), (1 << 60, 16, 16, 2, 1)])
def test_sizes_that_pass_64_bits(s1kv, tmp_path, n, heads, dim, layers, dtype):
    with pytest.raises(s1kv.S1KVError) as e:
        s1kv.prefix_file_info(q4_file(tmp_path / "a", b"", n, heads, dim, layers, dtype))
    assert e.value.status == s1kv.EINVAL


@pytest.mark.parametrize("dtype", ["int4", "Q4", "q8", "float16", "half", "", 3, None, "fp8"])
def test_pools_of_an_unknown_type(s1kv, dtype):
    with pytest.raises(s1kv.S1KVError) as e:
        s1kv.Pool(1, 2, 64, 4, 16, dtype=dtype, host_only=True)
    assert e.value.status == s1kv.EINVAL and "dtype" in str(e.value)


def test_pools_of_known_types(s1kv):
    import torch
    for dtypes, want in ((("f32", "fp32", "float32", 0, torch.float32), s1kv.DTYPE_F32),
                         (("bf16", "bfloat16", 1, torch.bfloat16), s1kv.DTYPE_BF16), (("q4", 2), s1kv.DTYPE_Q4)):
        for d in dtypes:
            pool = s1kv.Pool(1, 2, 64, 4, 16, dtype=d, host_only=True)
            assert pool.dtype == want
            pool.close()

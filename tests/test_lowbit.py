"""CPU tests of the low-bit operators: the plain forms against the format's
guarantees, and the calls that are refused before any kernel runs."""
import ctypes as C

import numpy as np
import pytest

from oracle import lowbit as LB


def rows(rng, n, d, kind):
    x = rng.standard_normal((n, d)).astype(np.float32)
    if kind == "offset":
        x = x * 0.01 + 300
    elif kind == "wide":
        x = x * np.exp(rng.uniform(-60, 60, (n, 1))).astype(np.float32)
    elif kind == "outlier":
        x[:, rng.integers(0, d)] *= 50
    return x


@pytest.mark.parametrize("kind", ["plain", "offset", "wide", "outlier"])
def test_rows_are_held_within_half_a_step(kind):
    x = rows(np.random.default_rng(1), 200, 96, kind)
    c, s, m = LB.q4_rows(x)
    assert c.min() >= 0 and c.max() <= 15
    held = m.astype(np.float64)[:, None] + s.astype(np.float64)[:, None] * (c - 8)
    # exact arithmetic bounds the error by s / 2; s itself is one fp32 rounding (2^-24) of its requirement
    assert (np.abs(held - x) <= s[:, None] * (0.5 + 16 * 2.0 ** -24)).all()


def test_constant_zero_and_unholdable_rows():
    x = np.zeros((6, 16), np.float32)
    x[1] = 3.3
    x[2, 5] = np.nan
    x[3, 0] = np.inf
    x[4] = 3.4e38
    x[5] = 1e-42
    held = LB.q4_values(x)
    assert (held[0] == 0).all() and np.abs(held[1] - 3.3).max() < 3.3 * 2 ** -12
    assert np.isnan(held[2:5]).all() and np.isfinite(held[5]).all()


def test_tokens_are_nearest():
    x = np.random.default_rng(2).standard_normal((50, 33)).astype(np.float32)
    c, s = LB.tokens8(x)
    assert (np.abs(c * s.astype(np.float64)[:, None] - x) <= s[:, None] * (0.5 + 2.0 ** -17)).all()
    assert (np.abs(c).max(-1) == 127).all()


@pytest.mark.parametrize("dim,bs,ok", [(128, 16, True), (64, 4, True), (8, 8, True), (256, 16, True), (264, 16, False),
                                       (12, 16, False), (128, 2, False), (128, 1, False)])
def test_q4_pool_shapes(s1kv, dim, bs, ok):
    if ok:
        s1kv.Pool(1, 2, dim, 4, bs, dtype="q4", host_only=True).close()
        return
    with pytest.raises(s1kv.S1KVError) as e:
        s1kv.Pool(1, 2, dim, 4, bs, dtype="q4", host_only=True)
    assert e.value.status == s1kv.EINVAL and "4-bit" in str(e.value)


def test_unknown_dtype_is_refused(s1kv):
    d = s1kv.PoolDesc(1, 1, 64, 16, 4, 3, 8, 0, 1e6, s1kv.POOL_HOST_ONLY, None)
    h = C.c_void_p()
    assert s1kv.lib().s1kv_pool_create(C.byref(d), 0, C.byref(h)) == s1kv.EINVAL


def test_noalloc_decode_refuses_q4(s1kv):
    L = s1kv.lib()
    assert L.s1kv_decode_attention_noalloc(64, 64, s1kv.DTYPE_Q4, 64, 1, 64, 16, 64, 4, 64, 1, 16, 64, 64, 1,
                                           None) == s1kv.EINVAL


def test_batch_gather_refuses_a_null_batch(s1kv):
    assert s1kv.lib().s1kv_batch_gather(None, 0, 0, None, None) == s1kv.EINVAL


@pytest.mark.parametrize("m,k,ld", [(-1, 16, 16), (4, 17, 16), (4, 16, 24), (4, 131073, 131088), (4, -1, 16)])
def test_quantize_tokens_refusals(s1kv, m, k, ld):
    assert s1kv.lib().s1kv_quantize_tokens(64, m, k, 64, ld, 64, None) == s1kv.EINVAL


def test_quantize_tokens_pointers(s1kv):
    L = s1kv.lib()
    assert L.s1kv_quantize_tokens(None, 4, 16, 64, 16, 64, None) == s1kv.EINVAL
    assert L.s1kv_quantize_tokens(64, 4, 16, 72, 16, 64, None) == s1kv.EINVAL
    assert L.s1kv_quantize_tokens(None, 0, 16, None, 16, None, None) == s1kv.OK


def group(s1kv, m, k, ns, xq=64, w=64, n_mats=None):
    L, n = s1kv.lib(), len(ns)
    vp, i64 = C.c_void_p, C.c_int64
    return L.s1kv_matmul_w8a8_group(xq, 64, m, k, n if n_mats is None else n_mats, (vp * n)(*[w] * n), (vp * n)(*[64] * n),
                                    (i64 * n)(*ns), (vp * n)(*[64] * n), None)


def test_matmul_w8a8_refusals(s1kv):
    assert group(s1kv, 4, 17, [8]) == s1kv.EINVAL
    assert group(s1kv, 4, 131088, [8]) == s1kv.EINVAL
    assert group(s1kv, -1, 16, [8]) == s1kv.EINVAL
    assert group(s1kv, 4, 16, [-8]) == s1kv.EINVAL
    assert group(s1kv, 4, 16, [8], xq=None) == s1kv.EINVAL
    assert group(s1kv, 4, 16, [8], xq=72) == s1kv.EINVAL
    assert group(s1kv, 4, 16, [8], w=68) == s1kv.EINVAL
    assert group(s1kv, 4, 16, [8] * 5) == s1kv.EINVAL
    assert group(s1kv, 4, 16, [8], n_mats=0) == s1kv.EINVAL
    assert s1kv.lib().s1kv_matmul_w8a8_group(64, 64, 4, 16, 1, None, None, None, None, None) == s1kv.EINVAL
    assert group(s1kv, 0, 16, [8, 8]) == s1kv.OK  # nothing to compute
    assert group(s1kv, 4, 16, [0, 0]) == s1kv.OK


def test_q4_prefix_file_is_read_on_the_host(s1kv, tmp_path):
    import struct

    from test_prefix_file import fnv1a64
    n, heads, dim = 3, 2, 16
    body = bytes(np.random.default_rng(0).integers(0, 120, 2 * n * heads * (dim // 2 + 4), dtype=np.uint8))

    def write(payload, d=dim):
        p = tmp_path / "q4.s1kv"
        p.write_bytes(struct.pack("<8s8I q f I Q", b"S1KVPFX\0", 1, 64, 1, heads, d, 16, 2, 0, n, 1e6, 0,
                                  fnv1a64(payload)) + payload)
        return p

    info = s1kv.prefix_file_info(write(body))
    assert info["dtype"] == s1kv.DTYPE_Q4 and info["n_tokens"] == n
    for payload, d in ((body[:-1], dim), (body, 12)):
        with pytest.raises(s1kv.S1KVError):
            s1kv.prefix_file_info(write(payload, d))


def test_linear_w8a8_refusals(s1kv):
    L = s1kv.lib()
    vp, i64 = C.c_void_p, C.c_int64
    args = lambda n: ((vp * 1)(64), (vp * 1)(64), (i64 * 1)(n), (vp * 1)(64))  # noqa: E731
    assert L.s1kv_w8a8_workspace(3, 17) == 3 * 32 + 16 and L.s1kv_w8a8_workspace(-1, 4) == 0
    assert L.s1kv_linear_w8a8_group(64, 3, 17, 64, 111, 1, *args(8), None) == s1kv.EINVAL  # workspace too small
    assert L.s1kv_linear_w8a8_group(64, 3, 17, 72, 112, 1, *args(8), None) == s1kv.EINVAL  # and not aligned
    assert L.s1kv_linear_w8a8_group(None, 3, 17, 64, 112, 1, *args(8), None) == s1kv.EINVAL
    assert L.s1kv_linear_w8a8_group(64, 3, 131073, 64, 1 << 40, 1, *args(8), None) == s1kv.EINVAL
    assert L.s1kv_linear_w8a8_group(64, 3, 17, 64, 112, 1, *args(0), None) == s1kv.OK  # nothing to compute

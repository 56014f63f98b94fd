"""GPU tests of the 4-bit cache and the 8-bit product where they can go wrong:
rows of equal values, scales far apart, and what the pool's other calls meet.

Tolerance of attention: as in test_gpu_4bit_8bit.py a weight is off by S 2^-21
at most, relative, for scores of up to S < 32 in log2 units: 1.5e-5; the sums
and the two fp16 parts of p s_v leave a few 2^-23 more.  So an output element
is within 2e-5 of sum_t p_t |v_t|, taken as its largest over the row's dims:
each row and head is held to its own size, whatever the others hold."""
import numpy as np
import pytest

from oracle import lowbit as LB
from test_gpu_4bit_8bit import dev, fill, kv, pool_of

pytestmark = pytest.mark.gpu
TOL = 2e-5


def check_rows(got, q, k, v, lens=None):
    """got [rows, Hq, D] against 64 bits on what the cache holds of k and v."""
    k, v = LB.q4_values(k), LB.q4_values(v)
    want, size = LB.attention64(q, k, v), LB.attention64(q, k, np.abs(v)).max(-1, keepdims=True)
    assert got.shape == want.shape and np.isfinite(want).all()
    assert np.isfinite(got).all(), "not finite"
    err = (np.abs(got - want) / np.maximum(size, 1e-300)).max()
    assert err <= TOL, err


def attend_and_check(s1kv, k, v, r, hq, seed=0, q=None):
    n, hkv, dim = k.shape
    if q is None:
        q = np.random.default_rng(seed).standard_normal((r, hq, dim)).astype(np.float32)
    pool = pool_of(s1kv, hkv, dim, -(-n // 16) + 4)
    fill(pool, [n], k, v)
    got = pool.attention(0, [0], [r], dev(q), hq).cpu().numpy()
    assert pool.check_device() == 0
    check_rows(got, q, k, v)


# ------------------------------------------------------ keys of scale zero --

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("r", [1, 3, 60, 170])
@pytest.mark.parametrize("kind", ["zeros", "ones", "value", "head", "group", "last", "tiny", "first"])
def test_keys_of_equal_values(s1kv, cuda, dim, r, kind):
    """K rows whose values are all the same are held with s = 0 (or a tiny s):
    their scores are m sum(q) alone."""
    rng = np.random.default_rng(80)
    hkv, hq, n = 2, 8, 193  # the last group of 32 keys holds one
    k, v = kv(rng, n, hkv, dim)
    if kind == "zeros":
        k[:] = 0
    elif kind == "ones":
        k[:] = 1
    elif kind == "value":
        k[:] = 3.3 / 8  # not a bf16 number
    elif kind == "head":
        k[:, 1] = 0
    elif kind == "group":
        k[32:64] = 0
        k[96:128, 0] = -0.5
    elif kind == "last":
        k[192] = 0
    elif kind == "tiny":
        k *= np.float32(1e-35)
    else:
        k[:40] = 0
    attend_and_check(s1kv, k, v, r, hq)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 33, 64])
def test_short_prompts_of_zero_keys(s1kv, cuda, dim, n):
    v = kv(np.random.default_rng(81), n, 1, dim)[1]
    attend_and_check(s1kv, np.zeros((n, 1, dim), np.float32), v, n, 4)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("r", [1, 150])
def test_keys_of_scales_far_apart(s1kv, cuda, dim, r):
    """Keys of 2^-40 beside ordinary ones in every group, and keys with a large
    common value beside a small spread (m / s of 2^9 and, seldom, 2^20)."""
    rng = np.random.default_rng(82)
    k, v = kv(rng, 300, 2, dim)
    k[::3] *= np.float32(2.0 ** -40)
    k[1::7] = k[1::7] * np.float32(2.0 ** -11) + np.float32(0.25)
    k[5::50] = np.float32(0.25)
    k[5::50, :, 0] += np.float32(2.0 ** -22)
    attend_and_check(s1kv, k, v, r, 8)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("r", [1, 40, 200])
@pytest.mark.parametrize("at,grow", [(230, 24), (230, 40), (230, 90), (100, 40), (299, 40), (0, 60)])
def test_a_large_key(s1kv, cuda, dim, r, at, grow):
    """One key 2^24 to 2^90 larger: a row that sees it gives it all its weight or
    none, rows before it are as they would be without."""
    rng = np.random.default_rng(79)
    k, v = kv(rng, 300, 2, dim)
    k[at] *= np.float32(2.0 ** grow)
    attend_and_check(s1kv, k, v, r, 8)


# ------------------------------------------------- values of far-off scales --

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("r", [1, 40, 200])
@pytest.mark.parametrize("at,grow", [(230, 16), (230, 20), (230, 40), (230, 70), (100, 30), (299, 60), (0, 40)])
def test_a_large_value_row(s1kv, cuda, dim, r, at, grow):
    """One V row 2^16 to 2^70 larger than the others: query rows before it do
    not see it and keep their precision, whatever the tile holds."""
    rng = np.random.default_rng(83)
    k, v = kv(rng, 300, 2, dim)
    v[at] *= np.float32(2.0 ** grow)
    attend_and_check(s1kv, k, v, r, 8)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hq", [4, 8])
@pytest.mark.parametrize("r", [1, 90])
@pytest.mark.parametrize("grow", [20, 40, 60])
@pytest.mark.parametrize("where", ["early", "late", "both"])
def test_a_large_value_row_that_weighs_little(s1kv, cuda, dim, hq, r, grow, where):
    """The large V rows are seen, but their scores lie 56 log2 units below the
    others': what they add is small, and the others keep their precision."""
    rng = np.random.default_rng(84)
    n, hkv = 600, 1
    u = rng.standard_normal(dim).astype(np.float32)
    u *= np.float32(np.sqrt(dim) / np.linalg.norm(u))
    side = np.ones(n, np.float32)
    for i in {"early": (3, 17), "late": (500,), "both": (0, 200, 509)}[where]:
        side[i] = -1
    top = 28 * np.log(2) / np.sqrt(dim)
    k = ((side[:, None] * u * top) + 0.01 * rng.standard_normal((n, dim))).astype(np.float32)[:, None]
    v = rng.standard_normal((n, hkv, dim)).astype(np.float32)
    v[side < 0] *= np.float32(2.0 ** grow)
    q = (np.tile(u, (r, hq, 1)) + 0.02 * rng.standard_normal((r, hq, dim))).astype(np.float32)
    attend_and_check(s1kv, k, v, r, hq, q=q)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("r", [1, 300])
@pytest.mark.parametrize("shape", ["rise", "fall", "constants", "huge", "offset"])
def test_value_rows_of_all_sizes(s1kv, cuda, dim, r, shape):
    """V rows that grow or shrink by 2^100 over the sequence, rows of equal
    values (s = 0) among others, rows next to fp32's end, rows of a large
    common value."""
    rng = np.random.default_rng(85)
    n = 500
    k, v = kv(rng, n, 2, dim)
    if shape in ("rise", "fall"):
        steps = np.linspace(-60, 40, n) * (1 if shape == "rise" else -1)
        v *= np.exp2(np.floor(steps)).astype(np.float32)[:, None, None]
    elif shape == "constants":
        v[::2] = np.float32(3.3)
        v[1::6] = 0
    elif shape == "huge":
        v *= np.float32(1e34)
        v[::5] = np.float32(3.3)
        v[3::5] = np.float32(1e36)
    else:
        v = v * np.float32(2.0 ** -10) + np.float32(4.0)
    attend_and_check(s1kv, k, v, r, 4)


@pytest.mark.parametrize("dim", [64, 128])
def test_long_chunks_with_large_value_rows(s1kv, cuda, dim):
    """As many chunks as SMs, so that none is split and sums are set aside on
    the way: V rows of 2^50 here and there, and a steady growth of 2^40."""
    rng = np.random.default_rng(86)
    hkv, hq, n, r = 8, 32, 1570, 1301
    k, v = kv(rng, n, hkv, dim)
    k *= np.float32(0.2)
    v[:, 2] *= np.exp2(np.floor(np.arange(n) * 41 / n)).astype(np.float32)[:, None]
    v[[700, 1400], 0] *= np.float32(2.0 ** 50)
    v[[300, 301, 1569], 5] *= np.float32(2.0 ** 24)
    q = rng.standard_normal((r, hq, dim)).astype(np.float32)
    pool = pool_of(s1kv, hkv, dim, 100)
    fill(pool, [n], k, v)
    got = pool.attention(0, [0], [r], dev(q), hq).cpu().numpy()
    for h in (0, 2, 5):
        heads = slice(4 * h, 4 * h + 4)
        check_rows(got[:, heads], q[:, heads], k[:, h:h + 1], v[:, h:h + 1])


@pytest.mark.parametrize("dim", [64, 128])
def test_long_decode_with_large_value_rows(s1kv, cuda, dim):
    """Rows split over CTAs: the splits' references differ by far."""
    rng = np.random.default_rng(87)
    k, v = kv(rng, 9000, 1, dim)
    v[[5, 4000, 8990]] *= np.float32(2.0 ** 40)
    v[3000:3500] *= np.float32(2.0 ** -50)
    attend_and_check(s1kv, k, v, 1, 4)
    attend_and_check(s1kv, k, v, 1, 12)
    attend_and_check(s1kv, k, v, 3, 4)


# ------------------------------------------------------- rows of wide spread --

@pytest.mark.parametrize("dim", [64, 128, 256, 40])
@pytest.mark.parametrize("rope", [False, True])
def test_rows_that_span_fp32(s1kv, cuda, dim, rope):
    """x - m passes fp32's largest at the low end: the codes are the format's."""
    rng = np.random.default_rng(88)
    n, hkv = 6, 2
    x = rng.standard_normal((n, hkv, dim)).astype(np.float32)
    x[0, 0] = np.linspace(-3.3e38, 3.3e38, dim)
    x[1, 1, ::3], x[1, 1, 5] = -3.2e38, 3.3e38
    x[2, 0, :2] = 3.3e38, -3.3e38
    x[3] *= np.float32(7e37)
    x[4, 1, -1] = -3.3e38
    pool = pool_of(s1kv, hkv, dim, 10)
    for i in range(n):  # (position 0: RoPE leaves the values as they are)
        with pool.batch([i], [1]) as b:
            one = dev(x[i:i + 1])
            b.rope_append(0, one, one) if rope else b.append(0, one, one)
            for which in (s1kv.K, s1kv.V):
                np.testing.assert_array_equal(b.gather(0, which).cpu().numpy(), LB.q4_values(x[i:i + 1]))


# ------------------------------------------------------- heads of a KV head --

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("g", [2, 4, 8, 9])
@pytest.mark.parametrize("r", [1, 20])
@pytest.mark.parametrize("factor", [2.0 ** 30, 2.0 ** 90, np.inf, np.nan])
def test_one_heads_query_leaves_the_others_alone(s1kv, cuda, dim, g, r, factor):
    """Query heads that share a KV head, one of them far larger or not finite:
    the others are held to their own precision."""
    rng = np.random.default_rng(89)
    hkv, n = 2, 150
    k, v = kv(rng, n, hkv, dim)
    q = rng.standard_normal((r, g * hkv, dim)).astype(np.float32)
    odd = [1, g * hkv - 1]
    rest = [h for h in range(g * hkv) if h not in odd]
    plain = q.copy()
    with np.errstate(invalid="ignore"):
        q[:, odd, 3:5] *= np.float32(factor)
    pool = pool_of(s1kv, hkv, dim, 14)
    fill(pool, [n], k, v)
    got = pool.attention(0, [0], [r], dev(q), g * hkv).cpu().numpy()
    for h in rest:
        check_rows(got[:, [h]], plain[:, [h]], k[:, [h // g]], v[:, [h // g]])
    if not np.isfinite(factor):
        assert np.isnan(got[:, odd]).all()


# ------------------------------------------------- batches open at one time --

def plain_rows(pool, kk, vv, q):
    """Attention of q's rows, the last tokens of kk, vv, as the pool holds them."""
    if pool.dtype == 2:
        kk, vv = LB.q4_values(kk), LB.q4_values(vv)
    elif pool.dtype == 1:
        kk, vv = (LB._bf16_rn(x) for x in (kk, vv))
    return LB.attention64(q, kk, vv)


@pytest.mark.parametrize("dtype", ["q4", "bf16", "f32"])
def test_decode_beside_an_open_batch_that_appends(s1kv, cuda, dtype):
    """One batch appends (its kernel lets the next start early), another that
    began before that append reads its tokens, right behind it."""
    rng = np.random.default_rng(90)
    hkv, hq, dim, n, new = 8, 32, 128, 900, 700
    k, v = kv(rng, 4 * n, hkv, dim)
    k2, v2 = kv(rng, 4 * new, hkv, dim)
    q = rng.standard_normal((5, hq, dim)).astype(np.float32)
    pool = s1kv.Pool(1, hkv, dim, 600, 16, dtype=dtype)
    with pool.batch([0, 1, 2, 3], [n] * 4, [0] * 4) as b:
        b.append(0, dev(k), dev(v))
    grow = pool.batch([0, 1, 2, 3], [new] * 4, [0] * 4)
    pool.fork(1, 9, n + new)  # shares blocks that `grow` fills
    read = pool.batch([0, 1, 2, 3, 9], None, [1] * 5)
    dk, dv, dq = dev(k2), dev(v2), dev(q)
    grow.append(0, dk, dv)
    got = read.attention(0, dq).cpu().numpy()
    grow.end()
    read.end()
    for row, i in enumerate((0, 1, 2, 3, 1)):
        kk = np.concatenate([k[i * n:(i + 1) * n], k2[i * new:(i + 1) * new]])
        vv = np.concatenate([v[i * n:(i + 1) * n], v2[i * new:(i + 1) * new]])
        want = plain_rows(pool, kk, vv, q[row:row + 1])
        assert np.abs(got[row] - want[0]).max() <= 2e-5 * np.abs(vv).max()


@pytest.mark.parametrize("dtype", ["q4", "bf16", "f32"])
def test_decode_of_a_sequence_named_twice(s1kv, cuda, dtype):
    rng = np.random.default_rng(91)
    hkv, hq, dim = 8, 32, 128
    k, v = kv(rng, 840, hkv, dim)
    q = rng.standard_normal((2, hq, dim)).astype(np.float32)
    pool = s1kv.Pool(1, hkv, dim, 80, 16, dtype=dtype)
    with pool.batch([0, 0], [400, 440], [1, 1]) as b:
        b.append(0, dev(k), dev(v))
        got = b.attention(0, dev(q)).cpu().numpy()
    for row, n in enumerate((400, 840)):
        want = plain_rows(pool, k[:n], v[:n], q[row:row + 1])
        assert np.abs(got[row] - want[0]).max() <= 2e-5 * np.abs(v).max()


# ----------------------------------------------------------------- products --

@pytest.mark.parametrize("m", [1, 2, 8, 20, 64, 200, 700])
@pytest.mark.parametrize("k", [512, 2048])
def test_products_one_behind_the_other(s1kv, cuda, m, k):
    """Calls without a pause, each quantising other tokens into the workspace
    that the one before used: every product is of its own tokens."""
    torch = cuda
    rng = np.random.default_rng(m + k)
    n, turns = 384, 12
    w = s1kv.quantize_channels(rng.standard_normal((k, n)).astype(np.float32))
    xs = [dev((rng.standard_normal((m, k)) * 3.0 ** i).astype(np.float32)) for i in range(turns)]
    outs = [torch.empty((m, n), device="cuda") for _ in xs]
    for _ in range(3):
        for x, o in zip(xs, outs):
            s1kv.matmul_w8a8(x, w, o)
        torch.cuda.synchronize()
        for x, o in zip(xs, outs):
            c, s = LB.tokens8(x.cpu().numpy())
            np.testing.assert_array_equal(o.cpu().numpy(), LB.product8(c, s, w.data.cpu().numpy()[:, :k], w.scales.cpu().numpy()))
            o.zero_()


# ----------------------------------------------- chunk batches side by side --

@pytest.mark.parametrize("dtype,dim,bs", [("q4", 40, 16), ("q4", 128, 8), ("f32", 64, 16), ("bf16", 40, 16)])
def test_chunk_batches_of_odd_shapes_keep_their_own_rows(s1kv, cuda, dtype, dim, bs):
    """Shapes without a chunk kernel plan their rows at the first attention
    call: another open batch's plan must not take their place."""
    rng = np.random.default_rng(92)
    hkv, hq = 2, 4
    pool = s1kv.Pool(2, hkv, dim, 100, bs, dtype=dtype)
    lens, rows = {0: 90, 1: 61}, {0: 7, 1: 11}
    kvs = {i: kv(rng, n, hkv, dim) for i, n in lens.items()}
    with pool.batch([0, 1], [90, 61], [0, 0]) as b:
        for layer in (0, 1):
            b.append(layer, *(dev(np.concatenate([kvs[0][j], kvs[1][j]])) for j in (0, 1)))
    q = {i: rng.standard_normal((r, hq, dim)).astype(np.float32) for i, r in rows.items()}
    open_ = {i: pool.batch([i], None, [rows[i]]) for i in (0, 1)}
    got = [(i, open_[i].attention(layer, dev(q[i])).cpu().numpy()) for layer in (0, 1) for i in (0, 1)]
    for b in open_.values():
        b.end()
    for i, o in got:
        want = plain_rows(pool, *kvs[i], q[i])
        assert np.abs(o - want).max() <= 2e-5 * np.abs(kvs[i][1]).max()
    assert pool.check_device() == 0


# ------------------------------------------------------------- prefix files --

LOAD = """
import re, sys
import torch
import s1kv

def status(key):
    return int(re.search(key + r":\\s+(\\d+) kB", open("/proc/self/status").read()).group(1)) * 1024

dtype, path, small, layers = sys.argv[1], sys.argv[2], sys.argv[3], int(sys.argv[4])
pool = s1kv.Pool(layers, 8, 128, 600, 16, dtype=dtype)
assert pool.prefix_load_v1(1, small) == 16
before = status("VmRSS")
assert pool.prefix_load_v1(2, path) == 4096
print(status("VmHWM") - before)
"""


@pytest.mark.parametrize("dtype,layers,most", [("q4", 16, 2.0), ("f32", 4, 2.6)])
def test_a_prefix_file_is_held_once(s1kv, cuda, tmp_path, dtype, layers, most):
    """Host memory of a load: the file, and its rows in fp32 where the pool
    takes those; a 4-bit file for a 4-bit pool is not widened."""
    import os
    import subprocess
    import sys
    torch = cuda
    pool = s1kv.Pool(layers, 8, 128, 600, 16, dtype=dtype)
    paths = []
    for seq, n in ((1, 16), (2, 4096)):
        with pool.batch([seq], [n], [0]) as b:
            for layer in range(layers):
                b.append(layer, *(torch.randn((n, 8, 128), device="cuda") for _ in range(2)))
        paths.append(tmp_path / f"{seq}.s1kv")
        pool.prefix_save_v1(seq, paths[-1], np.arange(n))
    size = os.path.getsize(paths[1])
    env = dict(os.environ, PYTHONPATH=os.path.dirname(os.path.dirname(s1kv.__file__)))
    r = subprocess.run([sys.executable, "-c", LOAD, dtype, str(paths[1]), str(paths[0]), str(layers)], env=env,
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert int(r.stdout) <= most * size + (32 << 20), (int(r.stdout), size)


# ------------------------------------------------------------ device memory --

@pytest.mark.parametrize("dtype", ["q4", "bf16"])
def test_device_bytes_are_what_the_pool_holds(s1kv, cuda, dtype):
    """Host-buffer steps and split rows of growing size: the statistic follows
    the device's free memory, and outgrown host-step buffers are given back."""
    torch = cuda
    hkv, hq, dim = 8, 32, 128
    sizes = (100, 900, 3000)
    pool = s1kv.Pool(1, hkv, dim, 3000, 16, dtype=dtype, max_seqs=300)
    h = [torch.randn((sizes[-1], x, dim)).pin_memory() for x in (hq, hkv, hkv)]
    out = torch.empty_like(h[0]).pin_memory()
    long = torch.randn((40000, hkv, dim), device="cuda")
    q = torch.randn((256, hq, dim), device="cuda")
    o = torch.empty_like(q)
    with pool.batch([999], [40000], [0]) as b:
        b.append(0, long, long)
    torch.cuda.synchronize()
    free, told = torch.cuda.mem_get_info()[0], pool.stats()["device_bytes"]
    slot = 0
    for i, n in enumerate(sizes):
        with pool.batch([i], [n]) as b:
            b.layer_host(0, *(x[:n] for x in h), out[:n], hq)
        torch.cuda.synchronize()
        slot = 4 * n * dim * (3 * hq + 2 * hkv)
        for s in range(1000, 1000 + (1, 16, 250)[i]):
            if not pool.length(s):
                pool.fork(999, s, 40000)
        seqs = list(range(1000, 1000 + (1, 16, 250)[i]))
        with pool.batch(seqs, None, [1] * len(seqs)) as b:
            b.attention(0, q[:len(seqs)], o[:len(seqs)])
        torch.cuda.synchronize()
        held = free - torch.cuda.mem_get_info()[0]
        assert abs(held - (pool.stats()["device_bytes"] - told)) <= 48 << 20
    grown = pool.stats()["device_bytes"] - told
    assert 2 * slot <= grown


# --------------------------------------------------- addresses and alignment --

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("g", [4, 8])
@pytest.mark.parametrize("r", [1, 50])
def test_pointers_of_four_bytes(s1kv, cuda, dim, g, r):
    """k, v, q and out that are aligned to their elements only; what lies
    before and behind out stays."""
    torch = cuda
    rng = np.random.default_rng(93)
    hkv, n = 2, 130
    k, v = kv(rng, n, hkv, dim)
    q = rng.standard_normal((r, g * hkv, dim)).astype(np.float32)

    def odd(x, fill=None):
        buf = torch.full((x.size + 2,), 7.0, device="cuda")
        t = buf[1:-1].view(x.shape)
        if fill is None:
            t.copy_(torch.from_numpy(x))
        return t, buf

    pool = pool_of(s1kv, hkv, dim, 14)
    with pool.batch([0], [n], [0]) as b:
        b.append(0, odd(k)[0], odd(v)[0])
        for which, x in ((s1kv.K, k), (s1kv.V, v)):
            np.testing.assert_array_equal(b.gather(0, which, odd(k, 0)[0]).cpu().numpy(), LB.q4_values(x))
    out, buf = odd(q, 0)
    with pool.batch([0], None, [r]) as b:
        b.attention(0, odd(q)[0], out)
    check_rows(out.cpu().numpy(), q, k, v)
    assert buf[0] == 7 and buf[-1] == 7


@pytest.mark.parametrize("dim", [64, 128])
def test_blocks_beyond_four_gigabytes(s1kv, cuda, dim):
    rng = np.random.default_rng(94)
    hkv, hq, n = 8, 16, 300
    blocks = (9 << 29) // (hkv * 16 * (dim // 2 + 4))  # 4.5 GB of K, and of V
    pool = s1kv.Pool(1, hkv, dim, blocks, 16, dtype="q4", max_seqs=4, max_seq_len=4096)  # (the last blocks come first)
    k, v = kv(rng, n, hkv, dim)
    q = rng.standard_normal((70, hq, dim)).astype(np.float32)
    fill(pool, [n], k, v)
    assert pool.block_table(0).min() > blocks - 40
    for which, x in ((s1kv.K, k), (s1kv.V, v)):
        np.testing.assert_array_equal(pool.gather(0, 0, which).cpu().numpy(), LB.q4_values(x))
    for r in (1, 70):
        check_rows(pool.attention(0, [0], [r], dev(q[:r]), hq).cpu().numpy(), q[:r], k, v)
    assert pool.check_device() == 0


@pytest.mark.parametrize("dim", [64, 128])
def test_chunks_over_long_contexts(s1kv, cuda, dim):
    """More tokens than a CTA keeps block ids of (16384), with and without the
    tiles split over CTAs."""
    rng = np.random.default_rng(95)
    hkv, hq, n = 4, 16, 19000
    k, v = kv(rng, n, hkv, dim)
    pool = pool_of(s1kv, hkv, dim, 1200)
    fill(pool, [n], k, v)
    for r in (5, 2600):
        q = rng.standard_normal((r, hq, dim)).astype(np.float32)
        got = pool.attention(0, [0], [r], dev(q), hq).cpu().numpy()
        for row in {0, r // 2, r - 1}:
            seen = n - r + row + 1
            check_rows(got[row:row + 1, :4], q[row:row + 1, :4], k[:seen, :1], v[:seen, :1])
            check_rows(got[row:row + 1, 12:], q[row:row + 1, 12:], k[:seen, 3:], v[:seen, 3:])

"""GPU tests of the 4-bit cache and the 8-bit product against their plain
64-bit forms (oracle/lowbit.py).

Tolerances.  What a pool holds and 8-bit codes are compared bit for bit.  An
attention output is within the repository's fp32 bound, 2e-5 of the largest
output, of the 64-bit result on the held values: with scores up to S in log2
units, q's two fp16 parts leave 2^-23 of each product, the fp32 sums and the
scales a few 2^-24, so a weight is off by about S 2^-21 relative; S stays
under 32 in these inputs, 32 * 2^-21 = 1.5e-5 at the very most and not for
all weights at once.  An 8-bit product is an exact integer with three fp32
roundings: compared bit for bit with the same three."""
import numpy as np
import pytest

from oracle import lowbit as LB

pytestmark = pytest.mark.gpu
TOL = 2e-5


def pool_of(s1kv, hkv, dim, blocks, bs=16, seed=0, **kw):
    order = np.random.default_rng(seed).permutation(blocks).astype(np.int32)
    return s1kv.Pool(kw.pop("layers", 1), hkv, dim, blocks, bs, dtype="q4", initial_free_list=order, **kw)


def dev(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def kv(rng, n, hkv, dim):
    k = rng.standard_normal((n, hkv, dim)).astype(np.float32)
    k *= (0.5 + 2 * rng.random((1, hkv, dim)) ** 4).astype(np.float32)
    return k, (rng.standard_normal((n, hkv, dim)) + 0.3).astype(np.float32)


def fill(pool, lens, k, v, layer=0):
    with pool.batch(list(range(len(lens))), lens, [0] * len(lens)) as b:
        b.append(layer, dev(k), dev(v))


def check_close(got, want, tol=TOL):
    assert got.shape == want.shape
    nan = np.isnan(want)
    assert np.array_equal(nan, np.isnan(got))
    if not nan.all():
        err = np.abs(got[~nan] - want[~nan]).max() / np.abs(want[~nan]).max()
        assert err <= tol, err


# ------------------------------------------------------------------ rows --

def edge_rows(rng, n, hkv, dim):
    x = rng.standard_normal((n, hkv, dim)).astype(np.float32)
    x[0] = 0
    x[1] = 3.3
    x[2, 0, dim // 2] = np.nan
    x[3, 0, 1] = -np.inf
    x[4] *= 1e-41
    x[5] = x[5] * 1e-3 + 1000
    x[6] *= 1e37
    x[7, 0] = 3.4e38
    x[8, 0] = np.linspace(-8, 7, dim)  # codes near ties
    x[8, 0, : min(dim, 16)] = np.arange(-8, 8)[: min(dim, 16)]
    x[9] = np.round(x[9] * 4) / 8
    return x


@pytest.mark.parametrize("dim,bs,hkv", [(128, 16, 2), (64, 16, 3), (8, 4, 1), (24, 8, 2), (200, 12, 1), (256, 16, 2)])
def test_append_holds_the_format(s1kv, cuda, dim, bs, hkv):
    rng = np.random.default_rng(dim)
    lens = [11, 1, 37]
    n = sum(lens)
    k, v = edge_rows(rng, n, hkv, dim), edge_rows(rng, n, hkv, dim)[::-1].copy()
    pool = pool_of(s1kv, hkv, dim, 24, bs)
    with pool.batch([0, 1, 2], lens, [0, 0, 0]) as b:
        b.append(0, dev(k), dev(v))
        got = [b.gather(0, w).cpu().numpy() for w in (s1kv.K, s1kv.V)]
    for g, x in zip(got, (k, v)):
        np.testing.assert_array_equal(g, LB.q4_values(x))
    t0 = 0
    for i, ln in enumerate(lens):  # by sequence, and the bytes in storage
        table = pool.block_table(i)
        for which, x in ((s1kv.K, k), (s1kv.V, v)):
            np.testing.assert_array_equal(pool.gather(0, i, which).cpu().numpy(), LB.q4_values(x[t0:t0 + ln]))
            c, s, m = LB.q4_rows(x[t0:t0 + ln])
            raw = pool.read_storage(0, which)
            for j, blk in enumerate(table):
                part = slice(j * bs, min((j + 1) * bs, ln))
                cnt = part.stop - part.start
                for h in range(hkv):
                    cc, ss, mm = np.zeros((bs, dim), np.int64), np.zeros(bs, np.float32), np.zeros(bs, np.float32)
                    cc[:cnt], ss[:cnt], mm[:cnt] = c[part, h], s[part, h], m[part, h]
                    np.testing.assert_array_equal(raw[blk, h], LB.q4_storage(cc, ss, mm, which, bs))
        t0 += ln
    assert pool.check_device() == 0


@pytest.mark.parametrize("dim,hkv,hq", [(128, 2, 8), (64, 3, 3), (40, 1, 5)])
def test_rope_append_is_rope_then_append(s1kv, cuda, dim, hkv, hq):
    rng = np.random.default_rng(5)
    lens = [17, 1, 30]
    n = sum(lens)
    k, v = kv(rng, n, hkv, dim)
    q = rng.standard_normal((n, hq, dim)).astype(np.float32)
    pool, plain = pool_of(s1kv, hkv, dim, 16), s1kv.Pool(1, hkv, dim, 16, 16)
    got, want = [], []
    for p, o in ((pool, got), (plain, want)):
        for off in (0, 1):  # a second append starts inside blocks
            with p.batch([0, 1, 2], lens) as b:
                o.append(b.rope_append(0, dev(k), dev(v), q=dev(q)).cpu().numpy())
                o += [b.gather(0, s1kv.K).cpu().numpy(), b.gather(0, s1kv.V).cpu().numpy()]
    for i in (0, 3):
        np.testing.assert_array_equal(got[i], want[i])
    for i in (1, 2, 4, 5):
        np.testing.assert_array_equal(got[i], LB.q4_values(want[i]))


@pytest.mark.parametrize("dim", [64, 128, 40])
def test_rope_append_of_q_in_place(s1kv, cuda, dim):
    rng = np.random.default_rng(7)
    n, hkv, hq = 700, 2, 6
    k, v = kv(rng, n, hkv, dim)
    q = dev(rng.standard_normal((n, hq, dim)).astype(np.float32))
    pool = pool_of(s1kv, hkv, dim, 100)
    with pool.batch([0], [n]) as b:
        want = b.rope_append(0, dev(k), dev(v), q)
    pool.truncate(0, 0)
    with pool.batch([0], [n]) as b:
        got = b.rope_append(0, dev(k), dev(v), q, q)
    np.testing.assert_array_equal(got.cpu().numpy(), want.cpu().numpy())


@pytest.mark.parametrize("dim", [64, 128])
def test_norm_rope_append_is_the_fp32_pools_rows(s1kv, cuda, dim):
    rng = np.random.default_rng(6)
    lens, hkv, hq = [33, 1, 16], 3, 6
    n = sum(lens)
    k, v = kv(rng, n, hkv, dim)
    q = rng.standard_normal((n, hq, dim)).astype(np.float32)
    qw, kw = (dev(rng.random(dim).astype(np.float32) + 0.5) for _ in range(2))
    out = []
    for p in (pool_of(s1kv, hkv, dim, 16), s1kv.Pool(1, hkv, dim, 16, 16)):
        with p.batch([0, 1, 2], lens) as b:
            qr = b.norm_rope_append(0, dev(k), dev(v), kw, q=dev(q), q_norm_weight=qw)
            out.append([qr.cpu().numpy(), b.gather(0, s1kv.K).cpu().numpy(), b.gather(0, s1kv.V).cpu().numpy()])
    np.testing.assert_array_equal(out[0][0], out[1][0])
    np.testing.assert_array_equal(out[0][1], LB.q4_values(out[1][1]))
    np.testing.assert_array_equal(out[0][2], LB.q4_values(v))


def test_single_call_append_and_bad_slots(s1kv, cuda):
    rng = np.random.default_rng(7)
    pool = pool_of(s1kv, 2, 64, 4)
    k, v = kv(rng, 3, 2, 64)
    _, slots = pool.reserve(9, 3)
    pool.append(0, k, v, slots)
    np.testing.assert_array_equal(pool.gather(0, 9, s1kv.K).cpu().numpy(), LB.q4_values(k))
    before = pool.read_storage(0, s1kv.V)
    pool.append(0, k, v, [64, -1, 1 << 30])  # beyond the 4 blocks: skipped and flagged
    np.testing.assert_array_equal(pool.read_storage(0, s1kv.V), before)
    with pytest.raises(s1kv.S1KVError) as e:
        pool.check_device()
    assert e.value.status == s1kv.EDEVICE
    with pytest.raises(s1kv.S1KVError):
        pool.read_storage(0, s1kv.K, 1, 16)


# ------------------------------------------------------------- attention --

def attend(s1kv, lens, qlens, hq, hkv, dim, seed, bs=16, scale=1.0, blocks=None):
    rng = np.random.default_rng(seed)
    k, v = kv(rng, sum(lens), hkv, dim)
    q = (scale * rng.standard_normal((sum(qlens), hq, dim))).astype(np.float32)
    need = sum(-(-n // bs) for n in lens)
    pool = pool_of(s1kv, hkv, dim, blocks or need + 5, bs, seed)
    fill(pool, lens, k, v)
    with pool.batch(list(range(len(lens))), None, qlens) as b:
        got = b.attention(0, dev(q)).cpu().numpy()
    want, t0, r0 = [], 0, 0
    for n, r in zip(lens, qlens):
        want.append(LB.attention64(q[r0:r0 + r], LB.q4_values(k[t0:t0 + n]), LB.q4_values(v[t0:t0 + n])))
        t0, r0 = t0 + n, r0 + r
    assert pool.check_device() == 0
    check_close(got, np.concatenate(want))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("g", [1, 2, 3, 4, 5, 7, 8, 9, 16, 20])
def test_decode_groups(s1kv, cuda, dim, g):
    attend(s1kv, [1, 15, 16, 17, 64, 65, 257, 700], [1] * 8, 2 * g, 2, dim, 10 + g)


def test_decode_long_rows_merge_in_two_levels(s1kv, cuda):
    attend(s1kv, [20001, 5], [1, 1], 4, 1, 128, 31)
    attend(s1kv, [9000], [1], 24, 1, 64, 32)


def test_decode_sharp_and_flat_scores(s1kv, cuda):
    # scale 4: scores reach some 25 log2 units and the running maximum moves; flat: 3000 near-equal weights
    attend(s1kv, [900], [1], 8, 2, 128, 33, scale=4.0)
    attend(s1kv, [3000], [1], 8, 2, 128, 34, scale=0.01)


@pytest.mark.parametrize("dim,bs,hq,hkv", [(40, 16, 4, 2), (128, 8, 8, 2), (64, 4, 3, 3), (256, 16, 2, 1), (8, 4, 2, 2),
                                           (64, 16, 33, 1)])
def test_other_shapes(s1kv, cuda, dim, bs, hq, hkv):
    attend(s1kv, [1, bs, 2 * bs + 1, 100], [1] * 4, hq, hkv, dim, 40)
    attend(s1kv, [1, bs, 2 * bs + 1, 50], [1, 2, bs, 5], hq, hkv, dim, 41)


@pytest.mark.parametrize("hq,hkv,dim", [(8, 2, 128), (4, 4, 128), (8, 1, 128), (4, 2, 64), (7, 1, 128), (12, 4, 64), (16, 1, 128)])
def test_chunks(s1kv, cuda, hq, hkv, dim):
    attend(s1kv, [300, 64, 1, 130, 515], [40, 64, 1, 129, 0], hq, hkv, dim, 50)
    attend(s1kv, [333], [333], hq, hkv, dim, 51)
    attend(s1kv, [1025, 20], [2, 3], hq, hkv, dim, 52)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shape", ["up", "down", "steps"])
def test_scores_that_rise(s1kv, cuda, dim, shape):
    """Scores over 60 log2 units, up or down the sequence or in jumps inside
    tiles, so that the running maximum moves again and again, for decode rows
    and chunks (scores stay within 32 of zero)."""
    rng = np.random.default_rng(65)
    hkv, hq, n = 1, 4, 700
    u = rng.standard_normal(dim).astype(np.float32)
    u *= np.float32(np.sqrt(dim) / np.linalg.norm(u))
    ramp = np.linspace(-1, 1, n)
    if shape == "down":
        ramp = ramp[::-1]
    elif shape == "steps":
        ramp = np.sign(np.sin(np.arange(n) / 23.0)) * np.linspace(0.1, 1, n)
    top = 28 * np.log(2) / np.sqrt(dim)  # q.k / sqrt(dim) in log2 units: 28 at the ends
    k = (ramp[:, None] * u * top)[:, None].astype(np.float32)
    v = rng.standard_normal((n, hkv, dim)).astype(np.float32)
    pool = pool_of(s1kv, hkv, dim, 50)
    fill(pool, [n], k, v)
    for r in (1, 200):
        q = np.tile(u, (r, hq, 1)) + 0.05 * rng.standard_normal((r, hq, dim)).astype(np.float32)
        got = pool.attention(0, [0], [r], dev(q), hq).cpu().numpy()
        check_close(got, LB.attention64(q, LB.q4_values(k), LB.q4_values(v)))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shape", ["up", "steps"])
def test_long_chunks(s1kv, cuda, dim, shape):
    """As many chunks as SMs, so that none is split and a chunk passes over up
    to 13 tiles: scores that rise by 56 log2 units and V rows that grow by
    2^12 on the way, so what earlier tiles left is brought to new references
    (scores stay within 32 of zero)."""
    rng = np.random.default_rng(66)
    hkv, hq, n, r = 8, 32, 1570, 1301
    u = rng.standard_normal(dim).astype(np.float32)
    u *= np.float32(np.sqrt(dim) / np.linalg.norm(u))
    ramp = np.linspace(-1, 1, n)
    if shape == "steps":
        ramp = np.sign(np.sin(np.arange(n) / 93.0)) * np.linspace(0.1, 1, n)
    k = np.repeat((ramp[:, None] * u * (28 * np.log(2) / np.sqrt(dim)))[:, None].astype(np.float32), hkv, 1)
    k[:, 1::2] *= np.float32(0.1)  # flat scores: every tile counts
    v = rng.standard_normal((n, hkv, dim)).astype(np.float32)
    v *= np.exp2(np.floor(np.arange(n) * 13 / n)).astype(np.float32)[:, None, None]
    q = np.tile(u, (r, hq, 1)) + 0.05 * rng.standard_normal((r, hq, dim)).astype(np.float32)
    pool = pool_of(s1kv, hkv, dim, 100)
    fill(pool, [n], k, v)
    got = pool.attention(0, [0], [r], dev(q), hq).cpu().numpy()
    for h in (0, 3, 6):
        heads = slice(4 * h, 4 * h + 4)
        check_close(got[:, heads], LB.attention64(q[:, heads], LB.q4_values(k[:, h:h + 1]), LB.q4_values(v[:, h:h + 1])))


def test_scales_far_apart(s1kv, cuda):
    """V rows of one sequence differing by 2^80 in size, the large ones seldom
    and early or late: the running power of two must follow."""
    rng = np.random.default_rng(60)
    n, hkv, dim, hq = 500, 2, 128, 8
    k, v = kv(rng, n, hkv, dim)
    v[:250] *= np.float32(2.0 ** -60)
    v[400, 1] *= np.float32(2.0 ** 20)
    q = rng.standard_normal((1, hq, dim)).astype(np.float32)
    pool = pool_of(s1kv, hkv, dim, 40)
    fill(pool, [n], k, v)
    for keep in (n, 200):  # all, then only the small rows
        pool.truncate(0, keep)
        got = pool.attention(0, [0], [1], dev(q), hq).cpu().numpy()
        want = LB.attention64(q, LB.q4_values(k[:keep]), LB.q4_values(v[:keep]))
        for h in range(hq):
            check_close(got[:, h], want[:, h])


@pytest.mark.parametrize("qlen", [1, 20, 100])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_lies_past_the_end_is_not_read(s1kv, cuda, qlen, dim):
    rng = np.random.default_rng(61)
    hkv, hq, n = 2, 8, 100
    k, v = kv(rng, 160, hkv, dim)
    k[n:], v[n:] = np.nan, np.inf
    q = rng.standard_normal((qlen, hq, dim)).astype(np.float32)
    pool = pool_of(s1kv, hkv, dim, 10)
    fill(pool, [160], k, v)
    pool.truncate(0, n)
    got = pool.attention(0, [0], [qlen], dev(q), hq).cpu().numpy()
    check_close(got, LB.attention64(q, LB.q4_values(k[:n]), LB.q4_values(v[:n])))


@pytest.mark.parametrize("qlen", [1, 60])
def test_a_spoilt_row_reaches_who_sees_it_only(s1kv, cuda, qlen):
    rng = np.random.default_rng(62)
    hkv, hq, dim, n = 2, 4, 128, 90
    k, v = kv(rng, n, hkv, dim)
    k[70, 0, 3] = np.nan
    v[80, 1, 5] = np.inf
    q = rng.standard_normal((qlen, hq, dim)).astype(np.float32)
    pool = pool_of(s1kv, hkv, dim, 10)
    fill(pool, [n], k, v)
    got = pool.attention(0, [0], [qlen], dev(q), hq).cpu().numpy()
    for i in range(qlen):
        seen = n - qlen + i
        assert np.isnan(got[i, :2]).all() == (seen >= 70) and np.isnan(got[i, :2]).any() == (seen >= 70)
        assert np.isnan(got[i, 2:]).all() == (seen >= 80) and np.isnan(got[i, 2:]).any() == (seen >= 80)


# ------------------------------------------------- the pool's other calls --

def test_fork_copy_on_write_and_prefix_cache(s1kv, cuda):
    rng = np.random.default_rng(70)
    hkv, dim, hq = 2, 128, 8
    k, v = kv(rng, 60, hkv, dim)
    k2, v2 = kv(rng, 2, hkv, dim)
    pool = pool_of(s1kv, hkv, dim, 16, layers=2)
    with pool.batch([0], [60], [0]) as b:
        for layer in (0, 1):
            b.append(layer, dev(k), dev(v))
    pool.prefix_insert(0, np.arange(60, dtype=np.int32))
    pool.fork(0, 1, 55)  # ends inside a block: its first append copies it
    with pool.batch([0, 1], [1, 1]) as b:
        for layer in (0, 1):
            b.append(layer, dev(k2), dev(v2))
    assert pool.stats()["cow_copies"] >= 1
    assert pool.prefix_match(2, np.arange(60, dtype=np.int32)) == 48
    for layer in (0, 1):
        for which, x, y in ((s1kv.K, k, k2), (s1kv.V, v, v2)):
            np.testing.assert_array_equal(pool.gather(layer, 0, which).cpu().numpy(), LB.q4_values(np.concatenate([x, y[:1]])))
            np.testing.assert_array_equal(pool.gather(layer, 1, which).cpu().numpy(),
                                          LB.q4_values(np.concatenate([x[:55], y[1:]])))
            np.testing.assert_array_equal(pool.gather(layer, 2, which).cpu().numpy(), LB.q4_values(x[:48]))


def test_prefix_files(s1kv, cuda, tmp_path):
    rng = np.random.default_rng(71)
    k, v = edge_rows(rng, 40, 2, 64), edge_rows(rng, 40, 2, 64)
    pool = pool_of(s1kv, 2, 64, 8, layers=2)
    with pool.batch([0], [40], [0]) as b:
        b.append(0, dev(k), dev(v))
        b.append(1, dev(v), dev(k))
    path = tmp_path / "q4.s1kv"
    pool.prefix_save_v1(0, path, np.arange(40))
    assert s1kv.prefix_file_info(path)["dtype"] == s1kv.DTYPE_Q4
    for other in (pool_of(s1kv, 2, 64, 9, 8, seed=3, layers=2), s1kv.Pool(2, 2, 64, 8, 16)):  # 4-bit (other blocks) and fp32
        assert other.prefix_load_v1(5, path, register=True) == 40
        for layer, pair in ((0, (k, v)), (1, (v, k))):
            for which in (0, 1):
                np.testing.assert_array_equal(other.gather(layer, 5, which).cpu().numpy(), LB.q4_values(pair[which]))
    raw = tmp_path / "raw"
    pool.prefix_save(0, raw)
    np.testing.assert_array_equal(np.fromfile(raw, np.float32).reshape(2, 2, 40, 2, 64)[0, 0], LB.q4_values(k))
    pool.prefix_load(6, 40, raw)
    np.testing.assert_array_equal(pool.gather(0, 6, 0).cpu().numpy(), LB.q4_values(LB.q4_values(k)))


def test_host_buffers_and_reference_interface(s1kv, cuda):
    torch = cuda
    rng = np.random.default_rng(72)
    hkv, hq, dim = 2, 8, 64
    k, v = kv(rng, 50, hkv, dim)
    q = rng.standard_normal((50, hq, dim)).astype(np.float32)
    pool, same = pool_of(s1kv, hkv, dim, 8), pool_of(s1kv, hkv, dim, 8)
    h = [torch.from_numpy(x).pin_memory() for x in (q, k, v)]
    out = torch.empty_like(h[0]).pin_memory()
    with pool.batch([0], [50]) as b:
        b.layer_host(0, *h, out, hq)
    torch.cuda.synchronize()
    with same.batch([0], [50]) as b:
        qr = b.rope_append(0, dev(k), dev(v), q=dev(q))
        want = b.attention(0, qr)
    assert torch.equal(out, want.cpu())
    ref = s1kv.KVBlockPool(hkv, dim, 8, dtype="q4")
    ref.append(1, k, v)
    np.testing.assert_array_equal(ref.get_v(1).cpu().numpy(), LB.q4_values(v))
    got = s1kv.gqa_attention_paged(q[:1], ref.get_k_view(1), ref.get_v_view(1), hq, hkv, dim).cpu().numpy()
    check_close(got, LB.attention64(q[:1], LB.q4_values(k), LB.q4_values(v)))


def test_exchange_of_one_rank(s1kv, cuda):
    rng = np.random.default_rng(73)
    hkv, hq, dim = 2, 8, 128
    k, v = kv(rng, 200, hkv, dim)
    q = rng.standard_normal((1, hq, dim)).astype(np.float32)
    pool = pool_of(s1kv, hkv, dim, 16)
    fill(pool, [200], k, v)
    ex = s1kv.PeerExchange(0, 1, 1, hq, dim)
    with pool.batch([0], None, [1]) as b:
        want = b.attention(0, dev(q)).cpu().numpy()
        ex.attention(b, 0, dev(q), 0, 1)
        got = ex.output(1).cpu().numpy()
    np.testing.assert_array_equal(got, want)
    ex.close()


def test_graph_replay_and_another_stream(s1kv, cuda):
    """A captured step (append, attention, product) replays on new inputs, on
    a stream of its own, and gives what plain calls give."""
    torch = cuda
    rng = np.random.default_rng(74)
    hkv, hq, dim, lens = 2, 8, 128, [100, 33]
    k, v = kv(rng, sum(lens), hkv, dim)
    pools = [pool_of(s1kv, hkv, dim, 16) for _ in range(2)]
    w = s1kv.quantize_channels(rng.standard_normal((hq * dim, 96)).astype(np.float32))
    stream = torch.cuda.Stream()
    for p in pools:
        fill(p, lens, k, v)
    sk, sv, sq = (torch.zeros((2, h, dim), device="cuda") for h in (hkv, hkv, hq))

    def step(b):
        b.append(0, sk, sv)
        return s1kv.matmul_w8a8(b.attention(0, sq).reshape(2, -1), w)

    with torch.cuda.stream(stream):
        b = pools[0].batch([0, 1], [1, 1])
        step(b)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(b)
    plain = pools[1].batch([0, 1], [1, 1])
    for i in range(3):
        new = [dev(rng.standard_normal(t.shape).astype(np.float32)) for t in (sk, sv, sq)]
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for t, x in zip((sk, sv, sq), new):
                t.copy_(x)
            graph.replay()
        stream.synchronize()
        got = out.clone()
        assert torch.equal(got, step(plain))
    b.end()
    plain.end()


def test_prompts_captured_on_two_streams_at_once(s1kv, cuda):
    """Chunk attention of two pools and prompt-sized products, captured into a
    graph each and replayed at once on two streams, again and again."""
    torch = cuda
    rng = np.random.default_rng(75)
    hkv, hq, dim, n = 4, 16, 64, 900
    w = s1kv.quantize_channels(rng.standard_normal((hq * dim, 5000)).astype(np.float32))
    runs = []
    for i in range(2):
        k, v = kv(rng, n, hkv, dim)
        pool = pool_of(s1kv, hkv, dim, 60)
        fill(pool, [n], k, v)
        q = dev(rng.standard_normal((n - 100, hq, dim)).astype(np.float32))
        b = pool.batch([0], None, [n - 100])
        o, y = torch.empty_like(q), torch.empty((n - 100, 5000), device="cuda")

        def step(b=b, q=q, o=o, y=y):
            b.attention(0, q, o)
            s1kv.matmul_w8a8(o.reshape(n - 100, -1), w, y)

        step()
        torch.cuda.synchronize()
        want = o.clone(), y.clone()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            b.end()
            b = pool.batch([0], None, [n - 100])
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step(b=b)
        runs.append((stream, graph, o, y, want, b, q))
    for _ in range(5):
        for stream, graph, o, y, *_ in runs:
            with torch.cuda.stream(stream):
                o.zero_(), y.zero_()
                graph.replay()
    torch.cuda.synchronize()
    for _, _, o, y, want, b, _ in runs:
        assert torch.equal(o, want[0]) and torch.equal(y, want[1])
        b.end()


# --------------------------------------------------------------- products --

@pytest.mark.parametrize("m,k", [(1, 1), (3, 16), (5, 33), (1, 4096), (130, 1000), (2, 131072)])
def test_token_codes(s1kv, cuda, m, k):
    rng = np.random.default_rng(k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    if m > 2:
        x[0] = 0
        x[1] = np.round(x[1] * 8) / 16  # many ties
        x[1, 0] = 127 / 16
        x[2] *= 1e-40
    q, s = s1kv.quantize_tokens(x)
    c, want = LB.tokens8(x)
    assert q.shape == (m, (k + 15) // 16 * 16)
    np.testing.assert_array_equal(s.cpu().numpy(), want)
    np.testing.assert_array_equal(q.cpu().numpy()[:, :k], c)
    assert (q.cpu().numpy()[:, k:] == 0).all()


PRODUCTS = [(1, 16, 1), (1, 1024, 2048), (1, 1020, 333), (1, 1022, 50), (1, 1040, 70), (2, 100, 77), (7, 48, 130), (8, 4096, 256), (9, 512, 300), (16, 2000, 129), (17, 64, 64),
            (33, 1000, 777), (64, 4096, 512), (65, 272, 200), (128, 128, 128), (129, 1040, 385), (256, 1536, 1000),
            (300, 4096, 520), (1000, 80, 50), (2049, 512, 640), (5, 131072, 40), (50, 600, 200), (100, 48, 11700), (3, 14336, 70),
            (34, 131072, 130), (20, 4096, 5200), (32, 512, 300), (11, 8192, 6200)]


@pytest.mark.parametrize("m,k,n", PRODUCTS)
def test_product(s1kv, cuda, m, k, n):
    rng = np.random.default_rng(m * 7 + k + n)
    x = rng.standard_normal((m, k)).astype(np.float32)
    w = rng.standard_normal((k, n)).astype(np.float32)
    wq = s1kv.quantize_channels(w)
    got = s1kv.matmul_w8a8(x, wq).cpu().numpy()
    c, s = LB.tokens8(x)
    np.testing.assert_array_equal(got, LB.product8(c, s, wq.data.cpu().numpy()[:, :k], wq.scales.cpu().numpy()))


@pytest.mark.parametrize("m,k,ns", [(4100, 272, [1500]), (257, 1040, [7201]), (700, 80, [5000]), (2000, 640, [1000, 130, 2001]),
                                    (9000, 16, [513])])
def test_product_of_prompts(s1kv, cuda, m, k, ns):
    """Tokens and channels enough for tiles over pairs of SMs, ragged in both."""
    rng = np.random.default_rng(m + k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    x[m - 1, 0], x[m // 2] = np.inf, 0
    ws = [s1kv.quantize_channels(rng.standard_normal((k, n)).astype(np.float32)) for n in ns]
    outs = s1kv.matmul_w8a8_group(x, ws)
    c, s = LB.tokens8(x)
    xq, sx = s1kv.quantize_tokens(x)
    for w, o in zip(ws, outs):
        want = LB.product8(c, s, w.data.cpu().numpy()[:, :k], w.scales.cpu().numpy())
        np.testing.assert_array_equal(o.cpu().numpy(), want)
        o.fill_(1.0)  # the caller's own codes
        s1kv.check(s1kv.lib().s1kv_matmul_w8a8(xq.data_ptr(), sx.data_ptr(), m, w.ld, w.data.data_ptr(), w.scales.data_ptr(), w.n,
                                               o.data_ptr(), s1kv._stream()))
        np.testing.assert_array_equal(o.cpu().numpy(), want)


@pytest.mark.parametrize("m", [1, 20, 200])
def test_product_at_the_integers_limits(s1kv, cuda, m):
    """Sums of 131072 products of 127: beyond 24 bits and next to 2^31."""
    torch = cuda
    k = 131072
    xq = torch.full((m, k), 127, dtype=torch.int8, device="cuda")
    w = torch.full((24, k), 127, dtype=torch.int8, device="cuda")
    w[1::2] = -127
    xq[-1, 1::2] = -128
    ones = torch.ones(max(m, 24), device="cuda")
    out = torch.empty((m, 24), device="cuda")
    s1kv.check(s1kv.lib().s1kv_matmul_w8a8(xq.data_ptr(), ones.data_ptr(), m, k, w.data_ptr(), ones.data_ptr(), 24,
                                           out.data_ptr(), s1kv._stream()))
    want = (xq.cpu().numpy().astype(np.int64) @ w.cpu().numpy().astype(np.int64).T).astype(np.float32)
    np.testing.assert_array_equal(out.cpu().numpy(), want)


@pytest.mark.parametrize("m", [1, 6, 40, 300])
def test_product_group_is_the_single_products(s1kv, cuda, m):
    torch = cuda
    rng = np.random.default_rng(m)
    k = 528
    x = dev(rng.standard_normal((m, k)).astype(np.float32))
    ws = [s1kv.quantize_channels(rng.standard_normal((k, n)).astype(np.float32)) for n in (256, 1, 77, 640)]
    guard = torch.full((m + 1, 77), 7.0, device="cuda")  # a row behind the last must stay
    outs = [torch.empty((m, w.n), device="cuda") for w in ws]
    outs[2] = guard[:m]
    got = s1kv.matmul_w8a8_group(x, ws, outs)
    for g, w in zip(got, ws):
        assert torch.equal(g, s1kv.matmul_w8a8(x, w))
    assert (guard[m] == 7).all()


@pytest.mark.parametrize("m", [3, 50, 400])
def test_product_of_spoilt_and_empty_tokens(s1kv, cuda, m):
    rng = np.random.default_rng(m)
    x = rng.standard_normal((m, 96)).astype(np.float32)
    x[0, 5], x[1, 7], x[2] = np.nan, -np.inf, 0
    got = s1kv.matmul_w8a8(x, s1kv.quantize_channels(rng.standard_normal((96, 40)).astype(np.float32))).cpu().numpy()
    assert np.isnan(got[:2]).all() and (got[2] == 0).all() and np.isfinite(got[3:]).all()


def test_product_python_refusals(s1kv, cuda):
    torch = cuda
    w = s1kv.quantize_channels(np.ones((32, 8), np.float32))
    x = torch.ones((4, 32), device="cuda")
    for bad in (torch.ones((4, 31), device="cuda"), torch.ones(32, device="cuda")):
        with pytest.raises(s1kv.S1KVError):
            s1kv.matmul_w8a8(bad, w)
    for out in (torch.empty((4, 9), device="cuda"), torch.empty((8, 4), device="cuda").t(), torch.empty((4, 8), dtype=torch.half, device="cuda")):
        with pytest.raises(s1kv.S1KVError):
            s1kv.matmul_w8a8(x, w, out)
    with pytest.raises(s1kv.S1KVError):
        s1kv.ChannelQuantizedTensor(w.data.t(), w.scales)
    with pytest.raises(s1kv.S1KVError):
        s1kv.ChannelQuantizedTensor(w.data, w.scales, 8)
    assert s1kv.matmul_w8a8(torch.empty((0, 32), device="cuda"), w).shape == (0, 8)


# ------------------------------------------------------ the whole layer step --

@pytest.mark.parametrize("lens,new", [([40, 7, 129], [1, 1, 1]), ([0, 64], [150, 33])])
def test_layer_step(s1kv, cuda, lens, new):
    """x -> 8-bit q/k/v products -> RoPE + 4-bit append -> attention -> 8-bit
    output product, against the same chain in numpy on what each stage holds."""
    rng = np.random.default_rng(sum(lens))
    hidden, hkv, hq, dim = 256, 2, 8, 64
    wq, wk, wv = (s1kv.quantize_channels(rng.standard_normal((hidden, h * dim)).astype(np.float32) / 8) for h in (hq, hkv, hkv))
    wo = s1kv.quantize_channels(rng.standard_normal((hq * dim, hidden)).astype(np.float32))
    pool = pool_of(s1kv, hkv, dim, 40)
    seqs = list(range(len(lens)))
    hist = kv(rng, sum(lens), hkv, dim)
    if sum(lens):
        with pool.batch(seqs, lens, [0] * len(lens)) as b:
            b.append(0, dev(hist[0]), dev(hist[1]))
    x = rng.standard_normal((sum(new), hidden)).astype(np.float32)
    with pool.batch(seqs, new) as b:
        q, k, v = s1kv.matmul_w8a8_group(x, [wq, wk, wv])
        qr = b.rope_append(0, k.view(-1, hkv, dim), v.view(-1, hkv, dim), q=q.view(-1, hq, dim))
        o = b.attention(0, qr)
        y = s1kv.matmul_w8a8(o.reshape(sum(new), -1), wo).cpu().numpy()
    c, s = LB.tokens8(x)
    prods = [LB.product8(c, s, w.data.cpu().numpy(), w.scales.cpu().numpy()) for w in (wq, wk, wv)]
    for a, b_ in zip((q, k, v), prods):
        np.testing.assert_array_equal(a.cpu().numpy(), b_)
    want, t0, r0 = [], 0, 0
    for n, r in zip(lens, new):
        rot = s1kv.apply_rope(prods[1][r0:r0 + r].reshape(r, hkv, dim), n).cpu().numpy()
        kk = LB.q4_values(np.concatenate([hist[0][t0:t0 + n], rot]))
        vv = LB.q4_values(np.concatenate([hist[1][t0:t0 + n], prods[2][r0:r0 + r].reshape(r, hkv, dim)]))
        want.append(LB.attention64(qr[r0:r0 + r].cpu().numpy(), kk, vv))
        t0, r0 = t0 + n, r0 + r
    check_close(o.cpu().numpy(), np.concatenate(want))
    c, s = LB.tokens8(o.reshape(sum(new), -1).cpu().numpy())
    np.testing.assert_array_equal(y, LB.product8(c, s, wo.data.cpu().numpy(), wo.scales.cpu().numpy()))

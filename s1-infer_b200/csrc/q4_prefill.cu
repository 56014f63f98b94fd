// q4_prefill.cu -- chunked-prefill attention over a 4-bit cache (format:
// q4.cuh) on tcgen05: query chunks of more than one token, row i of a
// sequence's q_len new tokens seeing tokens 0 .. (kv_len - q_len) + i.
//
//   score_t = q . (s_k c_t) + m_k sum(q),  out = sum_t (p_t s_v) c_t + sum_t p_t m_v
// with the centred codes c = u - 8.  s c is exact in fp16: seven significant
// codes are 3 bits, the eighth a power of two, s is 8 bits, fp16 has 11.  q
// and p s_v are each split into two fp16 parts (22 bits) and both parts are
// multiplied: fp32-level results for twice the tensor-core work of a bf16
// cache's prefill, 8 Hq D products a (query, visible token) in place of 4.
// V stands as plain codes and s_v goes to p: the tensor cores cut the bits of
// a product that lie below the running sum, and products of 15 bits lose a
// quarter of what products of 22 lose over the hundreds of steps of a sum.
// Bound: a tile's chain scores - softmax - sums; two tiles in turn keep the
// tensor cores busy 35% of the time and the issue slots 49% (a prompt of 4001
// tokens, 32 heads on 8 of 128: 317 us, 414e12 operations a second, 830e12 with
// both parts counted; 8650 cycles a pair of tiles, 4100 of products).  K/V bytes
// are a seventh of bf16's.
//
// A CTA takes a chunk of queries of one sequence and KV head as two tiles A
// and B of 128 accumulator rows, a row a (query, head) pair: 128 / G queries
// times the G query heads of the KV head (any G up to 128).
//   * Four warpgroups run the softmax, two per tile, two threads a row:
//     scores from TMEM, the online softmax in the exp2 domain (reference max
//     moved only past 2^8), p split and stored over the scores.
//   * One warpgroup widens K/V: a thread loads a token's codes straight from
//     its block (the next tile's loads are in flight while it waits for the
//     buffer), makes fp16 of them and writes the 128-byte-swizzled tiles the
//     MMAs read.  K's dims stand in the order 0 4 1 5 2 6 3 7 of each eight,
//     as they come out of a word; q is stored alike.
//   * One warp issues the MMAs: PV_A(t) S_A(t+1) PV_B(t) S_B(t+1), so one
//     tile's softmax runs under the other's products, and K and V need one
//     buffer each: K(t+1) is written under PV_A(t), V(t+1) under S_B(t+1).
// Few chunks over a long context: the tiles are split over CTAs as well, a
// second kernel joins the partial rows.
// Waits are bounded; a timeout raises an abort flag that every role polls
// and the device error word.  TMEM is freed on every path.
#include <cmath>

#include "q4.cuh"

namespace s1kv {
namespace {

constexpr uint32_t kSpin = 1u << 22;
constexpr int kM = 128, kN = 128;  // rows per tile, tokens per K/V tile
constexpr int kSoftmaxWarps = 16, kWidenWarps = 4, kMmaWarp = 20;  // two softmax threads a row
constexpr int kThreads = 32 * 24;  // (three idle warps complete the MMA's warpgroup)
// Registers by role.  At launch 80 a thread, 768 * 80 = 61440 in all;
// 512 * 96 + 128 * 64 + 128 * 32 = 61440.  Spilled registers cost dearly here:
// shared memory leaves the L1 cache too little for them.
constexpr int kRegsSoftmax = 96, kRegsWiden = 64, kRegsMma = 32;
constexpr int kFlush = 4;          // tiles a chain of sums in TMEM
constexpr int kColO = 256;         // TMEM: S_A [0, 128) S_B [128, 256) O_A O_B
constexpr int kTmemCols = 512;
constexpr float kRescaleAt = 8.0f;
constexpr int kMinExp = 20;         // least exponent (biased) scales are taken relative to
constexpr int kUp = 11;             // K's largest s stands as 2^11 .. 2^12 in its fp16 tile: 8 s below 2^15
constexpr int kVUp = 6;             // V's largest s counts as 2^6 .. 2^7 beside p: p s below 2^15
// A V row counts by the exponent of max(s, |m| / 2^kBelowM) where rows are uneven,
// some s kEven powers of two below the largest or more; kFar below it at least.
constexpr int kBelowM = 8, kEven = 6, kFar = 80, kAbove = 60;
// Keys of uneven scales: scores are summed in units of 2^kUnit / un, where neither
// m_k sum(q) of the largest keys overflows nor that of the smallest is lost.
constexpr int kUnit = 28, kMinExpK = 40;
constexpr int kIdsCached = 1024;   // block ids kept in shared memory (16K tokens)

template <int D>
struct Cfg {
    static constexpr int kAtoms = D / 64;             // 128-byte swizzle atoms across a row
    static constexpr int kQBytes = kAtoms * kM * 128;  // one part of one query tile
    static constexpr int kKBytes = kAtoms * kN * 128;
    static constexpr int kOffQ = 0;                    // A high, A low, B high, B low
    static constexpr int kOffK = 4 * kQBytes;
    static constexpr int kOffV = kOffK + kKBytes;
    static constexpr int kOffPar = kOffV + kKBytes;    // TilePar [2]
    static constexpr int kOffXch = kOffPar + 2 * (kN * 20 + 32);  // floats [4][2 halves][256 rows]
    static constexpr int kOffRef = kOffXch + 4 * 4 * 2 * kM * 2;  // float2 [512] (max, exponent)
    static constexpr int kOffIds = kOffRef + 512 * 8;
    static constexpr int kOffBar = kOffIds + kIdsCached * 4;
    // k_full k_empty v_full v_empty par_full[2] s_full[2] p_full[2] pv_done[2] drain q_full pair[8]
    static constexpr int kNumBars = 22;
    static constexpr int kOffMisc = kOffBar + kNumBars * 8 + 8;  // TMEM slot, abort flag, set-aside slot
    static constexpr int kSmem = kOffMisc + 16 + 1024;
};

__device__ __forceinline__ uint32_t su32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// Barriers and the abort flag are held as 32-bit shared addresses (registers
// are short).
__device__ __forceinline__ void bar_init(uint32_t b, uint32_t n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b), "r"(n) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t b, uint32_t phase) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(b), "r"(phase)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool bar_wait(uint32_t b, uint32_t phase) {
    for (uint32_t i = 0; i < kSpin; i++)
        if (bar_try(b, phase)) return true;
    return false;
}
__device__ __forceinline__ void bar_arrive(uint32_t b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(b) : "memory");
}
__device__ __forceinline__ int flag_get(uint32_t flag) {
    int v;
    asm volatile("ld.volatile.shared.b32 %0, [%1];" : "=r"(v) : "r"(flag) : "memory");
    return v;
}
__device__ __forceinline__ void flag_set(uint32_t flag, int v) {
    asm volatile("st.volatile.shared.b32 [%0], %1;" ::"r"(flag), "r"(v) : "memory");
}
__device__ __forceinline__ bool warp_wait(uint32_t b, uint32_t phase, uint32_t abort_flag) {
    bool ok = bar_try(b, phase);
    for (uint32_t i = 0; i < kSpin && !ok; i++) {
        ok = bar_try(b, phase);
        if (!ok && flag_get(abort_flag)) break;
    }
    if (!ok) flag_set(abort_flag, 1);
    return __all_sync(0xffffffffu, ok);
}
// Shared-memory descriptor, 128-byte swizzle (layout type 2), 8-row groups
// 1024 bytes apart: the low word holds the address and the leading offset,
// the high word is the same for all (64-bit descriptors kept for every K step
// spill; a low word is one addition).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo_bytes) {
    return ((addr >> 4) & 0x3FFF) | (lbo_bytes >> 4) << 16;
}
// kind::f16 instruction descriptor: fp16 A and B (0), fp32 D (1).
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, int b_mn_major) {
    return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Issued by one elected lane of a converged warp: D (TMEM) (+)= A B with A in
// shared memory (ss) or TMEM (ts), B in shared memory.
__device__ __forceinline__ void mma_ss_w(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "elect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kDescHi)
        : "memory");
}
__device__ __forceinline__ void mma_ts_w(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t.reg .b64 db;\n\tmov.b64 db, {%2, %5};\n\t"
        "elect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kDescHi)
        : "memory");
}
__device__ __forceinline__ void mma_commit_w(uint32_t b) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(b)
        : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 16 consecutive fp32 columns of this thread's TMEM lane; the wait is apart.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
          "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr));
}
// Waits for this thread's TMEM loads.  The registers pass through, so that
// nothing that uses them can be moved ahead of the wait.
__device__ __forceinline__ void tmem_ld_wait16(float* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
                 :);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void split_h2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack_h2(a - f.x, b - f.y);
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) { return __byte_perm(a, b, s); }

__device__ __forceinline__ uint32_t mul_h2(uint32_t a, __half2 b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), b);
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 <= e <= 127

// Byte offset of 16-byte chunk `chunk` of row `r` in a tile of `rows` rows
// held as 128B-swizzled atoms of 64 elements.
__device__ __forceinline__ uint32_t chunk_at(int r, int chunk, int rows) {
    return (uint32_t)((chunk >> 3) * rows * 128 + r * 128 + (((chunk & 7) ^ (r & 7)) << 4));
}

template <int REGS>
__device__ __forceinline__ void regs_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void regs_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

// A softmax thread's state: half of each tile's tokens of a row.  un: scores
// are in units of 1 / un (q was scaled by a power of two); qs: sum of the
// scaled q.
struct RowState {
    float m;
    float2 l, z;  // of this thread's even and odd tokens
    int E;
    float un, qs;
};
// The parameters of a tile's rows.
struct TilePar {
    float mk[kN], mv[kN];
    float sv[kN];   // s_v 2^(133 - E)
    float ev[kN];   // exponents of V less E, from -kFar to kAbove
    float fk[kN];   // K's token t stands in the tile as s_k c 2^-kUnit / fk[t], a power of two
    float f[4];     // 2^kUnit fk of all the tokens 32 g .. + 31 where uneven[g] is 0
    uint8_t uneven[4];  // 1: these tokens' s_k and m_k lie too far apart for one power of two (or s_k is 0), or V's exponents do
    int E;              // largest exponent of s_v so far
    int pad[2];
};

// 2^(m' - m): from what refers to m' to m; reference maxima are whole numbers.
__device__ __forceinline__ float from_max(float m_old, float m) {
    return m_old == m ? 1.0f : m - m_old < 127.0f ? pow2((int)(m_old - m)) : 0.0f;  // (0 from m' = -inf)
}
// 2^(m' - m) 2^(E' - E): from sums that refer to (m', E') to (m, E); never more than 1.
__device__ __forceinline__ float rebase(float m_old, int e_old, float m, int e) {
    const float k = (m_old - m) + (float)(e_old - e);
    return k > -127.0f ? pow2((int)fminf(k, 0.0f)) : 0.0f;  // (0 from m' = -inf)
}

// The first `cols` columns of this thread's P times a power of two (exact but
// for subnormals): its reference max rose after they were stored.
__device__ __forceinline__ void scale_p(uint32_t tS, int cols, float f) {
    tmem_st_wait();
    const __half2 f2 = __float2half2_rn(f);
#pragma unroll 1
    for (int c = 0; c < cols; c += 16) {
        float w[16];
        tmem_ld16(tS + c, w);
        tmem_ld_wait16(w);
        uint32_t y[16];
#pragma unroll
        for (int i = 0; i < 16; i++) y[i] = mul_h2(__float_as_uint(w[i]), f2);
        tmem_st16(tS + c, y);
    }
}

// Half a tile's scores of one row (64 tokens from token t0) -> P over them: of
// each 16 columns the first 8 take the high parts of p s_v, the others the low
// parts.  One pass, 16 columns at a time with the next 16 on their way.  The
// reference max (a whole number of log2 units) moves only when a score outgrows
// it by 2^8, seldom after the first tile: then what this tile has stored so far
// is scaled; at the end the row's two threads agree on the larger reference.
// (A pass of its own for the maximum, agreed on before the weights, took 2200
// of 5400 cycles a tile.)  The loop stays rolled: unrolled over all scores the
// code runs from beyond the instruction cache.  ANY: only tokens up to `last`
// (of this tile) are seen, the others may hold anything, NaN included; and K's
// rows may have any scales: the score is (v fk + m_k qs 2^-kUnit) (un 2^kUnit), so
// that m_k is not divided by a scale (0, for a row of equal values).  Else m_k qs
// / f joins v in units of 1 / (un f), one operation a score.  fresh: O starts anew with
// this tile.
// The reference is one for the weights p s_v, which must fit fp16: m follows the
// largest score plus V's exponent relative to E, so a V row that a token does not
// see, or hardly weighs, takes no bits from the others however large it is.
// Where the rows' exponents are even the scores alone will do.  Then p may pass
// 2^8, by as much as V's exponents lie below E.
template <bool ANY, int D>
__device__ __forceinline__ bool softmax_tile(uint32_t tS, uint32_t tO, const TilePar& par, int t0, int last, RowState& st,
                                             bool fresh, float* xch, int xch_other, uint32_t pair, uint32_t phase,
                                             uint32_t p_full, uint32_t abort_flag, int lane) {
    float v[2][16];
    float m = st.m;
    float2 l2 = st.l, z2 = st.z;
    tmem_ld16(tS, v[0]);
    if (par.E != st.E) {
        // E has risen: m falls by as much, which leaves the sums of p s_v as they
        // are, as far as l and z stay in range (l to 2^100, z to 2^113)
        const int el = (int)(__float_as_uint(l2.x + l2.y) >> 23) + 13, ez = (int)(__float_as_uint(fmaxf(fabsf(z2.x), fabsf(z2.y))) >> 23);
        const int room = max(min(min(par.E - st.E, 120), 240 - max(el, ez)), 0);
        const float f = pow2(room);
        m -= (float)room;
        l2 = make_float2(l2.x * f, l2.y * f);
        z2 = make_float2(z2.x * f, z2.y * f);
    }
#pragma unroll 1
    for (int c = 0; c < 64; c += 32) {
        const float f = ANY ? pow2(kUnit) : par.f[(t0 + c) / 32], qs = __fdividef(st.qs, f), un = st.un * f;
        const float2 qs2 = make_float2(qs, qs), un2 = make_float2(un, un);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int c0 = t0 + c + 16 * u;
            float2 x[8];
            float top = -INFINITY;
            tmem_ld_wait16(v[u]);
            if (u == 0 || c == 0) tmem_ld16(tS + c + 16 * u + 16, v[u ^ 1]);
            if (ANY && __all_sync(0xffffffffu, c0 > last)) {  // none of these rows sees any of the 16
                const uint32_t none[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                tmem_st8(tS + c + 16 * u, none);
                tmem_st8(tS + c + 16 * u + 8, none);
                continue;
            }
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float4 k = *reinterpret_cast<const float4*>(&par.mk[c0 + 2 * i]);
                x[i] = make_float2(v[u][2 * i], v[u][2 * i + 1]);
                x[i + 1] = make_float2(v[u][2 * i + 2], v[u][2 * i + 3]);
                if (ANY) {
                    const float4 fk = *reinterpret_cast<const float4*>(&par.fk[c0 + 2 * i]);
                    x[i] = __fmul2_rn(x[i], make_float2(fk.x, fk.y));
                    x[i + 1] = __fmul2_rn(x[i + 1], make_float2(fk.z, fk.w));
                }
                x[i] = __ffma2_rn(make_float2(k.x, k.y), qs2, x[i]);
                x[i + 1] = __ffma2_rn(make_float2(k.z, k.w), qs2, x[i + 1]);
                float2 w0 = x[i], w1 = x[i + 1];
                if (ANY) {
                    if (c0 + 2 * i > last) x[i].x = -INFINITY;
                    if (c0 + 2 * i + 1 > last) x[i].y = -INFINITY;
                    if (c0 + 2 * i + 2 > last) x[i + 1].x = -INFINITY;
                    if (c0 + 2 * i + 3 > last) x[i + 1].y = -INFINITY;
                    const float4 ev = *reinterpret_cast<const float4*>(&par.ev[c0 + 2 * i]);
                    w0 = __ffma2_rn(x[i], un2, make_float2(ev.x, ev.y));
                    w1 = __ffma2_rn(x[i + 1], un2, make_float2(ev.z, ev.w));
                }
                top = fmaxf(fmaxf(top, fmaxf(w0.x, w0.y)), fmaxf(w1.x, w1.y));
            }
            if (!ANY) top *= un;
            const bool raise = top > m + kRescaleAt;
            if (__any_sync(0xffffffffu, raise)) {
                const float mn = raise ? ceilf(top) : m, r = from_max(m, mn);
                l2 = make_float2(l2.x * r, l2.y * r);
                z2 = make_float2(z2.x * r, z2.y * r);
                scale_p(tS, c + 16 * u, r);
                m = mn;
            }
            const float nm = m == -INFINITY ? 0.0f : -m;  // nothing visible yet: p = 0
            const float2 nm2 = make_float2(nm, nm);
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float4 mv = *reinterpret_cast<const float4*>(&par.mv[c0 + 2 * i]);
                const float4 sv = *reinterpret_cast<const float4*>(&par.sv[c0 + 2 * i]);
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const float2 y = __ffma2_rn(x[i + w], un2, nm2);
                    float2 mm = w ? make_float2(mv.z, mv.w) : make_float2(mv.x, mv.y);
                    if (ANY) {  // 0 times what an unseen token holds
                        if (c0 + 2 * (i + w) > last) mm.x = 0.0f;
                        if (c0 + 2 * (i + w) + 1 > last) mm.y = 0.0f;
                    }
                    const float2 p = make_float2(ex2(y.x), ex2(y.y));
                    l2 = __fadd2_rn(l2, p);
                    z2 = __ffma2_rn(p, mm, z2);
                    const float2 ps = __fmul2_rn(p, w ? make_float2(sv.z, sv.w) : make_float2(sv.x, sv.y));
                    // the high part rounded, not cut: the low parts' signs then
                    // vary and what the sums cut from them cancels
                    const __half2 t = __floats2half2_rn(ps.x, ps.y);
                    const float2 tf = __half22float2(t), r = __ffma2_rn(tf, make_float2(-1.0f, -1.0f), ps);
                    hi[i + w] = *reinterpret_cast<const uint32_t*>(&t);
                    lo[i + w] = pack_h2(r.x, r.y);
                }
            }
            tmem_st8(tS + c + 16 * u, hi);
            tmem_st8(tS + c + 16 * u + 8, lo);
        }
    }
    *xch = m;
    __syncwarp();
    if (lane == 0) bar_arrive(pair);
    if (!warp_wait(pair, phase, abort_flag)) return false;
    const float other = xch[xch_other];
    const int e = par.E;
    if (!__all_sync(0xffffffffu, m == other && m == st.m && e == st.E)) {
        const float row_m = fmaxf(m, other), r = from_max(m, row_m), corr = rebase(st.m, st.E, row_m, e);
        l2 = make_float2(l2.x * r, l2.y * r);
        z2 = make_float2(z2.x * r, z2.y * r);
        if (__any_sync(0xffffffffu, r != 1.0f)) scale_p(tS, 64, r);
        if (!fresh && __any_sync(0xffffffffu, corr != 1.0f)) {  // this thread's half of O's columns
#pragma unroll 1
            for (int c = 0; c < D / 2; c += 16) {
                float ov[16];
                tmem_ld16(tO + c, ov);
                tmem_ld_wait16(ov);
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; i++) w[i] = __float_as_uint(ov[i] * corr);
                tmem_st16(tO + c, w);
            }
        }
        st.m = row_m;
        st.E = e;
    }
    tmem_st_wait();
    st.l = l2;
    st.z = z2;
    tc_fence_before();
    __syncwarp();
    if (lane == 0) bar_arrive(p_full);
    return true;
}

}  // namespace

struct PrefillQ4Params {
    const float* q;          // [rows][Hq][D] fp32, post-RoPE
    float* out;
    const int32_t* table;
    const PrefillSeq* seqs;
    const char* kbase;       // this layer's tiles
    const char* vbase;
    float* part_o;           // n_split > 1: [split][rows][Hq][D], unnormalised
    float* part_ml;          // [split][rows][Hq][2]  (max in log2 units, sum)
    int64_t n_rows;
    int32_t n_seqs, max_chunks, n_split;
    int32_t max_bps, max_blocks;
    int32_t Hq, Hkv, G, QT;  // QT = 128 / G queries a tile
    float* aside;            // [n_aside][D][256] sums set aside by running CTAs
    int32_t* aside_lock;     // [n_aside] 1 while a CTA holds the slot
    int32_t n_aside;
    float scale_log2;
    int* err;
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1) prefill_q4_kernel(const __grid_constant__ PrefillQ4Params p) {
    using C = Cfg<D>;
    constexpr int kTileBytes = 16 * (D / 2 + 4);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (-su32(smem_raw) & 1023u);  // (a sum: the compiler still sees shared memory)
    const uint32_t bars = su32(smem) + C::kOffBar;
    const uint32_t k_full = bars, k_empty = bars + 8, v_full = bars + 16, v_empty = bars + 24;
    const uint32_t par_full = bars + 32, s_full = bars + 48, p_full = bars + 64, pv_done = bars + 80;  // of two each
    const uint32_t drain = bars + 96, q_full = bars + 104, pairs = bars + 112;
    const uint32_t abort_flag = su32(smem) + C::kOffMisc + 4;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
    float* xch = reinterpret_cast<float*>(smem + C::kOffXch);
    volatile int* aside_slot = reinterpret_cast<volatile int*>(smem + C::kOffMisc + 8);
    TilePar* par = reinterpret_cast<TilePar*>(smem + C::kOffPar);
    static_assert(sizeof(TilePar) == kN * 20 + 32, "two tiles' parameters");
    int32_t* ids = reinterpret_cast<int32_t*>(smem + C::kOffIds);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // the chunks with the most visible tokens first, all sequences' and heads'
    // (a head after the other, the last one's long chunks start when the SMs run empty)
    const int h = blockIdx.x % p.Hkv, seq_i = blockIdx.x / p.Hkv % p.n_seqs;
    const int chunk = p.max_chunks - 1 - blockIdx.x / p.Hkv / p.n_seqs;
    pdl_wait_trigger();
    const PrefillSeq sm = p.seqs[seq_i];
    const int G = p.G, QT = p.QT, q0 = chunk * 2 * QT;
    if (q0 >= sm.q_len) return;  // uniform: no TMEM allocated yet
    const int prefix = sm.kv_len - sm.q_len;
    const int kv_end = min(sm.kv_len, prefix + q0 + 2 * QT);
    const int all_tiles = (kv_end + kN - 1) / kN;
    const int tb = (int)((int64_t)all_tiles * blockIdx.y / p.n_split), te = (int)((int64_t)all_tiles * (blockIdx.y + 1) / p.n_split);
    const int n_tiles = te - tb;
    const bool two_tiles = q0 + QT < sm.q_len;
    const int32_t* tab = p.table + (int64_t)sm.table_row * p.max_bps;
    const int n_blocks = (kv_end + 15) / 16, b0 = tb * (kN / 16);

    // ---- set-up ----
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)), "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        // the widening and softmax warps arrive once a warp, the MMA commits once
        for (int i = 0; i < C::kNumBars; i++)
            bar_init(bars + 8 * i, i == 0 || i == 2 || i == 4 || i == 5 ? (uint32_t)kWidenWarps : i == 8 || i == 9 ? 8u : i == 13 ? (uint32_t)kSoftmaxWarps : i > 13 ? 2u : 1u);
        flag_set(abort_flag, 0);
        // A slot for the sums that chains of tiles set aside.  One CTA fits an
        // SM and there are as many slots as SMs, so one is free
        // (without one the sums merely run on).
        int got = -1;
        if (n_tiles > kFlush) {
            uint32_t sm_id;
            asm volatile("mov.u32 %0, %%smid;" : "=r"(sm_id));
            for (int i = 0; i < p.n_aside && got < 0; i++) {
                const int at = (int)((sm_id + i) % p.n_aside);
                if (atomicCAS(&p.aside_lock[at], 0, 1) == 0) got = at;
            }
            __threadfence();  // what the slot's last CTA left lies behind
        }
        *aside_slot = got;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    auto lookup = [&](int b) -> int32_t {  // -1: no such block
        if (b >= n_blocks) return -1;
        const int32_t blk = tab[b];
        if ((uint32_t)blk >= (uint32_t)p.max_blocks) {
            atomicOr(p.err, kErrBounds);
            return -1;
        }
        return blk;
    };
    for (int i = tid; i < min(n_tiles * (kN / 16), kIdsCached); i += kThreads) ids[i] = lookup(b0 + i);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int slot = *aside_slot;
    const int chain = slot < 0 ? INT32_MAX : kFlush;  // tiles until O starts anew

    if (warp >= kMmaWarp) {
        regs_dec<kRegsMma>();
        if (warp == kMmaWarp) {
            // ================= MMA issuer =================
            constexpr uint32_t idS = idesc_f16(kM, kN, 0), idO = idesc_f16(kM, D, 1);
            const uint32_t dk = desc_lo(su32(smem + C::kOffK), 16), dv = desc_lo(su32(smem + C::kOffV), kN * 128);
            const uint32_t dq0 = desc_lo(su32(smem + C::kOffQ), 16);
            // (rolled: descriptors of every step at once would spill)
            auto issue_s = [&](int X) {
                const uint32_t dq = dq0 + (uint32_t)X * (2 * C::kQBytes / 16);
#pragma unroll 1
                for (int part = 1; part >= 0; part--)  // the small parts first: the sums are cut, not rounded
#pragma unroll 1
                    for (int a = 0; a < C::kAtoms; a++) {
                        const uint32_t da = dq + (uint32_t)part * (C::kQBytes / 16) + (uint32_t)a * (kM * 128 / 16);
                        const uint32_t db = dk + (uint32_t)a * (kN * 128 / 16);
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            mma_ss_w(tmem + X * 128, da + 2 * k, db + 2 * k, idS, part == 0 || a > 0 || k > 0);
                    }
                mma_commit_w(s_full + 8 * X);
            };
            auto issue_pv = [&](int X, bool fresh) {  // both parts of P, the small ones first
#pragma unroll 2
                for (int ks = 0; ks < 8; ks++) {
                    const uint32_t a = tmem + X * 128 + ks * 16, db = dv + ks * (16 * 128 / 16);
                    mma_ts_w(tmem + kColO + X * 128, a + 8, db, idO, !fresh || ks > 0);
                    mma_ts_w(tmem + kColO + X * 128, a, db, idO, true);
                }
                mma_commit_w(pv_done + 8 * X);
            };
            bool ok = n_tiles > 0 && warp_wait(q_full, 0, abort_flag) && warp_wait(k_full, 0, abort_flag);
            if (ok) {
                tc_fence_after();
                issue_s(0);
                if (two_tiles) issue_s(1);
                mma_commit_w(k_empty);
            }
            for (int t = 0; t < n_tiles && ok; t++) {
                const uint32_t ph = (uint32_t)(t & 1);
                const bool more = t + 1 < n_tiles;
                for (int X = 0; X < (two_tiles ? 2 : 1) && ok; X++) {
                    ok = warp_wait(p_full + 8 * X, ph, abort_flag) && (X || warp_wait(v_full, ph, abort_flag));
                    if (!ok) break;
                    tc_fence_after();
                    issue_pv(X, t % chain == 0);
                    if (X == (two_tiles ? 1 : 0)) mma_commit_w(v_empty);  // after the last product that reads V(t)
                    if (more) {  // S_X(t + 1) overwrites P_X(t), which PV_X(t) ahead of it reads
                        ok = X || warp_wait(k_full, ph ^ 1u, abort_flag);
                        if (!ok) break;
                        tc_fence_after();
                        issue_s(X);
                        if (X == (two_tiles ? 1 : 0)) mma_commit_w(k_empty);
                    }
                }
            }
            // everything issued has finished before TMEM is freed (bounded)
            mma_commit_w(drain);
            bar_wait(drain, 0);
        }
    } else if (warp >= kSoftmaxWarps) {
        // ================= widening: K, V and the rows' scales =================
        regs_dec<kRegsWiden>();
        const int i = tid - 32 * kSoftmaxWarps;  // this thread's token of a tile (K), token pair and half (V)
        const int vp = i & 63, vh = i >> 6;
        constexpr int NK = D / 32;  // 16-byte loads of a token's K codes; as many of half a V pair's
        uint4 kr[NK];  // one tile of K or V at a time: K's next loads wait for V's conversion, registers are short
        uint4 (&vr)[NK] = kr;
        uint32_t pk = 0, pv[4];  // this thread's token of K; V's tokens lane + 32 j (every warp works out the tile's largest s_v)
        int E = kMinExp;         // largest exponent of s_v so far
        auto block = [&](int t, int b) -> int32_t {  // block b of local tile t
            const int j = t * (kN / 16) + b;
            return j < kIdsCached ? ids[j] : lookup(b0 + j);
        };
        auto load_k = [&](int t) {
            const int32_t blk = block(t, i >> 4);
            pk = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int32_t b = block(t, 2 * j + (lane >> 4));
                pv[j] = b < 0 || (tb + t) * kN + 32 * j + lane >= kv_end
                            ? 0u
                            : *reinterpret_cast<const uint32_t*>(p.vbase + ((int64_t)b * p.Hkv + h) * kTileBytes + 16 * (D / 2) + (lane & 15) * 4);
            }
#pragma unroll
            for (int c = 0; c < NK; c++) kr[c] = make_uint4(0, 0, 0, 0);
            if (blk < 0) return;
            const int64_t off = ((int64_t)blk * p.Hkv + h) * kTileBytes;
            const uint4* src = reinterpret_cast<const uint4*>(p.kbase + off + (i & 15) * (D / 2));
#pragma unroll
            for (int c = 0; c < NK; c++) kr[c] = src[c];
            if ((tb + t) * kN + i < kv_end)  // rows past the end hold anything
                pk = *reinterpret_cast<const uint32_t*>(p.kbase + off + 16 * (D / 2) + (i & 15) * 4);
        };
        auto load_v = [&](int t) {
            const int32_t blk = block(t, vp >> 3);
#pragma unroll
            for (int c = 0; c < NK; c++) vr[c] = make_uint4(0, 0, 0, 0);
            if (blk < 0) return;
            const uint4* src = reinterpret_cast<const uint4*>(p.vbase + ((int64_t)blk * p.Hkv + h) * kTileBytes + (vp & 7) * D +
                                                              vh * (D / 2));
#pragma unroll
            for (int c = 0; c < NK; c++) vr[c] = src[c];
        };
        if (n_tiles > 0) load_k(0);
        for (int t = 0; t < n_tiles; t++) {
            const uint32_t ph = (uint32_t)(t & 1);
            if (t > 0 && !warp_wait(k_empty, ph ^ 1u, abort_flag)) break;
            // parameters of slot t & 1: the softmax of tile t - 2 is done with
            // them (S(t - 1), which k_empty tracks, was issued after it)
            TilePar& par_t = par[ph];
            const float2 ka = q4_unpack(pk);
            const int wi = warp & 3;
            uint32_t top_v = 0, low_v = 255;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float x = q4_unpack(pv[j]).x;
                const uint32_t e = x < INFINITY ? __float_as_uint(x) >> 23 : 0u;
                top_v = max(top_v, e);
                low_v = min(low_v, e);
            }
            E = max(E, (int)__reduce_max_sync(0xffffffffu, top_v));
            const float2 va = q4_unpack(wi == 0 ? pv[0] : wi == 1 ? pv[1] : wi == 2 ? pv[2] : pv[3]);
            const int ev = va.x < INFINITY ? (int)(__float_as_uint(fmaxf(va.x, fabsf(va.y) * (1.0f / (1 << kBelowM)))) >> 23) : 0;
            par_t.ev[i] = (float)min(max(ev - E, -kFar), kAbove);
            par_t.mk[i] = ka.y;
            par_t.mv[i] = va.y;
            // a V row that cannot be held (s = m = NaN) counts as zeros here: its NaN
            // reaches the rows that see it through m
            par_t.sv[i] = va.x < INFINITY ? va.x * pow2(127 + kVUp - E) : 0.0f;
            if (i == 0) par_t.E = E;
            // one power of two for the 32 tokens if their scales are within 2^20 of
            // the largest (8 of fp16's bits carry the code and s) and m / s is not so large
            // nor s so small that m qs / f could overflow; else one a token
            const bool held = ka.x < INFINITY;
            const uint32_t et = held ? __float_as_uint(ka.x) >> 23 : 0u, em = held ? __float_as_uint(fabsf(ka.y)) >> 23 : 0u;
            const uint32_t ek = __reduce_max_sync(0xffffffffu, et);
            const bool uneven = ek < 64 || __any_sync(0xffffffffu, held && (et + 20 < ek || em > ek + 40));
            const bool uneven_v = __any_sync(0xffffffffu, (int)low_v + kEven < E);
            const int kx = max((int)(uneven ? et : ek), kMinExpK);
            par_t.fk[i] = pow2(kx - 127 - kUp - kUnit);
            if (lane == 0) {
                par_t.f[wi] = pow2(kx - 127 - kUp);
                par_t.uneven[wi] = uneven || uneven_v;
            }
            const __half2 sk = __float2half2_rn(ka.x * pow2(127 + kUp - kx));
            uint8_t* kt = smem + C::kOffK;
#pragma unroll
            for (int c = 0; c < NK; c++) {
                const uint32_t w[4] = {kr[c].x, kr[c].y, kr[c].z, kr[c].w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t x[4];
                    q4_centred(w[j], x);
                    *reinterpret_cast<uint4*>(kt + chunk_at(i, 4 * c + j, kN)) =
                        make_uint4(mul_h2(x[0], sk), mul_h2(x[1], sk), mul_h2(x[2], sk), mul_h2(x[3], sk));
                }
            }
            load_v(t);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                bar_arrive(par_full + 8 * ph);
                bar_arrive(k_full);
            }
            if (t > 0 && !warp_wait(v_empty, ph ^ 1u, abort_flag)) break;
            uint8_t* vt = smem + C::kOffV;
            const int ta = 2 * vp;  // the pair's tokens: rows ta and ta + 1
#pragma unroll
            for (int c = 0; c < NK; c++) {
                const uint32_t w[4] = {vr[c].x, vr[c].y, vr[c].z, vr[c].w};
#pragma unroll
                for (int j = 0; j < 4; j += 2) {  // two quads: eight dims of both tokens
                    uint32_t x[4], y[4];
                    q4_centred(w[j], x);
                    q4_centred(w[j + 1], y);
                    const int chunk = vh * (D / 16) + 2 * c + j / 2;
                    *reinterpret_cast<uint4*>(vt + chunk_at(ta, chunk, kN)) =
                        make_uint4(prmt(x[0], x[1], 0x5410), prmt(x[2], x[3], 0x5410), prmt(y[0], y[1], 0x5410),
                                   prmt(y[2], y[3], 0x5410));
                    *reinterpret_cast<uint4*>(vt + chunk_at(ta + 1, chunk, kN)) =
                        make_uint4(prmt(x[0], x[1], 0x7632), prmt(x[2], x[3], 0x7632), prmt(y[0], y[1], 0x7632),
                                   prmt(y[2], y[3], 0x7632));
                }
            }
            if (t + 1 < n_tiles) load_k(t + 1);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(v_full);
        }
    } else {
        regs_inc<kRegsSoftmax>();
        // ================= softmax warps =================
        // Softmax warp w: tile X = w / 8, rows 32 (w % 4) .. + 31 of it (a row a
        // lane, as TMEM has it), tokens 64 half .. + 63 of every tile, half =
        // (w / 4) % 2.  Row 128 X + r is query X QT + r / G, head r % G.  The
        // two warps of 32 rows bring 16 of q's rows each, all in flight, each
        // scaled by the power of two that puts its largest |q| in [2^14, 2^15).
        const int X = warp >> 3, half = (warp >> 2) & 1, r = 32 * (warp & 3) + lane, qi = X * QT + r / G;
        const uint32_t pair = pairs + 8 * (4 * X + (warp & 3));  // of the two warps
        float* x_mine = xch + half * 2 * kM + X * kM + r;  // slot s: + s * 4 kM; the other half's:
        const int x_other = (half ? -2 : 2) * kM;
        const bool valid = r < QT * G && q0 + qi < sm.q_len;
        {
            const int mine = valid ? (sm.q_start + q0 + qi) * p.Hq + h * G + r % G : -1;
            uint8_t* hi_at = smem + C::kOffQ + 2 * X * C::kQBytes;
            // D / 4 lanes a row, four dims a lane; x[j]: row RW j + lane / LR of the 16
            constexpr int LR = D / 4, RW = 32 / LR, NJ = 16 / RW;
            const int d0 = 4 * (lane % LR);
            const bool vec = ((uintptr_t)p.q & 15) == 0;
            float4 x[NJ];
            float mx[NJ], sum[NJ];
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const int at = __shfl_sync(0xffffffffu, mine, 16 * half + RW * j + lane / LR);
                const float* src = p.q + (int64_t)at * D + d0;
                x[j] = at < 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
                     : vec    ? *reinterpret_cast<const float4*>(src)
                              : make_float4(src[0], src[1], src[2], src[3]);
            }
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                x[j] = make_float4(x[j].x * p.scale_log2, x[j].y * p.scale_log2, x[j].z * p.scale_log2, x[j].w * p.scale_log2);
                mx[j] = fmaxf(fmaxf(fabsf(x[j].x), fabsf(x[j].y)), fmaxf(fabsf(x[j].z), fabsf(x[j].w)));
                sum[j] = (x[j].x + x[j].y) + (x[j].z + x[j].w);
            }
            // all rows' maxima and sums at once: halve the rows a lane holds and the lanes that hold a row
#pragma unroll
            for (int n = NJ / 2; n > 0; n >>= 1) {
                const bool up = lane & (2 * n);
#pragma unroll
                for (int j = 0; j < n; j++) {
                    const float m_keep = up ? mx[j + n] : mx[j], m_give = up ? mx[j] : mx[j + n];
                    const float s_keep = up ? sum[j + n] : sum[j], s_give = up ? sum[j] : sum[j + n];
                    mx[j] = fmaxf(m_keep, __shfl_xor_sync(0xffffffffu, m_give, 2 * n));
                    sum[j] = s_keep + __shfl_xor_sync(0xffffffffu, s_give, 2 * n);
                }
            }
            mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], 1));
            sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 1);
            // lanes 2 j and 2 j + 1 (of a row's lanes) hold x[j]'s row
            const int qe = min(max((int)(__float_as_uint(mx[0]) >> 23), 40), 240);
            const float scale = __uint_as_float((uint32_t)(268 - qe) << 23);
            if (!(lane & 1)) {  // for both of the row's threads
                float* at = xch + 2 * 4 * kM + X * kM + 32 * (warp & 3) + 16 * half + RW * (lane % LR / 2) + lane / LR;
                at[0] = at[2 * kM] = __uint_as_float((uint32_t)(qe - 14) << 23);  // 1 / scale
                at[4 * kM] = at[6 * kM] = sum[0] * scale;
            }
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const float sc = __shfl_sync(0xffffffffu, scale, (lane & ~(LR - 1)) + 2 * j);
                // K's order of dims: an even lane takes 0 4 1 5 of eight, the next one 2 6 3 7
                const bool odd = lane & 1;
                const float g0 = __shfl_xor_sync(0xffffffffu, odd ? x[j].x : x[j].z, 1);
                const float g1 = __shfl_xor_sync(0xffffffffu, odd ? x[j].y : x[j].w, 1);
                uint2 hi, lo;
                split_h2((odd ? g0 : x[j].x) * sc, (odd ? x[j].z : g0) * sc, hi.x, lo.x);
                split_h2((odd ? g1 : x[j].y) * sc, (odd ? x[j].w : g1) * sc, hi.y, lo.y);
                const uint32_t at = chunk_at(32 * (warp & 3) + 16 * half + RW * j + lane / LR, lane % LR / 2, kM) + 8 * (lane & 1);
                *reinterpret_cast<uint2*>(hi_at + at) = hi;
                *reinterpret_cast<uint2*>(hi_at + C::kQBytes + at) = lo;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                bar_arrive(q_full);
                bar_arrive(pair);
            }
        }
        bool ok = warp_wait(pair, 0, abort_flag);
        const int row_limit = valid ? prefix + q0 + qi : kv_end - 1;  // last visible token
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t tS = tmem + lanes + X * 128 + 64 * half, tO = tmem + lanes + kColO + X * 128 + half * (D / 2);
        RowState st{-INFINITY, make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f), kMinExp, x_mine[2 * 4 * kM], x_mine[3 * 4 * kM]};
        const bool active = X == 0 || two_tiles;
        float4* aside = reinterpret_cast<float4*>(p.aside) + ((int64_t)slot * (D / 4) + half * (D / 8)) * (2 * kM) + X * kM + r;  // columns 4 c ..: + 256 c
        float2* ref = reinterpret_cast<float2*>(smem + C::kOffRef) + tid;  // what this thread's set-aside sums refer to
        for (int t = 0; active && ok && t < n_tiles; t++) {
            const uint32_t ph = (uint32_t)(t & 1);
            const bool fresh = t % chain == 0;
            if (fresh && t > 0 && (ok = warp_wait(pv_done + 8 * X, ph ^ 1u, abort_flag))) {
                tc_fence_after();
                // The tensor cores cut their sums instead of rounding them, so a
                // long chain drifts: set the sums aside with rounded additions
                // (in L2, nothing waited for) and start anew.  S_X(t) runs meanwhile.
                const float c = t > chain ? rebase(ref->x, __float_as_int(ref->y), st.m, st.E) : 1.0f;
                const bool add = t > chain && __all_sync(0xffffffffu, c == 1.0f);
                if (t > chain && !add) __threadfence();
#pragma unroll 1
                for (int d = 0; d < D / 8; d += 4) {
                    float ov[16];
                    tmem_ld16(tO + 4 * d, ov);
                    tmem_ld_wait16(ov);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float4* at = aside + (d + i) * (2 * kM);
                        float4 o = make_float4(ov[4 * i], ov[4 * i + 1], ov[4 * i + 2], ov[4 * i + 3]);
                        if (add) {
                            asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(o.x), "f"(o.y),
                                         "f"(o.z), "f"(o.w)
                                         : "memory");
                        } else {
                            if (t > chain) {
                                const float4 old = __ldcg(at);
                                o = make_float4(fmaf(old.x, c, o.x), fmaf(old.y, c, o.y), fmaf(old.z, c, o.z), fmaf(old.w, c, o.w));
                            }
                            __stcg(at, o);
                        }
                    }
                }
                *ref = make_float2(st.m, __int_as_float(st.E));
            }
            // S_X(t) done also means PV_X(t - 1) done: O_X and P_X are free
            if (!ok || !warp_wait(par_full + 8 * ph, (uint32_t)((t >> 1) & 1), abort_flag) || !warp_wait(s_full + 8 * X, ph, abort_flag)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const int base = (tb + t) * kN;
            // (the pair's phase 0 was q's)
            if (base + kN - 1 > prefix + q0 || *reinterpret_cast<const uint32_t*>(par[ph].uneven))  // some row of the chunk does not see all of it
                ok = softmax_tile<true, D>(tS, tO, par[ph], 64 * half, row_limit - base, st, fresh, x_mine + ph * 4 * kM, x_other, pair,
                                           ph ^ 1u, p_full + 8 * X, abort_flag, lane);
            else
                ok = softmax_tile<false, D>(tS, tO, par[ph], 64 * half, 0, st, fresh, x_mine + ph * 4 * kM, x_other, pair, ph ^ 1u,
                                            p_full + 8 * X, abort_flag, lane);
        }
        int tid_;  // (where the row lies is worked out anew, not kept over the loop)
        asm volatile("mov.u32 %0, %%tid.x;" : "=r"(tid_));
        const int X_ = tid_ >> 8, half_ = (tid_ >> 7) & 1, r_ = tid_ & 127, qi_ = X_ * QT + r_ / G;
        const bool valid_ = r_ < QT * G && q0 + qi_ < sm.q_len;
        const int at = (sm.q_start + q0 + qi_) * p.Hq + h * G + r_ % G;
        const bool split = p.n_split > 1, had = n_tiles > chain;
        const float c = had ? rebase(ref->x, __float_as_int(ref->y), st.m, st.E) : 1.0f;
        float4 old[8];  // the sums set aside
        if (had) {
            __threadfence();
#pragma unroll
            for (int i = 0; i < 8; i++) old[i] = __ldcg(aside + i * (2 * kM));
        }
        if (active && n_tiles > 0 && ok && warp_wait(pv_done + 8 * X_, (uint32_t)((n_tiles - 1) & 1), abort_flag)) {
            tc_fence_after();
            // the row's sums from its two threads
            const float l_mine = st.l.x + st.l.y, z_mine = st.z.x + st.z.y;
            x_mine[2 * 4 * kM] = l_mine;
            x_mine[3 * 4 * kM] = z_mine;
            __syncwarp();
            if (lane == 0) bar_arrive(pair);
            warp_wait(pair, (uint32_t)((n_tiles + 1) & 1), abort_flag);
            const float l = l_mine + x_mine[2 * 4 * kM + x_other], z = z_mine + x_mine[3 * 4 * kM + x_other];
            const float back = pow2(st.E - 127 - kVUp);
            // (a split's l of more than 2^40 goes into its reference: the join takes that for the scores' maximum)
            const int up = l > 1.0995116e12f && l < INFINITY ? (int)(__float_as_uint(l) >> 23) - 127 : 0;
            const float inv = split ? pow2(-up) : 1.0f / l;
            if (split && valid_ && half_ == 0) {
                p.part_ml[((int64_t)blockIdx.y * p.n_rows * p.Hq + at) * 2] = st.m + (float)up;
                p.part_ml[((int64_t)blockIdx.y * p.n_rows * p.Hq + at) * 2 + 1] = l * pow2(-up);
            }
            // Half rows go through this warp's part of q's tiles (every product
            // that read q is done), so that a row's columns are written together.
            float4* stage = reinterpret_cast<float4*>(smem + C::kOffQ) + (tid_ >> 5) * (32 * D / 8);
            constexpr int LR = D / 8;  // lanes a half row
#pragma unroll 1
            for (int d = 0; d < D / 8; d += 8) {
                float ov[32];
                if (had && d)
#pragma unroll
                    for (int i = 0; i < 8; i++) old[i] = __ldcg(aside + (d + i) * (2 * kM));
                tmem_ld16(tO + 4 * d, ov);
                tmem_ld16(tO + 4 * d + 16, ov + 16);
                tmem_ld_wait16(ov);
                tmem_ld_wait16(ov + 16);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float4 o = make_float4(ov[4 * i], ov[4 * i + 1], ov[4 * i + 2], ov[4 * i + 3]);
                    if (had)
                        o = make_float4(fmaf(old[i].x, c, o.x), fmaf(old[i].y, c, o.y), fmaf(old[i].z, c, o.z), fmaf(old[i].w, c, o.w));
                    stage[lane * LR + ((d + i) ^ (lane & 7))] = make_float4(fmaf(o.x, back, z) * inv, fmaf(o.y, back, z) * inv,
                                                                            fmaf(o.z, back, z) * inv, fmaf(o.w, back, z) * inv);
                }
            }
            __syncwarp();
            float* dst = (split ? p.part_o + (int64_t)blockIdx.y * p.n_rows * p.Hq * D : p.out) + half_ * (D / 2) + 4 * (lane % LR);
            const bool vec = ((uintptr_t)dst & 15) == 0;
            const int row_at = valid_ ? at : -1;
#pragma unroll 4
            for (int j = 0; j < 32; j += 32 / LR) {
                const int row = j + lane / LR, to = __shfl_sync(0xffffffffu, row_at, row);
                const float4 o = stage[row * LR + ((lane % LR) ^ (row & 7))];
                if (to < 0) continue;
                float* d = dst + (int64_t)to * D;
                if (vec)
                    *reinterpret_cast<float4*>(d) = o;
                else
                    d[0] = o.x, d[1] = o.y, d[2] = o.z, d[3] = o.w;
            }
        }
        if (active && n_tiles == 0 && valid_) {  // an empty share of a split
            const int64_t row = (int64_t)blockIdx.y * p.n_rows * p.Hq + at;
            for (int d = 0; d < D / 2; d++) p.part_o[row * D + half_ * (D / 2) + d] = 0.0f;
            p.part_ml[row * 2] = -INFINITY;
            p.part_ml[row * 2 + 1] = 0.0f;
        }
    }

    // ---- tear-down: every path frees TMEM ----
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && flag_get(abort_flag)) atomicOr(p.err, kErrTimeout);
    if (tid == 0 && slot >= 0) {  // every thread is done with the slot
        __threadfence();
        atomicExch(&p.aside_lock[slot], 0);
    }
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

// Joins the n_split partial rows of a split chunk: a warp a (row, head).
__global__ void __launch_bounds__(256) join_q4_kernel(const PrefillQ4Params p, int D) {
    pdl_wait_trigger();
    const int64_t rows = p.n_rows * p.Hq, row = blockIdx.x * (int64_t)8 + threadIdx.x / 32;
    const int lane = threadIdx.x & 31;
    if (row >= rows) return;
    float M = -INFINITY;
    for (int s = 0; s < p.n_split; s++) M = fmaxf(M, p.part_ml[(s * rows + row) * 2]);
    float L = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.n_split; s++) {
        const float ms = p.part_ml[(s * rows + row) * 2], f = ms == -INFINITY ? 0.0f : ex2(ms - M);
        L = fmaf(p.part_ml[(s * rows + row) * 2 + 1], f, L);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (lane + 32 * i < D) o[i] = fmaf(p.part_o[(s * rows + row) * D + lane + 32 * i], f, o[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (lane + 32 * i < D) p.out[row * D + lane + 32 * i] = o[i] / L;
}

bool prefill_q4_supported(int D, int G, int block_size) {
    return (D == 64 || D == 128) && block_size == 16 && G >= 1 && G <= kM;
}

template <int D>
static int launch_prefill(const PrefillQ4Params& p, cudaStream_t stream) {
    static std::atomic<uint64_t> attr_set{0};  // per device
    int st = once_per_device(attr_set, [] {
        S1KV_CUDA(cudaFuncSetAttribute(prefill_q4_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem));
        return S1KV_OK;
    });
    if (st) return st;
    if ((int64_t)p.n_seqs * p.max_chunks * p.Hkv > INT32_MAX) return set_error(S1KV_EINVAL, "attention: too many query chunks");
    const dim3 grid((unsigned)(p.n_seqs * p.max_chunks * p.Hkv), (unsigned)p.n_split);
    S1KV_CUDA(launch_pdl(prefill_q4_kernel<D>, grid, dim3(kThreads), Cfg<D>::kSmem, stream, p));
    g_launches++;
    if (p.n_split > 1) {
        const int64_t rows = p.n_rows * p.Hq;
        S1KV_CUDA(launch_pdl(join_q4_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, stream, p, D));
        g_launches++;
    }
    return S1KV_OK;
}

// `max_kv`: the longest context of the batch.
int launch_prefill_q4(s1kv_batch* b, int32_t layer, const float* q, float* out, int32_t Hq, float scale_log2, int32_t max_kv,
                      cudaStream_t stream) {
    s1kv_pool* pool = b->pool;
    PrefillQ4Params p{};
    p.q = q;
    p.out = out;
    p.table = pool->d_table;
    p.seqs = b->d_pseqs;
    p.kbase = pool->k + (size_t)layer * pool->layer_bytes;
    p.vbase = pool->v + (size_t)layer * pool->layer_bytes;
    p.n_rows = b->n_rows;
    p.n_seqs = b->n_seqs;
    p.max_bps = pool->max_bps;
    p.max_blocks = (int32_t)pool->desc.max_blocks;
    p.Hq = Hq;
    p.Hkv = pool->desc.num_kv_heads;
    p.G = Hq / p.Hkv;
    p.QT = kM / p.G;
    p.max_chunks = (b->max_qlen + 2 * p.QT - 1) / (2 * p.QT);
    p.scale_log2 = scale_log2;
    p.err = pool->d_err;
    if (b->n_seqs == 0 || p.max_chunks == 0) return S1KV_OK;
    // Fewer chunks than SMs: split their tiles, at least 4 a CTA, so that all
    // SMs have work (a chunk's K/V reading and products run on one SM else).
    const int D = pool->desc.head_dim;
    const int64_t ctas = std::max<int64_t>(1, (b->n_rows + 2 * p.QT - 1) / (2 * p.QT)) * p.Hkv;
    const int64_t tiles = (max_kv + kN - 1) / kN;
    p.n_split = (int32_t)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(148 / ctas, tiles / 4), 64));
    // slots for the sums that long chains set aside, one an SM
    int sms = 0;
    S1KV_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, pool->device));
    const size_t slots = (size_t)sms * D * 2 * kM * sizeof(float);
    if (!pool->aside.p) {
        const int st = pool->aside.ensure(slots + sms * sizeof(int32_t));
        if (st) return st;
        S1KV_CUDA(cudaMemset((char*)pool->aside.p + slots, 0, sms * sizeof(int32_t)));
        S1KV_CUDA(cudaDeviceSynchronize());
    }
    p.aside = (float*)pool->aside.p;
    p.aside_lock = (int32_t*)((char*)pool->aside.p + slots);
    p.n_aside = sms;
    if (p.n_split > 1) {
        const size_t rows = (size_t)p.n_split * p.n_rows * Hq;
        const int st = pool->scratch.ensure(rows * (D + 2) * sizeof(float));
        if (st) return st;
        p.part_o = (float*)pool->scratch.p;
        p.part_ml = p.part_o + rows * D;
    }
    return D == 128 ? launch_prefill<128>(p, stream) : launch_prefill<64>(p, stream);
}

}  // namespace s1kv

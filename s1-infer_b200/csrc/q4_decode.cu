// q4_decode.cu -- paged split-K GQA attention over a 4-bit cache (format:
// q4.cuh) on warp-level tensor-core instructions (mma.sync m16n8k16, fp16 x
// fp16 -> fp32).
//
// With c = u - 8 the centred codes, k = m_k + s_k c and v = m_v + s_v c:
//   score_t = s_k (q . c_t) + m_k sum(q)
//   out     = sum_t (p_t s_v) c_t + sum_t p_t m_v,   over sum_t p_t
// so the products run over small integers, exact in fp16, and the scales
// act on scores.  The codes are centred before the products: unsigned sums
// would cancel against 8 sum(q) and 8 sum(p s_v).  (K's raw codes as fp16
// subnormals, u 2^-24, need no arithmetic, but contexts of a few tokens were
// off by up to 1.2e-6, now 2e-7, for 4% more time.)
//
// Precision: q (times log2(e) / sqrt(D)) and p s_v are each split into two
// fp16 parts, 22 bits, of values scaled by a power of two that puts the
// largest of a head's q, or of its weights p s_v so far, at 2^15: scores and
// outputs carry fp32-level error, whatever other heads or V rows that hardly
// weigh hold (V rows down to 2^kFar below the largest).
//
// Layout: one 16-token tile of a KV head is 16 D / 2 + 64 bytes of K and as
// many of V, contiguous, and the storage order is the fragments' own: a lane's
// codes of the whole tile are two 16-byte reads of K and two of V (D = 128; V's
// meet four to a bank).  Each warp brings pairs of tiles, two bulk copies a
// tile, into a ring of its own in shared memory, kNS pairs ahead, and takes a
// pair at a time: what a step costs besides the codes (waits, the maximum's
// vote) is shared by 32 tokens.
//   K: lane (g, t) = (L / 4, L % 4) takes dims 32 t .. 32 t + 31 of tokens g
//      and g + 8.  The sum over dims does not care for their order, so q's
//      fragments simply follow K's: nibbles n and n + 4 of a word are the
//      halves of one fp16x2 register.
//   V: lane (g, t) takes dims 16 g .. 16 g + 15 of token pairs t and t + 4;
//      a word holds four dims of the two adjacent tokens.
//   (w & 0x000f000f) | 0x64006400 is 1024 + u in both halves, and one fp16x2
//   operation makes it u - 8 (q4_centred).
// Query heads fill the N = 8 side: up to four heads take one mma with both
// parts of q (or p) side by side in its columns, five to eight take two.
//
// Work: as the other decode kernels, a CTA takes one split-K item (row,
// token range) of one KV head, its 4 warps the range's tiles in turn; warps
// merge through shared memory, splits through combine.cuh.
//
// Bound: nothing is full (46% of the issue slots, ALU 45% with widening, memory
// 57% of the copy rate, 16 warps an SM that wait for their own chain of loads,
// products and votes): 64 rows of 8192 tokens, 32 heads on 8 of 128, 138 us, 4.1
// TB/s (bf16 pools: 314 us); 2 of 131072, 64 heads, 98 us, 2.9 TB/s.
#include <cmath>

#include "combine.cuh"
#include "q4.cuh"

namespace s1kv {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kNW = 4;
constexpr int kTile = 16;
constexpr int kMaxG = 128;             // query heads per KV head the merge's scratch covers (least: 36 G of 6912 floats)
constexpr float kRescaleAt = 8.0f;     // log2 units
constexpr int kMinExp = 8;             // least exponent (biased) V's rows are taken relative to
// A V row counts by the exponent of max(s, |m| / 2^kBelowM) where rows are uneven,
// some s kEven powers of two below the largest or more; kFar below it at least.
constexpr int kBelowM = 8, kEven = 6, kFar = 80, kAbove = 60;
constexpr uint32_t kSpin = 1u << 22;
constexpr int kNS = 3;                 // stages a warp, of two tiles each
// CTAs an SM, within 64K registers and 227 KB, as far as nothing spills in the
// loop (a fifth CTA for D = 128 with two stages a warp: 6% slower on 64 rows of
// up to 8192 tokens; a sixth for D = 64: 4% on 200 rows of 1024).
constexpr int ctas_per_sm(int D) { return D == 64 ? 5 : 4; }

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transpose of an 8x8 b16 matrix held as the warp's m8n8 fragment.
__device__ __forceinline__ uint32_t movt(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// (a, b) -> fp16 pair and the fp16 pair of what it leaves out.
__device__ __forceinline__ void split_h2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack_h2(a - f.x, b - f.y);
}
__device__ __forceinline__ uint32_t su32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t b, uint32_t n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(b), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_wait(uint32_t b, uint32_t phase) {
    for (uint32_t i = 0; i < kSpin; i++) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(b), "r"(phase)
            : "memory");
        if (ok) return true;
    }
    return false;
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t b) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(b)
                 : "memory");
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 <= e <= 127
// Biased exponent of x >= 0; 0 of a NaN.
__device__ __forceinline__ int exponent_of(float x) { return x < INFINITY ? (int)(__float_as_uint(x) >> 23) : 0; }
template <int NWD>
__device__ __forceinline__ void load_words(const char* at, uint32_t (&w)[NWD]) {
    if constexpr (NWD == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(at);
        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(at);
        w[0] = x.x, w[1] = x.y;
    }
}

}  // namespace

// D = 32 NWD; heads of one pass (NT = 1: up to 4, NT = 2: up to 8).
template <int D, int NT>
__global__ void __launch_bounds__(kNW * 32, ctas_per_sm(D)) decode_q4_kernel(const __grid_constant__ AttnParams p, int G) {
    constexpr int NWD = D / 32, KS = D / 16, GP = 4 * NT;
    constexpr int kTileBytes = kTile * (D / 2 + 4), kParams = kTile * (D / 2), kStage = 4 * kTileBytes;
    constexpr int kRing = kNW * kNS * kStage;
    static_assert(kRing >= kNW * GP * (D + 2) * 4, "the warps' partial rows lie over the rings");
    extern __shared__ __align__(128) char smem[];
    float* mo = reinterpret_cast<float*>(smem);  // [kNW][GP][D], over the rings once they are done
    float* mml = mo + kNW * GP * D;              // [kNW][GP][2]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const char* ring = smem + warp * kNS * kStage;
    const uint32_t bars = su32(smem) + kRing + warp * kNS * 8;
    int* flag = reinterpret_cast<int*>(smem + kRing + kNW * kNS * 8);
    const int gq = lane >> 2, tq = lane & 3;
    const int h = blockIdx.x % p.Hkv;  // (an item's heads together: the longest items of all heads come first)
    const WorkItem item = p.items[blockIdx.x / p.Hkv];
    const int tok0 = item.split * p.split_tokens;
    const int tok1 = min(tok0 + p.split_tokens, item.kv_len);
    const int n_tiles = (tok1 - tok0 + kTile - 1) / kTile;
    const int n_pairs = (n_tiles + 1) / 2;  // this warp: pairs warp, warp + kNW ..
    const int my_pairs = n_pairs > warp ? (n_pairs - warp + kNW - 1) / kNW : 0;
    const int32_t* tab = p.table + (int64_t)item.table_row * p.max_bps + (tok0 >> 4);

    int32_t my_blk = 0;
    auto fetch_ids = [&](int k) {  // block ids of this warp's pairs k .. k + 15, two a pair (-1: no second tile)
        const int tile = 2 * (warp + (k + (lane >> 1)) * kNW) + (lane & 1);
        my_blk = -1;
        if (tile < n_tiles) {
            my_blk = tab[tile];
            if ((uint32_t)my_blk >= (uint32_t)p.max_blocks) {
                atomicOr(p.err, kErrBounds);
                my_blk = 0;
            }
        }
    };
    auto issue = [&](int k, int it) {  // pair k of this warp into the stage of copy `it`
        // lanes 0 and 1 bring the pair's first and second tile
        const int32_t blk = __shfl_sync(kFull, my_blk, 2 * (k & 15) + (lane & 1));
        const bool both = __shfl_sync(kFull, blk, 1) >= 0;
        const uint32_t b = bars + (it % kNS) * 8;
        if (lane == 0) bar_expect(b, both ? kStage : kStage / 2);
        __syncwarp();
        if (lane < 2 && blk >= 0) {
            const int64_t off = ((int64_t)blk * p.Hkv + h) * kTileBytes;
            const uint32_t dst = su32(ring) + (it % kNS) * kStage + lane * 2 * kTileBytes;
            bulk_copy(dst, reinterpret_cast<const char*>(p.kbase) + off, kTileBytes, b);
            bulk_copy(dst + kTileBytes, reinterpret_cast<const char*>(p.vbase) + off, kTileBytes, b);
        }
    };
    if (lane == 0) {
        for (int i = 0; i < kNS; i++) bar_init(bars + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    fetch_ids(0);
    // Tiles that lie below the tokens this batch appends are requested before
    // the wait for the previous kernel: nothing that may still run writes them
    // (split_k_attention states why).
    const int n_first = min(kNS, my_pairs);
    int pre = 0;
    if (p.prewait)
        while (pre < n_first && tok0 + (warp + pre * kNW + 1) * 2 * kTile <= item.kv_len - p.prewait_margin) pre++;
    for (int k = 0; k < pre; k++) issue(k, k);
    pdl_wait();
    const RowMeta rm = p.rows[item.row];
    bool failed = false;
    int it0 = 0;  // copies consumed by earlier passes

    for (int g0 = 0; g0 < G; g0 += GP) {
        const int pairs = failed ? 0 : my_pairs;  // (the CTA's warps stay together whatever happens)
        if (g0 > 0) fetch_ids(0);
        for (int k = g0 > 0 ? 0 : pre; k < min(n_first, pairs); k++) issue(k, it0 + k);
        // q's fragments: column c of the N side is head g0 + c (NT = 2), or
        // head g0 + c % 4 with the high part in columns 0-3 and the low part
        // in 4-7 (NT = 1).  This lane's column and dims 8 NWD tq .. are one
        // contiguous piece of a row of q.
        const int head = NT == 1 ? gq & 3 : gq;
        const bool live = g0 + head < G;
        const float* qrow = p.q + ((int64_t)item.row * p.Hq + h * G + g0 + (live ? head : 0)) * D + 8 * NWD * tq;
        float x[8 * NWD];
        float amax = 0.0f, qsum = 0.0f;
        const bool vec = ((uintptr_t)p.q & 15) == 0;
#pragma unroll
        for (int d = 0; d < 8 * NWD; d += 4) {
            const float4 f = vec ? *reinterpret_cast<const float4*>(qrow + d) : make_float4(qrow[d], qrow[d + 1], qrow[d + 2], qrow[d + 3]);
            x[d] = f.x, x[d + 1] = f.y, x[d + 2] = f.z, x[d + 3] = f.w;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[d + e] = live ? x[d + e] * p.scale_log2 : 0.0f;
                amax = fmaxf(amax, fabsf(x[d + e]));
                qsum += x[d + e];
            }
        }
        qsum += __shfl_xor_sync(kFull, qsum, 1);
        qsum += __shfl_xor_sync(kFull, qsum, 2);
        amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 2));
        // power of two that puts the head's largest |q| in [2^14, 2^15)
        const int qe = min(max((int)(__float_as_uint(amax) >> 23), 40), 240);
        const float qscale = __uint_as_float((uint32_t)(127 + 14 + 127 - qe) << 23);
        const float unscale = __uint_as_float((uint32_t)(qe - 14) << 23);  // 1 / qscale
        uint32_t qf[NT][KS][2];
#pragma unroll
        for (int wi = 0; wi < NWD; wi++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const int d = 8 * wi + 2 * j + b;
                    uint32_t hi, lo;
                    split_h2(x[d] * qscale, x[d + 4] * qscale, hi, lo);
                    if (NT == 1) {
                        qf[0][2 * wi + j][b] = gq < 4 ? hi : lo;
                    } else {
                        qf[0][2 * wi + j][b] = hi;
                        qf[NT - 1][2 * wi + j][b] = lo;
                    }
                }
        // scale and sum(q) of the two heads whose scores this lane holds (columns 2 tq, 2 tq + 1);
        // NT = 2 is short of registers and reads them every step
        const float4* heads = reinterpret_cast<const float4*>(smem + kRing + kNW * kNS * 8 + 16) + 4 * warp;
        float4 hq;
        if (NT == 1) {
            hq = make_float4(__shfl_sync(kFull, unscale, 8 * tq & 31), __shfl_sync(kFull, qsum, 8 * tq & 31),
                             __shfl_sync(kFull, unscale, 8 * tq + 4 & 31), __shfl_sync(kFull, qsum, 8 * tq + 4 & 31));
        } else {
            if (tq == 0) reinterpret_cast<float2*>(const_cast<float4*>(heads))[gq] = make_float2(unscale, qsum);
            __syncwarp();
        }

        float o[KS][4];
#pragma unroll
        for (int mb = 0; mb < KS; mb++) o[mb][0] = o[mb][1] = o[mb][2] = o[mb][3] = 0.0f;
        // heads 2 tq, 2 tq + 1: reference max (log2 units, the same in the 8
        // lanes of a head), this lane's share of sum(p) and sum(p m_v)
        float m0 = -INFINITY, m1 = -INFINITY;
        float2 l2 = make_float2(0.f, 0.f), z2 = make_float2(0.f, 0.f);
        const float2 low = NT == 1 ? (tq < 2 ? make_float2(0.f, 0.f) : make_float2(-1.f, -1.f)) : make_float2(-1.f, -1.f);
        // V's scales are taken relative to 2^(E - 127), E the largest exponent of an s_v so far: vmul =
        // 2^(133 - E) puts the largest in [2^6, 2^7)
        float vmul = __uint_as_float((uint32_t)(260 - kMinExp) << 23);
        auto exponent_v = [&] { return 260 - (int)(__float_as_uint(vmul) >> 23); };  // E
        int k = 0;
        for (; k < pairs; k++) {
            const int it = it0 + k, stage = it % kNS;
            // Each lane polls for itself; a timeout goes into the vote below, so that
            // the warp leaves as one.
            const bool late = !bar_wait(bars + 8 * stage, (uint32_t)((it / kNS) & 1));
            const char* kt = ring + stage * kStage;
            const int rest = tok1 - (tok0 + (warp + k * kNW) * 2 * kTile);  // tokens of the pair: 32, fewer at the end

            if (NT == 2) hq = heads[tq];
            const float2 un2 = make_float2(hq.x, hq.z), qs2 = make_float2(hq.y, hq.w);
            // ---- scores: M = the 16 tokens of a tile, N = the 8 columns ----
            float2 x[2][2], va[2], vb[2];  // [tile][token gq, gq + 8] of heads (2 tq, 2 tq + 1); (s_v, m_v) of the tokens
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const char* at = kt + u * 2 * kTileBytes;
                uint32_t k0[NWD], k1[NWD];
                load_words<NWD>(at + gq * (D / 2) + tq * (4 * NWD), k0);
                load_words<NWD>(at + (gq + 8) * (D / 2) + tq * (4 * NWD), k1);
                const uint32_t* kp = reinterpret_cast<const uint32_t*>(at + kParams) + gq;
                const float2 ka = q4_unpack(kp[0]), kb = q4_unpack(kp[8]);
                float sa[4] = {0.f, 0.f, 0.f, 0.f}, sb[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int wi = 0; wi < NWD; wi++) {
                    uint32_t c0[4], c1[4];
                    q4_centred(k0[wi], c0);
                    q4_centred(k1[wi], c1);
#pragma unroll
                    for (int j = 0; j < 2; j++) {  // (small parts first: the sums are cut, not rounded)
                        float(&sum)[4] = j ? sb : sa;
                        const int ks = 2 * wi + j;
                        if (NT == 2) mma16816(sum, c0[2 * j], c1[2 * j], c0[2 * j + 1], c1[2 * j + 1], qf[NT - 1][ks][0], qf[NT - 1][ks][1]);
                        mma16816(sum, c0[2 * j], c1[2 * j], c0[2 * j + 1], c1[2 * j + 1], qf[0][ks][0], qf[0][ks][1]);
                    }
                }
                float2 s0 = __fadd2_rn(make_float2(sa[0], sa[1]), make_float2(sb[0], sb[1]));
                float2 s1 = __fadd2_rn(make_float2(sa[2], sa[3]), make_float2(sb[2], sb[3]));
                if (NT == 1) {  // high + low part of q
                    s0 = __fadd2_rn(s0, make_float2(__shfl_xor_sync(kFull, s0.x, 2), __shfl_xor_sync(kFull, s0.y, 2)));
                    s1 = __fadd2_rn(s1, make_float2(__shfl_xor_sync(kFull, s1.x, 2), __shfl_xor_sync(kFull, s1.y, 2)));
                }
                // s (q . c) + m sum(q)
                x[u][0] = __ffma2_rn(make_float2(ka.x, ka.x), __fmul2_rn(s0, un2), __fmul2_rn(make_float2(ka.y, ka.y), qs2));
                x[u][1] = __ffma2_rn(make_float2(kb.x, kb.x), __fmul2_rn(s1, un2), __fmul2_rn(make_float2(kb.y, kb.y), qs2));
            }
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint32_t* vp = reinterpret_cast<const uint32_t*>(kt + (2 * u + 1) * kTileBytes + kParams) + gq;
                va[u] = q4_unpack(vp[0]);
                vb[u] = q4_unpack(vp[8]);
            }
            if (rest < 2 * kTile) {  // rows past the end hold anything, NaN included: score -inf, s_v even with E, m_v 0
                const float2 past = make_float2(__uint_as_float((260u << 23) - __float_as_uint(vmul)), 0.0f);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    if (16 * u + gq >= rest) x[u][0] = make_float2(-INFINITY, -INFINITY), va[u] = past;
                    if (16 * u + gq + 8 >= rest) x[u][1] = make_float2(-INFINITY, -INFINITY), vb[u] = past;
                }
            }
            // the reference max of a head moves only when a score outgrows it
            // by 2^8, and E only when a V row outgrows it: both are rare, and so
            // are V rows of 2^kEven below E
            float mx0 = fmaxf(fmaxf(x[0][0].x, x[0][1].x), fmaxf(x[1][0].x, x[1][1].x));
            float mx1 = fmaxf(fmaxf(x[0][0].y, x[0][1].y), fmaxf(x[1][0].y, x[1][1].y));
            const float most = fmaxf(fmaxf(va[0].x, vb[0].x), fmaxf(va[1].x, vb[1].x));
            const float least = fminf(fminf(va[0].x, vb[0].x), fminf(va[1].x, vb[1].x));
            if (__any_sync(kFull, mx0 > m0 + kRescaleAt || mx1 > m1 + kRescaleAt || most * vmul >= 128.0f || least * vmul < 64.0f / (1 << kEven) ||
                                  late)) {
                if (__any_sync(kFull, late)) break;
                // The reference is one for the weights p s_v, which must fit fp16:
                // scores plus V's exponents relative to E (down to -kFar).  A V row
                // that is hardly weighed then takes no bits from the others,
                // however large it is; p may pass 2^8 by as much as V's exponents
                // lie below E.
                float c = 1.0f;
                const int d = (int)__reduce_max_sync(kFull, (unsigned)exponent_of(most)) - exponent_v();
                if (d > 0) {
                    // m falls by as much as E rises, which leaves the sums of p s_v as
                    // they are, as far as l and z stay in range (l to 2^100, z to 2^113)
                    const int u = max(exponent_of(fmaxf(l2.x, l2.y)) + 13, exponent_of(fmaxf(fabsf(z2.x), fabsf(z2.y))));
                    const int by = max(min(min(d, 120), 237 - (int)__reduce_max_sync(kFull, (unsigned)u)), 0);
                    const float g = pow2(by);
                    m0 -= (float)by;
                    m1 -= (float)by;
                    l2 = make_float2(l2.x * g, l2.y * g);
                    z2 = make_float2(z2.x * g, z2.y * g);
                    c = by - d < -126 ? 0.0f : pow2(by - d);
                    vmul = __uint_as_float(__float_as_uint(vmul) - ((uint32_t)d << 23));
                }
                mx0 = mx1 = -INFINITY;
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const float2 r = i ? vb[u] : va[u];
                        const int e = exponent_of(fmaxf(r.x, fabsf(r.y) * (1.0f / (1 << kBelowM)))) - exponent_v();
                        const float ev = (float)min(max(e, -kFar), kAbove);
                        mx0 = fmaxf(mx0, x[u][i].x + ev);
                        mx1 = fmaxf(mx1, x[u][i].y + ev);
                    }
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    mx0 = fmaxf(mx0, __shfl_xor_sync(kFull, mx0, off));
                    mx1 = fmaxf(mx1, __shfl_xor_sync(kFull, mx1, off));
                }
                const bool r0 = mx0 > m0 + kRescaleAt, r1 = mx1 > m1 + kRescaleAt;
                float c0 = r0 ? ex2(m0 - mx0) : 1.0f, c1 = r1 ? ex2(m1 - mx1) : 1.0f;  // 0 from m = -inf
                if (r0) m0 = mx0;
                if (r1) m1 = mx1;
                l2 = make_float2(l2.x * c0, l2.y * c1);
                z2 = make_float2(z2.x * c0, z2.y * c1);
                c0 *= c;
                c1 *= c;
#pragma unroll
                for (int mb = 0; mb < KS; mb++) {
                    o[mb][0] *= c0;
                    o[mb][1] *= c1;
                    o[mb][2] *= c0;
                    o[mb][3] *= c1;
                }
            }
            // p, then p s_v in two fp16 parts: rows of P^T, transposed in
            // registers into the B fragments of O^T += V^T P^T.  NT = 1: lanes
            // of columns 0-3 give the high part, of 4-7 the low part.
            const float2 nm = make_float2(-m0, -m1);
            auto weights = [&](float2 xs, float2 sm, uint32_t& first, uint32_t& second) {
                const float2 y = __fadd2_rn(xs, nm), pr = make_float2(ex2(y.x), ex2(y.y));
                l2 = __fadd2_rn(l2, pr);
                z2 = __ffma2_rn(pr, make_float2(sm.y, sm.y), z2);
                const float w = sm.x * vmul;
                const float2 ps = __fmul2_rn(pr, make_float2(w, w));
                const __half2 hi = __floats2half2_rn(ps.x, ps.y);
                const float2 r = __ffma2_rn(__half22float2(hi), low, ps);  // NT = 1, columns 0-3: ps itself
                second = pack_h2(r.x, r.y);
                first = *reinterpret_cast<const uint32_t*>(&hi);
            };
            uint32_t b0[2][2], b1[2][2];  // [tile][high, low (NT = 2)]: tokens 2 tq .. and 2 tq + 8 ..
#pragma unroll
            for (int u = 0; u < 2; u++) {
                uint32_t h0, e0, h1, e1;
                weights(x[u][0], va[u], h0, e0);
                weights(x[u][1], vb[u], h1, e1);
                if (NT == 1) {
                    b0[u][0] = movt(e0), b1[u][0] = movt(e1);
                } else {
                    b0[u][0] = movt(h0), b1[u][0] = movt(h1);
                    b0[u][1] = movt(e0), b1[u][1] = movt(e1);
                }
            }
            // ---- O^T += V^T P^T: M = 16 dims per m-block, K = 16 tokens.  The tensor
            // cores cut what lies below the running sum.  NT = 2 (two products a tile):
            // a pair's sum is taken apart, small parts first, and added with rounding
            // (2 rows of 131072 tokens: error 1.3e-6 -> 1e-7 for 97 against 92 us); NT = 1
            // stays within 3.3e-7 without. ----
#pragma unroll
            for (int u = 0; u < (NT == 1 ? 2 : 1); u++) {
                const char* at = kt + u * 2 * kTileBytes + kTileBytes;
                constexpr int NU = NT == 1 ? 1 : 2;
                uint32_t v0[NU][NWD], v1[NU][NWD];
#pragma unroll
                for (int i = 0; i < NU; i++) {
                    load_words<NWD>(at + i * 2 * kTileBytes + tq * D + gq * (4 * NWD), v0[i]);
                    load_words<NWD>(at + i * 2 * kTileBytes + (tq + 4) * D + gq * (4 * NWD), v1[i]);
                }
#pragma unroll
                for (int wi = 0; wi < NWD; wi++) {
                    uint32_t c0[NU][4], c1[NU][4];
#pragma unroll
                    for (int i = 0; i < NU; i++) {
                        q4_centred(v0[i][wi], c0[i]);
                        q4_centred(v1[i][wi], c1[i]);
                    }
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float(&acc)[4] = o[2 * wi + j];
                        if constexpr (NT == 1) {
                            mma16816(acc, c0[0][2 * j], c0[0][2 * j + 1], c1[0][2 * j], c1[0][2 * j + 1], b0[u][0], b1[u][0]);
                        } else {
                            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int part = 1; part >= 0; part--)
#pragma unroll
                                for (int i = 0; i < 2; i++)
                                    mma16816(sum, c0[i][2 * j], c0[i][2 * j + 1], c1[i][2 * j], c1[i][2 * j + 1], b0[i][part], b1[i][part]);
                            const float2 x0 = __fadd2_rn(make_float2(acc[0], acc[1]), make_float2(sum[0], sum[1]));
                            const float2 x1 = __fadd2_rn(make_float2(acc[2], acc[3]), make_float2(sum[2], sum[3]));
                            acc[0] = x0.x, acc[1] = x0.y, acc[2] = x1.x, acc[3] = x1.y;
                        }
                    }
                }
            }
            __syncwarp();  // the stage is read: its next pair may come
            if (k + kNS < pairs) {
                if (((k + kNS) & 15) == 0) fetch_ids(k + kNS);
                if (lane < 2) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                issue(k + kNS, it + kNS);
            }
        }

        if (k < pairs) {  // pair k did not come
            // copies still in flight land before the CTA exits (bounded)
            if (lane == 0) atomicOr(p.err, kErrTimeout);
            failed = true;
            for (int i = k; i < min(pairs, k + kNS); i++) bar_wait(bars + 8 * ((it0 + i) % kNS), (uint32_t)(((it0 + i) / kNS) & 1));
            m0 = m1 = -INFINITY;
            l2 = z2 = make_float2(0.f, 0.f);
        }
        it0 += pairs;
        float l0 = l2.x, l1 = l2.y, z0 = z2.x, z1 = z2.y;
        // ---- merge the warps through shared memory (over the rings) ----
        const float back = __uint_as_float((254u << 23) - __float_as_uint(vmul));  // 1 / vmul
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
            l0 += __shfl_xor_sync(kFull, l0, off);
            l1 += __shfl_xor_sync(kFull, l1, off);
            z0 += __shfl_xor_sync(kFull, z0, off);
            z1 += __shfl_xor_sync(kFull, z1, off);
        }
        // a sum of more than 2^40 goes into the reference: the merges take that for the scores' maximum
        const int up0 = l0 > 1.0995116e12f ? exponent_of(l0) - 127 : 0, up1 = l1 > 1.0995116e12f ? exponent_of(l1) - 127 : 0;
        const float down0 = pow2(-max(up0, 0)), down1 = pow2(-max(up1, 0));
        m0 += (float)max(up0, 0);
        m1 += (float)max(up1, 0);
        l0 *= down0;
        l1 *= down1;
#pragma unroll
        for (int mb = 0; mb < KS; mb++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (NT == 1) o[mb][i] += __shfl_xor_sync(kFull, o[mb][i], 2);
                o[mb][i] = fmaf(o[mb][i], back, i & 1 ? z1 : z0) * (i & 1 ? down1 : down0);
            }
        __syncthreads();  // every warp's tiles are consumed
        if (2 * tq < GP) {  // dims D / 8 gq + 2 mb (rows g) and + 1 (rows g + 8) of heads 2 tq, 2 tq + 1
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int hc = 2 * tq + i;
                float* dst = &mo[(warp * GP + hc) * D + (D / 8) * gq];
#pragma unroll
                for (int mb = 0; mb < KS; mb++) {
                    dst[2 * mb] = o[mb][i];
                    dst[2 * mb + 1] = o[mb][2 + i];
                }
                if (gq == 0) {
                    mml[(warp * GP + hc) * 2] = i ? m1 : m0;
                    mml[(warp * GP + hc) * 2 + 1] = i ? l1 : l0;
                }
            }
        }
        __syncthreads();
        const int64_t part = (int64_t)(rm.part_off + item.split) * p.Hkv + h;
        for (int idx = threadIdx.x; idx < min(GP, G - g0) * D; idx += kNW * 32) {
            const int g = idx / D, d = idx % D;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kNW; w++) M = fmaxf(M, mml[(w * GP + g) * 2]);
            float L = 0.0f, O = 0.0f;
#pragma unroll
            for (int w = 0; w < kNW; w++) {
                const float mw = mml[(w * GP + g) * 2];
                const float f = (mw == -INFINITY) ? 0.0f : ex2(mw - M);
                L = fmaf(mml[(w * GP + g) * 2 + 1], f, L);
                O = fmaf(mo[(w * GP + g) * D + d], f, O);
            }
            if (rm.n_split == 1) {
                store_out(p, item.row, h * G + g0 + g, d, D, O / L);
            } else {
                p.part_o[(part * G + g0 + g) * D + d] = O;
                if (d == 0) {
                    p.part_ml[(part * G + g0 + g) * 2] = M;
                    p.part_ml[(part * G + g0 + g) * 2 + 1] = L;
                }
            }
        }
        // before the next pass's copies overwrite the partial rows
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
    }
    pdl_trigger();
    if (p.counters && rm.n_split > 1) {
        finish_split_row(p, item.row, h, item.split, rm.n_split, G, D, flag, mo, kRing / 4);
    }
}

// ------------------------------------------------- any head_dim and block --
// One warp per (query row, query head), tokens in order: shapes the kernel
// above does not take (head_dim other than 64 and 128, blocks other than 16
// tokens, more than kMaxG query heads per KV head).
__global__ void attn_q4_generic_kernel(const AttnParams p) {
    const int G = p.Hq / p.Hkv, D = p.D, nq = D / 4, bs = p.block_size;
    const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31;
    const RowMeta rm = p.rows[row];
    const int32_t* tab = p.table + (int64_t)rm.table_row * p.max_bps;
    for (int g = threadIdx.x >> 5; g < G; g += blockDim.x >> 5) {
        const float* q = p.q + ((int64_t)row * p.Hq + h * G + g) * D;
        float qv[2][4], o[2][4];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int quad = lane + 32 * i;
                qv[i][e] = quad < nq ? q[4 * quad + e] : 0.0f;
                o[i][e] = 0.0f;
            }
        float m = -INFINITY, l = 0.0f;
        for (int j = 0; j < rm.kv_len; j++) {
            const int32_t blk = tab[j / bs];
            if ((uint32_t)blk >= (uint32_t)p.max_blocks) {
                if (lane == 0) atomicOr(p.err, kErrBounds);
                continue;
            }
            int t;
            const int64_t slot = (int64_t)blk * bs + j % bs;
            const char* kt = q4_tile(const_cast<void*>(p.kbase), slot, h, p.Hkv, bs, D, &t);
            const char* vt = q4_tile(const_cast<void*>(p.vbase), slot, h, p.Hkv, bs, D, &t);
            const float2 sk = q4_unpack(*reinterpret_cast<const uint32_t*>(kt + q4_param(t, bs, D)));
            const float2 sv = q4_unpack(*reinterpret_cast<const uint32_t*>(vt + q4_param(t, bs, D)));
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int quad = lane + 32 * i;
                if (quad >= nq) continue;
                const uint32_t c = *reinterpret_cast<const uint16_t*>(kt + q4_k_quad(t, quad, D));
#pragma unroll
                for (int e = 0; e < 4; e++) s = fmaf(qv[i][e], q4_value((c >> (4 * e)) & 15u, sk.x, sk.y), s);
            }
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(kFull, s, off);
            s *= p.scale_log2;
            const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.0f : ex2(m - mn), pj = ex2(s - mn);
            l = fmaf(l, c, pj);
            m = mn;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int quad = lane + 32 * i;
                if (quad >= nq) continue;
                const uint32_t cv = *reinterpret_cast<const uint16_t*>(vt + q4_v_quad(t, quad, D));
#pragma unroll
                for (int e = 0; e < 4; e++) o[i][e] = fmaf(pj, q4_value((cv >> (4 * e)) & 15u, sv.x, sv.y), o[i][e] * c);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int quad = lane + 32 * i;
            if (quad < nq)
#pragma unroll
                for (int e = 0; e < 4; e++) store_out(p, row, h * G + g, 4 * quad + e, D, o[i][e] / l);
        }
    }
}

bool decode_q4_supported(int D, int G, int block_size) {
    return (D == 64 || D == 128) && block_size == kTile && G >= 1 && G <= kMaxG;
}

int decode_q4_ctas_per_sm(int D) { return ctas_per_sm(D); }

template <int D, int NT>
static int launch_q4(const AttnParams& p, int G, cudaStream_t stream) {
    constexpr int smem = kNW * kNS * (4 * kTile * (D / 2 + 4) + 8) + 16 + kNW * 64;
    static std::atomic<uint64_t> attr_set{0};  // per device
    const int st = once_per_device(attr_set, [] {
        S1KV_CUDA(cudaFuncSetAttribute(decode_q4_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        return S1KV_OK;
    });
    if (st) return st;
    if ((int64_t)p.n_items * p.Hkv > INT32_MAX) return set_error(S1KV_EINVAL, "decode: too many work items");
    S1KV_CUDA(launch_pdl(decode_q4_kernel<D, NT>, dim3((unsigned)(p.n_items * p.Hkv)), dim3(kNW * 32), smem, stream, p, G));
    g_launches++;
    S1KV_CUDA(cudaGetLastError());
    return S1KV_OK;
}

int launch_decode_q4(const AttnParams& p, cudaStream_t stream) {
    if (p.n_rows <= 0) return S1KV_OK;
    const int G = p.Hq / p.Hkv;
    if (p.items && decode_q4_supported(p.D, G, p.block_size)) {
        if (p.D == 128) return G <= 4 ? launch_q4<128, 1>(p, G, stream) : launch_q4<128, 2>(p, G, stream);
        return G <= 4 ? launch_q4<64, 1>(p, G, stream) : launch_q4<64, 2>(p, G, stream);
    }
    attn_q4_generic_kernel<<<dim3((unsigned)p.n_rows, (unsigned)p.Hkv), 32 * std::min(G, 8), 0, stream>>>(p);
    g_launches++;
    S1KV_CUDA(cudaGetLastError());
    return S1KV_OK;
}

}  // namespace s1kv

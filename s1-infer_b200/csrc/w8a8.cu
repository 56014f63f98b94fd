// w8a8.cu -- products in 8-bit integers: tokens quantised to int8 with one
// scale each, times int8 weights with one scale per output channel.
//
//   s_m = fp32(max_k |x[m,k]| / 127), 1 for a row of zeros
//   xq[m,k] = the integer nearest to x[m,k] / s_m, ties to even
//   out[m,n] = fp32(sum_k xq[m,k] w[n,k]) * s_m * sw[n]
//
// The sum is exact in 32-bit integers (127 * 127 * K < 2^31 up to K =
// 131072), so its order is free and every run gives the same bits.  A row
// of x with a NaN or an infinity gets s_m = NaN and codes 0: its outputs are
// NaN, not a finite value made from the rest of the row.
//
// Weights are [N][K] rows of K bytes (an nn.Linear weight's own order; what
// s1kv_quantize_rows makes of it), K a multiple of 16 padded with zeros in x.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "internal.h"

namespace s1kv {
namespace {

constexpr int kMaxMats = 4;
constexpr int64_t kMaxK = 131072;

struct W8Mat {
    const int8_t* w;
    const float* scales;
    float* out;
    int N, tile0;
};
struct W8Group {
    W8Mat m[kMaxMats];
    int n;
};

// x / s to the nearest integer where fp32 cannot tell (next to a tie, or 1 / s
// overflowed), in 64 bits.
__device__ __noinline__ float token_code_near_tie(float x, float s) {
    return s > 0.0f ? (float)rint((double)x / (double)s) : 0.0f;
}

// Code of one value, -127 .. 127; inv = 1 / s.  The fp32 quotient is within
// 127 * 3 * 2^-24 = 2.3e-5 of the real one.
__device__ __forceinline__ int token_code(float x, float s, float inv) {
    const float q = x * inv;
    float n = rintf(q);
    if (!(fabsf(q - n) < 0.49995f)) n = token_code_near_tie(x, s);
    return (int)fminf(fmaxf(n, -127.0f), 127.0f);
}

__device__ __forceinline__ uint32_t token_codes4(float4 x, float s, float inv) {
    return (uint32_t)(token_code(x.x, s, inv) & 255) | (uint32_t)(token_code(x.y, s, inv) & 255) << 8 |
           (uint32_t)(token_code(x.z, s, inv) & 255) << 16 | (uint32_t)(token_code(x.w, s, inv) & 255) << 24;
}

// |x| of the largest, infinite once any is not finite.
__device__ __forceinline__ float top_of(float mx, float x) {
    const float a = fabsf(x);
    return a < INFINITY ? fmaxf(mx, a) : INFINITY;
}

// Maximum over the CTA's 256 threads; `part` is 8 floats of shared memory.
__device__ __forceinline__ float cta_max(float mx, float* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) mx = fmaxf(mx, part[i]);
    return mx;
}

__device__ __forceinline__ float token_scale(float mx) { return mx > 0.0f ? __fdiv_rn(mx, 127.0f) : 1.0f; }

// A row a CTA.  NV > 0: rows of up to 1024 NV values, a multiple of 4 and
// 16-byte aligned, stay in registers between the maximum and the codes (one
// read of x: 8001 rows of 4096 in 39 us, 4.2 TB/s); NV = 0: any row, read twice.
template <int NV>
__global__ void __launch_bounds__(256) quantize_tokens_kernel(const float* x, int64_t K, int8_t* q, int64_t ldq, float* scales) {
    pdl_wait_trigger();
    __shared__ float part[8];
    const int64_t m = blockIdx.x;
    const float* src = x + m * K;
    float mx = 0.0f;
    float4 v[NV > 0 ? NV : 1];
    if (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int k = 4 * (threadIdx.x + 256 * i);
            v[i] = k < K ? __ldcs(reinterpret_cast<const float4*>(src + k)) : make_float4(0.f, 0.f, 0.f, 0.f);
            mx = top_of(top_of(top_of(top_of(mx, v[i].x), v[i].y), v[i].z), v[i].w);
        }
    } else {
        for (int64_t k = threadIdx.x; k < K; k += 256) mx = top_of(mx, src[k]);
    }
    mx = cta_max(mx, part);
    const bool fine = mx < INFINITY;
    const float s = token_scale(mx), inv = __frcp_rn(s);
    if (threadIdx.x == 0) scales[m] = fine ? s : __uint_as_float(0x7FC00000u);
    if (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int k = 4 * (threadIdx.x + 256 * i);
            if (k < ldq) *reinterpret_cast<uint32_t*>(q + m * ldq + k) = fine ? token_codes4(v[i], s, inv) : 0u;
        }
    } else {
        for (int64_t k = threadIdx.x; k < ldq; k += 256)
            q[m * ldq + k] = (int8_t)(fine && k < K ? token_code(src[k], s, inv) : 0);
    }
}

int launch_quantize(const float* x, int64_t M, int64_t K, int8_t* q, int64_t ldq, float* scales, cudaStream_t stream) {
    const int nv = K % 4 || ((uintptr_t)x & 15) || ldq > 16384 ? 0 : ldq <= 1024 ? 1 : ldq <= 2048 ? 2 : ldq <= 4096 ? 4 : ldq <= 8192 ? 8 : 16;
    auto kern = nv == 0 ? quantize_tokens_kernel<0>
                        : nv == 1 ? quantize_tokens_kernel<1>
                                  : nv == 2 ? quantize_tokens_kernel<2>
                                  : nv == 4 ? quantize_tokens_kernel<4> : nv == 8 ? quantize_tokens_kernel<8> : quantize_tokens_kernel<16>;
    S1KV_CUDA(launch_pdl(kern, dim3((unsigned)M), dim3(256), 0, stream, x, K, q, ldq, scales));
    g_launches++;
    return S1KV_OK;
}

// ---------------------------------------------- few tokens: weight stream --
// Up to 8 NTILE tokens (NTILE = 1, 2 or 4): bound by the N K bytes of the
// weights.  mma.sync m16n8k32 on int8 with the channels on the 16-row side
// and the tokens on the 8-column side.  The sum over k does not care for the
// order of k, so a lane's fragments are simply 16 adjacent bytes of its
// channel's (and its token's) row: weights go from global memory to the
// instruction's registers in 16-byte loads, nothing is staged or shuffled.
// A CTA owns 16 channels, its 8 warps split K by 128-byte steps; the warps'
// integer sums meet in shared memory.  Behind this call's own token quantiser
// (EARLY) the first steps' weights are requested before the wait for it: the
// quantiser has waited for all that came before it and writes no weights.
// FUSED (one token of up to kFusedK values): each CTA quantises the token
// itself, from x through L2 into its shared memory: one launch instead of two.
// What runs before it may write anything, so its first weights are only
// brought to L2 before the wait.
// Three CTAs an SM with two steps in flight a warp stream better than two with
// four (8 tokens, K = 4096, 6144 channels: 7.8 against 11.0 us, 3.3 TB/s).
constexpr int kFusedK = 1024;  // four values a thread
constexpr int kGemvWarps = 8;
constexpr int kGemvPre = 2;  // 128-byte steps in flight a warp

__device__ __forceinline__ void imma16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NTILE, bool FUSED, bool EARLY>  // (neither: the caller's codes)
__global__ void __launch_bounds__(kGemvWarps * 32, 3)
    w8a8_gemv_kernel(const float* x, int x_len, const int8_t* xq, const float* sx, int M, int K, const __grid_constant__ W8Group grp) {
    __shared__ uint4 own[FUSED ? kFusedK / 16 : 1];  // the token's codes
    __shared__ float part[8], own_scale;
    __shared__ int red[kGemvWarps][16][8 * NTILE + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    int mi = 0;
#pragma unroll
    for (int i = 1; i < kMaxMats; i++)
        if (i < grp.n && (int)blockIdx.x >= grp.m[i].tile0) mi = i;
    const W8Mat& mat = grp.m[mi];
    const int n0 = ((int)blockIdx.x - mat.tile0) * 16;
    // rows past the last channel read the last one's bytes and are not stored
    const int8_t* w0 = mat.w + (int64_t)min(n0 + g, mat.N - 1) * K;
    const int8_t* w1 = mat.w + (int64_t)min(n0 + g + 8, mat.N - 1) * K;
    // step s of this warp: bytes 128 (warp + 8 s) .. + 127, in two 64-byte halves of 16 bytes a lane
    const int steps = ((K + 127) / 128 - warp + kGemvWarps - 1) / kGemvWarps;
    uint4 a[kGemvPre][2][2];
    auto fetch = [&](int s, uint4 (&r)[2][2]) {
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            const int k = 128 * (warp + kGemvWarps * s) + 64 * hf + 16 * t;
            const bool in = s < steps && k < K;
            r[hf][0] = in ? __ldcs(reinterpret_cast<const uint4*>(w0 + k)) : make_uint4(0, 0, 0, 0);
            r[hf][1] = in ? __ldcs(reinterpret_cast<const uint4*>(w1 + k)) : make_uint4(0, 0, 0, 0);
        }
    };
    auto fetch_first = [&] {
#pragma unroll
        for (int s = 0; s < kGemvPre; s++) fetch(s, a[s]);
    };
    if (EARLY) fetch_first();
    if (FUSED && t < 2 && 128 * warp < K)  // all of a warp's row pieces: one step
        asm volatile("prefetch.global.L2 [%0];" ::"l"((t ? w1 : w0) + 128 * warp));
    pdl_wait_trigger();
    if (!EARLY) fetch_first();
    if (FUSED) {
        const int k = 4 * threadIdx.x;
        const float4 v = k < x_len ? *reinterpret_cast<const float4*>(x + k) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float mx = cta_max(top_of(top_of(top_of(top_of(0.0f, v.x), v.y), v.z), v.w), part);
        const bool fine = mx < INFINITY;
        const float s = token_scale(mx), inv = __frcp_rn(s);
        if (threadIdx.x == 0) own_scale = fine ? s : __uint_as_float(0x7FC00000u);
        if (k < K) reinterpret_cast<uint32_t*>(own)[threadIdx.x] = fine ? token_codes4(v, s, inv) : 0u;
        __syncthreads();
    }
    int acc[NTILE][4] = {};
    for (int s0 = 0; s0 < steps; s0 += kGemvPre) {
#pragma unroll
        for (int u = 0; u < kGemvPre; u++) {
            const int s = s0 + u;
            if (s >= steps) break;
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const int k = 128 * (warp + kGemvWarps * s) + 64 * hf + 16 * t;
                const uint4 x = a[u][hf][0], y = a[u][hf][1];
#pragma unroll
                for (int nt = 0; nt < NTILE; nt++) {
                    // tokens past the last read the last one's bytes; their columns are not stored
                    const int64_t at = (int64_t)min(8 * nt + g, M - 1) * K + k;
                    const uint4 b = k >= K ? make_uint4(0, 0, 0, 0)
                                           : FUSED ? own[at >> 4] : *reinterpret_cast<const uint4*>(xq + at);
                    imma16832(acc[nt], x.x, y.x, x.y, y.y, b.x, b.y);
                    imma16832(acc[nt], x.z, y.z, x.w, y.w, b.z, b.w);
                }
            }
            fetch(s + kGemvPre, a[u]);
        }
    }
#pragma unroll
    for (int nt = 0; nt < NTILE; nt++)
#pragma unroll
        for (int i = 0; i < 4; i++) red[warp][g + (i >> 1) * 8][8 * nt + 2 * t + (i & 1)] = acc[nt][i];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * 8 * NTILE; i += kGemvWarps * 32) {
        const int n = i & 15, m = i >> 4;
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kGemvWarps; w++) sum += red[w][n][m];
        if (m < M && n0 + n < mat.N)
            mat.out[(int64_t)m * mat.N + n0 + n] = __fmul_rn(__fmul_rn((float)sum, FUSED ? own_scale : sx[m]), mat.scales[n0 + n]);
    }
}

// (Tokens' codes and scales, and x, are read by ordinary loads throughout: the
// kernel that writes them may run while this one waits, which the read-only
// path does not allow for.)
//
// -------------------------------------------------- many tokens: tcgen05 --
// tcgen05.mma kind::i8 with the 128 channels of a tile as M and NT = 64 or 128
// tokens as N, bound by the weights' bytes; a stored output row is 128 adjacent
// channels.  Roles: a TMA warp fills a ring of
// 128-byte deep stages (both operands K-major, 128B swizzle, rows past the
// end zero filled), one warp issues the MMAs, four warps take finished
// accumulators out of TMEM, scale and store them.
//   * Tiles enough for the machine: persistent CTAs, two accumulators in
//     TMEM so that a tile's output leaves while the next one's products run;
//     eight token tiles at a time share the weights through L2.
//   * Fewer tiles than SMs (few tokens): the K range of a tile is split over
//     a cluster of up to 8 CTAs, each rank sends its partial sums of a token
//     slice to that slice's owner through distributed shared memory, the
//     owner adds them (integers: any order, the same bits) and stores.
// Waits are bounded; a timeout raises an abort flag that every role polls
// and the error word; copies in flight are waited for, TMEM is freed.
constexpr uint32_t kSpin = 1u << 22;
constexpr int kCh = 128;             // channels a tile
constexpr int kKB = 128;             // bytes of K a stage
constexpr int kTcThreads = 192;      // TMA warp, MMA warp, 4 epilogue warps

template <int NT, bool SPLIT>
struct TcCfg {
    static constexpr int kStageBytes = kKB * (kCh + NT);
    // split tiles leave room for a second CTA on the SM
    static constexpr int kStages = SPLIT ? 3 : 6;
    static constexpr int kCols = (SPLIT ? 1 : 2) * NT;             // two accumulators for a chain of tiles
    static constexpr int kExchange = SPLIT ? kCh * NT * 4 : 0;     // [rank][token of the slice][channel] sums
    static constexpr int kOffX = kStages * kStageBytes;
    static constexpr int kOffScales = kOffX + kExchange;           // [4 warps][token]
    static constexpr int kOffBar = kOffScales + (SPLIT ? 0 : 4 * NT * 4);
    static constexpr int kNumBars = 2 * kStages + 5;
    static constexpr int kSmem = kOffBar + kNumBars * 8 + 16 + 1024;
};

struct TcParams {
    W8Group grp;       // tile0 counts tiles of 128 channels
    const float* sx;
    int M, k_blocks;   // stages of K
    int ch_tiles, tok_tiles;
    int early;         // this call's token quantiser runs before: weights may be read before the wait for it
};
struct TcMaps {
    CUtensorMap x, w[kMaxMats];
};

__device__ int g_w8a8_error;  // error word of this file's kernels (s1kv_device_check reads it)

__device__ __forceinline__ uint32_t su32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(b)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* b, uint32_t phase) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(su32(b)), "r"(phase)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t phase) {
    for (uint32_t i = 0; i < kSpin; i++)
        if (bar_try(b, phase)) return true;
    return false;
}
// The same for a whole warp, giving up when another role raised the flag; a
// timeout raises it.
__device__ __forceinline__ bool warp_wait(uint64_t* b, uint32_t phase, volatile int* abort_flag) {
    bool ok = false;
    for (uint32_t i = 0; i < kSpin && !ok; i++) {
        ok = bar_try(b, phase);
        if (!ok && *abort_flag) break;
    }
    if (!ok) *abort_flag = 1;
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ void tma2(uint32_t dst, const CUtensorMap* m, uint64_t* b, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(m), "r"(c0), "r"(c1), "r"(su32(b))
        : "memory");
}
// Shared-memory descriptor: K-major, 128-byte swizzle (layout type 2), 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t sdesc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
// kind::i8 instruction descriptor: signed 8-bit A and B (1), 32-bit integer D (2), both K-major.
__host__ __device__ constexpr uint32_t idesc_s8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Issued by one elected lane of a converged warp.
__device__ __forceinline__ void mma_i8_w(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_commit_w(uint64_t* b) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(su32(b))
        : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 16 consecutive 32-bit columns of this thread's TMEM lane, waited for.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, int (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

// The scales of n tokens from token m0 into this warp's part of shared memory
// (the kernel that wrote them may have run beside this one's start, so they are
// read by ordinary loads, which are slow next to every store of an output).
__device__ __forceinline__ void bring_scales(float* to, const float* sx, int m0, int n, int M) {
    __syncwarp();  // the last tile's are read
    for (int i = threadIdx.x & 31; i < n; i += 32) to[i] = m0 + i < M ? sx[m0 + i] : 0.0f;
    __syncwarp();
}
// A lane's channel of m_end tokens out of TMEM, scaled, to out (rows of N).
__device__ __forceinline__ void store_tile(uint32_t taddr, int m_end, const float* scales, float* out, int N, bool live, float sw) {
    for (int c = 0; c < m_end; c += 16) {
        int v[16];
        float sx[16];
#pragma unroll
        for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(sx + j) = *reinterpret_cast<const float4*>(scales + c + j);
        tmem_ld16(taddr + c, v);
#pragma unroll
        for (int j = 0; j < 16; j++)
            sx[j] = __fmul_rn(__fmul_rn((float)v[j], sx[j]), sw);
        float* at = out + (int64_t)c * N;
        if (live && c + 16 <= m_end) {
#pragma unroll
            for (int j = 0; j < 16; j++) __stcs(at + (int64_t)j * N, sx[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++)
                if (live && c + j < m_end) __stcs(at + (int64_t)j * N, sx[j]);
        }
    }
}

template <int NT, bool SPLIT>
__global__ void __launch_bounds__(kTcThreads, 1)
    w8a8_tc_kernel(const __grid_constant__ TcParams p, const __grid_constant__ TcMaps maps) {
    using C = TcCfg<NT, SPLIT>;
    constexpr int ST = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (-su32(smem_raw) & 1023u);  // (a sum: the compiler still sees shared memory)
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
    uint64_t* empty = full + ST;
    uint64_t* acc_full = empty + ST;    // [2]
    uint64_t* acc_empty = acc_full + 2;  // [2]
    uint64_t* drain = acc_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffBar + C::kNumBars * 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)), "r"(C::kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < C::kNumBars; i++) bar_init(&full[i], i == 2 * ST + 2 || i == 2 * ST + 3 ? 4u : 1u);  // acc_empty: one arrive a warp
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    if (SPLIT) {  // every rank runs before the first store into its shared memory
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // this CTA's tiles and its share of K
    const int cs = SPLIT ? (int)gridDim.y : 1, rank = SPLIT ? (int)blockIdx.y : 0;
    const int kb0 = (int)((int64_t)p.k_blocks * rank / cs), kb1 = (int)((int64_t)p.k_blocks * (rank + 1) / cs);
    const int n_tiles = p.ch_tiles * p.tok_tiles;
    auto tile_at = [&](int t, int& ch, int& tok) {  // eight token tiles side by side, their channels in turn
        const int per = 8 * p.ch_tiles, grp = t / per, in = t - grp * per, wide = min(8, p.tok_tiles - grp * 8);
        ch = in / wide;
        tok = grp * 8 + in - ch * wide;
    };
    auto mat_of = [&](int ch) {
        int mi = 0;
#pragma unroll
        for (int i = 1; i < kMaxMats; i++)
            if (i < p.grp.n && ch >= p.grp.m[i].tile0) mi = i;
        return mi;
    };

    if (warp == 0) {
        // ================= TMA producer =================
        int it = 0;  // stages used so far
        bool ok = true;
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.x) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.w[0]) : "memory");
        }
        // the weights of the first stages do not depend on this call's token
        // quantiser: requested before the wait for it
        int pre = 0;
        if (p.early) {
            int ch, tok;
            tile_at(blockIdx.x, ch, tok);
            const int mi = mat_of(ch), n0 = (ch - p.grp.m[mi].tile0) * kCh;
            pre = min(ST, kb1 - kb0);
            for (int s = 0; s < pre; s++)
                if (lane == 0) {
                    bar_expect(&full[s], C::kStageBytes);
                    tma2(su32(smem + s * C::kStageBytes), &maps.w[mi], &full[s], (kb0 + s) * kKB, n0);
                }
            __syncwarp();
        }
        pdl_wait();
        for (int t = blockIdx.x; t < n_tiles && ok; t += gridDim.x) {
            int ch, tok;
            tile_at(t, ch, tok);
            const int mi = mat_of(ch), n0 = (ch - p.grp.m[mi].tile0) * kCh;
            for (int kb = kb0; kb < kb1; kb++, it++) {
                const int s = it % ST;
                if (it >= ST && !(ok = warp_wait(&empty[s], (uint32_t)((it / ST - 1) & 1), abort_flag))) break;
                if (lane == 0) {
                    const uint32_t at = su32(smem + s * C::kStageBytes);
                    if (it >= pre) {
                        bar_expect(&full[s], C::kStageBytes);
                        tma2(at, &maps.w[mi], &full[s], kb * kKB, n0);
                    }
                    tma2(at + kCh * kKB, &maps.x, &full[s], kb * kKB, tok * NT);
                }
                __syncwarp();
            }
        }
        // every copy issued has landed before the CTA may exit (bounded)
        for (int i = max(0, it - ST); i < it; i++) bar_wait(&full[i % ST], (uint32_t)((i / ST) & 1));
    } else if (warp == 1) {
        // ================= MMA issuer =================
        constexpr uint32_t id = idesc_s8(kCh, NT);
        int it = 0, done = 0;  // stages consumed, tiles issued
        bool ok = true;
        for (int t = blockIdx.x; t < n_tiles && ok; t += gridDim.x, done++) {
            const int buf = done & 1;
            if (done >= 2 && !(ok = warp_wait(&acc_empty[buf], (uint32_t)((done / 2 - 1) & 1), abort_flag))) break;
            tc_fence_after();
            for (int kb = kb0; kb < kb1; kb++, it++) {
                const int s = it % ST;
                if (!(ok = warp_wait(&full[s], (uint32_t)((it / ST) & 1), abort_flag))) break;
                tc_fence_after();
                const uint64_t da = sdesc(su32(smem + s * C::kStageBytes)), db = sdesc(su32(smem + s * C::kStageBytes + kCh * kKB));
#pragma unroll
                for (int k = 0; k < kKB / 32; k++)  // 32 bytes of K an instruction
                    mma_i8_w(tmem + buf * NT, da + 2 * k, db + 2 * k, id, kb > kb0 || k > 0);
                mma_commit_w(&empty[s]);
            }
            if (ok) mma_commit_w(&acc_full[buf]);
        }
        // everything issued has finished before TMEM is freed (bounded)
        mma_commit_w(drain);
        bar_wait(drain, 0);
    } else {
        // ================= epilogue =================
        pdl_wait_trigger();  // the scales of the tokens, and outputs the kernel before may still read
        const int sub = warp & 3;  // the TMEM lanes 32 sub .. + 31 are this warp's
        const uint32_t lanes = (uint32_t)(32 * sub) << 16;
        float* scales = reinterpret_cast<float*>(smem + C::kOffScales) + sub * NT;
        int done = 0;
        for (int t = blockIdx.x; t < n_tiles; t += gridDim.x, done++) {
            const int buf = done & 1;
            int ch, tok;
            tile_at(t, ch, tok);
            const W8Mat& mat = p.grp.m[mat_of(ch)];
            const int n = (ch - mat.tile0) * kCh + 32 * sub + lane;
            const bool live = n < mat.N;
            const float sw = !SPLIT && live ? mat.scales[n] : 0.0f;
            if (!SPLIT) bring_scales(scales, p.sx, tok * NT, NT, p.M);
            if (!warp_wait(&acc_full[buf], (uint32_t)((done / 2) & 1), abort_flag)) break;
            tc_fence_after();
            if (!SPLIT) {
                store_tile(tmem + lanes + buf * NT, min(NT, p.M - tok * NT), scales, mat.out + (int64_t)tok * NT * mat.N + n,
                           mat.N, live, sw);
            } else {
                // columns [r * per, (r + 1) * per) of this tile are rank r's: [rank][column][channel]
                const int per = NT / cs;
                const uint32_t mine = su32(smem + C::kOffX) + (uint32_t)((rank * per * kCh + 32 * sub + lane) * 4);
                for (int c = 0; c < NT; c += 16) {
                    int v[16];
                    tmem_ld16(tmem + lanes + c, v);
#pragma unroll
                    for (int j0 = 0; j0 < 16; j0 += 8) {  // per is 8 or more
                        const int owner = (c + j0) / per;
                        uint32_t at;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                                     : "=r"(at)
                                     : "r"(mine + (uint32_t)((c + j0 - owner * per) * kCh * 4)), "r"(owner));
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at + j * kCh * 4), "r"(v[j0 + j]) : "memory");
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&acc_empty[buf]);
        }
    }

    // ---- tear-down: every path frees TMEM ----
    __syncthreads();
    if (SPLIT) {
        // this rank's slice: a token a warp, four channels a lane; the scales are
        // on their way while the other ranks' sums arrive
        pdl_wait();
        int ch, tok;
        tile_at(blockIdx.x, ch, tok);
        const W8Mat& mat = p.grp.m[mat_of(ch)];
        constexpr int kWarps = kTcThreads / 32, kMost = (NT / 2 + kWarps - 1) / kWarps;
        const int per = NT / cs, n = (ch - mat.tile0) * kCh + 4 * lane, m0 = tok * NT + rank * per;
        float sw[4], sm[kMost];
#pragma unroll
        for (int j = 0; j < 4; j++) sw[j] = n + j < mat.N ? mat.scales[n + j] : 0.0f;
#pragma unroll
        for (int i = 0; i < kMost; i++) {
            const int c = warp + kWarps * i;
            sm[i] = c < per && m0 + c < p.M ? p.sx[m0 + c] : 0.0f;
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        const int* got = reinterpret_cast<const int*>(smem + C::kOffX) + 4 * lane;
#pragma unroll
        for (int i = 0; i < kMost; i++) {
            const int c = warp + kWarps * i, m = m0 + c;
            if (c >= per || m >= p.M) break;
            int sum[4] = {0, 0, 0, 0};
            for (int r = 0; r < cs; r++) {
                const int4 v = *reinterpret_cast<const int4*>(got + (r * per + c) * kCh);
                sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
            }
            float* out = mat.out + (int64_t)m * mat.N + n;
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (n + j < mat.N) out[j] = __fmul_rn(__fmul_rn((float)sum[j], sm[i]), sw[j]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *abort_flag) atomicOr(&g_w8a8_error, kErrTimeout);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kCols) : "memory");
    }
}

// ------------------------------------ prompts: tcgen05 over pairs of SMs ----
// 256 channels by 256 tokens a pair of CTAs (cta_group::2): each brings its 128
// channels' weights and half of the tokens and holds its channels' sums of all
// the tokens, so a CTA moves 32 KB a stage from L2 where a tile of its own of
// 128 channels takes 48 KB.  The even rank's MMA warp issues for both; every
// copy counts on its barrier, its commits arrive at both.  Persistent, two
// accumulators, eight token tiles share the weights through L2, as above.
struct PairCfg {
    static constexpr int kTok = 256;
    static constexpr int kStageBytes = kKB * (kCh + kTok / 2);  // a CTA's part
    static constexpr int kStages = 6;
    static constexpr int kOffScales = kStages * kStageBytes;  // [4 warps][token]
    static constexpr int kOffBar = kOffScales + 4 * kTok * 4;
    static constexpr int kNumBars = 2 * kStages + 5;
    static constexpr int kSmem = kOffBar + kNumBars * 8 + 16 + 1024;
};

// The address of the pair's even rank's copy of a barrier.
__device__ __forceinline__ uint32_t lead_bar(uint64_t* b) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(su32(b)));
    return at;
}
__device__ __forceinline__ void tma2_pair(uint32_t dst, const CUtensorMap* m, uint32_t lead, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(m), "r"(c0), "r"(c1), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void mma_i8_pair_w(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_commit_pair_w(uint64_t* b) {  // arrives at both CTAs' barrier
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(su32(b)),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTcThreads, 1)
    w8a8_pair_kernel(const __grid_constant__ TcParams p, const __grid_constant__ TcMaps maps) {
    using C = PairCfg;
    constexpr int ST = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (-su32(smem_raw) & 1023u);  // (a sum: the compiler still sees shared memory)
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);  // [ST], the even rank's count for both
    uint64_t* empty = full + ST;
    uint64_t* acc_full = empty + ST;     // [2]
    uint64_t* acc_empty = acc_full + 2;  // [2], the even rank's count for both
    uint64_t* drain = acc_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffBar + C::kNumBars * 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = (int)(blockIdx.x & 1);

    if (tid == 0) {
        for (int i = 0; i < C::kNumBars; i++) bar_init(&full[i], i == 2 * ST + 2 || i == 2 * ST + 3 ? 8u : 1u);  // acc_empty: one arrive a warp
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    cluster_sync();  // both run and their barriers stand
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)), "r"(2 * C::kTok)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // TMEM is there in both before an MMA writes it
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    const int n_tiles = p.ch_tiles * p.tok_tiles, first = (int)(blockIdx.x >> 1), step = (int)(gridDim.x >> 1);
    auto tile_at = [&](int t, int& ch, int& tok) {  // eight token tiles side by side, their channels in turn
        const int per = 8 * p.ch_tiles, grp = t / per, in = t - grp * per, wide = min(8, p.tok_tiles - grp * 8);
        ch = in / wide;
        tok = grp * 8 + in - ch * wide;
    };
    auto mat_of = [&](int ch) {
        int mi = 0;
#pragma unroll
        for (int i = 1; i < kMaxMats; i++)
            if (i < p.grp.n && ch >= p.grp.m[i].tile0) mi = i;
        return mi;
    };

    if (warp == 0) {
        // ================= TMA producer: this CTA's channels and tokens =================
        int it = 0;  // stages used so far
        bool ok = true;
        int pre = 0;  // weights requested before the wait for this call's token quantiser
        auto load_w = [&](int s, int kb, int mi, int n0) {
            if (rank == 0) bar_expect(&full[s], 2 * C::kStageBytes);
            tma2_pair(su32(smem + s * C::kStageBytes), &maps.w[mi], lead_bar(&full[s]), kb * kKB, n0);
        };
        if (p.early) {
            int ch, tok;
            tile_at(first, ch, tok);
            const int mi = mat_of(ch);
            pre = min(ST, p.k_blocks);
            if (lane == 0)
                for (int s = 0; s < pre; s++) load_w(s, s, mi, (ch - p.grp.m[mi].tile0) * 2 * kCh + rank * kCh);
            __syncwarp();
        }
        pdl_wait();
        for (int t = first; t < n_tiles && ok; t += step) {
            int ch, tok;
            tile_at(t, ch, tok);
            const int mi = mat_of(ch), n0 = (ch - p.grp.m[mi].tile0) * 2 * kCh + rank * kCh, m0 = tok * C::kTok + rank * (C::kTok / 2);
            for (int kb = 0; kb < p.k_blocks; kb++, it++) {
                const int s = it % ST;
                if (it >= ST && !(ok = warp_wait(&empty[s], (uint32_t)((it / ST - 1) & 1), abort_flag))) break;
                if (lane == 0) {
                    if (it >= pre) load_w(s, kb, mi, n0);
                    tma2_pair(su32(smem + s * C::kStageBytes + kCh * kKB), &maps.x, lead_bar(&full[s]), kb * kKB, m0);
                }
                __syncwarp();
            }
        }
        // every copy issued has landed before a CTA of the pair may exit (bounded)
        if (rank == 0)
            for (int i = max(0, it - ST); i < it; i++) bar_wait(&full[i % ST], (uint32_t)((i / ST) & 1));
    } else if (warp == 1) {
        // ================= MMA issuer, for both =================
        if (rank == 0) {
            constexpr uint32_t id = idesc_s8(2 * kCh, C::kTok);
            int it = 0, done = 0;  // stages consumed, tiles issued
            bool ok = true;
            for (int t = first; t < n_tiles && ok; t += step, done++) {
                const int buf = done & 1;
                if (done >= 2 && !(ok = warp_wait(&acc_empty[buf], (uint32_t)((done / 2 - 1) & 1), abort_flag))) break;
                tc_fence_after();
                for (int kb = 0; kb < p.k_blocks; kb++, it++) {
                    const int s = it % ST;
                    if (!(ok = warp_wait(&full[s], (uint32_t)((it / ST) & 1), abort_flag))) break;
                    tc_fence_after();
                    const uint64_t da = sdesc(su32(smem + s * C::kStageBytes)), db = sdesc(su32(smem + s * C::kStageBytes + kCh * kKB));
#pragma unroll
                    for (int k = 0; k < kKB / 32; k++)  // 32 bytes of K an instruction
                        mma_i8_pair_w(tmem + buf * C::kTok, da + 2 * k, db + 2 * k, id, kb > 0 || k > 0);
                    mma_commit_pair_w(&empty[s]);
                }
                if (ok) mma_commit_pair_w(&acc_full[buf]);
            }
            // everything issued has finished before TMEM is freed (bounded)
            mma_commit_pair_w(drain);
            bar_wait(drain, 0);
        }
    } else {
        // ================= epilogue =================
        pdl_wait_trigger();  // the scales of the tokens, and outputs the kernel before may still read
        const int sub = warp & 3;  // the TMEM lanes 32 sub .. + 31 are this warp's
        const uint32_t lanes = (uint32_t)(32 * sub) << 16;
        float* scales = reinterpret_cast<float*>(smem + C::kOffScales) + sub * C::kTok;
        int done = 0;
        for (int t = first; t < n_tiles; t += step, done++) {
            const int buf = done & 1;
            int ch, tok;
            tile_at(t, ch, tok);
            const W8Mat& mat = p.grp.m[mat_of(ch)];
            const int n = (ch - mat.tile0) * 2 * kCh + rank * kCh + 32 * sub + lane;
            const bool live = n < mat.N;
            const float sw = live ? mat.scales[n] : 0.0f;
            bring_scales(scales, p.sx, tok * C::kTok, C::kTok, p.M);
            if (!warp_wait(&acc_full[buf], (uint32_t)((done / 2) & 1), abort_flag)) break;
            tc_fence_after();
            store_tile(tmem + lanes + buf * C::kTok, min(C::kTok, p.M - tok * C::kTok), scales, mat.out + (int64_t)tok * C::kTok * mat.N + n, mat.N, live, sw);
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
                asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(lead_bar(&acc_empty[buf])) : "memory");
        }
    }

    // ---- tear-down: every path frees TMEM; neither CTA leaves before the other is done ----
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (tid == 0 && *abort_flag) atomicOr(&g_w8a8_error, kErrTimeout);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * C::kTok) : "memory");
    }
}

// ---------------------------------------------------------------- launch --
std::atomic<uint64_t> g_used_on{0};  // devices a tcgen05 launch ran on (its error word may be set there)

int encode_rows(CUtensorMap* m, const int8_t* base, int64_t rows, int64_t K, int box_rows) {
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> cached{nullptr};
    PFN_cuTensorMapEncodeTiled_v12000 encode = cached.load(std::memory_order_acquire);
    if (!encode) {
        cudaDriverEntryPointQueryResult q;
        void* fn = nullptr;
        S1KV_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
        if (q != cudaDriverEntryPointSuccess || !fn)
            return set_error(S1KV_ECUDA, "matmul_w8a8: cuTensorMapEncodeTiled unavailable");
        encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
        cached.store(encode, std::memory_order_release);
    }
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)K};
    cuuint32_t box[2] = {(cuuint32_t)kKB, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    const CUresult r = encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(base), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(S1KV_EINVAL, "matmul_w8a8: tensor map rejected (%d)", (int)r);
    return S1KV_OK;
}

template <int NT, bool SPLIT>
int launch_tc(const int8_t* xq, const float* sx, int M, int K, const W8Group& grp, int ch_tiles, int cs, bool early,
              cudaStream_t stream) {
    auto kern = w8a8_tc_kernel<NT, SPLIT>;
    static std::atomic<uint64_t> attr_set{0};  // per device
    int st = once_per_device(attr_set, [&] {
        constexpr int bytes = TcCfg<NT, SPLIT>::kSmem;
        S1KV_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        return S1KV_OK;
    });
    if (st) return st;
    TcParams p{};
    p.grp = grp;
    p.sx = sx;
    p.early = early;
    p.M = M;
    p.k_blocks = (K + kKB - 1) / kKB;
    p.ch_tiles = ch_tiles;
    p.tok_tiles = (M + NT - 1) / NT;
    TcMaps maps;
    st = encode_rows(&maps.x, xq, M, K, NT);
    for (int i = 0; i < grp.n && !st; i++) st = encode_rows(&maps.w[i], grp.m[i].w, grp.m[i].N, K, kCh);
    if (st) return st;
    for (int i = grp.n; i < kMaxMats; i++) maps.w[i] = maps.w[0];
    int dev = 0;
    S1KV_CUDA(cudaGetDevice(&dev));
    if (dev < 64) g_used_on.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
    const int tiles = ch_tiles * p.tok_tiles;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = SPLIT ? dim3((unsigned)tiles, (unsigned)cs) : dim3((unsigned)std::min(tiles, 148));
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = TcCfg<NT, SPLIT>::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = (unsigned)cs;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = SPLIT ? 2 : 1;
    S1KV_CUDA(cudaLaunchKernelEx(&cfg, kern, p, maps));
    g_launches++;
    return S1KV_OK;
}

int launch_pair(const int8_t* xq, const float* sx, int M, int K, const W8Group& grp, int ch_tiles, bool early, cudaStream_t stream) {
    static std::atomic<uint64_t> attr_set{0};  // per device
    int st = once_per_device(attr_set, [&] {
        S1KV_CUDA(cudaFuncSetAttribute(w8a8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg::kSmem));
        return S1KV_OK;
    });
    if (st) return st;
    TcParams p{};
    p.grp = grp;
    p.sx = sx;
    p.early = early;
    p.M = M;
    p.k_blocks = (K + kKB - 1) / kKB;
    p.ch_tiles = ch_tiles;
    p.tok_tiles = (M + PairCfg::kTok - 1) / PairCfg::kTok;
    TcMaps maps;
    st = encode_rows(&maps.x, xq, M, K, PairCfg::kTok / 2);
    for (int i = 0; i < grp.n && !st; i++) st = encode_rows(&maps.w[i], grp.m[i].w, grp.m[i].N, K, kCh);
    if (st) return st;
    for (int i = grp.n; i < kMaxMats; i++) maps.w[i] = maps.w[0];
    int dev = 0;
    S1KV_CUDA(cudaGetDevice(&dev));
    if (dev < 64) g_used_on.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
    const unsigned pairs = (unsigned)std::min(ch_tiles * p.tok_tiles, 74);
    S1KV_CUDA(launch_pdl(w8a8_pair_kernel, dim3(2 * pairs), dim3(kTcThreads), PairCfg::kSmem, stream, p, maps));
    g_launches++;
    return S1KV_OK;
}

template <int NTILE, bool FUSED, bool EARLY>
int launch_gemv(const float* x, int x_len, const int8_t* xq, const float* sx, int M, int K, const W8Group& grp, int tiles,
                cudaStream_t stream) {
    S1KV_CUDA(launch_pdl(w8a8_gemv_kernel<NTILE, FUSED, EARLY>, dim3((unsigned)tiles), dim3(kGemvWarps * 32), 0, stream, x,
                         x_len, xq, sx, M, K, grp));
    g_launches++;
    return S1KV_OK;
}

// Which kernel, by the tokens: up to 8 the weight stream, and up to 32 while the
// weights are small (with the quantiser, in tiles beside it: 16 tokens, 25 MB 9.3
// us and 12.9, 59 MB 18.6 and 16.5, 67 MB 24.3 and 19.1; 32 tokens, 4 MB 6.0 and
// 8.0, 25 MB 13.7 and 12.3, 59 MB 29 and 16); above, the tensor-core tiles.
// NT is the least that holds the tokens (256 at most), halved down to 64 while
// there are fewer than 90 tiles (products alone: 256 tokens, K = 4096, 6144
// channels: 96 tiles of 128 tokens 12.7 us, 192 of 64 20.0; 4096 channels: 32
// tiles of 256 tokens 14.8, 128 of 64 11.3); then K is split over a cluster, at
// least two stages a CTA, two CTAs an SM, if the tiles are fewer than two thirds of
// the SMs (64 tokens, K = 4096: 48 tiles 9.4 us split in four, 10.8 unsplit; 112
// tiles 12.0 in two, 11.4 unsplit).  NT = 256 runs on pairs of SMs (8001 tokens, K
// = 4096, 14336 channels: 326 us, 2.9e15 operations a second, 88% of twice the bf16
// matrix rate; 442 us in tiles of 128 tokens of one SM; 8192^3: 3.3e15, 99%).
// x (optional, rows of x_len values): the tokens that xq and sx will hold; they
// are quantised here first, or by the weight stream itself.
int matmul_w8a8(const float* x, int x_len, int8_t* xq, float* sx, int M, int K, W8Group& grp, cudaStream_t stream) {
    int64_t channels = 0, tiles = 0;
    for (int i = 0; i < grp.n; i++) channels += grp.m[i].N;
    const bool stream_w = M <= 8 || (M <= 32 && channels * K <= (M <= 16 ? 48 : 20) << 20);
    const int rows = stream_w || K == 0 ? 16 : kCh;
    for (int i = 0; i < grp.n; i++) {
        grp.m[i].tile0 = (int)tiles;
        tiles += (grp.m[i].N + rows - 1) / rows;
    }
    int NT = M <= 64 ? 64 : M <= 128 ? 128 : 256;
    while (NT > 64 && tiles * ((M + NT - 1) / NT) < 90) NT /= 2;
    if (tiles * ((M + NT - 1) / NT) > INT32_MAX) return set_error(S1KV_EINVAL, "matmul_w8a8: more than 2^31 tiles");
    if (K == 0) {  // empty sums
        for (int i = 0; i < grp.n; i++)
            S1KV_CUDA(cudaMemsetAsync(grp.m[i].out, 0, sizeof(float) * (size_t)M * grp.m[i].N, stream));
        return S1KV_OK;
    }
    // One short token: a kernel of its own for the codes costs more than making
    // them in every CTA (K = 1024, 4096 channels: 3.3 us against 3.0; K = 2048:
    // 4.1 against 4.6), as long as all CTAs are resident at once.
    if (x && M == 1 && K <= kFusedK && tiles <= 3 * 148 && x_len % 4 == 0 && ((uintptr_t)x & 15) == 0)
        return launch_gemv<1, true, false>(x, x_len, nullptr, nullptr, M, K, grp, (int)tiles, stream);
    if (x) {
        const int st = launch_quantize(x, M, x_len, xq, K, sx, stream);
        if (st) return st;
    }
    if (M <= 8)
        return x ? launch_gemv<1, false, true>(nullptr, 0, xq, sx, M, K, grp, (int)tiles, stream)
                 : launch_gemv<1, false, false>(nullptr, 0, xq, sx, M, K, grp, (int)tiles, stream);
    if (stream_w && M <= 16)
        return x ? launch_gemv<2, false, true>(nullptr, 0, xq, sx, M, K, grp, (int)tiles, stream)
                 : launch_gemv<2, false, false>(nullptr, 0, xq, sx, M, K, grp, (int)tiles, stream);
    if (stream_w)
        return x ? launch_gemv<4, false, true>(nullptr, 0, xq, sx, M, K, grp, (int)tiles, stream)
                 : launch_gemv<4, false, false>(nullptr, 0, xq, sx, M, K, grp, (int)tiles, stream);
    const int k_blocks = (K + kKB - 1) / kKB;
    const int64_t all = tiles * ((M + NT - 1) / NT);
    if (NT == 64) {
        int cs = 1;
        while (cs < 8 && all <= 98 && all * cs * 2 <= 296 && k_blocks >= cs * 4) cs *= 2;
        return cs > 1 ? launch_tc<64, true>(xq, sx, M, K, grp, (int)tiles, cs, x != nullptr, stream)
                      : launch_tc<64, false>(xq, sx, M, K, grp, (int)tiles, 1, x != nullptr, stream);
    }
    if (NT == 128) return launch_tc<128, false>(xq, sx, M, K, grp, (int)tiles, 1, x != nullptr, stream);
    int pairs = 0;  // tiles of 256 channels
    for (int i = 0; i < grp.n; i++) {
        grp.m[i].tile0 = pairs;
        pairs += (grp.m[i].N + 2 * kCh - 1) / (2 * kCh);
    }
    return launch_pair(xq, sx, M, K, grp, pairs, x != nullptr, stream);
}

}  // namespace

int w8a8_take_error(int device, int* flags) {
    *flags = 0;
    if (device < 0 || device >= 64 || !(g_used_on.load(std::memory_order_relaxed) >> device & 1)) return S1KV_OK;
    int h = 0;
    S1KV_CUDA(cudaMemcpyFromSymbol(&h, g_w8a8_error, sizeof(int), 0, cudaMemcpyDeviceToHost));
    if (h) {
        const int zero = 0;
        S1KV_CUDA(cudaMemcpyToSymbol(g_w8a8_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice));
    }
    *flags = h;
    return S1KV_OK;
}
}  // namespace s1kv

using namespace s1kv;

extern "C" int s1kv_quantize_tokens(const float* x, int64_t M, int64_t K, int8_t* q, int64_t ldq, float* scales,
                                    void* stream) {
    if (M < 0 || K < 0 || M > INT32_MAX || K > kMaxK || ldq < K || ldq > kMaxK || ldq % 16)
        return set_error(S1KV_EINVAL, "quantize_tokens: rows of %lld values, ldq %lld (a multiple of 16, at least K, at most %lld)",
                         (long long)K, (long long)ldq, (long long)kMaxK);
    if (M == 0) return S1KV_OK;
    if ((K > 0 && !x) || (ldq > 0 && !q) || !scales) return set_error(S1KV_EINVAL, "quantize_tokens: null pointer");
    if ((uintptr_t)q & 15) return set_error(S1KV_EINVAL, "quantize_tokens: q must be 16-byte aligned");
    return launch_quantize(x, M, K, q, ldq, scales, (cudaStream_t)stream);
}

static int w8a8_group(const float* x, int64_t x_len, int8_t* xq, float* x_scales, int64_t M, int64_t K, int32_t n_mats,
                      const int8_t* const* w, const float* const* w_scales, const int64_t* N, float* const* out,
                      void* stream) {
    if (!w || !w_scales || !N || !out) return set_error(S1KV_EINVAL, "matmul_w8a8: null array");
    if (n_mats < 1 || n_mats > kMaxMats) return set_error(S1KV_EINVAL, "matmul_w8a8: 1 to %d matrices per call", kMaxMats);
    if (M < 0 || M > (1 << 30) || K < 0 || K > kMaxK || K % 16)
        return set_error(S1KV_EINVAL, "matmul_w8a8: M %lld, K %lld (a multiple of 16 up to %lld)", (long long)M, (long long)K,
                         (long long)kMaxK);
    W8Group grp = {};
    for (int i = 0; i < n_mats; i++) {
        if (N[i] < 0 || N[i] > (1 << 30)) return set_error(S1KV_EINVAL, "matmul_w8a8: bad shape");
        if (M == 0 || N[i] == 0) continue;
        if ((K > 0 && (!xq || !w[i])) || !x_scales || !w_scales[i] || !out[i])
            return set_error(S1KV_EINVAL, "matmul_w8a8: null pointer");
        if (((uintptr_t)xq | (uintptr_t)w[i]) & 15)
            return set_error(S1KV_EINVAL, "matmul_w8a8: xq and w must be 16-byte aligned");
        grp.m[grp.n++] = {w[i], w_scales[i], out[i], (int)N[i], 0};
    }
    if (grp.n == 0) return S1KV_OK;
    return matmul_w8a8(x, (int)x_len, xq, x_scales, (int)M, (int)K, grp, (cudaStream_t)stream);
}

extern "C" int s1kv_matmul_w8a8_group(const int8_t* xq, const float* x_scales, int64_t M, int64_t K, int32_t n_mats,
                                      const int8_t* const* w, const float* const* w_scales, const int64_t* N,
                                      float* const* out, void* stream) {
    return w8a8_group(nullptr, 0, const_cast<int8_t*>(xq), const_cast<float*>(x_scales), M, K, n_mats, w, w_scales, N, out,
                      stream);
}

extern "C" int64_t s1kv_w8a8_workspace(int64_t M, int64_t K) {
    if (M < 0 || M > (1 << 30) || K < 0 || K > kMaxK) return 0;
    return M * ((K + 15) / 16 * 16) + (4 * M + 15) / 16 * 16;
}

extern "C" int s1kv_linear_w8a8_group(const float* x, int64_t M, int64_t K, void* workspace, int64_t workspace_bytes,
                                      int32_t n_mats, const int8_t* const* w, const float* const* w_scales, const int64_t* N,
                                      float* const* out, void* stream) {
    if (M < 0 || M > (1 << 30) || K < 0 || K > kMaxK)
        return set_error(S1KV_EINVAL, "linear_w8a8: M %lld, K %lld (up to %lld)", (long long)M, (long long)K, (long long)kMaxK);
    if (M > 0 && K > 0 && !x) return set_error(S1KV_EINVAL, "linear_w8a8: null x");
    if (workspace_bytes < s1kv_w8a8_workspace(M, K) || (workspace_bytes > 0 && !workspace) || ((uintptr_t)workspace & 15))
        return set_error(S1KV_EINVAL, "linear_w8a8: needs %lld bytes of 16-byte aligned workspace",
                         (long long)s1kv_w8a8_workspace(M, K));
    const int64_t ld = (K + 15) / 16 * 16;
    int8_t* xq = (int8_t*)workspace;
    return w8a8_group(x, K, xq, (float*)(xq + M * ld), M, ld, n_mats, w, w_scales, N, out, stream);
}

extern "C" int s1kv_matmul_w8a8(const int8_t* xq, const float* x_scales, int64_t M, int64_t K, const int8_t* w,
                                const float* w_scales, int64_t N, float* out, void* stream) {
    return s1kv_matmul_w8a8_group(xq, x_scales, M, K, 1, &w, &w_scales, &N, &out, stream);
}

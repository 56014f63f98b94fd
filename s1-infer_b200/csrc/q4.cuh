// q4.cuh -- the 4-bit K/V row format (device code shared by the append,
// gather and attention kernels of S1KV_DTYPE_Q4 pools).
//
// A row is the D values x of one token and KV head.  With lo, hi its least
// and greatest value:
//   m = bf16(fp32((7 lo + 8 hi) / 15))          both to nearest even
//   s = fp32(max((hi - m) / 7, (m - lo) / 8)) rounded UP to bf16
//   code = 8 + nearest integer to (x - m) / s   (ties to even; 8 where s = 0 or NaN)
//   held value = fp32(m + s (code - 8))
// The codes -8 .. 7 around m reach lo and hi because s is rounded up, so
// every held value is within s / 2 of x, with no clipping, whatever the
// row's offset.  One (s, m) pair a row (4 bytes beside D / 2 bytes of codes)
// keeps K's scale and zero term out of the tensor-core products: they act
// on whole scores.  bf16 for both because its range is fp32's; the bound
// above holds for the rounded pair.  A row with a NaN or an infinity, or whose
// m or s passes bf16's largest (3.39e38), is held as s = m = NaN: the whole row
// reads back as NaN.
//
// Storage: one tile per (block, KV head), K and V apart:
//   codes  bs * D / 2 bytes, then the rows' params  bs * {bf16 s, bf16 m}.
//   K codes [token][D / 2]: nibble n of the row is value n (low first).
//   V codes [token pair][D / 4][2 tokens][2 bytes]: four values (a quad) of
//   a token are 16 bits, and a pair's tokens lie side by side in one 32-bit
//   word: that word holds, for four dims, the two adjacent tokens that one
//   fp16x2 register of a tensor-core fragment needs (K runs over dims, V
//   over tokens), and no byte belongs to two tokens, so tokens of one tile
//   may be appended by different threads, calls and launches.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"

namespace s1kv {

struct Q4Row {  // one row's parameters
    float s, m;
    uint32_t packed;  // bf16 s | bf16 m << 16, as stored
};

__device__ __forceinline__ uint32_t q4_bf16_rn(float f) {
    const uint32_t u = __float_as_uint(f);
    return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}

// (s, m) of a row from its extremes; `finite`: no value is NaN or infinite.
// In 64 bits so that each of the two fp32 values is the real number's
// rounding (the products by 1/15 and 1/7 are off by 2^-53).
__device__ __forceinline__ Q4Row q4_params(float lo, float hi, bool finite) {
    Q4Row r;
    const double l = lo, h = hi;
    const uint32_t mb = q4_bf16_rn(__double2float_rn((7.0 * l + 8.0 * h) * (1.0 / 15.0)));
    r.m = __uint_as_float(mb << 16);
    const double m = r.m;
    const float need = __double2float_rn(fmax((h - m) * (1.0 / 7.0), (m - l) * 0.125));
    const uint32_t sb = (__float_as_uint(need) + 0xFFFFu) >> 16;  // need >= 0: up
    r.s = __uint_as_float(sb << 16);
    if (!finite || !(r.s < INFINITY) || !(fabsf(r.m) < INFINITY)) {
        r.packed = 0x7FC07FC0u;
        r.s = r.m = __uint_as_float(0x7FC00000u);
        return r;
    }
    r.packed = sb | (mb << 16);
    return r;
}

// 0 .. 15; inv = 1 / s.  The fp32 quotient is within 2e-6 of the real one
// (|q| < 8.6, three roundings): only one this near a tie (or not finite,
// for a tiny s) is decided in 64 bits.
__device__ __forceinline__ uint32_t q4_code(float x, const Q4Row& r, float inv) {
    const float q = (x - r.m) * inv;
    float n = rintf(q);
    if (!(fabsf(q - n) < 0.49998f)) {
        n = 0.0f;
        if (r.s > 0.0f) n = (float)rint(((double)x - (double)r.m) / (double)r.s);
    }
    return (uint32_t)((int)fminf(fmaxf(n, -8.0f), 7.0f) + 8) & 15u;
}

__device__ __forceinline__ float q4_value(uint32_t code, float s, float m) {
    return fmaf(s, (float)((int)code - 8), m);  // the product is exact (8 x 4 bits): one rounding
}

__device__ __forceinline__ float2 q4_unpack(uint32_t packed) {  // (s, m)
    return make_float2(__uint_as_float(packed << 16), __uint_as_float(packed & 0xFFFF0000u));
}

__device__ __forceinline__ uint32_t q4_and_or(uint32_t w, uint32_t mask, uint32_t o) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(w), "r"(mask), "r"(o));  // (w & mask) | o
    return y;
}
// The eight codes of a word centred, u - 8, as fp16x2: nibble n of the low half
// and of the high half in out[n] (V: four dims of two tokens; K: dims n and
// n + 4 of eight).  0x6400 | u is the fp16 1024 + u, 0x6400 | 16 u is 1024 + 16 u.
__device__ __forceinline__ void q4_centred(uint32_t w, uint32_t (&out)[4]) {
    const __half2 one = __float2half2_rn(1.0f), m1032 = __float2half2_rn(-1032.0f);
    const __half2 sixteenth = __float2half2_rn(0.0625f), m72 = __float2half2_rn(-72.0f);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t x = w >> (8 * i);
        const uint32_t a = q4_and_or(x, 0x000F000Fu, 0x64006400u), b = q4_and_or(x, 0x00F000F0u, 0x64006400u);
        const __half2 ha = __hfma2(*reinterpret_cast<const __half2*>(&a), one, m1032);
        const __half2 hb = __hfma2(*reinterpret_cast<const __half2*>(&b), sixteenth, m72);
        out[2 * i] = *reinterpret_cast<const uint32_t*>(&ha);
        out[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&hb);
    }
}

// Bytes of one (block, KV head) tile and offsets inside it.
__host__ __device__ __forceinline__ int q4_tile_bytes(int bs, int D) { return bs * (D / 2 + 4); }
__device__ __forceinline__ int q4_k_quad(int t, int quad, int D) { return t * (D / 2) + quad * 2; }
__device__ __forceinline__ int q4_v_quad(int t, int quad, int D) { return (t >> 1) * D + quad * 4 + (t & 1) * 2; }
__device__ __forceinline__ int q4_param(int t, int bs, int D) { return bs * (D / 2) + t * 4; }

// Tile of (slot, head) in one layer's storage and the token's place in it.  (A
// pool has fewer than 2^31 slots: one 32-bit division.)
__device__ __forceinline__ char* q4_tile(void* base, int64_t slot, int h, int Hkv, int bs, int D, int* t) {
    const uint32_t blk = (uint32_t)slot / (uint32_t)bs;
    *t = (int)((uint32_t)slot - blk * (uint32_t)bs);
    return reinterpret_cast<char*>(base) + ((int64_t)blk * Hkv + h) * q4_tile_bytes(bs, D);
}

// Quantises one row held by `LANES` adjacent lanes of a warp, NQ quads a
// lane (quad lane_in_row + i * LANES; quads from nq on are absent), and
// stores it.  Every lane of the warp calls it; `store` is false for lanes
// whose row is absent or out of range.
template <int LANES, int NQ>
__device__ __forceinline__ void q4_store_row(const float (&x)[NQ][4], int nq, char* tile, int t, bool is_v, int bs, int D,
                                             bool store) {
    const int lr = threadIdx.x % LANES;
    float lo = INFINITY, hi = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < NQ; i++)
        if (lr + i * LANES < nq) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                lo = fminf(lo, x[i][e]);
                hi = fmaxf(hi, x[i][e]);
                bad |= !(fabsf(x[i][e]) < INFINITY);
            }
        }
    // a bad value spoils the row's maximum, which then spoils the row
    if (bad) hi = INFINITY;
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const Q4Row r = q4_params(lo, hi, hi < INFINITY);
    const float inv = __frcp_rn(r.s);
    if (!store) return;
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        const int quad = lr + i * LANES;
        if (quad >= nq) continue;
        uint32_t c = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) c |= q4_code(x[i][e], r, inv) << (4 * e);
        *reinterpret_cast<uint16_t*>(tile + (is_v ? q4_v_quad(t, quad, D) : q4_k_quad(t, quad, D))) = (uint16_t)c;
    }
    if (lr == 0) *reinterpret_cast<uint32_t*>(tile + q4_param(t, bs, D)) = r.packed;
}

// The same for a row held by LANES = D / 16 adjacent lanes, quads lane_in_row +
// i LANES (x[4 i ..]): a warp takes 512 / D rows, so the reductions and the
// 64-bit arithmetic of the parameters serve that many rows at once (a row a
// warp ran at a quarter of the speed).  Codes are made in packed fp32:
// (x - m) / s + 8, rounded by adding 1.5 * 2^23; a row with a value within
// 1e-4 of a tie is done again value by value.
template <int LANES>
__device__ __forceinline__ void q4_store_row16(const float (&x)[16], char* tile, int t, bool is_v, int bs, int D, bool store) {
    const int lr = threadIdx.x % LANES;
    float lo = x[0], hi = x[0];
    float2 bad2 = make_float2(0.f, 0.f);  // 0, or NaN from a value that is not finite
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        lo = fminf(fminf(lo, x[i]), x[i + 1]);
        hi = fmaxf(fmaxf(hi, x[i]), x[i + 1]);
        bad2 = __ffma2_rn(make_float2(x[i], x[i + 1]), make_float2(0.f, 0.f), bad2);
    }
    if (!(bad2.x + bad2.y == 0.0f)) hi = INFINITY;  // spoils the row's maximum, which then spoils the row
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const Q4Row r = q4_params(lo, hi, hi < INFINITY);
    const float inv = __frcp_rn(r.s);
    if (!store) return;
    const float2 m2 = make_float2(-r.m, -r.m), inv2 = make_float2(inv, inv), eight = make_float2(8.f, 8.f);
    const float kRound = 12582912.0f;  // 1.5 * 2^23
    const float2 up = make_float2(kRound, kRound), down = make_float2(-kRound, -kRound);
    float far = 0.0f;
    uint32_t c[4];
#pragma unroll
    for (int q = 0; q < 4; q++) {
        float u[4];
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            const float2 v = __ffma2_rn(__fadd2_rn(make_float2(x[4 * q + e], x[4 * q + e + 1]), m2), inv2, eight);
            const float2 n = __fadd2_rn(__fadd2_rn(v, up), down), d = __fadd2_rn(v, make_float2(-n.x, -n.y));
            far = fmaxf(fmaxf(far, fabsf(d.x)), fabsf(d.y));
            u[e] = n.x, u[e + 1] = n.y;
        }
        c[q] = (uint32_t)fmaf(4096.f, u[3], fmaf(256.f, u[2], fmaf(16.f, u[1], u[0])));
    }
    // (inv is not finite where s is 0 or too small to invert, or the row is spoilt;
    // m - lo passes fp32 where the row spans nearly all of it)
    if (!(far < 0.4999f) || !(fabsf(inv) < INFINITY) || !(r.m - lo < INFINITY)) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            c[q] = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) c[q] |= q4_code(x[4 * q + e], r, inv) << (4 * e);
        }
    }
    char* at = tile + (is_v ? q4_v_quad(t, lr, D) : q4_k_quad(t, lr, D));
    const int step = (is_v ? 4 : 2) * LANES;
#pragma unroll
    for (int q = 0; q < 4; q++) *reinterpret_cast<uint16_t*>(at + q * step) = (uint16_t)c[q];
    if (lr == 0) *reinterpret_cast<uint32_t*>(tile + q4_param(t, bs, D)) = r.packed;
}

}  // namespace s1kv

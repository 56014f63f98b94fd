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

// 0 .. 255 codes of one value; inv = 1 / s.  The fp32 quotient is within
// 127 * 3 * 2^-24 = 2.3e-5 of the real one: only one this near a tie (or not
// finite, for a tiny s) is decided in 64 bits.
__device__ __forceinline__ int token_code(float x, float s, float inv) {
    const float q = x * inv;
    float n = rintf(q);
    if (!(fabsf(q - n) < 0.49995f)) n = s > 0.0f ? (float)rint((double)x / (double)s) : 0.0f;
    return (int)fminf(fmaxf(n, -127.0f), 127.0f);
}

__global__ void __launch_bounds__(256) quantize_tokens_kernel(const float* __restrict__ x, int64_t M, int64_t K,
                                                              int8_t* __restrict__ q, int64_t ldq,
                                                              float* __restrict__ scales) {
    __shared__ float part[8];
    const int64_t m = blockIdx.x;
    const float* src = x + m * K;
    float mx = 0.0f;
    for (int64_t k = threadIdx.x; k < K; k += 256) {
        const float a = fabsf(src[k]);
        mx = a < INFINITY ? fmaxf(mx, a) : INFINITY;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) mx = fmaxf(mx, part[i]);
    const bool fine = mx < INFINITY;
    const float s = mx > 0.0f ? __fdiv_rn(mx, 127.0f) : 1.0f, inv = __frcp_rn(s);
    if (threadIdx.x == 0) scales[m] = fine ? s : __uint_as_float(0x7FC00000u);
    for (int64_t k = threadIdx.x; k < ldq; k += 256)
        q[m * ldq + k] = (int8_t)(fine && k < K ? token_code(src[k], s, inv) : 0);
}

// 64 x 64 outputs a CTA, 4 x 4 a thread, 64 bytes of K a step.
__global__ void __launch_bounds__(256) w8a8_tile_kernel(const int8_t* __restrict__ xq, const float* __restrict__ sx, int M,
                                                        int K, const __grid_constant__ W8Group grp) {
    __shared__ int xs[64][17], ws[64][17];
    int mi = 0;
#pragma unroll
    for (int i = 1; i < kMaxMats; i++)
        if (i < grp.n && (int)blockIdx.x >= grp.m[i].tile0) mi = i;
    const W8Mat& mat = grp.m[mi];
    const int n0 = ((int)blockIdx.x - mat.tile0) * 64, m0 = blockIdx.y * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += 64) {
        for (int i = threadIdx.x; i < 64 * 16; i += 256) {
            const int r = i >> 4, c = i & 15, k = k0 + 4 * c;
            xs[r][c] = m0 + r < M && k < K ? *reinterpret_cast<const int*>(xq + (int64_t)(m0 + r) * K + k) : 0;
            ws[r][c] = n0 + r < mat.N && k < K ? *reinterpret_cast<const int*>(mat.w + (int64_t)(n0 + r) * K + k) : 0;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 16; c++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(xs[ty * 4 + i][c], ws[tx + 16 * j][c], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int m = m0 + ty * 4 + i, n = n0 + tx + 16 * j;
            if (m < M && n < mat.N)
                mat.out[(int64_t)m * mat.N + n] = __fmul_rn(__fmul_rn((float)acc[i][j], sx[m]), mat.scales[n]);
        }
}

}  // namespace
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
    quantize_tokens_kernel<<<(unsigned)M, 256, 0, (cudaStream_t)stream>>>(x, M, K, q, ldq, scales);
    g_launches++;
    S1KV_CUDA(cudaGetLastError());
    return S1KV_OK;
}

extern "C" int s1kv_matmul_w8a8_group(const int8_t* xq, const float* x_scales, int64_t M, int64_t K, int32_t n_mats,
                                      const int8_t* const* w, const float* const* w_scales, const int64_t* N,
                                      float* const* out, void* stream) {
    if (!w || !w_scales || !N || !out) return set_error(S1KV_EINVAL, "matmul_w8a8: null array");
    if (n_mats < 1 || n_mats > kMaxMats) return set_error(S1KV_EINVAL, "matmul_w8a8: 1 to %d matrices per call", kMaxMats);
    if (M < 0 || M > (1 << 30) || K < 0 || K > kMaxK || K % 16)
        return set_error(S1KV_EINVAL, "matmul_w8a8: M %lld, K %lld (a multiple of 16 up to %lld)", (long long)M, (long long)K,
                         (long long)kMaxK);
    W8Group grp = {};
    int tiles = 0;
    for (int i = 0; i < n_mats; i++) {
        if (N[i] < 0 || N[i] > (1 << 30)) return set_error(S1KV_EINVAL, "matmul_w8a8: bad shape");
        if (M == 0 || N[i] == 0) continue;
        if ((K > 0 && (!xq || !w[i])) || !x_scales || !w_scales[i] || !out[i])
            return set_error(S1KV_EINVAL, "matmul_w8a8: null pointer");
        if (((uintptr_t)xq | (uintptr_t)w[i]) & 15)
            return set_error(S1KV_EINVAL, "matmul_w8a8: xq and w must be 16-byte aligned");
        grp.m[grp.n++] = {w[i], w_scales[i], out[i], (int)N[i], tiles};
        tiles += (int)((N[i] + 63) / 64);
    }
    if (grp.n == 0) return S1KV_OK;
    const int64_t row_tiles = (M + 63) / 64;
    for (int64_t r0 = 0; r0 < row_tiles; r0 += 65535) {  // grid.y's limit
        const int64_t m0 = r0 * 64, m = std::min<int64_t>(M - m0, 65535 * 64);
        W8Group g = grp;
        for (int i = 0; i < g.n; i++) g.m[i].out += m0 * g.m[i].N;
        w8a8_tile_kernel<<<dim3((unsigned)tiles, (unsigned)((m + 63) / 64)), 256, 0, (cudaStream_t)stream>>>(
            xq + m0 * K, x_scales + m0, (int)m, (int)K, g);
        g_launches++;
        S1KV_CUDA(cudaGetLastError());
    }
    return S1KV_OK;
}

extern "C" int s1kv_matmul_w8a8(const int8_t* xq, const float* x_scales, int64_t M, int64_t K, const int8_t* w,
                                const float* w_scales, int64_t N, float* out, void* stream) {
    return s1kv_matmul_w8a8_group(xq, x_scales, M, K, 1, &w, &w_scales, &N, &out, stream);
}

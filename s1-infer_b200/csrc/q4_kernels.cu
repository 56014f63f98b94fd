// q4_kernels.cu -- data movement of 4-bit pools (format: q4.cuh): append
// with and without RoPE, gather, and the byte rows of prefix files.
#include <algorithm>

#include "q4.cuh"

namespace s1kv {

constexpr int kSMs = 148;

// -------------------------------------------------------------- append ----
// A row (one token and head of k, v or, rotated only, q) per LANES lanes,
// one quad of values a lane: its extremes are two shuffle reductions, and
// K's 64 code bytes of a row (D = 128) leave as one segment.  RoPE
// (src/nn/RoPE.cpp:32-33: out1 = x1 c - x2 s, out2 = x2 c + x1 s, each
// operation rounded on its own) reads its partner quad D / 2 away through
// the L1 cache, before the quantisation.
template <int LANES, int NQ, bool ROPE>
__global__ void __launch_bounds__(256) append_q4_kernel(const AppendParams p) {
    pdl_wait_trigger();
    const int D = p.D, half = D / 2, nq = D / 4;
    constexpr int RPW = 32 / LANES;
    const int lane = threadIdx.x & 31, lr = lane % LANES;
    const int64_t kv_rows = p.n * p.Hkv, q_rows = ROPE && p.q_in ? p.n * p.Hq : 0, total = 2 * kv_rows + q_rows;
    const int64_t warp = blockIdx.x * (int64_t)(blockDim.x / 32) + threadIdx.x / 32, warps = (int64_t)gridDim.x * (blockDim.x / 32);
    for (int64_t u0 = warp * RPW; u0 < total; u0 += warps * RPW) {  // warp-uniform (shuffles inside)
        const int64_t u = u0 + lane / LANES;
        const bool have = u < total;
        const int part = u < kv_rows ? 0 : u < 2 * kv_rows ? 1 : 2;  // K, V, Q
        const int64_t th = part == 0 ? u : part == 1 ? u - kv_rows : u - 2 * kv_rows;
        const int H = part == 2 ? p.Hq : p.Hkv;
        const int64_t t = have ? th / H : 0;
        const int h = (int)(th - t * H);
        const float* src = (part == 0 ? p.k : part == 1 ? p.v : p.q_in) + (have ? th : 0) * D;
        const bool rot = ROPE && part != 1;
        const int32_t pos = rot && have ? p.pos[t] : 0;
        bool ok = have;
        if (rot && have && (uint64_t)pos >= (uint64_t)p.rope_cap) {
            if (lr == 0) atomicOr(p.err, kErrBounds);
            ok = false;
        }
        float x[NQ][4];
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            const int quad = lr + i * LANES, d = 4 * quad;
            x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.0f;
            if (quad >= nq || !ok) continue;
#pragma unroll
            for (int e = 0; e < 4; e++) x[i][e] = src[d + e];
            if (rot) {
                const bool first = d < half;
                const float* other = src + (first ? d + half : d - half);
                const float2* cs = p.rope + (int64_t)pos * half + (first ? d : d - half);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float2 c = __ldg(cs + e);
                    const float o = other[e];
                    x[i][e] = first ? __fsub_rn(__fmul_rn(x[i][e], c.x), __fmul_rn(o, c.y))
                                    : __fadd_rn(__fmul_rn(x[i][e], c.x), __fmul_rn(o, c.y));
                }
            }
        }
        char* tile = nullptr;
        int tt = 0;
        bool store = ok && part != 2;
        if (store) {
            const int32_t slot = p.slots[t];
            if ((uint64_t)slot >= (uint64_t)p.num_slots) {
                if (lr == 0) atomicOr(p.err, kErrBounds);
                store = false;
            } else {
                tile = q4_tile(part == 0 ? p.kpool : p.vpool, slot, h, p.Hkv, p.block_size, D, &tt);
            }
        }
        if (ok && part == 2)
#pragma unroll
            for (int i = 0; i < NQ; i++) {
                const int quad = lr + i * LANES;
                if (quad < nq)
#pragma unroll
                    for (int e = 0; e < 4; e++) p.q_out[th * D + 4 * quad + e] = x[i][e];
            }
        q4_store_row<LANES, NQ>(x, nq, tile, tt, part == 1, p.block_size, D, store);
    }
}

int launch_append_q4(const AppendParams& p, bool rope, cudaStream_t stream, bool pdl) {
    if (p.n <= 0) return S1KV_OK;
    const int64_t rows = 2 * p.n * p.Hkv + (rope && p.q_in ? p.n * p.Hq : 0);
    const int rpw = p.D == 64 ? 2 : 1;
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>((rows + 8 * rpw - 1) / (8 * rpw), kSMs * 16));
#define S1KV_APPEND(L, N, R)                                                                            \
    do {                                                                                               \
        if (pdl) S1KV_CUDA(launch_pdl(append_q4_kernel<L, N, R>, dim3(grid), dim3(256), 0, stream, p)); \
        else append_q4_kernel<L, N, R><<<grid, 256, 0, stream>>>(p);                                   \
    } while (0)
#define S1KV_APPEND_R(R)                       \
    do {                                       \
        if (p.D == 64) S1KV_APPEND(16, 1, R);  \
        else if (p.D <= 128) S1KV_APPEND(32, 1, R); \
        else S1KV_APPEND(32, 2, R);            \
    } while (0)
    if (rope) S1KV_APPEND_R(true);
    else S1KV_APPEND_R(false);
#undef S1KV_APPEND_R
#undef S1KV_APPEND
    g_launches++;
    S1KV_CUDA(cudaGetLastError());
    return S1KV_OK;
}

// -------------------------------------------------------------- gather ----
// One thread per quad: token i of a sequence (block-table row `trow`) or of
// a batch (`slots`), widened to fp32.
__global__ void gather_q4_kernel(const char* __restrict__ base, bool is_v, const int32_t* __restrict__ trow,
                                 const int32_t* __restrict__ slots, int64_t n, int bs, int Hkv, int D, int64_t num_slots,
                                 float* __restrict__ out, int* err) {
    const int nq = D / 4;
    const int64_t total = n * Hkv * nq;
    for (int64_t u = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; u < total; u += (int64_t)gridDim.x * blockDim.x) {
        const int quad = (int)(u % nq);
        const int64_t th = u / nq, i = th / Hkv;
        const int h = (int)(th - i * Hkv);
        const int64_t slot = slots ? slots[i] : (int64_t)trow[i / bs] * bs + i % bs;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if ((uint64_t)slot >= (uint64_t)num_slots) {
            atomicOr(err, kErrBounds);
        } else {
            int t;
            const char* tile = q4_tile(const_cast<char*>(base), slot, h, Hkv, bs, D, &t);
            const uint32_t c = *reinterpret_cast<const uint16_t*>(tile + (is_v ? q4_v_quad(t, quad, D) : q4_k_quad(t, quad, D)));
            const float2 sm = q4_unpack(*reinterpret_cast<const uint32_t*>(tile + q4_param(t, bs, D)));
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = q4_value((c >> (4 * e)) & 15u, sm.x, sm.y);
        }
        if (((uintptr_t)out & 15) == 0)
            *reinterpret_cast<float4*>(out + u * 4) = make_float4(v[0], v[1], v[2], v[3]);
        else
#pragma unroll
            for (int e = 0; e < 4; e++) out[u * 4 + e] = v[e];
    }
}

int launch_gather_q4(s1kv_pool* p, int32_t layer, const int32_t* trow, const int32_t* slots, int64_t n, int which,
                     float* out, cudaStream_t stream) {
    if (n <= 0) return S1KV_OK;
    const char* base = (which ? p->v : p->k) + (size_t)layer * p->layer_bytes;
    const int64_t total = n * p->desc.num_kv_heads * (p->desc.head_dim / 4);
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>((total + 255) / 256, kSMs * 16));
    gather_q4_kernel<<<grid, 256, 0, stream>>>(base, which != 0, trow, slots, n, p->desc.block_size, p->desc.num_kv_heads,
                                               p->desc.head_dim, p->num_slots, out, p->d_err);
    g_launches++;
    S1KV_CUDA(cudaGetLastError());
    return S1KV_OK;
}

// ------------------------------------------------------------ byte rows ----
// Rows as prefix files hold them: [token][head] of D / 2 code bytes in K's
// order, then the params.  TO_POOL writes rows into slots, else rows of a
// sequence are read.  One thread per 16 bits (a quad, or half the params).
template <bool TO_POOL>
__global__ void rows_q4_kernel(char* __restrict__ base, bool is_v, const int32_t* __restrict__ trow,
                               const int32_t* __restrict__ slots, int64_t n, int bs, int Hkv, int D, int64_t num_slots,
                               uint16_t* __restrict__ rows, int* err) {
    const int nq = D / 4, words = nq + 2;
    const int64_t total = n * Hkv * words;
    for (int64_t u = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; u < total; u += (int64_t)gridDim.x * blockDim.x) {
        const int w = (int)(u % words);
        const int64_t th = u / words, i = th / Hkv;
        const int64_t slot = slots ? slots[i] : (int64_t)trow[i / bs] * bs + i % bs;
        if ((uint64_t)slot >= (uint64_t)num_slots) {
            atomicOr(err, kErrBounds);
            continue;
        }
        int t;
        char* tile = q4_tile(base, slot, (int)(th - i * Hkv), Hkv, bs, D, &t);
        uint16_t* at = reinterpret_cast<uint16_t*>(
            tile + (w >= nq ? q4_param(t, bs, D) + 2 * (w - nq) : is_v ? q4_v_quad(t, w, D) : q4_k_quad(t, w, D)));
        if (TO_POOL) *at = rows[u];
        else rows[u] = *at;
    }
}

int launch_rows_q4(s1kv_pool* p, int32_t layer, const int32_t* trow, const int32_t* slots, int64_t n, int which,
                   void* rows, bool to_pool, cudaStream_t stream) {
    if (n <= 0) return S1KV_OK;
    char* base = (which ? p->v : p->k) + (size_t)layer * p->layer_bytes;
    const int64_t total = n * p->desc.num_kv_heads * (p->desc.head_dim / 4 + 2);
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>((total + 255) / 256, kSMs * 16));
    auto kern = to_pool ? rows_q4_kernel<true> : rows_q4_kernel<false>;
    kern<<<grid, 256, 0, stream>>>(base, which != 0, trow, slots, n, p->desc.block_size, p->desc.num_kv_heads,
                                   p->desc.head_dim, p->num_slots, (uint16_t*)rows, p->d_err);
    g_launches++;
    S1KV_CUDA(cudaGetLastError());
    return S1KV_OK;
}

}  // namespace s1kv

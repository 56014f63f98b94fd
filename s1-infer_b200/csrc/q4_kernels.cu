// q4_kernels.cu -- data movement of 4-bit pools (format: q4.cuh): append
// with and without RoPE, gather, and the byte rows of prefix files.
#include <algorithm>

#include "q4.cuh"

namespace s1kv {

constexpr int kSMs = 148;

// -------------------------------------------------------------- append ----
// A row (one token and head of k, v or, rotated only, q) on LANES lanes.
// LANES = D / 16 (D of 64, 128, 256): four quads of values a lane, LANES quads
// apart, so that a row's lanes read 16 LANES adjacent bytes at a time and a
// value's RoPE partner D / 2 away is the lane's own (17000 tokens of 8 heads of
// 128: 34.5 us, 4.6 TB/s, with RoPE 39.2; 16 contiguous values a lane and
// partners read again: 36.9 and 57.4).  LANES = 32, any other D: two quads a lane, 128 values apart,
// partners read through the L1 cache.  RoPE (src/nn/RoPE.cpp:32-33: out1 =
// x1 c - x2 s, out2 = x2 c + x1 s, each operation rounded on its own) comes
// before the quantisation.  Bound by the fp32 rows read (8 bytes a K and V
// value pair against 1 written) and by the instructions that find a row's
// parameters and codes, 56% of the issue slots.
template <int LANES, bool ROPE>
__global__ void __launch_bounds__(256, 5) append_q4_kernel(const AppendParams p) {
    pdl_wait_trigger();
    constexpr bool kWide = LANES < 32;
    constexpr int NQ = kWide ? 4 : 2, RPW = 32 / LANES;
    const int D = p.D, half = D / 2, nq = D / 4;
    const int lane = threadIdx.x & 31, lr = lane % LANES;
    const uint32_t kv_rows = (uint32_t)(p.n * p.Hkv), q_rows = ROPE && p.q_in ? (uint32_t)(p.n * p.Hq) : 0u;
    const uint32_t total = 2 * kv_rows + q_rows;  // (launch_append_q4 keeps it below 2^31)
    const uint32_t warp = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32, warps = gridDim.x * (blockDim.x / 32);
    for (uint32_t u0 = warp * RPW; u0 < total; u0 += warps * RPW) {  // warp-uniform (shuffles inside)
        const uint32_t u = u0 + lane / LANES;
        const bool have = u < total;
        const int part = u < kv_rows ? 0 : u < 2 * kv_rows ? 1 : 2;  // K, V, Q
        const uint32_t th = !have ? 0u : part == 0 ? u : part == 1 ? u - kv_rows : u - 2 * kv_rows;
        const uint32_t H = part == 2 ? p.Hq : p.Hkv, t = th / H;
        const int h = (int)(th - t * H);
        const float* src = (part == 0 ? p.k : part == 1 ? p.v : p.q_in) + (int64_t)th * D;
        const bool rot = ROPE && part != 1;
        const int32_t pos = rot && have ? p.pos[t] : 0;
        bool ok = have;
        if (rot && have && (uint64_t)pos >= (uint64_t)p.rope_cap) {
            if (lr == 0) atomicOr(p.err, kErrBounds);
            ok = false;
        }
        float x[4 * NQ];
        if constexpr (kWide) {  // 16-byte aligned (launch_append_q4)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float4 f = ok ? *reinterpret_cast<const float4*>(src + 4 * (lr + LANES * i)) : make_float4(0.f, 0.f, 0.f, 0.f);
                x[4 * i] = f.x, x[4 * i + 1] = f.y, x[4 * i + 2] = f.z, x[4 * i + 3] = f.w;
            }
            if (rot && ok) {
#pragma unroll
                for (int i = 0; i < 2; i++) {  // quads i and i + 2
                    const float4* cs = reinterpret_cast<const float4*>(p.rope + (int64_t)pos * half + 4 * (lr + LANES * i));
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const float4 c = __ldg(cs + e / 2);  // two (cos, sin)
                        float &a0 = x[4 * i + e], &a1 = x[4 * i + e + 1], &b0 = x[4 * i + 8 + e], &b1 = x[4 * i + 9 + e];
                        const float y0 = __fsub_rn(__fmul_rn(a0, c.x), __fmul_rn(b0, c.y));
                        const float y1 = __fsub_rn(__fmul_rn(a1, c.z), __fmul_rn(b1, c.w));
                        b0 = __fadd_rn(__fmul_rn(b0, c.x), __fmul_rn(a0, c.y));
                        b1 = __fadd_rn(__fmul_rn(b1, c.z), __fmul_rn(a1, c.w));
                        a0 = y0, a1 = y1;
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NQ; i++) {
                const int quad = lr + i * LANES, d = 4 * quad;
                x[4 * i] = x[4 * i + 1] = x[4 * i + 2] = x[4 * i + 3] = 0.0f;
                if (quad >= nq || !ok) continue;
#pragma unroll
                for (int e = 0; e < 4; e++) x[4 * i + e] = src[d + e];
                if (rot) {
                    const bool first = d < half;
                    const float* other = src + (first ? d + half : d - half);
                    const float2* cs = p.rope + (int64_t)pos * half + (first ? d : d - half);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float2 c = __ldg(cs + e);
                        const float a = __fmul_rn(x[4 * i + e], c.x), b = __fmul_rn(other[e], c.y);
                        x[4 * i + e] = first ? __fsub_rn(a, b) : __fadd_rn(a, b);
                    }
                }
            }
            if (ROPE) __syncwarp();  // a row's lanes have all read it (q_out may be q_in)
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
                if (quad >= nq) continue;
                float* dst = p.q_out + (int64_t)th * D + 4 * quad;
                if (kWide) *reinterpret_cast<float4*>(dst) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                else
#pragma unroll
                    for (int e = 0; e < 4; e++) dst[e] = x[4 * i + e];
            }
        if constexpr (kWide) {
            q4_store_row16<LANES>(x, tile, tt, part == 1, p.block_size, D, store);
        } else {
            const float y[2][4] = {{x[0], x[1], x[2], x[3]}, {x[4], x[5], x[6], x[7]}};
            q4_store_row<32, 2>(y, nq, tile, tt, part == 1, p.block_size, D, store);
        }
    }
}

int launch_append_q4(const AppendParams& all, bool rope, cudaStream_t stream, bool pdl) {
    // row numbers in 32 bits: a call of more than 2^31 rows goes in pieces
    const int64_t per = 2 * (int64_t)all.Hkv + (rope && all.q_in ? all.Hq : 0), most = ((int64_t)1 << 30) / per;
    const bool wide = (all.D == 64 || all.D == 128 || all.D == 256) &&
                      ((((uintptr_t)all.k | (uintptr_t)all.v | (uintptr_t)(all.q_in ? all.q_in : all.k) |
                         (uintptr_t)(all.q_in ? all.q_out : all.k)) & 15) == 0);
    const int lanes = wide ? all.D / 16 : 32;
    for (int64_t t0 = 0; t0 < all.n; t0 += most) {
        AppendParams p = all;
        p.n = std::min<int64_t>(most, all.n - t0);
        p.k += t0 * p.Hkv * p.D;
        p.v += t0 * p.Hkv * p.D;
        if (p.q_in) p.q_in += t0 * p.Hq * p.D, p.q_out += t0 * p.Hq * p.D;
        p.slots += t0;
        if (p.pos) p.pos += t0;
        const int64_t rows = p.n * per, per_cta = 8 * (32 / lanes);
        const int grid = (int)std::max<int64_t>(1, std::min<int64_t>((rows + per_cta - 1) / per_cta, kSMs * 16));
#define S1KV_APPEND(L, R)                                                                            \
    do {                                                                                             \
        if (pdl) S1KV_CUDA(launch_pdl(append_q4_kernel<L, R>, dim3(grid), dim3(256), 0, stream, p)); \
        else append_q4_kernel<L, R><<<grid, 256, 0, stream>>>(p);                                    \
    } while (0)
#define S1KV_APPEND_R(R)                    \
    do {                                    \
        if (lanes == 4) S1KV_APPEND(4, R);  \
        else if (lanes == 8) S1KV_APPEND(8, R);   \
        else if (lanes == 16) S1KV_APPEND(16, R); \
        else S1KV_APPEND(32, R);            \
    } while (0)
        if (rope) S1KV_APPEND_R(true);
        else S1KV_APPEND_R(false);
#undef S1KV_APPEND_R
#undef S1KV_APPEND
        g_launches++;
        S1KV_CUDA(cudaGetLastError());
    }
    return S1KV_OK;
}

// -------------------------------------------------------------- gather ----
// Token i of a sequence (block-table row `trow`) or of a batch (`slots`), widened
// to fp32: a warp eight (token, head) rows at a time, one quad a lane.  The
// rows' places are worked out by a lane each, their codes and parameters all
// requested before the first is widened (17000 tokens of 8 heads of 128: 16.6 us,
// 4.7 TB/s; 4 or 16 rows: 18.7).
constexpr int kGatherRows = 8;
__global__ void __launch_bounds__(256) gather_q4_kernel(const char* __restrict__ base, bool is_v, const int32_t* __restrict__ trow,
                                                        const int32_t* __restrict__ slots, uint32_t n_rows, uint32_t row0, int bs,
                                                        int Hkv, int D, int64_t num_slots, float* __restrict__ out, int* err) {
    const int nq = D / 4, lane = threadIdx.x & 31;
    const uint32_t warp = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32, warps = gridDim.x * (blockDim.x / 32);
    const bool vec = ((uintptr_t)out & 15) == 0;
    for (uint32_t r0 = warp * kGatherRows; r0 < n_rows; r0 += warps * kGatherRows) {
        // lane j looks row r0 + j up
        int64_t off = -1;
        int t = 0;
        if (lane < kGatherRows && r0 + lane < n_rows) {
            const uint32_t th = row0 + r0 + lane, i = th / Hkv;
            const int32_t slot = slots ? slots[i] : trow[i / bs] * bs + (int)(i % bs);
            if ((uint64_t)slot >= (uint64_t)num_slots) {
                atomicOr(err, kErrBounds);
            } else {
                const int32_t blk = slot / bs;
                t = slot - blk * bs;
                off = ((int64_t)blk * Hkv + (int)(th - i * Hkv)) * q4_tile_bytes(bs, D);
            }
        }
        for (int quad = lane; quad - lane < nq; quad += 32) {  // warp-uniform (shuffles inside)
            uint32_t c[kGatherRows], sm[kGatherRows];
#pragma unroll
            for (int j = 0; j < kGatherRows; j++) {
                const int64_t at = __shfl_sync(0xffffffffu, off, j);
                const int tt = __shfl_sync(0xffffffffu, t, j);
                c[j] = 0x8888u, sm[j] = 0;  // zeros where the slot is out of range
                if (at < 0 || quad >= nq) continue;
                sm[j] = *reinterpret_cast<const uint32_t*>(base + at + q4_param(tt, bs, D));
                c[j] = *reinterpret_cast<const uint16_t*>(base + at + (is_v ? q4_v_quad(tt, quad, D) : q4_k_quad(tt, quad, D)));
            }
#pragma unroll
            for (int j = 0; j < kGatherRows; j++) {
                if (r0 + j >= n_rows || quad >= nq) continue;
                const float2 p = q4_unpack(sm[j]);
                const float4 v = make_float4(q4_value(c[j] & 15u, p.x, p.y), q4_value((c[j] >> 4) & 15u, p.x, p.y),
                                             q4_value((c[j] >> 8) & 15u, p.x, p.y), q4_value(c[j] >> 12, p.x, p.y));
                float* dst = out + (int64_t)(r0 + j) * D + 4 * quad;
                if (vec) __stcs(reinterpret_cast<float4*>(dst), v);
                else dst[0] = v.x, dst[1] = v.y, dst[2] = v.z, dst[3] = v.w;
            }
        }
    }
}

int launch_gather_q4(s1kv_pool* p, int32_t layer, const int32_t* trow, const int32_t* slots, int64_t n, int which,
                     float* out, cudaStream_t stream) {
    if (n <= 0) return S1KV_OK;
    const char* base = (which ? p->v : p->k) + (size_t)layer * p->layer_bytes;
    const int64_t rows = n * p->desc.num_kv_heads;
    if (rows > UINT32_MAX) return set_error(S1KV_EINVAL, "gather: more than 2^32 rows");
    for (int64_t r0 = 0; r0 < rows; r0 += (int64_t)1 << 30) {
        const uint32_t part = (uint32_t)std::min<int64_t>((int64_t)1 << 30, rows - r0);
        const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(((int64_t)part + 8 * kGatherRows - 1) / (8 * kGatherRows), kSMs * 32));
        gather_q4_kernel<<<grid, 256, 0, stream>>>(base, which != 0, trow, slots, part, (uint32_t)r0, p->desc.block_size,
                                                   p->desc.num_kv_heads, p->desc.head_dim, p->num_slots,
                                                   out + r0 * p->desc.head_dim, p->d_err);
        g_launches++;
        S1KV_CUDA(cudaGetLastError());
    }
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

// Norms of the query and key heads, rotary embedding and the append to a paged KV cache, one pass over the qkv rows:
//     y = x * rsqrt(mean(x^2) + eps) * w            per head of HD values (optional)
//     (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)  for the rot/2 pairs of the token's own position
// query heads go to q_out (or back to their place), key and value heads to the slot of the token, in the cache's type.
//
// The pass is bound by HBM: it reads every qkv value once and writes it once, nothing else of size.  So one lane holds
// sixteen bytes of a head (HD / 8 lanes per head, one or two heads per warp), all loads of a warp's heads are issued
// before the first is used, and the tables' row of the token is read once per warp and serves all its heads.  The
// rotation's partner values come by shuffle in the input's 16-bit form (four shuffles, not eight); everything is
// computed in fp32 from the inputs and rounded once, to fp16 / bf16 or straight to e4m3.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "exl3_common.cuh"
#include "exl3_paged.cuh"

namespace exl3 {

struct AppendParams {
    void *qkv, *q_out;
    long long ld_qkv, ld_q;
    const void *q_weight, *k_weight;
    const float *cos, *sin;              // [max_pos][rot / 2]
    const long long *positions, *slots;  // [tokens]
    int tokens, qh, kvh, rot, max_pos, norm;
    float eps;
    void *k, *v;
    long long page_stride, head_stride, tok_stride;
    long long total_slots;
    int page_size;
    float k_inv_scale, v_inv_scale;
};

constexpr int kAppendWarps = 8;

template <typename T>
__device__ __forceinline__ void unpack8(const uint4 &u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = Type16<T>::to_float2(w[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

template <typename T, bool FP8>
__device__ __forceinline__ void store8(void *base, long long off, const float (&f)[8], float inv_scale) {
    if constexpr (FP8) {
        const uint2 r = make_uint2(e4m3x4(f[0] * inv_scale, f[1] * inv_scale, f[2] * inv_scale, f[3] * inv_scale),
                                   e4m3x4(f[4] * inv_scale, f[5] * inv_scale, f[6] * inv_scale, f[7] * inv_scale));
        *reinterpret_cast<uint2 *>(static_cast<unsigned char *>(base) + off) = r;
    } else {
        uint4 r;
        r.x = Type16<T>::pack(f[0], f[1]); r.y = Type16<T>::pack(f[2], f[3]);
        r.z = Type16<T>::pack(f[4], f[5]); r.w = Type16<T>::pack(f[6], f[7]);
        *reinterpret_cast<uint4 *>(static_cast<T *>(base) + off) = r;
    }
}

template <typename T, bool FP8, int HD, bool ADJACENT>
__global__ void __launch_bounds__(kAppendWarps * 32) qk_norm_rope_append_kernel(const __grid_constant__ AppendParams P) {
    constexpr int kLanes = HD / 8;            // lanes of a head
    constexpr int kPer = 32 / kLanes;         // heads of a warp
    constexpr int kBatch = 4;                 // heads in flight per lane
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane / kLanes, l = lane - sub * kLanes;
    const int heads = P.qh + 2 * P.kvh;
    const int t = blockIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");

    T *const row = static_cast<T *>(P.qkv) + (size_t)t * P.ld_qkv;
    const long long pos = __ldg(P.positions + t), slot = __ldg(P.slots + t);
    const bool pos_ok = pos >= 0 && pos < P.max_pos;         // otherwise the token is left as it is
    const bool slot_ok = slot >= 0 && slot < P.total_slots;  // otherwise nothing is appended

    // this lane's part of the table row, and its partner lane: half form: elements e and e +- rot/2, frequency
    // e mod rot/2; adjacent form: pairs inside the lane, frequencies 4 l .. 4 l + 3
    const int half = P.rot >> 1;
    const bool turn = 8 * l < P.rot;
    const bool upper = 8 * l >= half;
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { c[i] = 1.f; s[i] = 0.f; }
    if (turn && pos_ok) {
        if constexpr (ADJACENT) {
            const float4 c4 = __ldg(reinterpret_cast<const float4 *>(P.cos + pos * half + 4 * l));
            const float4 s4 = __ldg(reinterpret_cast<const float4 *>(P.sin + pos * half + 4 * l));
            c[0] = c4.x; c[1] = c4.y; c[2] = c4.z; c[3] = c4.w;
            s[0] = s4.x; s[1] = s4.y; s[2] = s4.z; s[3] = s4.w;
        } else {
            const long long at = pos * half + 8 * l - (upper ? half : 0);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float4 c4 = __ldg(reinterpret_cast<const float4 *>(P.cos + at) + i);
                const float4 s4 = __ldg(reinterpret_cast<const float4 *>(P.sin + at) + i);
                c[4 * i] = c4.x; c[4 * i + 1] = c4.y; c[4 * i + 2] = c4.z; c[4 * i + 3] = c4.w;
                s[4 * i] = s4.x; s[4 * i + 1] = s4.y; s[4 * i + 2] = s4.z; s[4 * i + 3] = s4.w;
            }
        }
    }
    const int shift = ADJACENT || !turn ? 0 : (upper ? -(half >> 3) : (half >> 3));
    const int partner = lane + shift;
    const float sign = upper ? 1.f : -1.f;

    long long dst_off = 0;
    if (slot_ok) {
        const long long page = slot / P.page_size;
        dst_off = page * P.page_stride + (slot - page * P.page_size) * P.tok_stride + 8 * l;
    }

    for (int u0 = warp * kPer; u0 < heads; u0 += kBatch * kAppendWarps * kPer) {
        uint4 x[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int h = u0 + j * kAppendWarps * kPer + sub;
            x[j] = h < heads ? *reinterpret_cast<const uint4 *>(row + (size_t)h * HD + 8 * l) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int first = u0 + j * kAppendWarps * kPer;           // uniform in the warp
            if (first >= heads) break;
            const int h = first + sub;
            float y[8], r = 1.f;
            unpack8<T>(x[j], y);
            if (P.norm) {
                float q = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) q += y[i] * y[i];
#pragma unroll
                for (int o = kLanes / 2; o; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
                r = rsqrtf(q * (1.f / HD) + P.eps);
            }
            uint4 px = make_uint4(0, 0, 0, 0);
            if constexpr (!ADJACENT) {
                px.x = __shfl_sync(0xffffffffu, x[j].x, partner);
                px.y = __shfl_sync(0xffffffffu, x[j].y, partner);
                px.z = __shfl_sync(0xffffffffu, x[j].z, partner);
                px.w = __shfl_sync(0xffffffffu, x[j].w, partner);
            }
            if (h >= heads || !pos_ok) continue;
            if (h >= P.qh + P.kvh) {                                  // value head
                if (slot_ok) store8<T, FP8>(P.v, dst_off + (h - P.qh - P.kvh) * P.head_stride, y, P.v_inv_scale);
                continue;
            }
            const bool is_q = h < P.qh;
            if (!is_q && !slot_ok) continue;
            const T *w = static_cast<const T *>(is_q ? P.q_weight : P.k_weight);
            const bool weighted = P.norm && w != nullptr;
            if (weighted) {
                float g[8];
                unpack8<T>(__ldg(reinterpret_cast<const uint4 *>(w + 8 * l)), g);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] *= r * g[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] *= r;
            }
            if (turn) {
                if constexpr (ADJACENT) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float a = y[2 * i], b = y[2 * i + 1];
                        y[2 * i] = a * c[i] - b * s[i];
                        y[2 * i + 1] = b * c[i] + a * s[i];
                    }
                } else {
                    float z[8];
                    unpack8<T>(px, z);
                    if (weighted) {
                        float g[8];
                        unpack8<T>(__ldg(reinterpret_cast<const uint4 *>(w + 8 * (l + shift))), g);
#pragma unroll
                        for (int i = 0; i < 8; ++i) z[i] *= r * g[i];
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) z[i] *= r;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = y[i] * c[i] + sign * z[i] * s[i];
                }
            }
            if (is_q)
                store8<T, false>(P.q_out, (long long)t * P.ld_q + (long long)h * HD + 8 * l, y, 1.f);
            else
                store8<T, FP8>(P.k, dst_off + (h - P.qh) * P.head_stride, y, P.k_inv_scale);
        }
    }
}

template <typename T, bool FP8, int HD>
static cudaError_t launch_append(const AppendParams &P, bool adjacent, cudaStream_t st) {
    auto kernel = adjacent ? qk_norm_rope_append_kernel<T, FP8, HD, true> : qk_norm_rope_append_kernel<T, FP8, HD, false>;
    return launch_pdl(kernel, dim3(P.tokens), dim3(kAppendWarps * 32), 0, st, P);
}

}  // namespace exl3

extern "C" int exl3_qk_norm_rope_append(void *qkv, long long ld_qkv, void *q_out, long long ld_q_out, const void *q_weight,
                                        const void *k_weight, int norm, float eps, const void *cos, const void *sin,
                                        int rot_dim, int interleaved, int max_pos, const void *positions, const void *slots,
                                        int tokens, int q_heads, int is_bf16, const exl3_paged_cache *cache, void *stream) {
    using namespace exl3;
    if (!cache || !positions || !slots || !qkv || (rot_dim && (!cos || !sin))) return EXL3_E_NULL;
    int rc = check_cache(*cache, is_bf16, false);
    if (rc != EXL3_OK) return rc;
    const int hd = cache->head_dim, kvh = cache->kv_heads;
    if (tokens < 0 || q_heads <= 0 || q_heads > 65535 || (ld_qkv & 7) || ld_qkv < (long long)(q_heads + 2 * kvh) * hd ||
        rot_dim < 0 || rot_dim > hd || (rot_dim & 15) || max_pos <= 0 || (norm && !(eps >= 0.f)))
        return EXL3_E_SHAPE;
    if (q_out && ((ld_q_out & 7) || ld_q_out < (long long)q_heads * hd)) return EXL3_E_SHAPE;
    if (!aligned(qkv, 16) || !aligned(q_out, 16) || !aligned(q_weight, 16) || !aligned(k_weight, 16) || !aligned(cos, 16) ||
        !aligned(sin, 16) || !aligned(positions, 8) || !aligned(slots, 8))
        return EXL3_E_ALIGN;
    if (tokens == 0) return EXL3_OK;
    AppendParams P = {};
    P.qkv = qkv; P.ld_qkv = ld_qkv;
    P.q_out = q_out ? q_out : qkv; P.ld_q = q_out ? ld_q_out : ld_qkv;
    P.q_weight = q_weight; P.k_weight = k_weight;
    P.cos = (const float *)cos; P.sin = (const float *)sin;
    P.positions = (const long long *)positions; P.slots = (const long long *)slots;
    P.tokens = tokens; P.qh = q_heads; P.kvh = kvh; P.rot = rot_dim; P.max_pos = max_pos; P.norm = norm; P.eps = eps;
    P.k = cache->k_pages; P.v = cache->v_pages;
    P.page_stride = cache->page_stride; P.head_stride = cache->head_stride; P.tok_stride = cache->token_stride;
    P.page_size = cache->page_size;
    P.total_slots = (long long)cache->num_pages * cache->page_size;
    P.k_inv_scale = 1.f / cache->k_scale; P.v_inv_scale = 1.f / cache->v_scale;
    const bool fp8 = cache->dtype == EXL3_KV_E4M3, adj = interleaved != 0;
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (hd == 256)
        e = is_bf16 ? (fp8 ? launch_append<__nv_bfloat16, true, 256>(P, adj, st) : launch_append<__nv_bfloat16, false, 256>(P, adj, st))
                    : (fp8 ? launch_append<__half, true, 256>(P, adj, st) : launch_append<__half, false, 256>(P, adj, st));
    else
        e = is_bf16 ? (fp8 ? launch_append<__nv_bfloat16, true, 128>(P, adj, st) : launch_append<__nv_bfloat16, false, 128>(P, adj, st))
                    : (fp8 ? launch_append<__half, true, 128>(P, adj, st) : launch_append<__half, false, 128>(P, adj, st));
    if (e != cudaSuccess) return EXL3_E_LAUNCH;
    return launch_status();
}

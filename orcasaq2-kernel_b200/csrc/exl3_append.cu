// Norms of the query and key heads, rotary embedding and the append to a paged KV cache, one pass over the qkv rows:
//     y = x * rsqrt(mean(x^2) + eps) * w            per head of HD values (optional)
//     (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)  for the rot/2 pairs of the token's own position
// query heads go to q_out (or back to their place), key and value heads to the slot of the token, in the cache's type.
//
// The pass is bound by HBM: it reads every qkv value once and writes it once, nothing else of size.  One lane holds
// sixteen bytes of a head (HD / 8 lanes per head, one or two heads per warp), and the loads of four heads are issued
// before the first is used.  What it takes to stay at that bound is few instructions per value: weight, cosine and sine
// are multiplied once per token and kind of head (a = w_i c_i, b = +- w_partner s_i), a head then costs
// r (x a + x_partner b) in packed fp32, the partner values come by shuffle in the input's 16-bit form, and four heads'
// sums of squares are reduced together (ten shuffles instead of twenty), while the loads of the next four are in flight.
// 16384 tokens of 24 / 4 heads of 256: 100 us, 5.5 TB/s, 85 % of the measured copy rate (one head after the other with
// its weights read beside it: 163 us).  Few tokens take a CTA each instead of a warp, since then latency counts.
// Everything is computed in fp32 from the inputs and rounded once, to fp16 / bf16 or straight to e4m3.
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
    float k_scale, v_scale;              // e4m3 pools hold value / scale
};

constexpr int kAppendWarps = 8;
constexpr int kFewTokens = 1024;

template <typename T>
__device__ __forceinline__ void unpack8(const uint4 &u, float2 (&f)[4]) {
    f[0] = Type16<T>::to_float2(u.x); f[1] = Type16<T>::to_float2(u.y);
    f[2] = Type16<T>::to_float2(u.z); f[3] = Type16<T>::to_float2(u.w);
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

// e4m3: the quotient itself (times the reciprocal, values at the border between two e4m3 numbers went to the wrong one, and a
// scale below 2^-128 has no reciprocal).
template <typename T, bool FP8>
__device__ __forceinline__ void store8(void *base, long long off, const float2 (&f)[4], float scale) {
    if constexpr (FP8) {
        const uint2 r = make_uint2(e4m3x4(f[0].x / scale, f[0].y / scale, f[1].x / scale, f[1].y / scale),
                                   e4m3x4(f[2].x / scale, f[2].y / scale, f[3].x / scale, f[3].y / scale));
        *reinterpret_cast<uint2 *>(static_cast<unsigned char *>(base) + off) = r;
    } else {
        const uint4 r = make_uint4(Type16<T>::pack(f[0].x, f[0].y), Type16<T>::pack(f[1].x, f[1].y),
                                   Type16<T>::pack(f[2].x, f[2].y), Type16<T>::pack(f[3].x, f[3].y));
        *reinterpret_cast<uint4 *>(static_cast<T *>(base) + off) = r;
    }
}

// Sums of four values over groups of kLanes lanes, in every lane.
template <int kLanes>
__device__ __forceinline__ void reduce4(float (&q)[4], int lane) {
    // each step of the first two halves the number of values a lane carries: lane bits 0 and 1 say which it keeps
    const bool b0 = lane & 1, b1 = lane & 2;
    float k0 = b0 ? q[1] : q[0], k1 = b0 ? q[3] : q[2];
    k0 += __shfl_xor_sync(0xffffffffu, b0 ? q[0] : q[1], 1);
    k1 += __shfl_xor_sync(0xffffffffu, b0 ? q[2] : q[3], 1);
    float v = b1 ? k1 : k0;
    v += __shfl_xor_sync(0xffffffffu, b1 ? k0 : k1, 2);
#pragma unroll
    for (int o = 4; o < kLanes; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int base = lane & ~3;                                // lanes base .. base + 3 have the sums of values 0 .. 3
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = __shfl_sync(0xffffffffu, v, base + j);
}

// This lane's cosines and signed sines at position pos.
template <bool ADJACENT>
__device__ __forceinline__ void table_row(const AppendParams &P, long long pos, int l, int half, bool upper, float2 (&c)[4], float2 (&s)[4]) {
    if constexpr (ADJACENT) {
        const float4 c4 = __ldg(reinterpret_cast<const float4 *>(P.cos + pos * half + 4 * l));
        const float4 s4 = __ldg(reinterpret_cast<const float4 *>(P.sin + pos * half + 4 * l));
        c[0] = make_float2(c4.x, c4.x); c[1] = make_float2(c4.y, c4.y); c[2] = make_float2(c4.z, c4.z); c[3] = make_float2(c4.w, c4.w);
        s[0] = make_float2(-s4.x, s4.x); s[1] = make_float2(-s4.y, s4.y); s[2] = make_float2(-s4.z, s4.z); s[3] = make_float2(-s4.w, s4.w);
    } else {
        const long long at = pos * half + 8 * l - (upper ? half : 0);
        const float sign = upper ? 1.f : -1.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float4 c4 = __ldg(reinterpret_cast<const float4 *>(P.cos + at) + i);
            const float4 s4 = __ldg(reinterpret_cast<const float4 *>(P.sin + at) + i);
            c[2 * i] = make_float2(c4.x, c4.y); c[2 * i + 1] = make_float2(c4.z, c4.w);
            s[2 * i] = make_float2(sign * s4.x, sign * s4.y); s[2 * i + 1] = make_float2(sign * s4.z, sign * s4.w);
        }
    }
}
// Cosines times this lane's weights, sines times its partner's.
template <typename T, bool ADJACENT>
__device__ __forceinline__ void weigh(const T *w, int l, int shift, float2 (&a)[4], float2 (&b)[4]) {
    float2 g[4], p[4];
    unpack8<T>(__ldg(reinterpret_cast<const uint4 *>(w + 8 * l)), g);
    unpack8<T>(__ldg(reinterpret_cast<const uint4 *>(w + 8 * (l + shift))), p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = mul2(a[i], g[i]);
        b[i] = mul2(b[i], ADJACENT ? make_float2(g[i].y, g[i].x) : p[i]);
    }
}

// Few tokens: a CTA per token, its eight warps share the heads of all kinds, and what a head needs beside its values
// (weights, its partner's too) is read with it: more instructions per value, but one load latency from end to end.
template <typename T, bool FP8, int HD, bool ADJACENT>
__global__ void __launch_bounds__(kAppendWarps * 32) append_token_kernel(const __grid_constant__ AppendParams P) {
    constexpr int kLanes = HD / 8;            // lanes of a head
    constexpr int kPer = 32 / kLanes;         // heads of a warp
    constexpr int kFly = 4;                   // heads in flight per lane
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane / kLanes, l = lane - sub * kLanes;
    const int heads = P.qh + 2 * P.kvh, t = blockIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");

    T *const row = static_cast<T *>(P.qkv) + (size_t)t * P.ld_qkv + 8 * l;
    const long long pos = __ldg(P.positions + t), slot = __ldg(P.slots + t);
    const bool pos_ok = pos >= 0 && pos < P.max_pos, slot_ok = slot >= 0 && slot < P.total_slots;
    const int half = P.rot >> 1;
    const bool turn = 8 * l < P.rot, upper = 8 * l >= half;
    const int shift = ADJACENT || !turn ? 0 : (upper ? -(half >> 3) : (half >> 3));
    float2 c[4], s[4];                        // per element, the sine with the sign of its term
#pragma unroll
    for (int i = 0; i < 4; ++i) { c[i] = make_float2(1.f, 1.f); s[i] = make_float2(0.f, 0.f); }
    if (turn && pos_ok) table_row<ADJACENT>(P, pos, l, half, upper, c, s);
    long long dst_off = 0;
    if (slot_ok) {
        const long long page = slot / P.page_size;
        dst_off = page * P.page_stride + (slot - page * P.page_size) * P.tok_stride + 8 * l;
    }
#pragma unroll 1
    for (int u0 = warp * kPer; u0 < heads; u0 += kFly * kAppendWarps * kPer) {
        uint4 x[kFly];
#pragma unroll
        for (int j = 0; j < kFly; ++j) {
            const int h = u0 + j * kAppendWarps * kPer + sub;
            x[j] = h < heads ? *reinterpret_cast<const uint4 *>(row + (size_t)h * HD) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < kFly; ++j) {
            const int first = u0 + j * kAppendWarps * kPer;          // uniform in the warp
            if (first >= heads) break;
            const int h = first + sub;
            float2 y[4], z[4];
            float r = 1.f;
            unpack8<T>(x[j], y);
            if (P.norm) {
                float2 q = make_float2(0.f, 0.f);
#pragma unroll
                for (int i = 0; i < 4; ++i) q = fma2(y[i], y[i], q);
                float sum = q.x + q.y;
#pragma unroll
                for (int o = kLanes / 2; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                r = rsqrtf(sum * (1.f / HD) + P.eps);
            }
            if constexpr (!ADJACENT) {
                uint4 px;
                px.x = __shfl_sync(0xffffffffu, x[j].x, lane + shift);
                px.y = __shfl_sync(0xffffffffu, x[j].y, lane + shift);
                px.z = __shfl_sync(0xffffffffu, x[j].z, lane + shift);
                px.w = __shfl_sync(0xffffffffu, x[j].w, lane + shift);
                unpack8<T>(px, z);
            }
            if (h >= heads || !pos_ok) continue;
            if (h >= P.qh + P.kvh) {                                 // value head
                if (!slot_ok) continue;
                const long long to = dst_off + (h - P.qh - P.kvh) * P.head_stride;
                if constexpr (FP8) store8<T, true>(P.v, to, y, P.v_scale);
                else *reinterpret_cast<uint4 *>(static_cast<T *>(P.v) + to) = x[j];
                continue;
            }
            const bool is_q = h < P.qh;
            if (!is_q && !slot_ok) continue;
            const T *const w = static_cast<const T *>(is_q ? P.q_weight : P.k_weight);
            float2 a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { a[i] = c[i]; b[i] = s[i]; }
            if (P.norm && w) weigh<T, ADJACENT>(w, l, shift, a, b);
            const float2 rr = make_float2(r, r);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 m = mul2(y[i], a[i]), other = ADJACENT ? make_float2(y[i].y, y[i].x) : z[i];
                y[i] = mul2(turn ? fma2(other, b[i], m) : m, rr);
            }
            if (is_q)
                store8<T, false>(P.q_out, (long long)t * P.ld_q + (long long)h * HD + 8 * l, y, 1.f);
            else
                store8<T, FP8>(P.k, dst_off + (h - P.qh) * P.head_stride, y, P.k_scale);
        }
    }
}

// Many tokens: a warp per token.
template <typename T, bool FP8, int HD, bool ADJACENT>
__global__ void __launch_bounds__(kAppendWarps * 32, 3) append_stream_kernel(const __grid_constant__ AppendParams P) {
    constexpr int kLanes = HD / 8;            // lanes of a head
    constexpr int kPer = 32 / kLanes;         // heads of a warp
    constexpr int kFly = 4;                   // heads in flight per lane
    const int lane = threadIdx.x & 31;
    const int sub = lane / kLanes, l = lane - sub * kLanes;
    const int t = blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    if (t >= P.tokens) return;

    T *const row = static_cast<T *>(P.qkv) + (size_t)t * P.ld_qkv + 8 * l;
    const long long at_pos = __ldg(P.positions + t), slot = __ldg(P.slots + t);
    const bool slot_ok = slot >= 0 && slot < P.total_slots;  // otherwise nothing is appended
    if (at_pos < 0 || at_pos >= P.max_pos) return;           // the token is left as it is
    const int pos = (int)at_pos;

    // this lane's part of the table row, and its partner lane: half form: elements e and e +- rot/2, frequency
    // e mod rot/2; adjacent form: pairs inside the lane, frequencies 4 l .. 4 l + 3
    const int half = P.rot >> 1;
    const bool turn = 8 * l < P.rot, upper = 8 * l >= half;
    const int shift = ADJACENT || !turn ? 0 : (upper ? -(half >> 3) : (half >> 3));
    long long dst_off = 0;
    if (slot_ok) {
        const long long page = slot / P.page_size;
        dst_off = page * P.page_stride + (slot - page * P.page_size) * P.tok_stride + 8 * l;
    }

    // The heads in batches of kFly units of this warp (a unit: kPer heads), all of a kind: query, key, value.  The loads of
    // a batch are issued before the one ahead of it is worked on.
    const int units_q = (P.qh + kPer - 1) / kPer, units_kv = (P.kvh + kPer - 1) / kPer;
    const int nq = (units_q + kFly - 1) / kFly, nk = slot_ok ? (units_kv + kFly - 1) / kFly : 0, batches = nq + 2 * nk;
    const auto kind_of = [&](int n, int &u0) {               // kind of batch n, its first unit
        const int kind = n < nq ? 0 : n < nq + nk ? 1 : 2;
        u0 = (n - (kind == 0 ? 0 : kind == 1 ? nq : nq + nk)) * kFly;
        return kind;
    };
    const auto load = [&](int n, uint4 (&x)[kFly]) {
        int u0;
        const int kind = kind_of(n, u0), heads = kind ? P.kvh : P.qh;
        const T *const from = row + (size_t)(kind == 0 ? 0 : kind == 1 ? P.qh : P.qh + P.kvh) * HD;
#pragma unroll
        for (int j = 0; j < kFly; ++j) {
            const int h = (u0 + j) * kPer + sub;
            x[j] = h < heads ? *reinterpret_cast<const uint4 *>(from + (size_t)h * HD) : make_uint4(0, 0, 0, 0);
        }
    };
    uint4 x[kFly], ahead[kFly];
    load(0, ahead);
    float2 a[4], b[4];                                       // y = r (x a + x_partner b)
    const auto factors = [&](const T *w) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { a[i] = make_float2(1.f, 1.f); b[i] = make_float2(0.f, 0.f); }
        if (turn) table_row<ADJACENT>(P, pos, l, half, upper, a, b);
        if (P.norm && w) weigh<T, ADJACENT>(w, l, shift, a, b);
    };
#pragma unroll 1
    for (int n = 0; n < batches; ++n) {
        int u0;
        const int kind = kind_of(n, u0), heads = kind ? P.kvh : P.qh;
#pragma unroll
        for (int j = 0; j < kFly; ++j) x[j] = ahead[j];
        if (n + 1 < batches) load(n + 1, ahead);
        if (kind == 2) {
#pragma unroll
            for (int j = 0; j < kFly; ++j) {
                const int h = (u0 + j) * kPer + sub;
                if (h >= heads) continue;
                if constexpr (FP8) {
                    float2 y[4];
                    unpack8<T>(x[j], y);
                    store8<T, true>(P.v, dst_off + h * P.head_stride, y, P.v_scale);
                } else {
                    *reinterpret_cast<uint4 *>(static_cast<T *>(P.v) + dst_off + h * P.head_stride) = x[j];
                }
            }
            continue;
        }
        if (n == 0 || n == nq) factors(static_cast<const T *>(kind ? P.k_weight : P.q_weight));
        float r[kFly] = {1.f, 1.f, 1.f, 1.f};
        if (P.norm) {
#pragma unroll
            for (int j = 0; j < kFly; ++j) {
                float2 y[4], q = make_float2(0.f, 0.f);
                unpack8<T>(x[j], y);
#pragma unroll
                for (int i = 0; i < 4; ++i) q = fma2(y[i], y[i], q);
                r[j] = q.x + q.y;
            }
            reduce4<kLanes>(r, lane);
#pragma unroll
            for (int j = 0; j < kFly; ++j) r[j] = rsqrtf(r[j] * (1.f / HD) + P.eps);
        }
#pragma unroll
        for (int j = 0; j < kFly; ++j) {
            const int h = (u0 + j) * kPer + sub;
            float2 y[4], z[4];
            unpack8<T>(x[j], y);
            if constexpr (ADJACENT) {
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = make_float2(y[i].y, y[i].x);
            } else {
                uint4 px;
                px.x = __shfl_sync(0xffffffffu, x[j].x, lane + shift);
                px.y = __shfl_sync(0xffffffffu, x[j].y, lane + shift);
                px.z = __shfl_sync(0xffffffffu, x[j].z, lane + shift);
                px.w = __shfl_sync(0xffffffffu, x[j].w, lane + shift);
                unpack8<T>(px, z);
            }
            const float2 rr = make_float2(r[j], r[j]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // (a rotated pair only: an infinity times a zero sine must not reach the others)
                const float2 m = mul2(y[i], a[i]);
                y[i] = mul2(turn ? fma2(z[i], b[i], m) : m, rr);
            }
            if (h >= heads) continue;
            if (kind == 0)
                store8<T, false>(P.q_out, (long long)t * P.ld_q + (long long)h * HD + 8 * l, y, 1.f);
            else
                store8<T, FP8>(P.k, dst_off + h * P.head_stride, y, P.k_scale);
        }
    }
}

template <typename T, bool FP8, int HD>
static cudaError_t launch_append(const AppendParams &P, bool adjacent, cudaStream_t st) {
    // Measured with 24 / 4 heads of 256 (us, a CTA per token against a warp per token): 4.2 / 10.4 at 5 tokens, 10.7 / 11.7 at
    // 1024 into an e4m3 cache, 14.3 / 14.4 at 1024 and 24.6 / 20.6 at 2048 into an fp16 one, 163 / 100 at 16384.  The crossing
    // lies at about 1024 for 16-bit caches and somewhat above for e4m3 ones, where the one threshold for both costs up to 1 us.
    if (P.tokens <= kFewTokens) {
        auto kernel = adjacent ? append_token_kernel<T, FP8, HD, true> : append_token_kernel<T, FP8, HD, false>;
        return launch_pdl(kernel, dim3(P.tokens), dim3(kAppendWarps * 32), 0, st, P);
    }
    auto kernel = adjacent ? append_stream_kernel<T, FP8, HD, true> : append_stream_kernel<T, FP8, HD, false>;
    return launch_pdl(kernel, dim3((P.tokens + kAppendWarps - 1) / kAppendWarps), dim3(kAppendWarps * 32), 0, st, P);
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
    if (tokens < 0 || tokens > (1 << 27) || q_heads <= 0 || q_heads > 65535 || (ld_qkv & 7) || ld_qkv < (long long)(q_heads + 2 * kvh) * hd ||
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
    P.k_scale = cache->k_scale; P.v_scale = cache->v_scale;
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

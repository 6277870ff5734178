// Attention of a tree of drafted tokens over a paged KV cache (exl3_tree_attn): one warp per draft and query head.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "exl3_common.cuh"
#include "exl3_paged.cuh"

namespace exl3 {

struct TreeParams {
    const void *q;
    void *out;
    long long q_stride, out_stride;
    const void *k, *v;
    long long page_stride, head_stride, tok_stride;
    const int *block_table, *seq_lens, *starts;
    const long long *mask;
    int bt_stride, width, num_pages, page_size;
    int batch, tokens, max_drafts, qh, kvh, G;
    float scale_log2, v_scale;
};

template <typename T, bool FP8, int HD>
__global__ void __launch_bounds__(128) tree_attn_kernel(const __grid_constant__ TreeParams P) {
    constexpr int kPer = HD / 32;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = blockIdx.z, i = blockIdx.y, h = blockIdx.x * 4 + warp;
    const int first = max(0, min(P.starts[b], P.tokens));
    const int n = max(0, min(P.starts[b + 1], P.tokens) - first);
    if (i >= n || i >= P.max_drafts || h >= P.qh) return;
    const int len = (int)min((long long)max(P.seq_lens[b], 0), (long long)P.width * P.page_size);
    const int ctx = len - n;
    const unsigned long long m = P.mask ? (unsigned long long)P.mask[first + i] : (i == 63 ? ~0ull : (2ull << i) - 1);
    const T *q = static_cast<const T *>(P.q) + (size_t)(first + i) * P.q_stride + (size_t)h * HD;
    float x[kPer], o[kPer], top = -INFINITY, sum = 0.f;
    for (int d = 0; d < kPer; ++d) { x[d] = (float)q[lane + 32 * d]; o[d] = 0.f; }
    for (int t = 0; t < len; ++t) {
        if (t >= ctx && !(m >> (t - ctx) & 1)) continue;
        const int page = P.block_table[(size_t)b * P.bt_stride + t / P.page_size];
        if (page < 0 || page >= P.num_pages) continue;
        const size_t off = (size_t)page * P.page_stride + (size_t)(h / P.G) * P.head_stride + (size_t)(t % P.page_size) * P.tok_stride;
        float s = 0.f, v[kPer];
        for (int d = 0; d < kPer; ++d) {
            if constexpr (FP8) {
                s += x[d] * (float)static_cast<const __nv_fp8_e4m3 *>(P.k)[off + lane + 32 * d];
                v[d] = (float)static_cast<const __nv_fp8_e4m3 *>(P.v)[off + lane + 32 * d];
            } else {
                s += x[d] * (float)static_cast<const T *>(P.k)[off + lane + 32 * d];
                v[d] = (float)static_cast<const T *>(P.v)[off + lane + 32 * d];
            }
        }
        for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
        s *= P.scale_log2;
        const float up = fmaxf(top, s);
        const float c = top == -INFINITY ? 0.f : exp2f(top - up), p = s == -INFINITY ? 0.f : exp2f(s - up);
        top = up;
        sum = sum * c + p;
        for (int d = 0; d < kPer; ++d) o[d] = o[d] * c + p * v[d];
    }
    const float inv = sum == 0.f ? 0.f : P.v_scale / sum;
    T *out = static_cast<T *>(P.out) + (size_t)(first + i) * P.out_stride + (size_t)h * HD;
    for (int d = 0; d < kPer; ++d) out[lane + 32 * d] = (T)(o[d] * inv);
}

}  // namespace exl3

extern "C" size_t exl3_tree_attn_workspace_bytes(int batch, int q_heads, int max_drafts, const exl3_paged_cache *cache) {
    return 0;
}

extern "C" int exl3_tree_attn(const void *q, long long q_stride, void *out, long long out_stride, const void *block_table,
                              int table_stride, int table_width, const void *seq_lens, const void *starts,
                              const void *mask, int batch, int tokens, int max_drafts, int q_heads, float scale,
                              int is_bf16, const exl3_paged_cache *cache, void *workspace, size_t workspace_bytes,
                              void *stream) {
    using namespace exl3;
    if (!q || !out || !block_table || !seq_lens || !starts || !cache) return EXL3_E_NULL;
    const int rc = check_cache(*cache, is_bf16, true);
    if (rc != EXL3_OK) return rc;
    const int hd = cache->head_dim, kvh = cache->kv_heads;
    if (batch < 0 || batch > 65535 || tokens < 0 || q_heads <= 0 || q_heads > 65535 || q_heads % kvh || table_width <= 0 ||
        table_stride < table_width || (long long)table_width * cache->page_size > INT32_MAX || (q_stride & 7) ||
        (out_stride & 7) || q_stride < (long long)q_heads * hd || out_stride < (long long)q_heads * hd ||
        max_drafts < 1 || max_drafts > EXL3_TREE_MAX_DRAFTS)
        return EXL3_E_SHAPE;
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(block_table, 4) || !aligned(seq_lens, 4) || !aligned(starts, 4) ||
        !aligned(mask, 8))
        return EXL3_E_ALIGN;
    if (batch == 0 || tokens == 0) return EXL3_OK;
    TreeParams P = {};
    P.q = q; P.out = out; P.q_stride = q_stride; P.out_stride = out_stride;
    P.k = cache->k_pages; P.v = cache->v_pages;
    P.page_stride = cache->page_stride; P.head_stride = cache->head_stride; P.tok_stride = cache->token_stride;
    P.block_table = (const int *)block_table; P.seq_lens = (const int *)seq_lens; P.starts = (const int *)starts;
    P.mask = (const long long *)mask;
    P.bt_stride = table_stride; P.width = table_width; P.num_pages = cache->num_pages; P.page_size = cache->page_size;
    P.batch = batch; P.tokens = tokens; P.max_drafts = max_drafts; P.qh = q_heads; P.kvh = kvh; P.G = q_heads / kvh;
    P.scale_log2 = scale * cache->k_scale * 1.4426950408889634f; P.v_scale = cache->v_scale;
    const bool fp8 = cache->dtype == EXL3_KV_E4M3;
    auto kernel = is_bf16 ? (hd == 256 ? (fp8 ? tree_attn_kernel<__nv_bfloat16, true, 256> : tree_attn_kernel<__nv_bfloat16, false, 256>)
                                       : (fp8 ? tree_attn_kernel<__nv_bfloat16, true, 128> : tree_attn_kernel<__nv_bfloat16, false, 128>))
                          : (hd == 256 ? (fp8 ? tree_attn_kernel<__half, true, 256> : tree_attn_kernel<__half, false, 256>)
                                       : (fp8 ? tree_attn_kernel<__half, true, 128> : tree_attn_kernel<__half, false, 128>));
    if (launch_pdl(kernel, dim3((q_heads + 3) / 4, max_drafts, batch), dim3(128), 0, (cudaStream_t)stream, P) != cudaSuccess)
        return EXL3_E_LAUNCH;
    return launch_status();
}

// What the kernels over paged KV caches share: the 16-bit value types, the checks of a cache description.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "exl3_common.cuh"

namespace exl3 {

template <typename T>
struct Type16;
template <>
struct Type16<__half> {
    static __device__ __forceinline__ float2 to_float2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};
template <>
struct Type16<__nv_bfloat16> {
    static __device__ __forceinline__ float2 to_float2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};

// Two fp32 operations at a time.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// Head size, strides, alignment and scales of a paged cache; the values around it are fp16, or bf16 when is_bf16.
// tiles: the tokens of a page are read in tiles of sixteen.
inline int check_cache(const exl3_paged_cache &c, int is_bf16, bool tiles) {
    if (!c.k_pages || !c.v_pages) return EXL3_E_NULL;
    if (c.head_dim != 128 && c.head_dim != 256) return EXL3_E_UNSUPPORTED;
    if (c.dtype != EXL3_KV_E4M3 && c.dtype != (is_bf16 ? EXL3_KV_BF16 : EXL3_KV_F16)) return EXL3_E_UNSUPPORTED;
    const long long amask = c.dtype == EXL3_KV_E4M3 ? 15 : 7;
    if (c.num_pages <= 0 || c.page_size <= 0 || c.kv_heads <= 0 || c.kv_heads > 65535 || (tiles && (c.page_size & 15)) ||
        c.page_stride <= 0 || c.head_stride <= 0 || c.token_stride < c.head_dim || (c.page_stride & amask) ||
        (c.head_stride & amask) || (c.token_stride & amask) || !(c.k_scale > 0.f) || !(c.v_scale > 0.f) ||
        c.k_scale > 3e38f || c.v_scale > 3e38f)
        return EXL3_E_SHAPE;
    if (!aligned(c.k_pages, 16) || !aligned(c.v_pages, 16)) return EXL3_E_ALIGN;
    return EXL3_OK;
}

}  // namespace exl3

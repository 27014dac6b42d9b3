// Eight consecutive elements of a row, loaded and stored as f32 whatever the row's type.
#pragma once

#include "common.hpp"

namespace th {

struct kv_f8 { float v[8]; };

template <typename X>
__device__ __forceinline__ kv_f8 kv_load8(const X* p) {
    kv_f8 r;
    if constexpr (sizeof(X) == 4) {
        const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
        r = kv_f8{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
    } else {
        typedef X x8 __attribute__((ext_vector_type(8)));
        const x8 a = *(const x8*)p;
#pragma unroll
        for (int i = 0; i < 8; i++) r.v[i] = (float)a[i];
    }
    return r;
}

template <typename Y>
__device__ __forceinline__ void kv_put8(Y* p, const kv_f8& r) {
    if constexpr (sizeof(Y) == 4) {
        ((float4*)p)[0] = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
        ((float4*)p)[1] = make_float4(r.v[4], r.v[5], r.v[6], r.v[7]);
    } else {
        typedef Y y8 __attribute__((ext_vector_type(8)));
        y8 a;
#pragma unroll
        for (int i = 0; i < 8; i++) a[i] = (Y)r.v[i];
        *(y8*)p = a;
    }
}

__device__ __forceinline__ void kv_store8(void* base, th_dtype dt, size_t at, const kv_f8& r) {
    if (dt == TH_F32) kv_put8((float*)base + at, r);
    else if (dt == TH_F16) kv_put8((_Float16*)base + at, r);
    else kv_put8((__bf16*)base + at, r);
}

__device__ __forceinline__ void kv_store1(void* base, th_dtype dt, size_t at, float v) {
    if (dt == TH_F32) ((float*)base)[at] = v;
    else if (dt == TH_F16) ((_Float16*)base)[at] = (_Float16)v;
    else ((__bf16*)base)[at] = (__bf16)v;
}

}  // namespace th

// pieces.hpp - pieces of 8 neighbouring elements of a row, fp32 or bf16, at any
// address that is a multiple of the element's size.
#pragma once

#include "common.hpp"

namespace jh {

struct f32x8_t {
    float v[8];
};

// 8 elements of a row at any address that is a multiple of the element's size
template <typename T>
__device__ __forceinline__ f32x8_t load8(const T* p) {
    f32x8_t r;
    if constexpr (sizeof(T) == 4) {
        const f32x4_t a = reinterpret_cast<const f32x4_any_t*>(p)[0].v, b = reinterpret_cast<const f32x4_any_t*>(p)[1].v;
#pragma unroll
        for (int i = 0; i < 4; ++i) r.v[i] = a[i], r.v[4 + i] = b[i];
    } else {
        const u32x4_t u = reinterpret_cast<const u32x4_any2_t*>(p)->v;
#pragma unroll
        for (int i = 0; i < 4; ++i) r.v[2 * i] = bf16_lo(u[i]), r.v[2 * i + 1] = bf16_hi(u[i]);
    }
    return r;
}
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const uint16_t* p) { return bf16_lo(*p); }

__device__ __forceinline__ void store8(float* p, const f32x8_t& r) {
    reinterpret_cast<f32x4_any_t*>(p)[0].v = f32x4_t{r.v[0], r.v[1], r.v[2], r.v[3]};
    reinterpret_cast<f32x4_any_t*>(p)[1].v = f32x4_t{r.v[4], r.v[5], r.v[6], r.v[7]};
}
__device__ __forceinline__ void store8(uint16_t* p, const f32x8_t& r) {
    reinterpret_cast<u32x4_any2_t*>(p)->v = u32x4_t{pack_bf16x2(r.v[0], r.v[1]), pack_bf16x2(r.v[2], r.v[3]),
                                                    pack_bf16x2(r.v[4], r.v[5]), pack_bf16x2(r.v[6], r.v[7])};
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(uint16_t* p, float v) { *p = (uint16_t)pack_bf16x2(v, 0.0f); }

// the first n of 8 elements, n = 1 .. 8; those behind are `rest`
template <typename T>
__device__ __forceinline__ f32x8_t load_piece(const T* p, int n, float rest = 0.0f) {
    if (n == 8) return load8(p);
    f32x8_t r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = i < n ? load1(p + i) : rest;
    return r;
}
template <typename T>
__device__ __forceinline__ void store_piece(T* p, const f32x8_t& r, int n) {
    if (n == 8) {
        store8(p, r);
    } else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < n) store1(p + i, r.v[i]);
    }
}

// A piece as it lies in memory.  Loads that are to be under way together are written
// as load_raw, their values taken afterwards: a conversion beside the load, in the branch
// of whole pieces, makes the compiler wait for each before the next.
template <typename T>
struct Raw8 {
    u32x4_t v[sizeof(T) / 2];
};
__device__ __forceinline__ uint32_t bits1(const float* p) { return __float_as_uint(*p); }
__device__ __forceinline__ uint32_t bits1(const uint16_t* p) { return *p; }
// the first n of 8 elements, n = 1 .. 8; those behind have the bits `rest`
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw(const T* p, int n, uint32_t rest = 0) {
    Raw8<T> r;
    if (n == 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = reinterpret_cast<const u32x4_any2_t*>(p)[i].v;
    } else {
        uint32_t e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i < n ? bits1(p + i) : rest;
        if constexpr (sizeof(T) == 4) {
            r.v[0] = u32x4_t{e[0], e[1], e[2], e[3]};
            r.v[1] = u32x4_t{e[4], e[5], e[6], e[7]};
        } else {
            r.v[0] = u32x4_t{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
        }
    }
    return r;
}
__device__ __forceinline__ f32x8_t values(const Raw8<float>& r) {
    f32x8_t x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = __uint_as_float(r.v[i / 4][i % 4]);
    return x;
}
__device__ __forceinline__ f32x8_t values(const Raw8<uint16_t>& r) {
    f32x8_t x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x.v[2 * i] = bf16_lo(r.v[0][i]), x.v[2 * i + 1] = bf16_hi(r.v[0][i]);
    return x;
}

// the larger of two, NaN where one is NaN (fmaxf drops it): one instruction on gfx950
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

}  // namespace jh

// kv4_cache.hip - rows into the 4-bit key/value cache and back (layout in
// kv4.hpp).  No counterpart in the reference.
//
// Writing a row x of D values:
//   s = bf16((max x - min x) * fp32(1/15)),  m = bf16(min x),
//   c = clamp(rint((x - m) / s), 0, 15)          (0 where s = 0)
// The rounded s and m are the ones that the codes are formed with, so a value
// is off by half a step and, at the row's ends, by what s and m were rounded.
// A row with a NaN or an infinity, or whose range passes fp32 or minimum bf16, is
// kept as NaN throughout: its codes could not say where.
//
// Bound by HBM: rows are read once and their codes, a quarter of bf16 rows or an
// eighth of fp32 ones, written once.  A row is 16 (D = 128) or 8 (D = 64) lanes
// of 8 values, so its minimum and maximum are four or three exchanges within 16
// lanes; a wave has neighbouring tokens of one head, whose value codes share the
// 8-byte groups of 4 tokens.  Ragged prompts of up to 2048 tokens, 16 sequences, 8
// heads of 128, fp32: 37 us, 4.7 TB/s, and 19 us, 5.2 TB/s, for the read of the
// same rows; one token each of 64 sequences: 4.3 and 2.9 us.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "kv4.hpp"
#include "launch.hpp"

namespace jh {
namespace {

constexpr int THREADS = 256;

struct RowsIn {
    const void* p;
    int64_t token_stride, head_stride;
};
__device__ __forceinline__ void load8(const float* p, float* v) {
    const f32x4_t a = reinterpret_cast<const f32x4_any_t*>(p)[0].v, b = reinterpret_cast<const f32x4_any_t*>(p)[1].v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
}
__device__ __forceinline__ void load8(const uint16_t* p, float* v) {
    const u32x4_t u = reinterpret_cast<const u32x4_any2_t*>(p)->v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(u[i]), v[2 * i + 1] = bf16_hi(u[i]);
}

// f over the LANES neighbouring lanes that hold a row, by lane permutations within
// rows of 16 lanes: with the lane beside, the two beside, the mirror image in 8, in 16
template <int LANES, typename F>
__device__ __forceinline__ float over_row(float v, F f) {
    const auto with = [&](auto ctrl) {
        const int u = __float_as_int(v);
        v = f(v, __int_as_float(__builtin_amdgcn_update_dpp(u, u, decltype(ctrl)::value, 0xf, 0xf, false)));
    };
    with(std::integral_constant<int, 0xb1>{});
    with(std::integral_constant<int, 0x4e>{});
    with(std::integral_constant<int, 0x141>{});
    if constexpr (LANES == 16) with(std::integral_constant<int, 0x140>{});
    return v;
}

// A row's codes of this lane's 8 values, and its scale and minimum.  A quotient is
// the product with 1 / s, corrected by its remainder: that is the division's own
// rounding wherever nothing leaves the normal numbers, since s has 8 bits (a
// correctly rounded reciprocal and one correction give the correctly rounded
// quotient but for divisors whose bits are all ones, a theorem of Markstein's).
template <int LANES>
__device__ __forceinline__ uint32_t quantise(const float* v, uint32_t* code) {
    float lo = v[0], hi = v[0];
    bool fine = fabsf(v[0]) <= FLT_MAX;
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        lo = fminf(lo, v[i]);
        hi = fmaxf(hi, v[i]);
        fine = fine && fabsf(v[i]) <= FLT_MAX;
    }
    if (!fine) hi = __builtin_inff();  // kept by fmaxf, and the range with it
    lo = over_row<LANES>(lo, [](float a, float b) { return fminf(a, b); });
    hi = over_row<LANES>(hi, [](float a, float b) { return fmaxf(a, b); });
    const float range = (hi - lo) * (1.0f / 15.0f);
    const uint32_t meta = pack_bf16x2(range, lo);
    const float s = bf16_lo(meta), m = bf16_hi(meta);
    if (!(range <= FLT_MAX) || !(fabsf(m) <= FLT_MAX)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) code[i] = 0;
        return 0x7fc07fc0u;
    }
    const auto coded = [](float t) { return (uint32_t)fminf(fmaxf(rintf(t), 0.0f), 15.0f); };
    if (s > 0x1p-100f && s < 0x1p100f) {
        const float r = 1.0f / s;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = v[i] - m, t = d * r;
            code[i] = coded(__builtin_fmaf(__builtin_fmaf(-t, s, d), r, t));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) code[i] = s > 0.0f ? coded(__fdiv_rn(v[i] - m, s)) : 0u;
    }
    return meta;
}

// grid: x heads within blocks of tokens of a sequence, y sequences; a block has
// THREADS / LANES neighbouring tokens of a head, and neighbouring blocks the heads
// of the same tokens, whose rows lie side by side
template <typename T, int D>
__global__ __launch_bounds__(THREADS) void kv4_append_kernel(KV4View c, KV4Batch b, RowsIn k, RowsIn v) {
    constexpr int LANES = D / 8, TOKENS = THREADS / LANES;
    const int h = blockIdx.x % c.heads, lane = threadIdx.x % LANES;
    const int block = blockIdx.x / c.heads, blocks = gridDim.x / c.heads;
    const int seq = blockIdx.y;
    const int n = kv4_count(b, seq), first = kv4_first(b, seq), len = kv4_scalar(b.lens + seq);
    for (int64_t i0 = (int64_t)block * TOKENS; i0 < n; i0 += (int64_t)blocks * TOKENS) {
        const int i = (int)i0 + (int)threadIdx.x / LANES;
        if (i >= n) continue;
        float x[8], y[8];
        load8(static_cast<const T*>(k.p) + (first + i) * k.token_stride + h * k.head_stride + 8 * lane, x);
        load8(static_cast<const T*>(v.p) + (first + i) * v.token_stride + h * v.head_stride + 8 * lane, y);
        const int64_t at = (int64_t)len - n + i;  // a row before the sequence's begin is dropped
        const int page = at >= 0 && at <= INT32_MAX ? kv4_page(c, b, seq, (int)at) : -1;
        if (page < 0) continue;
        const int off = (int)at & (c.page_size - 1);
        const int64_t row = kv4_row(c, page, h, off);
        uint32_t code[8];
        uint32_t meta = quantise<LANES>(x, code);
        uint32_t word = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) word |= code[e] << (4 * (e / 2) + 16 * (e % 2));
        reinterpret_cast<uint32_t*>(c.k)[row * (D / 8) + lane] = word;
        if (lane == 0) c.k_meta[row] = meta;
        meta = quantise<LANES>(y, code);
        // the four tokens' groups of 8 bytes: two of them for 8 values
        uint16_t* held = reinterpret_cast<uint16_t*>(c.v) + (row - off % 4) * (D / 4) + off % 4;
#pragma unroll
        for (int g = 0; g < 2; ++g)
            held[4 * (2 * lane + g)] = (uint16_t)(code[4 * g] | code[4 * g + 1] << 4 | code[4 * g + 2] << 8 | code[4 * g + 3] << 12);
        if (lane == 0) c.v_meta[row] = meta;
    }
}

__device__ __forceinline__ void store8(float* p, const float* v) {
    reinterpret_cast<f32x4_t*>(p)[0] = f32x4_t{v[0], v[1], v[2], v[3]};
    reinterpret_cast<f32x4_t*>(p)[1] = f32x4_t{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void store8(uint16_t* p, const float* v) {
    *reinterpret_cast<u32x4_t*>(p) = u32x4_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                             pack_bf16x2(v[6], v[7])};
}

// the same rows as values; a row before the sequence's begin is 0, one on a
// page that the pool does not have NaN
template <typename T, int D>
__global__ __launch_bounds__(THREADS) void kv4_read_kernel(KV4View c, KV4Batch b, T* k, T* v) {
    constexpr int LANES = D / 8, TOKENS = THREADS / LANES;
    const int h = blockIdx.x % c.heads, lane = threadIdx.x % LANES;
    const int block = blockIdx.x / c.heads, blocks = gridDim.x / c.heads;
    const int seq = blockIdx.y;
    const int n = kv4_count(b, seq), first = kv4_first(b, seq), len = kv4_scalar(b.lens + seq);
    for (int64_t i0 = (int64_t)block * TOKENS; i0 < n; i0 += (int64_t)blocks * TOKENS) {
        const int i = (int)i0 + (int)threadIdx.x / LANES;
        if (i >= n) continue;
        const int64_t at = (int64_t)len - n + i;
        const int page = at >= 0 && at <= INT32_MAX ? kv4_page(c, b, seq, (int)at) : -1;
        float x[8], y[8];
        if (page < 0) {
            const float none = at < 0 ? 0.0f : __builtin_nanf("");
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = y[e] = none;
        } else {
            const int off = (int)at & (c.page_size - 1);
            const int64_t row = kv4_row(c, page, h, off);
            const uint32_t word = reinterpret_cast<const uint32_t*>(c.k)[row * (D / 8) + lane];
            uint32_t meta = c.k_meta[row];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[e] = __builtin_fmaf(bf16_lo(meta), (float)(word >> (4 * (e / 2) + 16 * (e % 2)) & 15u), bf16_hi(meta));
            meta = c.v_meta[row];
            const uint16_t* held = reinterpret_cast<const uint16_t*>(c.v) + (row - off % 4) * (D / 4) + off % 4;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const uint32_t u = held[4 * (2 * lane + g)];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    y[4 * g + e] = __builtin_fmaf(bf16_lo(meta), (float)(u >> (4 * e) & 15u), bf16_hi(meta));
            }
        }
        const int64_t to = ((int64_t)(first + i) * c.heads + h) * D + 8 * lane;
        store8(k + to, x);
        store8(v + to, y);
    }
}

template <int D>
dim3 rows_grid(const KV4View& c, const KV4Batch& b) {
    const int tokens = THREADS / (D / 8);
    const int rows = std::max(1, std::min(b.max_q, b.tokens));
    // below 2^24 blocks in x
    const int blocks = std::min((rows - 1) / tokens + 1, std::max(1, (1 << 23) / c.heads));
    return dim3((unsigned)(blocks * c.heads), (unsigned)b.batch);
}

}  // namespace

hipError_t launch_kv4_append(int dtype, const KV4View& c, const KV4Batch& b, const void* k, int64_t k_token,
                             int64_t k_head, const void* v, int64_t v_token, int64_t v_head, hipStream_t s) {
    const RowsIn ki{k, k_token, k_head}, vi{v, v_token, v_head};
    if (c.D == 128) {
        const dim3 g = rows_grid<128>(c, b);
        if (dtype == JH_F32)
            kv4_append_kernel<float, 128><<<g, THREADS, 0, s>>>(c, b, ki, vi);
        else
            kv4_append_kernel<uint16_t, 128><<<g, THREADS, 0, s>>>(c, b, ki, vi);
    } else {
        const dim3 g = rows_grid<64>(c, b);
        if (dtype == JH_F32)
            kv4_append_kernel<float, 64><<<g, THREADS, 0, s>>>(c, b, ki, vi);
        else
            kv4_append_kernel<uint16_t, 64><<<g, THREADS, 0, s>>>(c, b, ki, vi);
    }
    return hipGetLastError();
}

hipError_t launch_kv4_read(int dtype, const KV4View& c, const KV4Batch& b, void* k, void* v, hipStream_t s) {
    if (c.D == 128) {
        const dim3 g = rows_grid<128>(c, b);
        if (dtype == JH_F32)
            kv4_read_kernel<float, 128><<<g, THREADS, 0, s>>>(c, b, static_cast<float*>(k), static_cast<float*>(v));
        else
            kv4_read_kernel<uint16_t, 128><<<g, THREADS, 0, s>>>(c, b, static_cast<uint16_t*>(k), static_cast<uint16_t*>(v));
    } else {
        const dim3 g = rows_grid<64>(c, b);
        if (dtype == JH_F32)
            kv4_read_kernel<float, 64><<<g, THREADS, 0, s>>>(c, b, static_cast<float*>(k), static_cast<float*>(v));
        else
            kv4_read_kernel<uint16_t, 64><<<g, THREADS, 0, s>>>(c, b, static_cast<uint16_t*>(k), static_cast<uint16_t*>(v));
    }
    return hipGetLastError();
}

}  // namespace jh

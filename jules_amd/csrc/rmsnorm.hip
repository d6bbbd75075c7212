// rmsnorm.hip - the residual's addition with the root-mean-square norm, rows
// out as fp32, bf16 or int8 with a scale for each row (the A and scale_A of
// jules_hip_matmul_w8a8).  No counterpart in the reference.
//
//   h = x + r,  r' = round(h),  y_j = h_j w_j / sqrt(sum h^2 / N + eps)
//   int8: s = max|y| / 127,  q_j = rint(y_j / s)
// The norm's factor is one number for the row, so max|y| = max|h w| times it
// and q_j = rint(h_j w_j * 127 / max|h w|): one reduction over the row gives
// both numbers, and the codes do not depend on the factor's rounding.
//
// Bound by HBM: a row is read once, held in registers as h, and written once.
// h and h w are fp32; the sum of squares is fp64, so that no row that fp32
// holds overflows or vanishes in it (a convert and an fma an element, far
// below what the loads cost).
#include <algorithm>
#include <cfloat>

#include "common.hpp"
#include "launch.hpp"

namespace jh {
namespace {

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

struct __attribute__((packed, aligned(1))) u32x2_any1_t {
    u32x2_t v;
};

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

// the larger of two, NaN where one is NaN (fmaxf drops it): one instruction on gfx950
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// sum and largest of the group's values, the same order for every row.  The waves'
// parts alternate between two places, so that one barrier a row is enough: a wave
// that writes a place again has passed the barrier after which it was read.
struct RowStats {
    double sum;
    float top;
};
template <int G>
__device__ __forceinline__ RowStats reduce_row(RowStats a, int turn) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        a.sum += __shfl_xor(a.sum, o);
        a.top = larger(a.top, __shfl_xor(a.top, o));
    }
    if constexpr (G > 64) {
        __shared__ RowStats parts[2][G / 64];
        RowStats* part = parts[turn & 1];
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = a;
        __syncthreads();
        a = part[0];
#pragma unroll
        for (int w = 1; w < G / 64; ++w) {
            a.sum += part[w].sum;
            a.top = larger(a.top, part[w].top);
        }
    }
    return a;
}

// What the row's numbers come to: the norm's factor, and for int8 rows the
// scale and the factor from h w to codes.
struct RowFactors {
    float rstd, scale, lift, inv;
    bool bad;
};
__device__ __forceinline__ RowFactors row_factors(RowStats a, int N, float eps) {
    RowFactors f;
    f.rstd = (float)(1.0 / sqrt(a.sum / (double)N + (double)eps));
    // 127 / top overflows below 2^-121: tiny rows are lifted by a power of two
    f.lift = a.top < 0x1p-100f ? 0x1p100f : 1.0f;
    f.inv = a.top > 0.0f ? 127.0f / (a.top * f.lift) : 0.0f;
    // a NaN or an infinity in the row: the sum of squares says so; h w past fp32, or
    // no number for the weight's sake: the largest does
    f.bad = !(a.sum <= DBL_MAX) || !(a.top <= FLT_MAX);
    f.scale = f.bad ? __builtin_nanf("") : a.top * f.rstd / 127.0f;
    if (!f.bad && a.top == 0.0f) f.scale = 0.0f;
    return f;
}

struct NormArgs {
    const void *x, *r;
    const float* w;
    void *r_out, *out;
    float* scale;
    int M, N, out_dtype;
    float eps;
};

// up to 8 elements of the row from j on are written (n of them)
template <typename RT, bool RES>
__device__ __forceinline__ void write_piece(const NormArgs& a, const RowFactors& f, int64_t at, const f32x8_t& h,
                                            const f32x8_t& w, int n) {
    if (RES && a.r_out) {
        RT* p = static_cast<RT*>(a.r_out) + at;
        if (n == 8) {
            store8(p, h);
        } else {
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (i < n) store1(p + i, h.v[i]);
        }
    }
    if (a.out_dtype == JH_I8) {
        int8_t* p = static_cast<int8_t*>(a.out) + at;
        uint32_t u[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int q = f.bad ? 0 : (int)rintf(h.v[i] * w.v[i] * f.lift * f.inv);
            u[i / 4] |= (uint32_t)(q & 255) << (8 * (i % 4));
        }
        if (n == 8) {
            reinterpret_cast<u32x2_any1_t*>(p)->v = u32x2_t{u[0], u[1]};
        } else {
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (i < n) p[i] = (int8_t)(u[i / 4] >> (8 * (i % 4)));
        }
    } else {
        f32x8_t y;
#pragma unroll
        for (int i = 0; i < 8; ++i) y.v[i] = h.v[i] * f.rstd * w.v[i];
        if (a.out_dtype == JH_F32) {
            float* p = static_cast<float*>(a.out) + at;
            if (n == 8) {
                store8(p, y);
            } else {
#pragma unroll
                for (int i = 0; i < 7; ++i)
                    if (i < n) store1(p + i, y.v[i]);
            }
        } else {
            uint16_t* p = static_cast<uint16_t*>(a.out) + at;
            if (n == 8) {
                store8(p, y);
            } else {
#pragma unroll
                for (int i = 0; i < 7; ++i)
                    if (i < n) store1(p + i, y.v[i]);
            }
        }
    }
}

template <typename XT, typename RT, bool RES>
__device__ __forceinline__ f32x8_t read_piece(const NormArgs& a, int64_t at, int n) {
    f32x8_t h;
    if (n == 8) {
        h = load8(static_cast<const XT*>(a.x) + at);
        if constexpr (RES) {
            const f32x8_t r = load8(static_cast<const RT*>(a.r) + at);
#pragma unroll
            for (int i = 0; i < 8; ++i) h.v[i] += r.v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            h.v[i] = 0.0f;
            if (i < n) {
                h.v[i] = load1(static_cast<const XT*>(a.x) + at + i);
                if constexpr (RES) h.v[i] += load1(static_cast<const RT*>(a.r) + at + i);
            }
        }
    }
    return h;
}
__device__ __forceinline__ f32x8_t read_weight(const float* w, int j, int n) {
    if (n == 8) return load8(w + j);
    f32x8_t r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = i < n ? w[j + i] : 0.0f;
    return r;
}

__device__ __forceinline__ void count(RowStats* s, const f32x8_t& h, const f32x8_t& w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        s->sum = __builtin_fma((double)h.v[i], (double)h.v[i], s->sum);
        s->top = larger(s->top, fabsf(h.v[i] * w.v[i]));
    }
}

// G threads a row, NP pieces of 8 neighbouring elements a thread; a block holds
// 256 / G rows, or one row of more threads, and goes on to others with the weight
// in its registers
template <typename XT, typename RT, bool RES, int G, int NP>
__global__ __launch_bounds__(G < 256 ? 256 : G) void add_rmsnorm_kernel(NormArgs a) {
    constexpr int ROWS = G < 256 ? 256 / G : 1;
    const int tid = G < 256 ? threadIdx.x % G : threadIdx.x;
    constexpr bool KEEP = G * NP < 4096;  // 1024 threads with 4 pieces have no registers for it
    f32x8_t w[KEEP ? NP : 1];
    const auto weight = [&](int t) {
        const int j = 8 * (tid + G * t), n = min(8, a.N - j);
        return n > 0 ? read_weight(a.w, j, n) : f32x8_t{};
    };
    if constexpr (KEEP) {
#pragma unroll
        for (int t = 0; t < NP; ++t) w[t] = weight(t);
    }
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * ROWS + (G < 256 ? threadIdx.x / G : 0); row < a.M;
         row += (int64_t)gridDim.x * ROWS, ++turn) {
        const int64_t at = row * a.N;
        f32x8_t h[NP];
        RowStats s{0.0, 0.0f};
#pragma unroll
        for (int t = 0; t < NP; ++t) {
            const int j = 8 * (tid + G * t), n = min(8, a.N - j);
            if (n > 0) h[t] = read_piece<XT, RT, RES>(a, at + j, n);
        }
#pragma unroll
        for (int t = 0; t < NP; ++t)
            if (8 * (tid + G * t) < a.N) count(&s, h[t], KEEP ? w[KEEP ? t : 0] : weight(t));
        s = reduce_row<G>(s, turn);
        const RowFactors f = row_factors(s, a.N, a.eps);
        if (a.out_dtype == JH_I8 && tid == 0) a.scale[row] = f.scale;
#pragma unroll
        for (int t = 0; t < NP; ++t) {
            const int j = 8 * (tid + G * t), n = min(8, a.N - j);
            if (n > 0) write_piece<RT, RES>(a, f, at + j, h[t], KEEP ? w[KEEP ? t : 0] : weight(t), n);
        }
    }
}

// rows longer than a block holds: read twice.  x and r are read before r' is
// written by the same thread, so r' may be r or x here too.
template <typename XT, typename RT, bool RES>
__global__ __launch_bounds__(1024) void add_rmsnorm_long_kernel(NormArgs a) {
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x, ++turn) {
        const int64_t at = row * a.N;
        RowStats s{0.0, 0.0f};
        for (int64_t j = 8 * (int64_t)threadIdx.x; j < a.N; j += 8 * 1024) {
            const int n = (int)min((int64_t)8, a.N - j);
            count(&s, read_piece<XT, RT, RES>(a, at + j, n), read_weight(a.w, (int)j, n));
        }
        s = reduce_row<1024>(s, turn);
        const RowFactors f = row_factors(s, a.N, a.eps);
        if (a.out_dtype == JH_I8 && threadIdx.x == 0) a.scale[row] = f.scale;
        for (int64_t j = 8 * (int64_t)threadIdx.x; j < a.N; j += 8 * 1024) {
            const int n = (int)min((int64_t)8, a.N - j);
            const f32x8_t h = read_piece<XT, RT, RES>(a, at + j, n);
            write_piece<RT, RES>(a, f, at + j, h, read_weight(a.w, (int)j, n), n);
        }
    }
}

template <typename XT, typename RT, bool RES, int G, int NP>
void launch(const NormArgs& a, int blocks, hipStream_t s) {
    constexpr int ROWS = G < 256 ? 256 / G : 1;
    const int64_t rows = ((int64_t)a.M + ROWS - 1) / ROWS;
    add_rmsnorm_kernel<XT, RT, RES, G, NP><<<(unsigned)std::min((int64_t)blocks, rows), G < 256 ? 256 : G, 0, s>>>(a);
}

// Few threads with many elements each keep the most rows in flight: 8192 rows of
// 8192 bf16 take 87 us (5.4 TB/s) with 256 threads of 32 elements, 165 us with
// 1024 of 8, of which a CU holds one row at a time.  Up to two rows a CU 1024
// threads are the faster, a row being done sooner (8 rows: 5.2 us).  Four blocks a
// CU, as many as are resident, read the weight once each; a block a row: 98 us.
// Rows of odd width, at 4-byte addresses: 4.8 TB/s (1999 of 5001 fp32, 34 us).
template <typename XT, typename RT, bool RES>
hipError_t launch(const NormArgs& a, hipStream_t s) {
    if (a.N <= 512)
        launch<XT, RT, RES, 64, 1>(a, 8192, s);
    else if (a.N <= 2048)
        launch<XT, RT, RES, 256, 1>(a, 2048, s);
    else if (a.M <= 512 && a.N <= 8192)
        launch<XT, RT, RES, 1024, 1>(a, 512, s);
    else if (a.N <= 4096)
        launch<XT, RT, RES, 256, 2>(a, 1024, s);
    else if (a.N <= 8192)
        launch<XT, RT, RES, 256, 4>(a, 1024, s);
    else if (a.N <= 16384)
        launch<XT, RT, RES, 512, 4>(a, 512, s);
    else if (a.N <= 32768)
        launch<XT, RT, RES, 1024, 4>(a, 512, s);
    else
        add_rmsnorm_long_kernel<XT, RT, RES><<<(unsigned)std::min(a.M, 2048), 1024, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_add_rmsnorm(int x_dtype, int r_dtype, int out_dtype, const void* x, const void* r, const float* w,
                              void* r_out, void* out, float* scale, int M, int N, float eps, hipStream_t s) {
    const NormArgs a{x, r, w, r_out, out, scale, M, N, out_dtype, eps};
    if (!r) return x_dtype == JH_F32 ? launch<float, float, false>(a, s) : launch<uint16_t, uint16_t, false>(a, s);
    if (x_dtype == JH_F32)
        return r_dtype == JH_F32 ? launch<float, float, true>(a, s) : launch<float, uint16_t, true>(a, s);
    return r_dtype == JH_F32 ? launch<uint16_t, float, true>(a, s) : launch<uint16_t, uint16_t, true>(a, s);
}

}  // namespace jh

// rotary.hip - rotary positions of one or several axes, and their backward
// pass.  No counterpart in the reference.
//
//   a_p = positions[axis(p)][t] * inv_freq[p],  p = 0 .. R/2 - 1
//   (u, w) -> (u cos a - w sin a, u sin a + w cos a)
// on the pairs (u, w) = x[p], x[p + R/2] or x[2p], x[2p + 1]; elements R .. D-1
// stay as they are.  The rotation's transpose is the rotation by -a, which is
// all of the backward pass.
//
// Bound by HBM: every element is read and written once.  An angle is needed
// once a token and pair but used by all heads, so a block first puts the
// cosines and sines of its tokens into LDS.  The angle is formed in fp64 and
// reduced to a fraction of a turn there, which is then rounded to fp32: at position
// 10^6 an fp32 angle is off by 0.03, this one by 10^-7.  bf16, 2 x 8000 tokens, 40 heads of 128:
// 64 us, 5.1 TB/s; 8 x 4096, 32 heads of 128 with half of each rotated: 107 us,
// 5.0 TB/s, a copy's rate; 8 tokens: 3.4 us.
#include <algorithm>

#include "common.hpp"
#include "launch.hpp"

namespace jh {
namespace {

constexpr int THREADS = 256;

struct RotaryArgs {
    const void* x;
    void* out;
    const int32_t* pos;
    const double* freq;
    const int32_t* axis;  // or null: axis 0
    int64_t xs[3], os[3];  // strides of batch, head, token
    int64_t tokens;        // B * S
    int axes, H, S, D, R;
    int tb, hc;  // tokens and heads of a block
    float sign;
    bool copy;  // elements R .. D-1 are not in place already
};

// V neighbouring elements at any address that is a multiple of the element's size
template <int V>
__device__ __forceinline__ void load(const float* p, float* v) {
    if constexpr (V == 1) {
        v[0] = *p;
    } else {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const f32x4_t q = reinterpret_cast<const f32x4_any_t*>(p)[i].v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * i + j] = q[j];
        }
    }
}
template <int V>
__device__ __forceinline__ void load(const uint16_t* p, float* v) {
    if constexpr (V == 1) {
        v[0] = bf16_lo(*p);
    } else {
#pragma unroll
        for (int i = 0; i < V / 8; ++i) {
            const u32x4_t q = reinterpret_cast<const u32x4_any2_t*>(p)[i].v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[8 * i + 2 * j] = bf16_lo(q[j]), v[8 * i + 2 * j + 1] = bf16_hi(q[j]);
        }
    }
}
template <int V>
__device__ __forceinline__ void store(float* p, const float* v) {
    if constexpr (V == 1) {
        *p = v[0];
    } else {
#pragma unroll
        for (int i = 0; i < V / 4; ++i)
            reinterpret_cast<f32x4_any_t*>(p)[i].v = f32x4_t{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
    }
}
template <int V>
__device__ __forceinline__ void store(uint16_t* p, const float* v) {
    if constexpr (V == 1) {
        *p = (uint16_t)pack_bf16x2(v[0], 0.0f);
    } else {
#pragma unroll
        for (int i = 0; i < V / 8; ++i)
            reinterpret_cast<u32x4_any2_t*>(p)[i].v =
                u32x4_t{pack_bf16x2(v[8 * i], v[8 * i + 1]), pack_bf16x2(v[8 * i + 2], v[8 * i + 3]),
                        pack_bf16x2(v[8 * i + 4], v[8 * i + 5]), pack_bf16x2(v[8 * i + 6], v[8 * i + 7])};
    }
}

// V pairs, or V elements behind the rotated ones, a thread and step
template <typename XT, typename OT, int V, bool HALF>
__global__ __launch_bounds__(THREADS) void rotary_kernel(RotaryArgs a) {
    extern __shared__ float angles[];  // cosines [tb][R/2], sines [tb][R/2]
    const int half = a.R / 2;
    float* cosines = angles;
    float* sines = angles + a.tb * half;
    const int64_t t0 = (int64_t)blockIdx.x * a.tb;
    const int tb = (int)min((int64_t)a.tb, a.tokens - t0);
    for (int i = threadIdx.x; i < tb * half; i += THREADS) {
        const int t = i / half, p = i - t * half;
        const int ax = a.axis ? a.axis[p] : 0;
        float c = __builtin_nanf(""), s = c;  // an axis that is none
        if (ax >= 0 && ax < a.axes) {
            const double turns = (double)a.pos[ax * a.tokens + t0 + t] * (a.freq[p] * 0.15915494309189533577);
            sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        }
        cosines[t * half + p] = c;
        sines[t * half + p] = a.sign * s;
    }
    __syncthreads();
    const int rot = half / V, pieces = rot + (a.copy ? (a.D - a.R) / V : 0);
    const int h0 = blockIdx.y * a.hc, hc = min(a.hc, a.H - h0);
    // items: (token, head, piece), neighbouring pieces on neighbouring threads
    const int lanes = THREADS / pieces;  // (token, head) in flight; 0 where a row has more pieces than threads
    const int first = lanes ? (int)threadIdx.x / pieces : 0, step = lanes ? lanes : 1;
    if (lanes && first >= lanes) return;
    for (int i = first; i < tb * hc; i += step) {
        const int t = i / hc, h = h0 + i - t * hc;
        const int64_t token = t0 + t, b = token / a.S, s = token - b * a.S;
        const XT* x = static_cast<const XT*>(a.x) + b * a.xs[0] + h * a.xs[1] + s * a.xs[2];
        OT* o = static_cast<OT*>(a.out) + b * a.os[0] + h * a.os[1] + s * a.os[2];
        for (int piece = lanes ? (int)threadIdx.x % pieces : (int)threadIdx.x; piece < pieces;
             piece += lanes ? pieces : THREADS) {
            if (piece >= rot) {
                const int j = a.R + (piece - rot) * V;
                float v[V];
                load<V>(x + j, v);
                store<V>(o + j, v);
                continue;
            }
            const int p = piece * V;
            float v[2 * V], r[2 * V];
            if constexpr (HALF) {
                load<V>(x + p, v);
                load<V>(x + half + p, v + V);
            } else if constexpr (V == 1) {
                load<1>(x + 2 * p, v);
                load<1>(x + 2 * p + 1, v + 1);
            } else {
                load<2 * V>(x + 2 * p, v);
            }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float c = cosines[t * half + p + k], sn = sines[t * half + p + k];
                constexpr int ui = HALF ? 1 : 2, wo = HALF ? V : 1;
                const float u = v[ui * k], w = v[ui * k + wo];
                r[ui * k] = __builtin_fmaf(u, c, -(w * sn));
                r[ui * k + wo] = __builtin_fmaf(u, sn, w * c);
            }
            if constexpr (HALF) {
                store<V>(o + p, r);
                store<V>(o + half + p, r + V);
            } else if constexpr (V == 1) {
                store<1>(o + 2 * p, r);
                store<1>(o + 2 * p + 1, r + 1);
            } else {
                store<2 * V>(o + 2 * p, r);
            }
        }
    }
}

template <typename XT, typename OT, int V>
hipError_t launch(bool half, const RotaryArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((a.tokens + a.tb - 1) / a.tb), (unsigned)((a.H + a.hc - 1) / a.hc));
    const size_t lds = (size_t)a.tb * a.R * sizeof(float);
    if (half)
        rotary_kernel<XT, OT, V, true><<<grid, THREADS, lds, s>>>(a);
    else
        rotary_kernel<XT, OT, V, false><<<grid, THREADS, lds, s>>>(a);
    return hipGetLastError();
}

template <typename XT, typename OT>
hipError_t launch(bool half, const RotaryArgs& a, int v, hipStream_t s) {
    return v == 8 ? launch<XT, OT, 8>(half, a, s) : launch<XT, OT, 1>(half, a, s);
}

}  // namespace

hipError_t launch_rotary(int x_dtype, int out_dtype, bool half, bool inverse, const void* x, const int64_t* xs,
                         void* out, const int64_t* os, const int32_t* pos, const double* freq, const int32_t* axis,
                         int axes, int B, int H, int S, int D, int R, hipStream_t s) {
    RotaryArgs a{x, out, pos, freq, axis, {xs[0], xs[1], xs[2]}, {os[0], os[1], os[2]}, (int64_t)B * S, axes, H, S, D, R,
                 1, H, inverse ? -1.0f : 1.0f, x != out};
    // 8 pairs a thread where the rotated and the other elements divide by it
    const int v = (R / 2) % 8 == 0 && (D - R) % 8 == 0 ? 8 : 1;
    const int pieces = R / 2 / v + (a.copy ? (D - R) / v : 0);
    const int lanes = std::max(1, THREADS / pieces);
    if (a.tokens * H * pieces < (int64_t)2048 * THREADS)
        a.hc = std::min(H, lanes);  // few tokens: one step a thread, on as many blocks as there are
    else
        // up to four steps a thread, and 16 tokens: with R = 1024 their angles take the 64 KB of LDS that a
        // launch gets unasked
        a.tb = std::max(1, std::min(16, 1024 / std::min(1024, H * pieces)));
    // fewer than 2^24 blocks of 256 threads (at most 2^27 tokens, so tb stays within 16)
    while ((a.tokens + a.tb - 1) / a.tb >= (1 << 24)) a.tb *= 2;
    if (x_dtype == JH_F32)
        return out_dtype == JH_F32 ? launch<float, float>(half, a, v, s) : launch<float, uint16_t>(half, a, v, s);
    return out_dtype == JH_F32 ? launch<uint16_t, float>(half, a, v, s) : launch<uint16_t, uint16_t>(half, a, v, s);
}

}  // namespace jh

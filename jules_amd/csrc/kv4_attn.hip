// kv4_attn.hip - attention over the paged key/value cache held in 4 bits (layout
// in kv4.hpp), for one token of a sequence, some drafted ones, or a chunk of a
// prompt.  No counterpart in the reference, whose attention has no cache.
//
//   o = softmax(scale q K^T) V,  K = m_k + s_k c_k,  V = m_v + s_v c_v
// New token i of the n of a sequence of length L is at position L - n + i and
// sees the keys up to its own.  A code becomes the bf16 number C = 1 + c/16, exactly, by
// one shift and one and-or for two codes, and the rest of the dequantisation is
// left to where it is one number a key:
//   q . K  = 16 s_k (q . C - sum q) + m_k sum q
//   sum p V = 16 (sum P' C - MID sum P') + sum p (m_v + 7.5 s_v),
//   P' = bf16(p s_v),  MID = 1 + 7.5/16
// -sum q is the accumulator that the first product starts from.  P' is rounded
// once and both of its sums take the rounded number, so what its rounding is
// multiplied by is the code's distance from the middle of the row's range, about
// the value's distance from the row's mean: the error is that of an attention
// with bf16 probabilities.  (With MID = 1 it was 0.0049 of the output at 8192
// keys of unit variance, with this one 0.0020; bf16 outputs alone are 0.0017.)
//
// One wave holds 16 rows (new tokens x heads of the group) times RT, and takes 32 keys
// at a time.  Both products are transposed, S^T = K Q^T and O^T = V^T P^T: the
// scores of a row then lie in the four lanes that also hold that row's P as the
// second product's operand, 4 neighbouring keys of each 16, and the softmax
// needs no exchange between lanes but for the row's maximum when it grows.
// Keys and values go from memory to the matrix cores through registers alone.
#include <algorithm>
#include <cfloat>

#include "kv4.hpp"
#include "launch.hpp"

namespace jh {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int KEYS = 32;     // keys of a step
constexpr int WAVES = 4;     // waves of a workgroup
constexpr float MID = 1.0f + 7.5f / 16.0f;  // C of the middle of a row's range
constexpr float GROW = 8.0f; // a row's reference grows when a score passes it by this (log2)

struct AttnArgs {
    KV4View c;
    KV4Batch b;
    const uint16_t* q;
    int64_t q_token, q_head;
    uint16_t* o;
    float* lse;
    float* part;    // splits > 1: sums [row][split][D], then (reference, sum) [row][split]
    float scale;
    int heads_q, group;
    int splits, chunk;  // keys of a split, a multiple of KEYS * WAVES; the last has all the rest
};

// C of the low nibble of each half, bits 3-6 of a bf16 1.x
struct CodeMask {
    uint32_t keep, one;
};
// The two constants in registers, a vector and a scalar one, as one and-or
// takes them: as literals they are an and and an or.
__device__ __forceinline__ CodeMask code_mask() {
    CodeMask m{0x00780078u, 0x3f803f80u};
    asm volatile("" : "+v"(m.keep));
    asm volatile("" : "+s"(m.one));
    return m;
}
__device__ __forceinline__ uint32_t codes(CodeMask m, uint32_t w, int j) {
    const uint32_t x = j == 0 ? w << 3 : w >> (4 * j - 3);
    return (x & m.keep) | m.one;
}
__device__ __forceinline__ bf16x8_t operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(bf16x8_t, u32x4_t{a, b, c, d});
}

// one step's keys and values as they lie in memory: this lane's part of 2 x 16 tokens
template <int D>
struct Raw {
    uint32_t k[2][D / 32], v[2][D / 32];
    u32x4_t km[2], vm[2];
};

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
    if constexpr (N == 4) {
        const u32x4_t u = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = u[i];
    } else {
        const u32x2_t u = *reinterpret_cast<const u32x2_t*>(p);
        w[0] = u[0], w[1] = u[1];
    }
}

// the value of code 7.5 of a row
__device__ __forceinline__ float middle(uint32_t meta) {
    return __builtin_fmaf(7.5f, bf16_lo(meta), bf16_hi(meta));
}

// Rows of one wave: RT tiles of 16, its running sums, and the step over 32 keys.
// A row's scores are taken relative to `ref`, which moves to the largest score so
// far when one passes it by GROW; `limit` is GROW, and lower than any score
// before the row's first key.
template <int D, int RT>
struct Rows {
    static constexpr int KI = D / 32;  // products over elements of a key tile
    static constexpr int VI = D / 16;  // tiles of 16 elements of the output
    bf16x8_t q[RT][KI];
    float qsum[RT];   // sum of the row's q
    f32x4_t acc[RT][VI];
    f32x4_t psum[RT]; // sum of P', the same number four times
    float ref[RT], limit[RT], l[RT], pm[RT];
    int last[RT];     // position of the row's token: the last key it sees

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
#pragma unroll
            for (int i = 0; i < VI; ++i) acc[r][i] = f32x4_t{0, 0, 0, 0};
            psum[r] = f32x4_t{0, 0, 0, 0};
            limit[r] = -FLT_MAX;
            ref[r] = l[r] = pm[r] = 0.0f;
        }
    }

    // One step: keys base .. base + 31.  `mask`: some of them are not seen by some
    // row, or lie behind the sequence's end, or on no page of the pool.
    __device__ __forceinline__ void step(Raw<D>& raw, CodeMask m, float kscale, bool mask, int base, bool bad0, bool bad1) {
        f32x4_t x[RT][2];
#pragma unroll
        for (int r = 0; r < RT; ++r) x[r][0] = x[r][1] = f32x4_t{-qsum[r], -qsum[r], -qsum[r], -qsum[r]};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < KI; ++i) {
                const uint32_t w = raw.k[t][i];
                const bf16x8_t kc = operand(codes(m, w, 0), codes(m, w, 1), codes(m, w, 2), codes(m, w, 3));
#pragma unroll
                for (int r = 0; r < RT; ++r)
                    x[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kc, q[r][i], x[r][t], 0, 0, 0);
            }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float c1 = bf16_lo(raw.km[t][e]) * (16.0f * kscale), cm = bf16_hi(raw.km[t][e]) * kscale;
#pragma unroll
                for (int r = 0; r < RT; ++r)
                    x[r][t][e] = __builtin_fmaf(c1, x[r][t][e], __builtin_fmaf(cm, qsum[r], -ref[r]));
            }
        if (mask) {
            // an unseen key counts for nothing, whatever its scale and minimum
            // hold: where its value's are no numbers they become 0, and the rows
            // that see it NaN
            const int g = (threadIdx.x >> 4) & 3;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool none = (t ? bad1 : bad0) || !(fabsf(middle(raw.vm[t][e])) <= FLT_MAX);
                    raw.vm[t][e] = none ? 0u : raw.vm[t][e];
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const float y = none ? __builtin_nanf("") : x[r][t][e];
                        x[r][t][e] = base + 16 * t + 4 * g + e > last[r] ? -__builtin_inff() : y;
                    }
                }
        }
        float top[RT];
        bool grow = false;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            top[r] = -__builtin_inff();
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) top[r] = fmaxf(top[r], x[r][t][e]);
            grow = grow || top[r] > limit[r];
        }
        if (__any(grow)) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                float high = fmaxf(top[r], __shfl_xor(top[r], 16));
                high = fmaxf(high, __shfl_xor(high, 32));
                const bool none = high == -__builtin_inff();  // no key so far
                const bool begun = limit[r] == GROW;
                const float up = begun ? fmaxf(high, 0.0f) : none ? 0.0f : high;
                const float down = begun ? __builtin_amdgcn_exp2f(-up) : 0.0f;
                limit[r] = none ? limit[r] : GROW;
                ref[r] += up;
                l[r] *= down;
                pm[r] *= down;
                psum[r] *= down;
#pragma unroll
                for (int i = 0; i < VI; ++i) acc[r][i] *= down;
                x[r][0] -= up;
                x[r][1] -= up;
            }
        }
        bf16x8_t pb[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            uint32_t pw[2][2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float pv[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = __builtin_amdgcn_exp2f(x[r][t][e]);
                    l[r] += p;
                    pm[r] = __builtin_fmaf(p, middle(raw.vm[t][e]), pm[r]);
                    pv[e] = p * bf16_lo(raw.vm[t][e]);
                }
                pw[t][0] = pack_bf16x2(pv[0], pv[1]);
                pw[t][1] = pack_bf16x2(pv[2], pv[3]);
            }
            pb[r] = operand(pw[0][0], pw[0][1], pw[1][0], pw[1][1]);
            const bf16x8_t ones = operand(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
            psum[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pb[r], psum[r], 0, 0, 0);
        }
        // 8-byte groups of this lane: 4 tokens by 4 elements, tokens (0, 1) then (2, 3)
#pragma unroll
        for (int u = 0; u < D / 64; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bf16x8_t vc = operand(codes(m, raw.v[0][2 * u], e), codes(m, raw.v[0][2 * u + 1], e),
                                            codes(m, raw.v[1][2 * u], e), codes(m, raw.v[1][2 * u + 1], e));
#pragma unroll
                for (int r = 0; r < RT; ++r)
                    acc[r][4 * u + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vc, pb[r], acc[r][4 * u + e], 0, 0, 0);
            }
    }

    // what the lane's four parts of a row add up to; after it `acc` holds sums
    // of p V relative to `ref`, which is lower than any other's without a key
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            ref[r] = limit[r] == GROW ? ref[r] : -FLT_MAX;
            l[r] += __shfl_xor(l[r], 16);
            l[r] += __shfl_xor(l[r], 32);
            pm[r] += __shfl_xor(pm[r], 16);
            pm[r] += __shfl_xor(pm[r], 32);
#pragma unroll
            for (int i = 0; i < VI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[r][i][e] = __builtin_fmaf(16.0f, acc[r][i][e] - MID * psum[r][e], pm[r]);
        }
    }
};

// Workgroup: one sequence, one head of keys, some rows, one range of keys.
// SHARE: the four waves hold the same RT * 16 rows and take steps in turn, their
// sums are added through LDS; otherwise each has RT * 16 rows of its own.
template <int D, int RT, bool SHARE>
__global__ __launch_bounds__(64 * WAVES, RT == 1 ? 3 : RT == 2 ? 2 : 1) void kv4_attn_kernel(AttnArgs a) {
    constexpr int VI = D / 16, WROWS = RT * 16, BROWS = SHARE ? WROWS : WROWS * WAVES;
    const int lane = threadIdx.x & 63, n16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int split = blockIdx.x % a.splits, h = blockIdx.y;
    const int row_block = blockIdx.x / a.splits, row_blocks = gridDim.x / a.splits;
    const float kscale = a.scale * LOG2E;
    const CodeMask mask = code_mask();
    for (int seq = blockIdx.z; seq < a.b.batch; seq += gridDim.z) {
        const int n = kv4_count(a.b, seq), first = kv4_first(a.b, seq);
        const int len = min(max(0, a.b.lens[seq]), INT32_MAX - 2 * KEYS);
        // positions from here on are on no page; one of them is enough to say so
        const int64_t room = (int64_t)a.b.max_pages << a.c.page_shift;
        const int rows = n * a.group;  // at most tokens * heads_q
        for (int64_t r64 = (int64_t)row_block * BROWS; r64 < rows; r64 += (int64_t)row_blocks * BROWS) {
            const int r0 = (int)r64, w0 = r0 + (SHARE ? 0 : wave * WROWS);
            Rows<D, RT> R;
            R.clear();
            int seen = 0;         // keys that the block's rows, this wave's where they are its own, see
            int least = INT32_MAX;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const int row = w0 + 16 * r + n16;
                R.last[r] = -1;
                R.qsum[r] = 0.0f;
#pragma unroll
                for (int i = 0; i < R.KI; ++i) R.q[r][i] = operand(0, 0, 0, 0);
                if (row < rows) {
                    const int i = row / a.group, head = h * a.group + row % a.group;
                    R.last[r] = len - n + i;
                    const uint16_t* q = a.q + (first + i) * a.q_token + head * a.q_head + g * (D / 4);
#pragma unroll
                    for (int j = 0; j < R.KI; ++j) {
                        const u32x4_t u = reinterpret_cast<const u32x4_t*>(q)[j];
                        R.q[r][j] = __builtin_bit_cast(bf16x8_t, u);
#pragma unroll
                        for (int e = 0; e < 4; ++e) R.qsum[r] += bf16_lo(u[e]) + bf16_hi(u[e]);
                    }
                }
                R.qsum[r] += __shfl_xor(R.qsum[r], 16);
                R.qsum[r] += __shfl_xor(R.qsum[r], 32);
            }
            if (w0 < rows) {
                const int top = min(rows, w0 + WROWS) - 1;
                seen = max(0, len - n + top / a.group + 1);
                least = len - n + w0 / a.group + 1;  // keys that all of them see
            }
            const int64_t k0 = (int64_t)split * a.chunk;
            const int64_t end = min((int64_t)seen, room + KEYS);
            const int64_t k1 = split == a.splits - 1 ? end : min(end, k0 + a.chunk);
            const int step = SHARE ? KEYS * WAVES : KEYS;
            for (int64_t base64 = k0 + (SHARE ? wave * KEYS : 0); base64 < k1; base64 += step) {
                const int base = (int)base64;
                Raw<D> raw;
                bool bad[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int at = __builtin_amdgcn_readfirstlane(base + 16 * t);
                    int page = at < len ? kv4_page(a.c, a.b, seq, at) : 0;
                    bad[t] = page < 0;
                    const int64_t row = kv4_row(a.c, max(page, 0), h, at & (a.c.page_size - 1));
                    load_words<D / 32>(a.c.k + row * (D / 2) + n16 * (D / 2) + g * (D / 8), raw.k[t]);
                    load_words<D / 32>(a.c.v + row * (D / 2) + g * (2 * D) + n16 * (D / 8), raw.v[t]);
                    raw.km[t] = *reinterpret_cast<const u32x4_t*>(a.c.k_meta + row + 4 * g);
                    raw.vm[t] = *reinterpret_cast<const u32x4_t*>(a.c.v_meta + row + 4 * g);
                }
                R.step(raw, mask, kscale, base + KEYS > least || bad[0] || bad[1], base, bad[0], bad[1]);
            }
            R.finish();

            if constexpr (SHARE) {
                // the four waves' sums, one tile of rows after the other, in wave order
                __shared__ float sums[WAVES][16][D + 4];
                __shared__ float refs[WAVES][16], ls[WAVES][16];
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    __syncthreads();
                    if (g == 0) refs[wave][n16] = R.ref[r], ls[wave][n16] = R.l[r];
                    // O^T: element VI * (4 g + e) + i of row n16
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int i = 0; i < VI; ++i) sums[wave][n16][VI * (4 * g + e) + i] = R.acc[r][i][e];
                    __syncthreads();
                    // 16 threads a row, D / 16 elements each
                    const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * VI;
                    float ref = refs[0][row];
#pragma unroll
                    for (int w = 1; w < WAVES; ++w) ref = fmaxf(ref, refs[w][row]);
                    float l = 0.0f, v[VI] = {};
#pragma unroll
                    for (int w = 0; w < WAVES; ++w) {
                        const float f = __builtin_amdgcn_exp2f(refs[w][row] - ref);
                        l = __builtin_fmaf(ls[w][row], f, l);
#pragma unroll
                        for (int i = 0; i < VI; ++i) v[i] = __builtin_fmaf(sums[w][row][d0 + i], f, v[i]);
                    }
                    const int qrow = r0 + 16 * r + row;
                    if (qrow < rows) {
                        const int64_t to = (int64_t)(first + qrow / a.group) * a.heads_q + h * a.group + qrow % a.group;
                        if (a.splits > 1) {
                            float* p = a.part + (to * a.splits + split) * D + d0;
#pragma unroll
                            for (int i = 0; i < VI; i += 4)
                                *reinterpret_cast<f32x4_t*>(p + i) = f32x4_t{v[i], v[i + 1], v[i + 2], v[i + 3]};
                            if (d0 == 0) {
                                float* m = a.part + (int64_t)a.b.tokens * a.heads_q * a.splits * D + (to * a.splits + split) * 2;
                                m[0] = ref, m[1] = l;
                            }
                        } else {
                            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                            uint32_t w[VI / 2];
#pragma unroll
                            for (int i = 0; i < VI / 2; ++i) w[i] = pack_bf16x2(v[2 * i] * inv, v[2 * i + 1] * inv);
                            uint16_t* p = a.o + to * D + d0;
                            if constexpr (VI == 8)
                                *reinterpret_cast<u32x4_t*>(p) = u32x4_t{w[0], w[1], w[2], w[3]};
                            else
                                *reinterpret_cast<u32x2_t*>(p) = u32x2_t{w[0], w[1]};
                            if (a.lse && d0 == 0)
                                a.lse[to] = l == 0.0f ? -__builtin_inff() : (ref + __log2f(l)) * LN2;
                        }
                    }
                }
                __syncthreads();
            } else {
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const int row = w0 + 16 * r + n16;
                    if (row >= rows) continue;
                    const int64_t to = (int64_t)(first + row / a.group) * a.heads_q + h * a.group + row % a.group;
                    const float l = R.l[r], inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int d0 = VI * (4 * g + e);
                        if (a.splits > 1) {
                            float* p = a.part + (to * a.splits + split) * D + d0;
#pragma unroll
                            for (int i = 0; i < VI; i += 4)
                                *reinterpret_cast<f32x4_t*>(p + i) =
                                    f32x4_t{R.acc[r][i][e], R.acc[r][i + 1][e], R.acc[r][i + 2][e], R.acc[r][i + 3][e]};
                        } else {
                            uint32_t w[VI / 2];
#pragma unroll
                            for (int i = 0; i < VI / 2; ++i)
                                w[i] = pack_bf16x2(R.acc[r][2 * i][e] * inv, R.acc[r][2 * i + 1][e] * inv);
                            uint16_t* p = a.o + to * D + d0;
                            if constexpr (VI == 8)
                                *reinterpret_cast<u32x4_t*>(p) = u32x4_t{w[0], w[1], w[2], w[3]};
                            else
                                *reinterpret_cast<u32x2_t*>(p) = u32x2_t{w[0], w[1]};
                        }
                    }
                    if (g == 0) {
                        if (a.splits > 1) {
                            float* m = a.part + (int64_t)a.b.tokens * a.heads_q * a.splits * D + (to * a.splits + split) * 2;
                            m[0] = R.ref[r], m[1] = l;
                        } else if (a.lse) {
                            a.lse[to] = l == 0.0f ? -__builtin_inff() : (R.ref[r] + __log2f(l)) * LN2;
                        }
                    }
                }
            }
        }
    }
}

// the splits' sums, in their order; 16 threads a row
template <int D>
__global__ __launch_bounds__(256) void kv4_join_kernel(AttnArgs a) {
    constexpr int VI = D / 16;
    const int64_t first = a.b.cu_q ? min(max(a.b.cu_q[0], 0), a.b.tokens) : 0;
    const int64_t end = a.b.cu_q ? min(max(a.b.cu_q[a.b.batch], 0), a.b.tokens) : a.b.tokens;
    const float* meta = a.part + (int64_t)a.b.tokens * a.heads_q * a.splits * D;
    for (int64_t to = first * a.heads_q + blockIdx.x * 16 + (threadIdx.x >> 4); to < end * a.heads_q;
         to += (int64_t)gridDim.x * 16) {
        const int d0 = (threadIdx.x & 15) * VI;
        float ref = -FLT_MAX;
        for (int s = 0; s < a.splits; ++s) ref = fmaxf(ref, meta[(to * a.splits + s) * 2]);
        float l = 0.0f, v[VI] = {};
        for (int s = 0; s < a.splits; ++s) {
            const float* m = meta + (to * a.splits + s) * 2;
            const float f = __builtin_amdgcn_exp2f(m[0] - ref);
            l = __builtin_fmaf(m[1], f, l);
            const float* p = a.part + (to * a.splits + s) * D + d0;
#pragma unroll
            for (int i = 0; i < VI; ++i) v[i] = __builtin_fmaf(p[i], f, v[i]);
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint32_t w[VI / 2];
#pragma unroll
        for (int i = 0; i < VI / 2; ++i) w[i] = pack_bf16x2(v[2 * i] * inv, v[2 * i + 1] * inv);
        uint16_t* p = a.o + to * D + d0;
        if constexpr (VI == 8)
            *reinterpret_cast<u32x4_t*>(p) = u32x4_t{w[0], w[1], w[2], w[3]};
        else
            *reinterpret_cast<u32x2_t*>(p) = u32x2_t{w[0], w[1]};
        if (a.lse && d0 == 0) a.lse[to] = l == 0.0f ? -__builtin_inff() : (ref + __log2f(l)) * LN2;
    }
}

struct Plan {
    int rt;        // tiles of 16 rows a wave holds
    bool share;    // the workgroup's waves share them
    int row_blocks, splits, chunk;
};

// Rows of a sequence and key head decide the tile; the keys are split until
// there are about 8 workgroups a CU, or down to 256 keys.
Plan plan(int D, int batch, int heads_kv, int group, int max_q, int max_len) {
    Plan p;
    const int64_t rows = (int64_t)max_q * group;
    p.rt = rows <= 16 ? 1 : rows <= 32 || D == 128 ? 2 : 4;  // what a wave's registers hold
    p.share = rows <= 64;
    const int64_t brows = p.share ? p.rt * 16 : p.rt * 16 * WAVES;
    p.row_blocks = (int)std::min((int64_t)65536, (rows + brows - 1) / brows);
    const int64_t groups = std::max((int64_t)1, (int64_t)batch * heads_kv * p.row_blocks);
    const int64_t want = std::max((int64_t)1, 2048 / groups);
    const int unit = KEYS * WAVES;
    int64_t chunk = std::max((int64_t)256, ((int64_t)max_len + want - 1) / want);
    chunk = (chunk + unit - 1) / unit * unit;
    p.splits = (int)std::max((int64_t)1, ((int64_t)max_len + chunk - 1) / chunk);
    p.chunk = (int)std::min(chunk, (int64_t)INT32_MAX / unit * unit);
    return p;
}

template <int D>
hipError_t launch(const AttnArgs& a, const Plan& p, hipStream_t s) {
    const dim3 grid((unsigned)(p.row_blocks * p.splits), (unsigned)a.c.heads, (unsigned)std::min(a.b.batch, 65535));
    constexpr int T = 64 * WAVES;
    constexpr int MOST = D == 128 ? 2 : 4;
    if (!p.share)
        kv4_attn_kernel<D, MOST, false><<<grid, T, 0, s>>>(a);
    else if (p.rt == 4)
        kv4_attn_kernel<D, MOST, true><<<grid, T, 0, s>>>(a);
    else if (p.rt == 2)
        kv4_attn_kernel<D, 2, true><<<grid, T, 0, s>>>(a);
    else
        kv4_attn_kernel<D, 1, true><<<grid, T, 0, s>>>(a);
    if (p.splits > 1) {
        const int64_t rows = (int64_t)a.b.tokens * a.heads_q;
        kv4_join_kernel<D><<<(unsigned)std::min((int64_t)65536, (rows + 15) / 16), 256, 0, s>>>(a);
    }
    return hipGetLastError();
}

}  // namespace

size_t kv4_attn_workspace_size(int batch, int tokens, int heads_q, int heads_kv, int D, int max_q, int max_len) {
    const Plan p = plan(D, batch, heads_kv, heads_q / heads_kv, max_q, max_len);
    return p.splits > 1 ? (size_t)tokens * heads_q * p.splits * (D + 2) * sizeof(float) : 0;
}

hipError_t launch_kv4_attn(float scale, const KV4View& c, const KV4Batch& b, const uint16_t* q, int64_t q_token,
                           int64_t q_head, uint16_t* o, float* lse, int heads_q, int max_len, void* ws, hipStream_t s) {
    const int group = heads_q / c.heads;
    const Plan p = plan(c.D, b.batch, c.heads, group, b.max_q, max_len);
    const AttnArgs a{c, b, q, q_token, q_head, o, lse, static_cast<float*>(ws), scale, heads_q, group, p.splits, p.chunk};
    return c.D == 128 ? launch<128>(a, p, s) : launch<64>(a, p, s);
}

}  // namespace jh

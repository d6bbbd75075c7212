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
// (the values' lowest codes of each 16 bits are not shifted, and C = 1 + c/128, with
// 128 for 16: a sixteenth of the shifts less, 272 us for 273 over 15627 keys of chunks,
// 1291 for 1304 over 65536).
// -sum q is the accumulator that the first product starts from.  P' is rounded
// once and both of its sums take the rounded number, so what its rounding is
// multiplied by is the code's distance from the middle of the row's range, about
// the value's distance from the row's mean: the error is that of an attention
// with bf16 probabilities.  (With MID = 1 it was 0.0049 of the output at 8192
// keys of unit variance, with this one 0.0023; bf16 outputs alone are 0.0017.)
// The accumulators hold sum P' C, of which MID sum P' is by far the larger part and
// grows with the keys, and with it their roundings: taken out at the end alone, it
// made errors of 0.007 of the output at 65536 keys a wave and 0.015 at 131072.  So
// it is taken out every CENTER steps, of 1024 keys, and the error is 0.0024 from
// there to 262144 keys: an instruction an accumulator and 32 steps (chunks over
// 15627 keys 272 us for 270).
//
// One wave holds 16 rows (new tokens x heads of the group) times RT, and takes 32 keys
// at a time.  Both products are transposed, S^T = K Q^T and O^T = V^T P^T: the
// scores of a row then lie in the four lanes that also hold that row's P as the
// second product's operand, 4 neighbouring keys of each 16, and the softmax
// needs no exchange between lanes but for the row's maximum when it grows.
// Keys and values go from memory to the matrix cores through registers alone.
//
// Bound, one new token and 8 heads a key head, 64 sequences of 8192 keys: HBM, 5.1
// TB/s (112 us with the join); of 4096: 4.7 TB/s (61 us).  A short text of one sequence: what one
// CU takes in, 27 bytes/ns (1000 keys 10.5 us, 128 keys 5.3 us, 1 key 5.4 us).  From 32 rows on:
// vector instructions, a score's scale, exponential and rounding and a code's shift
// and and-or, about 290 beside 34 of the matrix cores' for 32 rows and 32 keys: chunks
// of 1024 tokens over 8192 keys, 8 sequences, 32 heads, D 128, 780 to 810 TFLOP/s on
// two cards, D 64 680.  What follows names both sides as they were when compared.
// Keys and values converted once for a workgroup, through LDS, were no faster (314
// us to 311 over 15627 keys; D 64 1034 to 829): the conversion saved went into
// writing and reading.  Keys as bytes, of which e4m3 holds 0 to 15 exactly, and q as
// two parts of bytes need fewer conversions (269 us to 293 a call), but that
// product adds in fewer bits: the log-sum-exp's error was 10^-5 and not 4 10^-7.
#include <algorithm>
#include <cfloat>

#include "kv4.hpp"
#include "launch.hpp"

namespace jh {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int KEYS = 32;     // keys of a step
constexpr int WAVES = 4;     // waves of a workgroup
constexpr int CENTER = 32;   // steps between two times that the middle's part leaves a wave's sums
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
    int turn;           // sequences after which the same part meets the same shader engine
};

// C of the low nibble of each half, bits 3-6 of a bf16 1.x
struct CodeMask {
    uint32_t keep, low, one;
};
// The two constants in registers, a vector and a scalar one, as one and-or
// takes them: as literals they are an and and an or.
__device__ __forceinline__ CodeMask code_mask() {
    CodeMask m{0x00780078u, 0x000f000fu, 0x3f803f80u};
    asm volatile("" : "+v"(m.keep));
    asm volatile("" : "+v"(m.low));
    asm volatile("" : "+s"(m.one));
    return m;
}
__device__ __forceinline__ uint32_t codes(CodeMask m, uint32_t w, int j) {
    const uint32_t x = j == 0 ? w << 3 : w >> (4 * j - 3);
    return (x & m.keep) | m.one;
}
// the value's, whose lowest code stays where it is: 1 + c/128
__device__ __forceinline__ uint32_t value_codes(CodeMask m, uint32_t w, int j) {
    return j == 0 ? (w & m.low) | m.one : codes(m, w, j);
}
__device__ __forceinline__ bf16x8_t operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(bf16x8_t, u32x4_t{a, b, c, d});
}

// where a step's two halves of 16 tokens lie: row indexes in the pool (of page 0
// where the table has no page), and which halves are on no page
struct Place {
    uint64_t row[2];
    bool bad[2];
};
// A sequence's row of the table: the step's two entries by scalar loads, which
// nothing waits for before `place` looks at them.
template <bool P16>  // pages of 16 tokens: the halves may be on two pages
struct Pages {
    const int32_t* row;
    int last;          // largest index
    int shift, inside; // page_shift, page_size - 1
    uint32_t pages, page_rows, head_row;  // rows of a page, and before the head's in it

    __device__ __forceinline__ void entries(int base, int (&page)[2]) const {
        page[0] = kv4_scalar(row + min(base >> shift, last));
        if (P16) page[1] = kv4_scalar(row + min((base + 16) >> shift, last));
    }
    // len: positions from there on are behind the sequence's end, their page is
    // not looked at
    __device__ __forceinline__ Place place(int base, int len, const int (&page)[2]) const {
        Place p;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int at = base + 16 * t;
            if (t && !P16) {
                p.row[1] = p.row[0] + 16;
                p.bad[1] = p.bad[0] & (at < len);
                break;
            }
            const bool fine = ((uint32_t)page[t] < pages) & ((at >> shift) <= last);
            p.bad[t] = !fine & (at < len);
            p.row[t] = (uint64_t)(fine ? (uint32_t)page[t] : 0u) * page_rows + (head_row + (uint32_t)(at & inside));
        }
        return p;
    }
};

// this lane's part of a step's keys, or values: codes, and scales and minimums of
// 4 neighbouring tokens of each half
template <int D>
struct Raw {
    uint32_t w[2][D / 32];
    u32x4_t meta[2];

    // at: this lane's bytes in 16 tokens' codes, 16 g its bytes in their metas.  Both
    // are made anew here, so that the loads take them as 32-bit offsets of a
    // scalar address and not as a 64-bit one kept in registers.
    __device__ __forceinline__ void load(const uint8_t* codes, const uint32_t* metas, const Place& p, uint32_t at, uint32_t g16) {
        asm volatile("" : "+v"(at), "+v"(g16));
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint8_t* c = codes + p.row[t] * (D / 2) + at;
            if constexpr (D == 128) {
                const u32x4_t u = *reinterpret_cast<const u32x4_t*>(c);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[t][i] = u[i];
            } else {
                const u32x2_t u = *reinterpret_cast<const u32x2_t*>(c);
                w[t][0] = u[0], w[t][1] = u[1];
            }
            meta[t] = *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint8_t*>(metas + p.row[t]) + g16);
        }
    }
};

// The four lanes that hold a row differ in bits 4 and 5 of their number: v_permlane
// 16 and 32 swaps put a value beside its partner's.
template <typename F>
__device__ __forceinline__ float over_row(float v, F f) {
    const uint32_t u = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const uint32_t w = __float_as_uint(v);
    const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row_sum(float v) {
    return over_row(v, [](float a, float b) { return a + b; });
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
    float qsum[RT], qscaled[RT];  // sum of the row's q, and that times the scale
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

    // Scores of the step's keys base .. base + 31, relative to `ref`.
    // q_at: with one tile of rows, this lane's operands of the queries in LDS.
    __device__ __forceinline__ void scores(const Raw<D>& k, CodeMask m, float kscale16, f32x4_t (&x)[RT][2],
                                           const u32x4_t* q_at) const {
#pragma unroll
        for (int r = 0; r < RT; ++r) x[r][0] = x[r][1] = f32x4_t{-qsum[r], -qsum[r], -qsum[r], -qsum[r]};
#pragma unroll
        for (int i = 0; i < KI; ++i) {
            bf16x8_t kc[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint32_t w = k.w[t][i];
                kc[t] = operand(codes(m, w, 0), codes(m, w, 1), codes(m, w, 2), codes(m, w, 3));
            }
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                // volatile: read at each step, not once and kept
                const bf16x8_t qi = RT == 1 ? __builtin_bit_cast(
                                                  bf16x8_t, *reinterpret_cast<const volatile u32x4_t*>(q_at + 64 * i))
                                            : q[r][i];
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    x[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kc[t], qi, x[r][t], 0, 0, 0);
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float c1 = bf16_lo(k.meta[t][e]) * kscale16, cm = bf16_hi(k.meta[t][e]);
#pragma unroll
                for (int r = 0; r < RT; ++r)
                    x[r][t][e] = __builtin_fmaf(c1, x[r][t][e], __builtin_fmaf(cm, qscaled[r], -ref[r]));
            }
    }

    // Where some of the keys are not seen by some row, or lie behind the
    // sequence's end, or on no page of the pool: an unseen key counts for nothing,
    // whatever its scale and minimum hold; where its value's are no numbers they
    // become 0, and the rows that see it NaN.
    __device__ __forceinline__ void mask(f32x4_t (&x)[RT][2], Raw<D>& v, const Place& p, int base) const {
        const int g = (threadIdx.x >> 4) & 3;
        float nan = __builtin_nanf(""), unseen = -__builtin_inff();
        asm volatile("" : "+v"(nan), "+v"(unseen));  // constants for here, not kept in registers
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool none = p.bad[t] || !(fabsf(middle(v.meta[t][e])) <= FLT_MAX);
                v.meta[t][e] = none ? 0u : v.meta[t][e];
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const float y = none ? nan : x[r][t][e];
                    x[r][t][e] = base + 16 * t + 4 * g + e > last[r] ? unseen : y;
                }
            }
    }

    // The reference moves where a score passes it; x becomes the scores' powers.
    __device__ __forceinline__ void rescale(f32x4_t (&x)[RT][2]) {
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
                const float high = over_row(top[r], [](float a, float b) { return fmaxf(a, b); });
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
    }

    // probabilities, their sums, and the sums of them times the values
    __device__ __forceinline__ void values(f32x4_t (&x)[RT][2], const Raw<D>& v, CodeMask m) {
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
                    pm[r] = __builtin_fmaf(p, middle(v.meta[t][e]), pm[r]);
                    pv[e] = p * bf16_lo(v.meta[t][e]);
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
                const bf16x8_t vc = operand(value_codes(m, v.w[0][2 * u], e), value_codes(m, v.w[0][2 * u + 1], e),
                                            value_codes(m, v.w[1][2 * u], e), value_codes(m, v.w[1][2 * u + 1], e));
#pragma unroll
                for (int r = 0; r < RT; ++r)
                    acc[r][4 * u + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vc, pb[r], acc[r][4 * u + e], 0, 0, 0);
            }
    }

    // all rows see a position that is on no page
    __device__ __forceinline__ void spoil() {
#pragma unroll
        for (int r = 0; r < RT; ++r) l[r] = __builtin_nanf("");
    }

    // Elements 4 u of the lane's groups have the lowest codes; the middle of a row's
    // range is code 7.5.
    static __device__ __forceinline__ constexpr float unit(int i) { return i % 4 == 0 ? 128.0f : 16.0f; }
    // The middle's part leaves `acc`: what stays of C is the code's distance from it,
    // whose sum does not grow with the keys' number but with its root.
    __device__ __forceinline__ void center() {
        float mid[2] = {-(1.0f + 7.5f / 128.0f), -(1.0f + 7.5f / 16.0f)};
        asm volatile("" : "+s"(mid[0]), "+s"(mid[1]));  // constants for here, not kept in registers
#pragma unroll
        for (int r = 0; r < RT; ++r) {
#pragma unroll
            for (int i = 0; i < VI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[r][i][e] = __builtin_fmaf(mid[i % 4 != 0], psum[r][e], acc[r][i][e]);
            psum[r] = f32x4_t{0, 0, 0, 0};
        }
    }

    // what the lane's four parts of a row add up to; after it `acc` holds sums
    // of p V relative to `ref`, which is lower than any other's without a key
    __device__ __forceinline__ void finish() {
        center();
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            ref[r] = limit[r] == GROW ? ref[r] : -FLT_MAX;
            l[r] = row_sum(l[r]);
            pm[r] = row_sum(pm[r]);
#pragma unroll
            for (int i = 0; i < VI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[r][i][e] = __builtin_fmaf(unit(i), acc[r][i][e], pm[r]);
        }
    }
};

// row of the outputs of a sequence and key head's row
__device__ __forceinline__ int64_t out_row(const AttnArgs& a, int h, int first, int row) {
    return (int64_t)(first + row / a.group) * a.heads_q + h * a.group + row % a.group;
}
// reference and sum of a row's split, behind all sums
__device__ __forceinline__ float* part_meta(const AttnArgs& a, int D, int64_t to, int split) {
    return a.part + (int64_t)a.b.tokens * a.heads_q * a.splits * D + (to * a.splits + split) * 2;
}

// Sums of row `to`: the output itself, or with splits this split's.
template <int N>
__device__ __forceinline__ void write_row(const AttnArgs& a, int D, int64_t to, int split, int d0, const float* v,
                                          float ref, float l) {
    if (a.splits > 1) {
        float* p = a.part + (to * a.splits + split) * D + d0;
#pragma unroll
        for (int i = 0; i < N; i += 4) *reinterpret_cast<f32x4_t*>(p + i) = f32x4_t{v[i], v[i + 1], v[i + 2], v[i + 3]};
        if (d0 == 0) {
            float* m = part_meta(a, D, to, split);
            m[0] = ref, m[1] = l;
        }
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = pack_bf16x2(v[2 * i] * inv, v[2 * i + 1] * inv);
    uint16_t* p = a.o + to * D + d0;
    if constexpr (N == 8)
        *reinterpret_cast<u32x4_t*>(p) = u32x4_t{w[0], w[1], w[2], w[3]};
    else
        *reinterpret_cast<u32x2_t*>(p) = u32x2_t{w[0], w[1]};
    if (a.lse && d0 == 0) a.lse[to] = l == 0.0f ? -__builtin_inff() : (ref + __log2f(l)) * LN2;
}

// The rows' sums after the last step.  O^T: lane (n16, g) has elements
// VI * (4 g + e) + i of row n16.
template <int D, int RT, bool SHARE>
__device__ __forceinline__ void write(const AttnArgs& a, const Rows<D, RT>& R, int tid, int wave, int split, int h,
                                      int first, int rows, int r0, int w0) {
    constexpr int VI = D / 16;
    const int n16 = tid & 15, g = (tid >> 4) & 3;
    if constexpr (SHARE) {
        // the four waves' sums, one tile of rows after the other, in wave order
        __shared__ float sums[WAVES][16][D + 4];
        __shared__ float refs[WAVES][16], ls[WAVES][16];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            __syncthreads();
            if (g == 0) refs[wave][n16] = R.ref[r], ls[wave][n16] = R.l[r];
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < VI; ++i) sums[wave][n16][VI * (4 * g + e) + i] = R.acc[r][i][e];
            __syncthreads();
            // 16 threads a row, D / 16 elements each
            const int row = tid >> 4, d0 = (tid & 15) * VI;
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
            if (qrow < rows) write_row<VI>(a, D, out_row(a, h, first, qrow), split, d0, v, ref, l);
        }
        __syncthreads();
    } else {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int row = w0 + 16 * r + n16;
            if (row >= rows) continue;
            const int64_t to = out_row(a, h, first, row);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v[VI];
#pragma unroll
                for (int i = 0; i < VI; ++i) v[i] = R.acc[r][i][e];
                write_row<VI>(a, D, to, split, VI * (4 * g + e), v, R.ref[r], R.l[r]);
            }
        }
    }
}

// Workgroup: one sequence, one head of keys, some rows, one range of keys.
// SHARE: the four waves hold the same RT * 16 rows and take steps in turn, their
// sums are added through LDS; otherwise each has RT * 16 rows of its own.
template <int D, int RT, bool SHARE, bool P16>
__global__ __launch_bounds__(64 * WAVES, RT == 1 ? 4 : RT == 2 && D == 64 ? 3 : 2) void kv4_attn_kernel(AttnArgs a) {
    constexpr int WROWS = RT * 16, BROWS = SHARE ? WROWS : WROWS * WAVES;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    // neighbouring workgroups have the heads of the same pages
    const int h = blockIdx.x % a.c.heads, part = blockIdx.x / a.c.heads;
    const int row_blocks = gridDim.x / a.c.heads / a.splits;
    const float kscale = a.scale * LOG2E, kscale16 = 16.0f * kscale;
    const CodeMask mask = code_mask();
    const int seq = blockIdx.y;
    // Workgroups are dealt to an XCD's four shader engines in turn.  The last
    // splits of short sequences are empty, and so are the last rows of those
    // with few new tokens: which part a workgroup has moves on as the turn
    // comes round, or an engine would get the same ones of all (64 sequences
    // of 512 to 8192 keys in 4 splits: 83 us, so 68).
    const int parts = a.splits * row_blocks, mine = (part + seq / a.turn) % parts;
    const int split = mine % a.splits, row_block = mine / a.splits;
    const int n = kv4_count(a.b, seq), first = kv4_first(a.b, seq);
    const int len = min(max(0, kv4_scalar(a.b.lens + seq)), INT32_MAX - 2 * KEYS * WAVES);
    // positions from here on are on no page; one of them is enough to say so
    const int64_t room = (int64_t)a.b.max_pages << a.c.page_shift;
    const Pages<P16> pages{a.b.table + (int64_t)seq * a.b.max_pages, a.b.max_pages - 1, a.c.page_shift,
                           a.c.page_size - 1, (uint32_t)a.c.num_pages, (uint32_t)a.c.heads * a.c.page_size,
                           (uint32_t)h * a.c.page_size};
    const int rows = n * a.group;  // at most tokens * heads_q
    for (int64_t r64 = (int64_t)row_block * BROWS; r64 < rows; r64 += (int64_t)row_blocks * BROWS) {
        const int r0 = (int)r64, w0 = r0 + (SHARE ? 0 : wave * WROWS);
        // Lane (n16, g): row n16 of 16, keys 4 g .. 4 g + 3 of 16.  The thread's
        // index is taken anew here and after the steps: what follows from it is
        // not kept in registers where it is not used.
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        const int lane = tid & 63, n16 = lane & 15, g = lane >> 4;
        // this lane's bytes of 16 tokens' keys and values
        const uint32_t k_at = n16 * (D / 2) + g * (D / 8), v_at = g * (2 * D) + n16 * (D / 8);
        // keys that the wave's rows see, and that all of them see
        int seen = 0, least = INT32_MAX;
        if (w0 < rows) {
            const int top = min(rows, w0 + WROWS) - 1;
            seen = max(0, len - n + top / a.group + 1);
            least = len - n + w0 / a.group + 1;
        }
        const int end = (int)min((int64_t)seen, room + KEYS);
        const int k0 = (int)min((int64_t)end, (int64_t)split * a.chunk);
        const int k1 = split == a.splits - 1 ? end : (int)min((int64_t)end, (int64_t)k0 + a.chunk);
        if (a.splits > 1 && k0 >= k1) {
            // no keys for this split: it says so, its sums are not read
            const int i = SHARE ? tid : lane;
            if (i < WROWS && w0 + i < rows) {
                const int64_t to = out_row(a, h, first, w0 + i);
                float* m = part_meta(a, D, to, split);
                float none = -FLT_MAX;
                asm volatile("" : "+v"(none));  // a constant for here, not kept in a register
                m[0] = none, m[1] = 0.0f;
            }
            continue;
        }
        const int step = SHARE ? KEYS * WAVES : KEYS;
        int base = __builtin_amdgcn_readfirstlane(k0 + (SHARE ? wave * KEYS : 0));  // all well below 2^31
        Raw<D> k, v;
        int page[2];
        Place here{};
        bool loaded = base < k1;
        if (loaded) {
            pages.entries(base, page);
            here = pages.place(base, len, page);
            k.load(a.c.k, a.c.k_meta, here, k_at, 16 * g);
            v.load(a.c.v, a.c.v_meta, here, v_at, 16 * g);
        }
        Rows<D, RT> R;
        R.clear();
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
            R.qsum[r] = row_sum(R.qsum[r]);
            R.qscaled[r] = R.qsum[r] * kscale;
        }
        // one tile of rows: the second product's operand from LDS, in the order
        // of the lanes, leaves room for a fourth wave on each SIMD
        __shared__ u32x4_t q_lds[RT == 1 ? 64 * (D / 32) : 1];
        if constexpr (RT == 1) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) q_lds[lane + 64 * i] = __builtin_bit_cast(u32x4_t, R.q[0][i]);
            __syncthreads();
        }
        const u32x4_t* q_at = q_lds + lane;
        f32x4_t x[RT][2];
        const int whole = min(k1, least - KEYS + 1);  // steps up to there: all rows see all keys
        if (base < whole) {
            bool bad = here.bad[0] | here.bad[1];
            // The next step's keys are loaded once this step's are scores, its
            // values once this step's are summed, into the same registers.  A wave
            // with scores goes first at the vector unit, so that the other's
            // matrix products come to run beside its softmax: 277 us with it, 294
            // without (chunks of 1024 tokens, 15627 keys; D 64, 65536 keys: 757, 819); first with the
            // keys' product too: 312 to 330.
            for (base += step; base < whole; base += step) {
                if (base / step % CENTER == 0) R.center();  // here, where no scores or values wait in registers
                pages.entries(base, page);
                __builtin_amdgcn_sched_barrier(0);  // asked for here, looked at after the scores
                R.scores(k, mask, kscale16, x, q_at);
                here = pages.place(base, len, page);
                k.load(a.c.k, a.c.k_meta, here, k_at, 16 * g);
                __builtin_amdgcn_s_setprio(1);
                R.rescale(x);
                R.values(x, v, mask);
                __builtin_amdgcn_s_setprio(0);
                v.load(a.c.v, a.c.v_meta, here, v_at, 16 * g);
                bad = bad | here.bad[0] | here.bad[1];
            }
            R.scores(k, mask, kscale16, x, q_at);
            R.rescale(x);
            R.values(x, v, mask);
            if (bad) R.spoil();
            loaded = false;
        }
        for (; base < k1; base += step) {
            if (!loaded) {
                pages.entries(base, page);
                here = pages.place(base, len, page);
                k.load(a.c.k, a.c.k_meta, here, k_at, 16 * g);
                v.load(a.c.v, a.c.v_meta, here, v_at, 16 * g);
            }
            loaded = false;
            R.scores(k, mask, kscale16, x, q_at);
            __builtin_amdgcn_s_setprio(1);
            R.mask(x, v, here, base);
            R.rescale(x);
            R.values(x, v, mask);
            __builtin_amdgcn_s_setprio(0);
        }
        R.finish();
        int tid2 = threadIdx.x;
        asm volatile("" : "+v"(tid2));
        write<D, RT, SHARE>(a, R, tid2, wave, split, h, first, rows, r0, w0);
    }
}

// the splits' sums, 16 threads for a row's D elements and PARTS such groups for a
// row, each every PARTS-th split; the groups' sums are added in order through LDS
template <int D, int PARTS>
__global__ __launch_bounds__(256) void kv4_join_kernel(AttnArgs a) {
    constexpr int VI = D / 16, ROWS = 16 / PARTS;
    const int first = kv4_first(a.b, 0), end = kv4_first(a.b, a.b.batch);
    const float* meta = a.part + (int64_t)a.b.tokens * a.heads_q * a.splits * D;
    const int group = threadIdx.x >> 4, part = group % PARTS, d0 = (threadIdx.x & 15) * VI;
    const int64_t last = (int64_t)end * a.heads_q;
    __shared__ float sums[16][D + 4], refs[16], ls[16];
    for (int64_t r0 = (int64_t)first * a.heads_q + blockIdx.x * ROWS; r0 < last; r0 += (int64_t)gridDim.x * ROWS) {
        const int64_t to = r0 + group / PARTS;
        float ref = -FLT_MAX, l = 0.0f, v[VI] = {};
        if (to < last)
            for (int s = part; s < a.splits; s += PARTS) {
                const float* m = meta + (to * a.splits + s) * 2;
                if (m[1] == 0.0f) continue;  // no keys, no sums
                const float* p = a.part + (to * a.splits + s) * D + d0;
                const float high = fmaxf(ref, m[0]);
                const float f = __builtin_amdgcn_exp2f(ref - high), g = __builtin_amdgcn_exp2f(m[0] - high);
                ref = high;
                l = __builtin_fmaf(m[1], g, l * f);
#pragma unroll
                for (int i = 0; i < VI; ++i) v[i] = __builtin_fmaf(p[i], g, v[i] * f);
            }
        __syncthreads();  // the rows before have been read
        if (d0 == 0) refs[group] = ref, ls[group] = l;
#pragma unroll
        for (int i = 0; i < VI; ++i) sums[group][d0 + i] = v[i];
        __syncthreads();
        for (int i = threadIdx.x; i < ROWS * D; i += 256) {
            const int g0 = i / D * PARTS, d = i % D;
            const int64_t row = r0 + i / D;
            if (row >= last) break;
            float high = refs[g0];
#pragma unroll
            for (int p = 1; p < PARTS; ++p) high = fmaxf(high, refs[g0 + p]);
            float total = 0.0f, o = 0.0f;
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                const float f = __builtin_amdgcn_exp2f(refs[g0 + p] - high);
                total = __builtin_fmaf(ls[g0 + p], f, total);
                o = __builtin_fmaf(sums[g0 + p][d], f, o);
            }
            o = total == 0.0f ? 0.0f : o / total;
            a.o[row * D + d] = (uint16_t)pack_bf16x2(o, 0.0f);
            if (a.lse && d == 0) a.lse[row] = total == 0.0f ? -__builtin_inff() : (high + __log2f(total)) * LN2;
        }
    }
}

struct Plan {
    int rt;        // tiles of 16 rows a wave holds
    bool share;    // the workgroup's waves share them
    int row_blocks, splits, chunk;
};

// Rows of a sequence and key head decide the tile.  The keys are split until
// the card is full: 8 workgroups a CU of one tile (64 sequences of 512 to 8192
// keys: 82 us whole, 78 + 5 in 2 splits, 68 + 5 in 4, 66 + 7 in 8), fewer of more
// tiles, whose start and end cost more (131072 keys, 40 rows of 64: 23 + 5 us
// in 64 splits, 27 + 5 in 48, 24 + 6 in 96, 21 + 7 in 128; 15627 keys of 3022
// new tokens: 315 us whole, 382 + 32 in 2).  A split costs a second launch too:
// none below 1024 keys (1000 keys: 10 us whole, 7 + 3 in 4 splits).
// With a max_q of the longest sequence the splits' sums are 35 MB at most.  One that is
// too small (a single token's, for a prompt's rows) would ask for splits of rows
// that fill the card by themselves, and for gigabytes: no more than WORKSPACE.
constexpr int64_t WORKSPACE = int64_t(256) << 20;
Plan plan(int D, int batch, int tokens, int heads_kv, int group, int max_q, int max_len) {
    Plan p;
    const int64_t rows = (int64_t)std::max(1, std::min(max_q, tokens)) * group;
    p.rt = rows <= 16 ? 1 : rows <= 32 || D == 128 ? 2 : rows <= 48 ? 3 : 4;  // what a wave's registers hold
    p.share = rows <= 64;
    const int64_t brows = p.share ? p.rt * 16 : p.rt * 16 * WAVES;
    // below 2^24 workgroups of 256 threads; a workgroup goes on to the rows that are left
    p.row_blocks = (int)std::min((int64_t)std::max(1, (1 << 22) / heads_kv), (rows + brows - 1) / brows);
    const int64_t groups = (int64_t)batch * heads_kv * p.row_blocks;
    const int full = p.rt == 1 ? 2048 : p.rt == 2 ? p.share ? 1024 : 512 : 256;
    const int64_t each = (int64_t)tokens * heads_kv * group * (D + 2) * (int64_t)sizeof(float);
    const int64_t want = std::max((int64_t)1, std::min(full / groups, WORKSPACE / each));
    const int unit = KEYS * WAVES;
    int64_t chunk = std::max((int64_t)1024, ((int64_t)max_len + want - 1) / want);
    chunk = (chunk + unit - 1) / unit * unit;
    p.splits = (int)std::max((int64_t)1, ((int64_t)max_len + chunk - 1) / chunk);
    p.chunk = (int)std::min(chunk, (int64_t)INT32_MAX / unit * unit);
    return p;
}

template <int D, bool P16>
hipError_t launch(const AttnArgs& a, const Plan& p, hipStream_t s) {
    const dim3 grid((unsigned)(p.row_blocks * p.splits * a.c.heads), (unsigned)a.b.batch);
    constexpr int T = 64 * WAVES, MOST = D == 128 ? 2 : 4;
    if (!p.share)
        kv4_attn_kernel<D, MOST, false, P16><<<grid, T, 0, s>>>(a);
    else if (p.rt == 4)
        kv4_attn_kernel<D, MOST, true, P16><<<grid, T, 0, s>>>(a);
    else if (p.rt == 3)
        kv4_attn_kernel<D, D == 128 ? MOST : 3, true, P16><<<grid, T, 0, s>>>(a);
    else if (p.rt == 2)
        kv4_attn_kernel<D, 2, true, P16><<<grid, T, 0, s>>>(a);
    else
        kv4_attn_kernel<D, 1, true, P16><<<grid, T, 0, s>>>(a);
    const int64_t rows = (int64_t)a.b.tokens * a.heads_q;
    if (p.splits > 4)
        kv4_join_kernel<D, 16><<<(unsigned)std::min((int64_t)1 << 20, rows), 256, 0, s>>>(a);
    else if (p.splits > 1)
        kv4_join_kernel<D, 4><<<(unsigned)std::min((int64_t)1 << 20, (rows + 3) / 4), 256, 0, s>>>(a);
    return hipGetLastError();
}

template <int D>
hipError_t launch(const AttnArgs& a, const Plan& p, hipStream_t s) {
    return a.c.page_size == 16 ? launch<D, true>(a, p, s) : launch<D, false>(a, p, s);
}

}  // namespace

size_t kv4_attn_workspace_size(int batch, int tokens, int heads_q, int heads_kv, int D, int max_q, int max_len) {
    const Plan p = plan(D, batch, tokens, heads_kv, heads_q / heads_kv, max_q, max_len);
    return p.splits > 1 ? (size_t)tokens * heads_q * p.splits * (D + 2) * sizeof(float) : 0;
}

hipError_t launch_kv4_attn(float scale, const KV4View& c, const KV4Batch& b, const uint16_t* q, int64_t q_token,
                           int64_t q_head, uint16_t* o, float* lse, int heads_q, int max_len, void* ws, hipStream_t s) {
    const int group = heads_q / c.heads;
    const Plan p = plan(c.D, b.batch, b.tokens, c.heads, group, b.max_q, max_len);
    const AttnArgs a{c, b, q, q_token, q_head, o, lse, static_cast<float*>(ws), scale, heads_q, group, p.splits, p.chunk,
                     p.splits * p.row_blocks % 4 == 0 ? 1 : p.splits * p.row_blocks % 2 == 0 ? 2 : 4};
    return c.D == 128 ? launch<128>(a, p, s) : launch<64>(a, p, s);
}

}  // namespace jh

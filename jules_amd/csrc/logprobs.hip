// logprobs.hip - log probabilities of given tokens, with the log-sum-exp, the
// entropy and the most likely alternatives of each row of logits, and the
// gradient with respect to the logits.  No counterpart in the reference, whose
// fusedCrossEntropyLoss (rowops.hip) gives one mean loss of fp32 rows.
//
//   z = scale x,  m = max z,  s = sum e^(z - m),  w = sum e^(z - m) (z - m)
//   lse = m + ln s,  logp = z_t - m - ln s,  entropy = ln s - w / s
//
// One pass over a row: every thread keeps the maximum and the sums of its own
// pieces of 8 neighbouring elements, the sums relative to its maximum, and the
// block joins them at the end.  Bound by HBM: 4096 x 50257 bf16 73 us, 5.7 TB/s,
// where a plain read of as many bytes gets 5.1 to 6.3.  What that took:
//   64 registers, for 32 waves a CU (90 us; 147 with one block of 1024 threads);
//   whole turns of 4 pieces without checks, their loads under way together (72 us;
//   checks around each load made the compiler wait for it before the next);
//   512 threads a row, not 1024: what a wave spends on joining is as much as it
//   spends on 100 elements a thread.
//
// The k alternatives are the first in the order (value falling, index rising).
// Each thread also keeps its largest value and the first of its pieces that has
// it.  The k-th of these pairs (value, piece) bounds what can be among the first
// k, since k threads hold an element at least as far in front; only those k
// threads can hold more.  They read their pieces again and put the elements that
// reach the bound in LDS, where each counts those before it.  No row, whatever its
// values, has more of them than k threads have elements.  4096 x 50257 bf16 take 89,
// 97 and 205 us with 1, 20 and 64 alternatives, 2048 x 50257 fp32 74 us with 5
// (5.6 TB/s); there the six barriers between these steps cost most.
//
// A row may be split over blocks, whose results, their k alternatives among them,
// are then joined by a second kernel.
//
//   dx_j = scale (g ([j = t] - p_j) - gh p_j (ln p_j + entropy)),  p = e^(z - lse)
#include <algorithm>
#include <cfloat>

#include "launch.hpp"
#include "pieces.hpp"

namespace jh {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// where a distance from the maximum is -infinity: e^ of it is 0, and so is its product with that
constexpr float FAR = -1e30f;
constexpr int MAX_PARTS = 64;
// keys in LDS, 64 KB of it less the other shared values
constexpr int MAX_KEYS = 8064;

// a float's place in an order of unsigned numbers, 0 where nothing is; -0 is +0
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
    return __uint_as_float(o ^ ((int32_t)o < 0 ? 0x80000000u : 0xffffffffu));
}
// key of (value falling, place rising)
__device__ __forceinline__ uint64_t key_of(float v, uint32_t place) { return (uint64_t)order_of(v) << 32 | (0xffffffffu - place); }
__device__ __forceinline__ uint32_t place_of(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

// The largest of three, NaN where one is NaN.  As an instruction of its own: the
// builtin's operands are first multiplied by 1 to quieten NaNs, an instruction an element.
__device__ __forceinline__ float largest(float a, float b, float c) {
    float r;
    asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// maximum, and the sums relative to it: e^((x - m) scale), and that times its exponent in powers of 2
struct Sums {
    float m, s, w;
};
__device__ __forceinline__ Sums no_sums() { return Sums{-FLT_MAX, 0.0f, 0.0f}; }
// relative to a maximum m at least as large; c2 = scale log2(e)
__device__ __forceinline__ void raise(Sums* a, float m, float c2) {
    const float d = larger((a->m - m) * c2, FAR), f = __builtin_amdgcn_exp2f(d);
    a->w = f * __builtin_fmaf(d, a->s, a->w);
    a->s *= f;
    a->m = m;
}
__device__ __forceinline__ Sums join(Sums a, Sums b, float c2) {
    const float m = larger(a.m, b.m);
    raise(&a, m, c2);
    raise(&b, m, c2);
    return Sums{m, a.s + b.s, a.w + b.w};
}

struct LogprobArgs {
    const void* logits;
    const int32_t* tokens;
    float *logp, *lse, *entropy;  // null: not wanted
    int32_t* top_ids;
    float* top_logp;
    int64_t stride;
    float scale, c2;
    int M, N, top, parts, width;  // width: elements of a part, a multiple of 8
    // of split rows: [M][parts] sums, [M][parts][top] keys
    Sums* sums;
    uint64_t* keys;
};

// ln of the sum; what a row of nothing but -infinity gets: probability 0 everywhere, no entropy
struct RowNumbers {
    float m, log_s, entropy;
    bool bad, none;  // a NaN or +infinity; nothing but -infinity
};
__device__ __forceinline__ RowNumbers row_numbers(const Sums& a) {
    RowNumbers r;
    r.bad = !(a.s <= FLT_MAX);
    r.none = a.s == 0.0f;
    r.m = a.m;
    r.log_s = logf(a.s);
    r.entropy = r.bad ? __builtin_nanf("") : r.none ? 0.0f : fmaxf(r.log_s - LN2 * (a.w / a.s), 0.0f);
    return r;
}
__device__ __forceinline__ float log_prob(const RowNumbers& r, float x, float scale) {
    return r.bad ? __builtin_nanf("") : r.none ? -INFINITY : (x - r.m) * scale - r.log_s;
}
template <typename T>
__device__ __forceinline__ void write_row(const LogprobArgs& a, int64_t row, const RowNumbers& r) {
    if (a.lse) a.lse[row] = r.bad ? __builtin_nanf("") : r.none ? -INFINITY : __builtin_fmaf(r.m, a.scale, r.log_s);
    if (a.entropy) a.entropy[row] = r.entropy;
    if (a.logp) {
        const int t = a.tokens[row];
        float v = 0.0f;  // a negative token: none
        if (t >= a.N)
            v = __builtin_nanf("");
        else if (t >= 0)
            v = log_prob(r, load1(static_cast<const T*>(a.logits) + row * a.stride + t), a.scale);
        a.logp[row] = v;
    }
}
__device__ __forceinline__ void write_top(const LogprobArgs& a, int64_t row, int rank, uint64_t key, const RowNumbers& r) {
    const int64_t at = row * a.top + rank;
    a.top_ids[at] = r.bad ? -1 : (int32_t)place_of(key);
    a.top_logp[at] = log_prob(r, value_of((uint32_t)(key >> 32)), a.scale);
}

// how many of n keys in LDS come before this one
__device__ __forceinline__ int rank_of(uint64_t key, const uint64_t* keys, int n) {
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < n; ++i) rank += keys[i] > key;
    return rank;
}

// A thread's largest value, the first of its pieces that has it (-1: no pieces), and the
// largest of its other pieces' largest values
struct Likeliest {
    float best, next;
    int piece;
};

// A part's alternatives, their keys in LDS, in any order.  Returns how many reached the
// bound (see above), the `top` first among them.  keys has room for the elements of
// `top` threads, and for one of each thread.
template <typename T, int BT>
__device__ __forceinline__ int find_top(uint64_t* keys, const T* x, int first, int len, int top, const Likeliest& l) {
    __shared__ uint32_t groups[64];
    __shared__ int found[2];
    __shared__ uint64_t threshold;
    __shared__ uint32_t group_threshold;
    const int tid = threadIdx.x;
    const uint64_t own = l.piece < 0 ? 0 : key_of(l.best, (uint32_t)l.piece);
    uint32_t g = (uint32_t)(own >> 32);
#pragma unroll
    for (int o = 1; o < BT / 64; o <<= 1) g = max(g, (uint32_t)__shfl_xor((int)g, o));
    if (tid % (BT / 64) == 0) groups[tid / (BT / 64)] = g;
    if (tid < 2) found[tid] = 0;
    if (tid == 0) threshold = 0;
    __syncthreads();
    if (tid < 64) {
        // a number that at least `top` of 64 groups reach, so at least as many threads: the
        // largest with its first bits, until no more than that reach it
        g = groups[tid];
        uint32_t at = 0;
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
            const int reach = __popcll(__ballot(g >= (at | bit)));
            if (reach >= top) at |= bit;
            if (reach == top) break;
        }
        if (tid == 0) group_threshold = at;
    }
    __syncthreads();
    // the top-th of the threads' best
    if (own && (uint32_t)(own >> 32) >= group_threshold) keys[atomicAdd(&found[0], 1)] = own;
    __syncthreads();
    const int threads = found[0];
    if (tid < threads && rank_of(keys[tid], keys, threads) == top - 1) threshold = keys[tid];
    __syncthreads();
    // those threads' elements that reach it, mostly of one piece each; where a thread may have
    // more, its wave reads all of its pieces together
    const uint64_t bound = threshold;
    const auto take = [&](int piece) {
        const int n = min(8, len - 8 * piece);
        const f32x8_t v = values(load_raw(x + 8 * piece, n));
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n && key_of(v.v[i], (uint32_t)piece) >= bound)
                keys[atomicAdd(&found[1], 1)] = key_of(v.v[i], (uint32_t)(first + 8 * piece + i));
    };
    const bool reaches = own && own >= bound;
    const bool more = reaches && order_of(l.next) >= (uint32_t)(bound >> 32);
    if (reaches && !more) take(l.piece);
    for (uint64_t left = __ballot(more); left; left &= left - 1) {
        const int thread = (tid & ~63) + __builtin_ctzll(left);
        for (int piece = thread + BT * (tid & 63); 8 * piece < len; piece += BT * 64) take(piece);
    }
    __syncthreads();
    return found[1];
}

// -infinity as an element's bits
template <typename T>
constexpr uint32_t kNothing = sizeof(T) == 4 ? 0xff800000u : 0xff80u;

// pieces b, b + BT, .. of the thread's part
template <int BT, bool TOP, typename T, int B>
__device__ __forceinline__ void add_pieces(const Raw8<T> (&raw)[B], int b, float c2, Sums* mine, Likeliest* l) {
    f32x8_t v[B];
    float m = mine->m;
#pragma unroll
    for (int t = 0; t < B; ++t) {
        v[t] = values(raw[t]);
        const float* e = v[t].v;
        const float top = largest(largest(e[0], e[1], e[2]), largest(e[3], e[4], e[5]), largest(e[6], e[7], e[7]));
        m = larger(m, top);
        if constexpr (TOP) {
            l->next = __builtin_amdgcn_fmed3f(l->next, l->best, top);  // next <= best: the second of the three
            if (top > l->best || l->piece < 0) l->best = top, l->piece = b + BT * t;
        }
    }
    raise(mine, m, c2);
#pragma unroll
    for (int t = 0; t < B; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = larger((v[t].v[i] - m) * c2, FAR), e = __builtin_amdgcn_exp2f(d);
            mine->s += e;
            mine->w = __builtin_fmaf(e, d, mine->w);
        }
}

// BT threads for a part of a row, in turns of B pieces each.  Dynamic LDS with TOP: launch_parts()
template <typename T, int BT, bool TOP>
__global__ __launch_bounds__(BT, 8) void logprobs_kernel(LogprobArgs a) {
    constexpr int WAVES = BT / 64, B = 4;
    __shared__ Sums wave_sums[WAVES];
    extern __shared__ uint64_t keys[];
    const int tid = threadIdx.x, part = blockIdx.y;
    const int first = part * a.width, len = min(a.width, a.N - first);
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.logits) + row * a.stride + first;
        Sums mine = no_sums();
        Likeliest l{-INFINITY, -INFINITY, -1};
        int b = tid;
        for (; 8 * (b + BT * (B - 1)) + 8 <= len; b += B * BT) {
            Raw8<T> raw[B];
#pragma unroll
            for (int t = 0; t < B; ++t) raw[t] = load_raw(x + 8 * (b + BT * t), 8);
            add_pieces<BT, TOP>(raw, b, a.c2, &mine, &l);
        }
        if (8 * (b + BT) + 8 <= len) {
            const Raw8<T> raw[2] = {load_raw(x + 8 * b, 8), load_raw(x + 8 * (b + BT), 8)};
            add_pieces<BT, TOP>(raw, b, a.c2, &mine, &l);
            b += 2 * BT;
        }
#pragma unroll 1
        for (; 8 * b < len; b += BT) {
            const Raw8<T> raw[1] = {load_raw(x + 8 * b, min(8, len - 8 * b), kNothing<T>)};
            add_pieces<BT, TOP>(raw, b, a.c2, &mine, &l);
        }
        // the wave's, relative to its maximum, then the block's
        float m = mine.m;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = larger(m, __shfl_xor(m, o));
        raise(&mine, m, a.c2);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            mine.s += __shfl_xor(mine.s, o);
            mine.w += __shfl_xor(mine.w, o);
        }
        if ((tid & 63) == 0) wave_sums[tid >> 6] = mine;
        __syncthreads();
        Sums all = wave_sums[tid % WAVES];
#pragma unroll
        for (int o = 1; o < WAVES; o <<= 1)
            all = join(all, Sums{__shfl_xor(all.m, o), __shfl_xor(all.s, o), __shfl_xor(all.w, o)}, a.c2);
        const int64_t item = row * a.parts + part;
        if (TOP || tid == 0) {
            const RowNumbers r = row_numbers(all);
            if (tid == 0) {
                if (a.parts > 1)
                    a.sums[item] = all;
                else
                    write_row<T>(a, row, r);
            }
            if constexpr (TOP) {
                uint64_t* part_keys = a.parts > 1 ? a.keys + item * a.top : nullptr;
                // no order where there is a NaN or +infinity
                const int n = r.bad ? 0 : find_top<T, BT>(keys, x, first, len, a.top, l);
                if (tid < a.top && (r.bad || tid >= n)) {  // a part may be shorter than `top`, a row not
                    if (part_keys)
                        part_keys[tid] = 0;
                    else
                        write_top(a, row, tid, 0, r);
                }
                for (int i = tid; i < n; i += BT) {
                    const uint64_t key = keys[i];
                    const int rank = rank_of(key, keys, n);
                    if (rank >= a.top) continue;
                    if (part_keys)
                        part_keys[rank] = key;
                    else
                        write_top(a, row, rank, key, r);
                }
            }
        }
        __syncthreads();  // the shared values are the next row's
    }
}

// Rows that were split: a block each.  Every part's keys are sorted, so the smallest of
// the parts' k/parts-th bounds the row's k-th from below: few keys reach it.
template <typename T>
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogprobArgs a) {
    extern __shared__ uint64_t keys[];
    __shared__ int found;
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const int n = a.parts * a.top, lane = threadIdx.x & 63;
        const uint64_t* row_keys = a.keys + row * n;
        uint64_t bound = ~(uint64_t)0;
        if (lane < a.parts && a.top) bound = row_keys[lane * a.top + (a.top - 1) / a.parts];
        Sums all = lane < a.parts ? a.sums[row * a.parts + lane] : no_sums();
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            all = join(all, Sums{__shfl_xor(all.m, o), __shfl_xor(all.s, o), __shfl_xor(all.w, o)}, a.c2);
            const uint64_t other = __shfl_xor(bound, o);
            bound = other < bound ? other : bound;
        }
        const RowNumbers r = row_numbers(all);
        if (threadIdx.x == 0) write_row<T>(a, row, r);
        if (!a.top) continue;
        if (r.bad) {
            if (threadIdx.x < a.top) write_top(a, row, threadIdx.x, 0, r);
            continue;
        }
        if (threadIdx.x == 0) found = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += 256) {
            const uint64_t key = row_keys[i];
            if (key && key >= bound) keys[atomicAdd(&found, 1)] = key;
        }
        __syncthreads();
        const int reached = found;
        for (int i = threadIdx.x; i < reached; i += 256) {
            const int rank = rank_of(keys[i], keys, reached);
            if (rank < a.top) write_top(a, row, rank, keys[i], r);
        }
        __syncthreads();
    }
}

// How rows are split, and the threads of a block.  Few long rows are split for the chip's
// sake: 64 x 128256 bf16 take 33 us whole, 20 in parts; 512 x 128256 49 and 35.  Below 65536
// the second launch costs the caller more than it gives (64 x 32000 fp32: 16 us and 20).
// A wave a row up to 8192 elements: 16384 x 8000 bf16 52.6 us, with 256 threads 57.9; 65536 x
// 1000 38 and 85; with many alternatives their keys leave few such blocks a CU.  1024 threads
// where a block a CU is all there is.
struct Split {
    int parts, width, threads;
};
Split split_of(int M, int N, int top) {
    // what the keys in LDS allow: `top` threads' elements
    const int most = top ? MAX_KEYS / (8 * top) * (8 * 512) : N;
    int parts = N / most + (N % most != 0);
    if (M <= 512 && N >= 65536) parts = std::max(parts, std::min(1024 / M, N / 8192));
    parts = std::min(std::max(parts, 1), MAX_PARTS);
    const int width = (N / parts + (N % parts != 0) + 7) / 8 * 8;
    const int threads = width <= 8192 && top <= 8 ? 64 : width <= 8192 ? 256 : M * parts > 256 || width <= 16384 ? 512 : 1024;
    return Split{N / width + (N % width != 0), width, threads};
}

template <typename T, int BT>
void launch_parts(const LogprobArgs& a, hipStream_t s) {
    // the runtime takes fewer than 2^32 threads a launch
    const dim3 grid((unsigned)std::min(a.M, (1 << 20) / a.parts), (unsigned)a.parts);
    if (a.top) {
        const int turns = a.width / (8 * BT) + (a.width % (8 * BT) != 0);
        logprobs_kernel<T, BT, true><<<grid, BT, sizeof(uint64_t) * std::max(BT, 8 * turns * a.top), s>>>(a);
    } else {
        logprobs_kernel<T, BT, false><<<grid, BT, 0, s>>>(a);
    }
}

template <typename T>
hipError_t launch(const LogprobArgs& a, int threads, hipStream_t s) {
    if (threads == 64)
        launch_parts<T, 64>(a, s);
    else if (threads == 256)
        launch_parts<T, 256>(a, s);
    else if (threads == 512)
        launch_parts<T, 512>(a, s);
    else
        launch_parts<T, 1024>(a, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.parts == 1) return e;
    logprobs_join_kernel<T><<<(unsigned)std::min(a.M, 1 << 20), 256, sizeof(uint64_t) * a.parts * a.top, s>>>(a);
    return hipGetLastError();
}

// ---- gradient ------------------------------------------------------------------

struct GradArgs {
    const void* logits;
    const int32_t* tokens;
    const float *lse, *entropy, *dlogp, *dentropy;  // entropy and dentropy null: no gradient of the entropy
    void* dlogits;
    int64_t stride, out_stride;
    float scale;
    int M, N;
};

// the log of a probability below all fp32 numbers: e^ of it is 0, and its product with what
// reaches the entropy stays within fp32, so that the two are 0 together
constexpr float GONE = -150.0f;

// BT threads for 32 bytes each of a row; a row's blocks side by side (rows side by side: 177 us
// for 4096 x 50257 bf16 instead of 148)
template <typename T>
constexpr int kGradPieces = 4 / (int)sizeof(T);

template <typename T, int BT>
__global__ __launch_bounds__(BT) void logprobs_bwd_kernel(GradArgs a) {
    constexpr int PIECES = kGradPieces<T>;
    const int first = 8 * ((int)blockIdx.x * BT * PIECES + (int)threadIdx.x);
    for (int64_t row = blockIdx.y; row < a.M; row += gridDim.y) {
        const T* x = static_cast<const T*>(a.logits) + row * a.stride;
        T* out = static_cast<T*>(a.dlogits) + row * a.out_stride;
        Raw8<T> raw[PIECES];
#pragma unroll
        for (int t = 0; t < PIECES; ++t) {
            const int j = first + 8 * BT * t, n = min(8, a.N - j);
            if (n > 0) raw[t] = load_raw(x + j, n);
        }
        const int token = a.tokens[row];
        const float lse = a.lse[row], entropy = a.entropy ? a.entropy[row] : 0.0f;
        // a row of nothing but -infinity has no gradient, whatever reaches it
        const bool none = lse == -INFINITY;
        float g = token < 0 || none ? 0.0f : a.dlogp[row] * a.scale;
        const float gh = !a.dentropy || none ? 0.0f : a.dentropy[row] * a.scale;
        if (token >= a.N) g = __builtin_nanf("");
#pragma unroll
        for (int t = 0; t < PIECES; ++t) {
            const int j = first + 8 * BT * t, n = min(8, a.N - j);
            if (n <= 0) continue;
            const f32x8_t v = values(raw[t]);
            f32x8_t y;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float log = none ? GONE : larger(__builtin_fmaf(v.v[i], a.scale, -lse), GONE);
                const float p = __builtin_amdgcn_exp2f(log * LOG2E);
                y.v[i] = -p * __builtin_fmaf(gh, log + entropy, g);
                if (j + i == token) y.v[i] += g;
            }
            store_piece(out + j, y, n);
        }
    }
}

template <typename T, int BT>
hipError_t launch_grad(const GradArgs& a, hipStream_t s) {
    constexpr int W = 8 * BT * kGradPieces<T>;
    const int blocks = (a.N + W - 1) / W;  // of a row, at most 1024
    logprobs_bwd_kernel<T, BT><<<dim3((unsigned)blocks, (unsigned)std::min({a.M, 65535, (1 << 23) / blocks})), BT, 0, s>>>(a);
    return hipGetLastError();
}
// rows of one wave's width in waves of their own: 65536 x 1000 bf16 keep half of 256 threads idle
template <typename T>
hipError_t launch_grad(const GradArgs& a, hipStream_t s) {
    return a.N <= 4096 ? launch_grad<T, 64>(a, s) : launch_grad<T, 256>(a, s);
}

}  // namespace

size_t token_logprobs_workspace_size(int M, int N, int top) {
    const Split p = split_of(M, N, top);
    return p.parts == 1 ? 0 : (size_t)M * p.parts * (sizeof(uint64_t) * top + 16);
}

hipError_t launch_token_logprobs(int dtype, const void* logits, int64_t stride, float scale, const int32_t* tokens, float* logp,
                                 float* lse, float* entropy, int top, int32_t* top_ids, float* top_logp, int M, int N, void* ws,
                                 hipStream_t s) {
    const Split p = split_of(M, N, top);
    LogprobArgs a{logits, tokens, logp, lse, entropy, top_ids, top_logp, stride, scale, scale * LOG2E,
                  M, N, top, p.parts, p.width, nullptr, nullptr};
    if (p.parts > 1) {
        a.keys = static_cast<uint64_t*>(ws);
        a.sums = reinterpret_cast<Sums*>(a.keys + (size_t)M * p.parts * top);
    }
    return dtype == JH_F32 ? launch<float>(a, p.threads, s) : launch<uint16_t>(a, p.threads, s);
}

hipError_t launch_token_logprobs_bwd(int dtype, const void* logits, int64_t stride, float scale, const int32_t* tokens,
                                     const float* lse, const float* entropy, const float* dlogp, const float* dentropy,
                                     void* dlogits, int64_t out_stride, int M, int N, hipStream_t s) {
    const GradArgs a{logits, tokens, lse, entropy, dlogp, dentropy, dlogits, stride, out_stride, scale, M, N};
    return dtype == JH_F32 ? launch_grad<float>(a, s) : launch_grad<uint16_t>(a, s);
}

}  // namespace jh

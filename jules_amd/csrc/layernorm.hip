// layernorm.hip - layer norm of a training step: forward with the residual's
// addition and dropout (philox.hpp), and backward with the gradients of the
// norm's weight and bias.  No counterpart in the reference, whose fusedLayerNorm
// (rowops.hip) is fp32 and forward only.
//
//   h = r + drop(x),  y_j = (h_j - mean) rstd gamma_j + beta_j,
//   mean = sum h / N,  rstd = 1 / sqrt(sum (h - mean)^2 / N + eps)
//
//   n_j = (h_j - mean) rstd,  a_j = dy_j gamma_j
//   dr_j = rstd (a_j - sum a / N - n_j sum a n / N) + dh_j,  dx = drop(dr)
//   dgamma_j = sum over rows of dy_j n_j,  dbeta_j = sum over rows of dy_j
//
// A row is read once, held in registers, and written once: bound by HBM.  A call of
// 32768 x 4096 bf16 with a residual and dropout takes 203 us forward (5.3 TB/s; 260 while
// the loads of x and r were waited for one by one), 259 us backward (5.2 TB/s; 454 so).
// Rows over 16384 elements, which no block holds, are read again after each sum, and for
// the columns: 2048 x 32768 bf16 184 us forward (2.9 TB/s of the bytes needed), 235
// backward, fp32 320 and 439.
//
// The mean is summed in 64 bits and so are the squares of the distances from it: no
// row whose distances stay within fp32 overflows or cancels in them, for a convert and
// an addition an element.
//
// Backward: a group of threads goes over many rows with its columns' two sums in
// registers, so dy and h are read once for the row's gradient and the columns'; a
// block leaves one row of partial sums in the workspace, and a second kernel adds
// those in order.  As many blocks as are resident: 512 of 512 threads at 4096 columns
// (256: 301 us, 1024: 263).  No atomics: the results do not depend on timing.
#include <algorithm>

#include "launch.hpp"
#include "philox.hpp"

namespace jh {
namespace {

// Sum over the G threads of a group (blocks of 256 threads hold 256 / G groups
// where G is less), the same order for every row.  The waves' parts alternate
// between two places, so that one barrier is enough: a wave that writes a place
// again has passed the barrier after which it was read.
template <int G, int K, typename T>
__device__ __forceinline__ void reduce_group(T (&a)[K], int& turn) {
#pragma unroll
    for (int o = G < 64 ? G / 2 : 32; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) a[k] += __shfl_xor(a[k], o);
    if constexpr (G > 64) {
        __shared__ T parts[2][G / 64][K];
        T(*part)[K] = parts[turn & 1];
        ++turn;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) part[threadIdx.x >> 6][k] = a[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            a[k] = part[0][k];
#pragma unroll
            for (int w = 1; w < G / 64; ++w) a[k] += part[w][k];
        }
    }
}

struct ForwardArgs {
    const void *x, *r;
    const float *gamma, *beta;  // null: ones, zeros
    void *h_out, *out;
    float *mean, *rstd;  // null: not kept
    Dropout drop;
    int M, N, h_dtype, out_dtype;
    float eps;
};

__device__ __forceinline__ f32x8_t load_vector(const float* v, int j, int n, float none) {
    if (v) return load_piece(v + j, n);
    f32x8_t r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = none;
    return r;
}

// x and r of a piece as they lie in memory, and h of them
template <typename XT, typename RT, bool RES>
struct RawH {
    Raw8<XT> x;
    Raw8<RT> r;
    __device__ __forceinline__ void load(const ForwardArgs& a, int64_t row, int j, int n) {
        x = load_raw(static_cast<const XT*>(a.x) + row * a.N + j, n);
        if constexpr (RES) r = load_raw(static_cast<const RT*>(a.r) + row * a.N + j, n);
    }
    __device__ __forceinline__ f32x8_t h(const ForwardArgs& a, const DropKey& key, int64_t row, int j) const {
        f32x8_t h = values(x);
        if (a.drop.t) h = drop8(h, key, a.drop, (uint32_t)row, (uint32_t)j / 8);
        if constexpr (RES) {
            const f32x8_t v = values(r);
#pragma unroll
            for (int i = 0; i < 8; ++i) h.v[i] += v.v[i];
        }
        return h;
    }
};
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t at, const f32x8_t& v, int n) {
    if (dtype == JH_F32)
        store_piece(static_cast<float*>(p) + at, v, n);
    else
        store_piece(static_cast<uint16_t*>(p) + at, v, n);
}
// h and y of a piece.  The weight and the bias are loaded before the piece's stores: a load
// behind stores waits for them too, the counter of both being one.
__device__ __forceinline__ void write_y(const ForwardArgs& a, int64_t row, int j, int n, const f32x8_t& h, float mean, float rstd) {
    const int64_t at = row * a.N + j;
    const f32x8_t g = load_vector(a.gamma, j, n, 1.0f), b = load_vector(a.beta, j, n, 0.0f);
    f32x8_t y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y.v[i] = __builtin_fmaf((h.v[i] - mean) * rstd, g.v[i], b.v[i]);
    if (a.h_out) store_any(a.h_out, a.h_dtype, at, h, n);
    store_any(a.out, a.out_dtype, at, y, n);
}

__device__ __forceinline__ double sum8(const f32x8_t& h, int n) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += i < n ? (double)h.v[i] : 0.0;
    return s;
}
// of the distances from the mean in fp32, which are exact where that is far from zero
__device__ __forceinline__ double squares8(const f32x8_t& h, float mean, int n) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double d = i < n ? (double)(h.v[i] - mean) : 0.0;
        s = __builtin_fma(d, d, s);
    }
    return s;
}
// squares about `mean`, which is `center` rounded
__device__ __forceinline__ float row_rstd(double squares, double center, float mean, int N, float eps) {
    const double e = center - (double)mean, var = squares / (double)N - e * e;
    return (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + (double)eps));
}

// G threads a row, NP pieces of 8 neighbouring elements a thread
template <typename XT, typename RT, bool RES, int G, int NP>
__global__ __launch_bounds__(G < 256 ? 256 : G) void add_layernorm_kernel(ForwardArgs a) {
    constexpr int ROWS = G < 256 ? 256 / G : 1;
    const int tid = G < 256 ? threadIdx.x % G : threadIdx.x;
    const DropKey key = a.drop.t ? drop_key(a.drop) : DropKey{};
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * ROWS + (G < 256 ? threadIdx.x / G : 0); row < a.M;
         row += (int64_t)gridDim.x * ROWS) {
        RawH<XT, RT, RES> raw[NP];
        f32x8_t h[NP];
        double s[1] = {0.0};
#pragma unroll
        for (int t = 0; t < NP; ++t) {
            const int j = 8 * (tid + G * t), n = min(8, a.N - j);
            if (n > 0) raw[t].load(a, row, j, n);
        }
#pragma unroll
        for (int t = 0; t < NP; ++t) {
            const int j = 8 * (tid + G * t), n = min(8, a.N - j);
            if (n <= 0) continue;
            h[t] = raw[t].h(a, key, row, j);
            s[0] += sum8(h[t], n);
        }
        reduce_group<G>(s, turn);
        const double center = s[0] / (double)a.N;
        const float mean = (float)center;
        s[0] = 0.0;
#pragma unroll
        for (int t = 0; t < NP; ++t) {
            const int n = min(8, a.N - 8 * (tid + G * t));
            if (n > 0) s[0] += squares8(h[t], mean, n);
        }
        reduce_group<G>(s, turn);
        const float rstd = row_rstd(s[0], center, mean, a.N, a.eps);
        if (tid == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
        float center32 = mean;  // the distances are formed again, rather than kept in registers
        asm volatile("" : "+v"(center32));
#pragma unroll
        for (int t = 0; t < NP; ++t) {
            const int j = 8 * (tid + G * t), n = min(8, a.N - j);
            if (n > 0) write_y(a, row, j, n, h[t], center32, rstd);
        }
    }
}

// rows longer than a block holds: read three times.  An element of x and r is last
// read by the thread that then writes it, so the outputs may be the inputs here too.
template <typename XT, typename RT, bool RES>
__global__ __launch_bounds__(1024) void add_layernorm_long_kernel(ForwardArgs a) {
    const DropKey key = a.drop.t ? drop_key(a.drop) : DropKey{};
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const auto pieces = [&](auto&& f) {
            for (int64_t j = 8 * (int64_t)threadIdx.x; j < a.N; j += 8 * 1024) {
                const int n = (int)min((int64_t)8, a.N - j);
                RawH<XT, RT, RES> raw;
                raw.load(a, row, (int)j, n);
                f((int)j, n, raw.h(a, key, row, (int)j));
            }
        };
        double s[1] = {0.0};
        pieces([&](int, int n, const f32x8_t& h) { s[0] += sum8(h, n); });
        reduce_group<1024>(s, turn);
        const double center = s[0] / (double)a.N;
        const float mean = (float)center;
        s[0] = 0.0;
        pieces([&](int, int n, const f32x8_t& h) { s[0] += squares8(h, mean, n); });
        reduce_group<1024>(s, turn);
        const float rstd = row_rstd(s[0], center, mean, a.N, a.eps);
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
        pieces([&](int j, int n, const f32x8_t& h) { write_y(a, row, j, n, h, mean, rstd); });
    }
}

template <typename XT, typename RT, bool RES, int G, int NP>
void launch_forward(const ForwardArgs& a, hipStream_t s) {
    constexpr int ROWS = G < 256 ? 256 / G : 1;
    const int64_t rows = ((int64_t)a.M + ROWS - 1) / ROWS;
    add_layernorm_kernel<XT, RT, RES, G, NP><<<(unsigned)std::min((int64_t)1 << 20, rows), G < 256 ? 256 : G, 0, s>>>(a);
}

// A block a row, none of its threads idle at the widths' upper ends, and as few of them as
// the registers allow, for the most rows in flight (dropout and residual, bf16): 65536 x 1024
// in waves of their own 104 us, 256 threads a row, half of them idle, 167; 32768 x 2048 with
// 256 threads of 8 elements 114, waves of 32 126; x 4096 with 256 of 16 199, 512 of 8 236; 8192
// x 8192 with 256 of 32 110, 512 of 16 126; 4096 x 16384 with 1024 of 16 133, 512 of 32 155.
// One rule for both types; in fp32 16384 x 4096 take 198 us (5.4 TB/s), 4096 x 16384 251 (4.3),
// and 8192 x 8192 217 (4.9) with 256 of 32, whose 182 registers leave two blocks a CU, where 512 of 16
// take 207, 1024 of 8 232 (bf16 118, 125 and 157 in those runs).
template <typename XT, typename RT, bool RES>
hipError_t launch_forward(const ForwardArgs& a, hipStream_t s) {
    if (a.N <= 128)
        launch_forward<XT, RT, RES, 16, 1>(a, s);
    else if (a.N <= 512)
        launch_forward<XT, RT, RES, 64, 1>(a, s);
    else if (a.N <= 1024)
        launch_forward<XT, RT, RES, 64, 2>(a, s);
    else if (a.N <= 2048)
        launch_forward<XT, RT, RES, 256, 1>(a, s);
    else if (a.N <= 4096)
        launch_forward<XT, RT, RES, 256, 2>(a, s);
    else if (a.N <= 8192)
        launch_forward<XT, RT, RES, 256, 4>(a, s);
    else if (a.N <= 16384)
        launch_forward<XT, RT, RES, 1024, 2>(a, s);
    else
        add_layernorm_long_kernel<XT, RT, RES><<<(unsigned)std::min(a.M, 2048), 1024, 0, s>>>(a);
    return hipGetLastError();
}
template <typename XT>
hipError_t launch_forward(const ForwardArgs& a, hipStream_t s) {
    if (!a.r) return launch_forward<XT, XT, false>(a, s);
    return a.h_dtype == JH_F32 ? launch_forward<XT, float, true>(a, s) : launch_forward<XT, uint16_t, true>(a, s);
}

// ---- backward -----------------------------------------------------------------

struct BackwardArgs {
    const void *dy, *h, *dh;  // dh null: none
    const float *mean, *rstd, *gamma;
    void *dx, *dr;   // either may be null: not wanted
    float* partial;  // [blocks][2][N]: sums of dy n and of dy over the block's rows; null: not wanted
    Dropout drop;
    int M, N;
};

// dy, h and dh of a piece as they lie in memory
template <typename XT, typename HT>
struct RawGrad {
    Raw8<XT> dy;
    Raw8<HT> h, dh;
    __device__ __forceinline__ void load(const BackwardArgs& a, int64_t row, int j, int n, bool with_dh) {
        const int64_t at = row * a.N + j;
        dy = load_raw(static_cast<const XT*>(a.dy) + at, n);
        h = load_raw(static_cast<const HT*>(a.h) + at, n);
        if (with_dh && a.dh) dh = load_raw(static_cast<const HT*>(a.dh) + at, n);
    }
    __device__ __forceinline__ f32x8_t norm(float mean, float rstd) const {
        f32x8_t r = values(h);
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = (r.v[i] - mean) * rstd;
        return r;
    }
    // sums of a = dy gamma and of a n; dy is 0 behind the row's end, where the mean alone times
    // rstd may be past fp32: 0 times that is left out
    __device__ __forceinline__ static void add(float (&c)[2], float a, float norm) {
        c[0] += a;
        c[1] = a == 0.0f ? c[1] : __builtin_fmaf(a, norm, c[1]);
    }
    // dr and dx of the piece
    __device__ __forceinline__ void write(const BackwardArgs& a, const DropKey& key, int64_t row, int j, int n, const f32x8_t& norm,
                                          const f32x8_t& gamma, float rstd, float c1, float c2) const {
        const int64_t at = row * a.N + j;
        const f32x8_t y = values(dy);
        f32x8_t g;
#pragma unroll
        for (int i = 0; i < 8; ++i) g.v[i] = rstd * (__builtin_fmaf(y.v[i], gamma.v[i], -c1) - norm.v[i] * c2);
        if (a.dh) {
            const f32x8_t more = values(dh);
#pragma unroll
            for (int i = 0; i < 8; ++i) g.v[i] += more.v[i];
        }
        if (a.dr) store_piece(static_cast<HT*>(a.dr) + at, g, n);
        if (a.dx) {
            if (a.drop.t) g = drop8(g, key, a.drop, (uint32_t)row, (uint32_t)j / 8);
            store_piece(static_cast<XT*>(a.dx) + at, g, n);
        }
    }
};

// SUMS: the columns' sums of the block's rows go to a.partial
template <typename XT, typename HT, int G, int NP, bool SUMS>
__device__ __forceinline__ void backward_rows(const BackwardArgs& a, int block, int blocks) {
    constexpr int ROWS = G < 256 ? 256 / G : 1;
    const int tid = G < 256 ? threadIdx.x % G : threadIdx.x, group = G < 256 ? threadIdx.x / G : 0;
    const DropKey key = a.drop.t ? drop_key(a.drop) : DropKey{};
    int turn = 0;
    constexpr bool KEEP = NP == 1;  // more pieces: no registers to spare for the weight
    f32x8_t gamma[KEEP ? NP : 1], sum_n[NP], sum_y[NP];
    const auto weight = [&](int t) {
        const int j = 8 * (tid + G * t), n = min(8, a.N - j);
        return n > 0 ? load_vector(a.gamma, j, n, 1.0f) : f32x8_t{};
    };
#pragma unroll
    for (int t = 0; t < NP; ++t) {
        if constexpr (KEEP) gamma[t] = weight(t);
        sum_n[t] = sum_y[t] = f32x8_t{};
    }
    struct Row {
        RawGrad<XT, HT> raw[NP];
        float mean, rstd;
    };
    const auto load = [&](int64_t row) {
        Row r;
        r.mean = a.mean[row];
        r.rstd = a.rstd[row];
#pragma unroll
        for (int t = 0; t < NP; ++t) {
            const int j = 8 * (tid + G * t), n = min(8, a.N - j);
            if (n > 0) r.raw[t].load(a, row, j, n, true);
        }
        return r;
    };
    // Of 1024 threads a CU holds one block: its next row's loads are under way while this one's
    // sums meet (1999 x 5001 fp32 28 us, 33 without; 8192 x 8192 bf16 127 and 134).  Smaller blocks
    // have others beside them and lose by it (32768 x 4096: 272 and 256).
    constexpr bool AHEAD = NP == 1 && G == 1024;
    const int64_t step = (int64_t)blocks * ROWS;
    int64_t row = (int64_t)block * ROWS + group;
    Row now, next;
    if (AHEAD && row < a.M) now = load(row);
    for (; row < a.M; row += step) {
        if constexpr (!AHEAD) now = load(row);
        RawGrad<XT, HT>(&raw)[NP] = now.raw;
        const float mean = now.mean, rstd = now.rstd;
        float c[2] = {0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < NP; ++t) {
            if (8 * (tid + G * t) >= a.N) continue;
            const f32x8_t dy = values(raw[t].dy), norm = raw[t].norm(mean, rstd), w = KEEP ? gamma[KEEP ? t : 0] : weight(t);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                RawGrad<XT, HT>::add(c, dy.v[i] * w.v[i], norm.v[i]);
                if constexpr (SUMS) {
                    sum_n[t].v[i] = __builtin_fmaf(dy.v[i], norm.v[i], sum_n[t].v[i]);
                    sum_y[t].v[i] += dy.v[i];
                }
            }
        }
        if (AHEAD && row + step < a.M) next = load(row + step);
        reduce_group<G>(c, turn);
        const float c1 = c[0] / (float)a.N, c2 = c[1] / (float)a.N;
        f32x8_t w = KEEP ? gamma[0] : weight(0);  // before the stores of the piece before, see write_y
#pragma unroll
        for (int t = 0; t < NP; ++t) {
            const int j = 8 * (tid + G * t), n = min(8, a.N - j);
            if (n <= 0) continue;
            const f32x8_t g = w;
            if (t + 1 < NP) w = KEEP ? gamma[KEEP ? t + 1 : 0] : weight(t + 1);
            raw[t].write(a, key, row, j, n, raw[t].norm(mean, rstd), g, rstd, c1, c2);
        }
        if constexpr (AHEAD) now = next;
    }
    if (!SUMS || !a.partial) return;
    float* out = a.partial + (int64_t)block * 2 * a.N;
    if constexpr (ROWS > 1) {
        // the block's groups, in order
        constexpr int W = 8 * G * NP;
        __shared__ float sums[ROWS][2][W];
#pragma unroll
        for (int t = 0; t < NP; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sums[group][0][8 * (tid + G * t) + i] = sum_n[t].v[i];
                sums[group][1][8 * (tid + G * t) + i] = sum_y[t].v[i];
            }
        __syncthreads();
        for (int k = threadIdx.x; k < 2 * W; k += 256) {
            const int which = k / W, j = k % W;
            if (j >= a.N) continue;
            float s = 0.0f;
            for (int g = 0; g < ROWS; ++g) s += sums[g][which][j];
            out[which * (int64_t)a.N + j] = s;
        }
    } else {
#pragma unroll
        for (int t = 0; t < NP; ++t) {
            const int j = 8 * (tid + G * t), n = min(8, a.N - j);
            if (n <= 0) continue;
            store_piece(out + j, sum_n[t], n);
            store_piece(out + a.N + j, sum_y[t], n);
        }
    }
}

template <typename XT, typename HT, int G, int NP>
__global__ __launch_bounds__(G < 256 ? 256 : G) void add_layernorm_bwd_kernel(BackwardArgs a) {
    backward_rows<XT, HT, G, NP, true>(a, blockIdx.x, gridDim.x);
}

// Few rows: blocks from a.first on; the first row_blocks take a row each (256 / G rows),
// the others all rows of 64 columns, whose sums they leave in dgamma and dbeta: dy and h are read twice,
// out of the caches, and there is one launch and no workspace.
template <typename XT, typename HT, int G, int NP>
__global__ __launch_bounds__(G < 256 ? 256 : G) void add_layernorm_bwd_few_kernel(BackwardArgs a, int first, int row_blocks,
                                                                                 float* dgamma, float* dbeta) {
    constexpr int WAVES = G < 256 ? 4 : G / 64;
    const int block = first + blockIdx.x;
    if (block < row_blocks) {
        backward_rows<XT, HT, G, NP, false>(a, block, row_blocks);
        return;
    }
    // 8 pieces a wave, 8 rows: lane = 8 row + piece
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int j0 = 64 * (block - row_blocks), j = j0 + 8 * (lane & 7), n = min(8, a.N - j);
    f32x8_t sum_n{}, sum_y{};
    if (n > 0) {
#pragma unroll 2
        for (int row = 8 * wave + (lane >> 3); row < a.M; row += 8 * WAVES) {
            RawGrad<XT, HT> raw;
            raw.load(a, row, j, n, false);
            const f32x8_t dy = values(raw.dy), norm = raw.norm(a.mean[row], a.rstd[row]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sum_n.v[i] = __builtin_fmaf(dy.v[i], norm.v[i], sum_n.v[i]);
                sum_y.v[i] += dy.v[i];
            }
        }
    }
    __shared__ float sums[WAVES][2][64];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int o = 8; o < 64; o <<= 1) {
            sum_n.v[i] += __shfl_xor(sum_n.v[i], o);
            sum_y.v[i] += __shfl_xor(sum_y.v[i], o);
        }
        if (lane < 8) {
            sums[wave][0][8 * lane + i] = sum_n.v[i];
            sums[wave][1][8 * lane + i] = sum_y.v[i];
        }
    }
    __syncthreads();
    if (threadIdx.x >= 128) return;
    float* out = threadIdx.x < 64 ? dgamma : dbeta;
    if (!out || j0 + lane >= a.N) return;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s += sums[w][threadIdx.x >> 6][lane];
    out[j0 + lane] = s;
}

// rows longer than a block holds: dy, h are read twice, and once more for the columns
template <typename XT, typename HT>
__global__ __launch_bounds__(1024) void add_layernorm_bwd_long_kernel(BackwardArgs a) {
    const DropKey key = a.drop.t ? drop_key(a.drop) : DropKey{};
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const float mean = a.mean[row], rstd = a.rstd[row];
        const auto pieces = [&](bool with_dh, auto&& f) {
            for (int64_t j = 8 * (int64_t)threadIdx.x; j < a.N; j += 8 * 1024) {
                const int n = (int)min((int64_t)8, a.N - j);
                RawGrad<XT, HT> raw;
                raw.load(a, row, (int)j, n, with_dh);
                f((int)j, n, raw, raw.norm(mean, rstd), load_vector(a.gamma, (int)j, n, 1.0f));
            }
        };
        float c[2] = {0.0f, 0.0f};
        pieces(false, [&](int, int, const RawGrad<XT, HT>& raw, const f32x8_t& norm, const f32x8_t& gamma) {
            const f32x8_t dy = values(raw.dy);
#pragma unroll
            for (int i = 0; i < 8; ++i) RawGrad<XT, HT>::add(c, dy.v[i] * gamma.v[i], norm.v[i]);
        });
        reduce_group<1024>(c, turn);
        const float c1 = c[0] / (float)a.N, c2 = c[1] / (float)a.N;
        pieces(true, [&](int j, int n, const RawGrad<XT, HT>& raw, const f32x8_t& norm, const f32x8_t& gamma) {
            raw.write(a, key, row, j, n, norm, gamma, rstd, c1, c2);
        });
    }
}
// the columns' sums of rows blockIdx.y, blockIdx.y + gridDim.y, .. of long rows
template <typename XT, typename HT>
__global__ __launch_bounds__(256) void layernorm_columns_kernel(BackwardArgs a) {
    for (int64_t j = 8 * ((int64_t)blockIdx.x * 256 + threadIdx.x); j < a.N; j += 8 * 256 * (int64_t)gridDim.x) {
        const int n = (int)min((int64_t)8, a.N - j);
        f32x8_t sum_n{}, sum_y{};
        for (int64_t row = blockIdx.y; row < a.M; row += gridDim.y) {
            RawGrad<XT, HT> raw;
            raw.load(a, row, (int)j, n, false);
            const f32x8_t dy = values(raw.dy), norm = raw.norm(a.mean[row], a.rstd[row]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sum_n.v[i] = __builtin_fmaf(dy.v[i], norm.v[i], sum_n.v[i]);
                sum_y.v[i] += dy.v[i];
            }
        }
        float* out = a.partial + (int64_t)blockIdx.y * 2 * a.N + j;
        store_piece(out, sum_n, n);
        store_piece(out + a.N, sum_y, n);
    }
}

// dgamma, dbeta = the partial rows' sums: a wave adds every 16th row of 64 columns,
// 8 loads under way together
__global__ __launch_bounds__(1024) void layernorm_fold_kernel(const float* partial, int parts, float* dgamma, float* dbeta,
                                                              int N) {
    __shared__ float sums[16][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t width = 2 * (int64_t)N;
    for (int64_t j0 = 64 * (int64_t)blockIdx.x; j0 < width; j0 += 64 * (int64_t)gridDim.x) {
        const int64_t j = j0 + lane;
        float s = 0.0f;
        if (j < width) {
#pragma unroll 8
            for (int p = wave; p < parts; p += 16) s += partial[p * width + j];
        }
        sums[wave][lane] = s;
        __syncthreads();
        if (wave == 0 && j < width) {
#pragma unroll
            for (int w = 1; w < 16; ++w) s += sums[w][lane];
            float* out = j < N ? dgamma : dbeta;
            if (out) out[j < N ? j : j - N] = s;
        }
        __syncthreads();
    }
}

// How many blocks, and with them partial rows, the backward pass has: what is resident.
// 65536 x 1024 bf16 in waves of their own: 1024 blocks 132 us, 512 144; with 256 threads a row,
// as at 2048: 144 and 238; 32768 x 4096: 512 blocks 255, 256 301; 8192 x 8192: 256 127, 192 139.
int backward_blocks(int M, int N) {
    if (N <= 1024) {
        const int rows = N <= 128 ? 16 : 4;
        return std::min(M / rows + (M % rows != 0), 1024);
    }
    return std::min(M, N <= 2048 ? 1024 : N <= 4096 ? 512 : N <= 16384 ? 256 : 64);
}

template <typename XT, typename HT, int G, int NP>
void launch_backward(const BackwardArgs& a, int blocks, hipStream_t s) {
    add_layernorm_bwd_kernel<XT, HT, G, NP><<<(unsigned)blocks, G < 256 ? 256 : G, 0, s>>>(a);
}
// The columns' sums take 16 registers a piece, so the threads hold fewer than forward:
// 32768 x 4096 bf16 with 512 of 8 elements 256 us, 256 of 16 275 at best; 8192 x 8192 with 1024
// of 8 127, 512 of 16 136; 4096 x 16384 with 1024 of 16 151, 512 of 32 178.  fp32: 16384 x 4096 251 us
// (5.3 TB/s), 8192 x 8192 255 (5.3), 4096 x 16384 294 (4.6).
template <typename XT, typename HT>
void launch_backward(const BackwardArgs& a, int blocks, hipStream_t s) {
    if (a.N <= 128) {
        launch_backward<XT, HT, 16, 1>(a, blocks, s);
    } else if (a.N <= 512) {
        launch_backward<XT, HT, 64, 1>(a, blocks, s);
    } else if (a.N <= 1024) {
        launch_backward<XT, HT, 64, 2>(a, blocks, s);
    } else if (a.N <= 2048) {
        launch_backward<XT, HT, 256, 1>(a, blocks, s);
    } else if (a.N <= 4096) {
        launch_backward<XT, HT, 512, 1>(a, blocks, s);
    } else if (a.N <= 8192) {
        launch_backward<XT, HT, 1024, 1>(a, blocks, s);
    } else if (a.N <= 16384) {
        // 1024 threads have the registers for 2 pieces in bf16 alone
        if constexpr (sizeof(XT) + sizeof(HT) == 4)
            launch_backward<XT, HT, 1024, 2>(a, blocks, s);
        else
            launch_backward<XT, HT, 512, 4>(a, blocks, s);
    } else {
        // the columns first: dx and dr may be dy and dh
        if (a.partial)
            layernorm_columns_kernel<XT, HT><<<dim3((unsigned)std::min(a.N / 2048 + (a.N % 2048 != 0), 65535), blocks), 256, 0, s>>>(a);
        if (a.dx || a.dr) add_layernorm_bwd_long_kernel<XT, HT><<<(unsigned)std::min(a.M, 2048), 1024, 0, s>>>(a);
    }
}

// Where the columns' sums read dy and h again rather than leave partial sums: the second
// launch and the workspace cost the caller 4.5 us (64 x 1024: 14.5 us against 18.9), reading
// again costs more than that from some thousand rows on (2000 x 1024: 25 against 18.7).  One
// rule for both types: 512 x 8192 bf16 18.4 us against 20.7, fp32 28.0 against 25.5, where it loses;
// 400 x 16384 24.7 against 29.4, fp32 37.4 against 45.3.
bool backward_few(int M, int N) { return N <= 16384 && (M <= 512 || (M <= 2048 && M * N <= 1 << 20)); }

template <typename XT, typename HT, int G, int NP>
void launch_few(const BackwardArgs& a, float* dgamma, float* dbeta, hipStream_t s) {
    constexpr int ROWS = G < 256 ? 256 / G : 1, BT = G < 256 ? 256 : G;
    const int rows = a.dx || a.dr ? (a.M + ROWS - 1) / ROWS : 0;
    const int columns = dgamma || dbeta ? (a.N + 63) / 64 : 0;
    if (rows && columns && a.dx == a.dy) {  // the columns have to have read dy
        add_layernorm_bwd_few_kernel<XT, HT, G, NP><<<columns, BT, 0, s>>>(a, rows, rows, dgamma, dbeta);
        add_layernorm_bwd_few_kernel<XT, HT, G, NP><<<rows, BT, 0, s>>>(a, 0, rows, dgamma, dbeta);
    } else if (rows + columns) {
        add_layernorm_bwd_few_kernel<XT, HT, G, NP><<<rows + columns, BT, 0, s>>>(a, 0, rows, dgamma, dbeta);
    }
}
template <typename XT, typename HT>
void launch_few(const BackwardArgs& a, float* dgamma, float* dbeta, hipStream_t s) {
    if (a.N <= 512)
        launch_few<XT, HT, 64, 1>(a, dgamma, dbeta, s);
    else if (a.N <= 2048)
        launch_few<XT, HT, 256, 1>(a, dgamma, dbeta, s);
    else if (a.N <= 8192)
        launch_few<XT, HT, 1024, 1>(a, dgamma, dbeta, s);
    else
        launch_few<XT, HT, 1024, 2>(a, dgamma, dbeta, s);
}

// f<XT, HT>() by the types
template <typename F>
void by_types(int x_dtype, int h_dtype, F&& f) {
    if (x_dtype == JH_F32)
        h_dtype == JH_F32 ? f(0.0f, 0.0f) : f(0.0f, (uint16_t)0);
    else
        h_dtype == JH_F32 ? f((uint16_t)0, 0.0f) : f((uint16_t)0, (uint16_t)0);
}

}  // namespace

hipError_t launch_add_layernorm(int x_dtype, int h_dtype, int out_dtype, const Dropout& drop, const void* x, const void* r,
                                const float* gamma, const float* beta, void* h_out, void* out, float* mean, float* rstd, int M,
                                int N, float eps, hipStream_t s) {
    const ForwardArgs a{x, r, gamma, beta, h_out, out, mean, rstd, drop, M, N, h_dtype, out_dtype, eps};
    return x_dtype == JH_F32 ? launch_forward<float>(a, s) : launch_forward<uint16_t>(a, s);
}

size_t add_layernorm_bwd_workspace_size(int M, int N) {
    return backward_few(M, N) ? 0 : (size_t)backward_blocks(M, N) * 2 * (size_t)N * sizeof(float);
}

hipError_t launch_add_layernorm_bwd(int x_dtype, int h_dtype, const Dropout& drop, const void* dy, const void* h, const void* dh,
                                    const float* mean, const float* rstd, const float* gamma, void* dx, void* dr, float* dgamma,
                                    float* dbeta, int M, int N, void* ws, hipStream_t s) {
    const bool columns = dgamma || dbeta;
    const BackwardArgs a{dy, h, dh, mean, rstd, gamma, dx, dr, columns ? static_cast<float*>(ws) : nullptr, drop, M, N};
    if (M > 0 && backward_few(M, N)) {
        by_types(x_dtype, h_dtype, [&](auto x, auto g) { launch_few<decltype(x), decltype(g)>(a, dgamma, dbeta, s); });
        return hipGetLastError();
    }
    const int blocks = backward_blocks(M, N);
    if (M > 0)  // no rows: the columns' sums are 0
        by_types(x_dtype, h_dtype, [&](auto x, auto g) { launch_backward<decltype(x), decltype(g)>(a, blocks, s); });
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !columns) return e;
    layernorm_fold_kernel<<<(unsigned)std::min((2 * (int64_t)N + 63) / 64, (int64_t)2048), 1024, 0, s>>>(a.partial, blocks, dgamma,
                                                                                                  dbeta, N);
    return hipGetLastError();
}

}  // namespace jh

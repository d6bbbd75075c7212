// dropout.hip - dropout whose mask is made from a counter each time and never
// stored (philox.hpp), with a residual's addition or without; its backward pass
// is the same call on the gradient.  No counterpart in the reference.
//
//   out = [residual +] (kept ? x * scale : 0)
//
// A thread takes a piece of 8 neighbouring elements of a row, one counter each.  Bound by
// HBM, in bf16 alone (4 bytes an element) nearly as much by the rounds' products: 32768 x
// 4096 bf16 onto an fp32 residual 225 us, 6.0 TB/s; bf16 alone 92 us, 5.8 TB/s.  A block for
// every 256 pieces: 2048 blocks that go on to others take 257 us and 100.
#include <algorithm>

#include "launch.hpp"
#include "philox.hpp"

namespace jh {
namespace {

template <typename XT, typename OT, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(Dropout d, const XT* x, const OT* r, OT* out, int M, int N) {
    const int pieces = N / 8 + (N % 8 != 0);
    const DropKey key = d.t ? drop_key(d) : DropKey{};  // t = 0: rng may be null, and every element is kept
    // a thread's pieces lie `stride` apart, in rows and pieces: one division for all of them
    const uint32_t stride = gridDim.x * 256, first = blockIdx.x * 256 + threadIdx.x;
    const int rows_on = (int)(stride / (uint32_t)pieces), pieces_on = (int)(stride % (uint32_t)pieces);
    int64_t row = first / (uint32_t)pieces;
    int piece = (int)(first % (uint32_t)pieces);
    while (row < M) {
        const int n = min(8, N - 8 * piece);
        const int64_t at = row * N + 8 * (int64_t)piece;
        const Raw8<XT> raw = load_raw(x + at, n);
        Raw8<OT> old;
        if constexpr (RES) old = load_raw(r + at, n);
        f32x8_t y = values(raw);
        if (d.t) y = drop8(y, key, d, (uint32_t)row, (uint32_t)piece);
        if constexpr (RES) {
            const f32x8_t v = values(old);
#pragma unroll
            for (int i = 0; i < 8; ++i) y.v[i] += v.v[i];
        }
        store_piece(out + at, y, n);
        row += rows_on;
        piece += pieces_on;
        if (piece >= pieces) {
            piece -= pieces;
            ++row;
        }
    }
}

template <typename XT, typename OT>
hipError_t launch(const Dropout& d, const void* x, const void* r, void* out, int M, int N, hipStream_t s) {
    const int64_t blocks = ((int64_t)M * (N / 8 + (N % 8 != 0)) + 255) / 256;
    const unsigned grid = (unsigned)std::min(blocks, (int64_t)1 << 20);
    if (r)
        dropout_kernel<XT, OT, true><<<grid, 256, 0, s>>>(d, static_cast<const XT*>(x), static_cast<const OT*>(r),
                                                          static_cast<OT*>(out), M, N);
    else
        dropout_kernel<XT, OT, false><<<grid, 256, 0, s>>>(d, static_cast<const XT*>(x), nullptr, static_cast<OT*>(out), M, N);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_dropout(int x_dtype, int out_dtype, const Dropout& d, const void* x, const void* residual, void* out, int M,
                          int N, hipStream_t s) {
    if (x_dtype == JH_F32)
        return out_dtype == JH_F32 ? launch<float, float>(d, x, residual, out, M, N, s)
                                   : launch<float, uint16_t>(d, x, residual, out, M, N, s);
    return out_dtype == JH_F32 ? launch<uint16_t, float>(d, x, residual, out, M, N, s)
                               : launch<uint16_t, uint16_t>(d, x, residual, out, M, N, s);
}

}  // namespace jh

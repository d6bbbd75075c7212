// philox.hpp - dropout's random bits, from a counter and a key, so that no mask
// is stored: the backward pass makes the same bits again.
//
// Philox4x32 with 10 rounds (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011): four 32-bit words from a counter of four
// and a key of two.  Element (i, j) of [M, N] takes half word j % 8 (the low half
// of each word first) of the words at the counter (j / 8, i, low and high word of
// rng[1] + offset), key (low and high word of rng[0]): it depends on nothing but
// the element's place and the three numbers, so kernels of any type and launch
// shape agree.  It is dropped where the half word is below t = round(65536 p) and
// multiplied by 65536 / (65536 - t) elsewhere, whose expectation is exact.
//
// 16 bits an element, not 32: the rounds' wide products run at a quarter of the
// rate of the other instructions, and a piece of 8 elements takes one counter
// instead of two.
#pragma once

#include "launch.hpp"
#include "pieces.hpp"

namespace jh {

struct DropKey {
    uint32_t k0, k1, o0, o1;
};
__device__ __forceinline__ DropKey drop_key(const Dropout& d) {
    const uint64_t seed = (uint64_t)d.rng[0], at = (uint64_t)d.rng[1] + d.offset;
    return DropKey{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)at, (uint32_t)(at >> 32)};
}

__device__ __forceinline__ u32x4_t philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u32x4_t{c0, c1, c2, c3};
}

// x of elements 8 piece .. 8 piece + 7 of a row: dropped ones 0 whatever they
// hold, the others scaled
__device__ __forceinline__ f32x8_t drop8(const f32x8_t& x, const DropKey& k, const Dropout& d, uint32_t row, uint32_t piece) {
    const u32x4_t w = philox(piece, row, k.o0, k.o1, k.k0, k.k1);
    f32x8_t r;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t bits = i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu;
        r.v[i] = bits >= d.t ? x.v[i] * d.scale : 0.0f;
    }
    return r;
}

}  // namespace jh

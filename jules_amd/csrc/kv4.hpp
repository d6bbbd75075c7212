// kv4.hpp - the key/value cache held in 4 bits: its layout, as the kernels that
// write (kv4_cache.hip) and read it (kv4_cache.hip, kv4_attn.hip) see it.
//
// A row is the D values of one token and key/value head: a scale s and a
// minimum m, both bf16 (one 32-bit word, s low), and D codes of 4 bits; code c
// stands for m + s c.  A page holds `page` tokens of every head:
//   k  [pages][heads][page][D/2 bytes]: row-major.  32-bit word w of a row has
//      elements 8w .. 8w+7: bits 4j .. 4j+3 hold 2j, bits 16+4j .. 16+4j+3 hold
//      2j+1, so that (word >> 4j) & 0x000f000f is a pair in order;
//   v  [pages][heads][page/4][D/4][8 bytes]: 4 tokens by 4 elements.  Token t of
//      the four has bits 16t .. 16t+15, element e of the four bits 4e .. 4e+3
//      of those, so that the pairs of the same mask are two tokens' values of
//      one element;
//   k_meta, v_meta  [pages][heads][page] words.
// The matrix product that reads the keys contracts over elements and the one
// that reads the values over tokens: with these orders both take their
// operands straight from 16-byte loads, a shift, an and and an or for two codes.
#pragma once

#include "common.hpp"
#include "launch.hpp"

namespace jh {

// One number of a call's table, lens or cu_q, the same address in all lanes, by a
// scalar load: it takes no place among the vector loads in flight.
__device__ __forceinline__ int kv4_scalar(const int32_t* p) {
    return *reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p));
}

// row index of token `off` of a page and head
__device__ __forceinline__ int64_t kv4_row(const KV4View& c, int page, int head, int off) {
    return ((int64_t)page * c.heads + head) * c.page_size + off;
}

// first packed row of sequence `seq`, and how many are its; never past the
// arrays, whatever cu_q holds
__device__ __forceinline__ int kv4_first(const KV4Batch& b, int seq) {
    return b.cu_q ? min(max(kv4_scalar(b.cu_q + seq), 0), b.tokens) : seq * b.max_q;
}
__device__ __forceinline__ int kv4_count(const KV4Batch& b, int seq) {
    if (!b.cu_q) return b.max_q;
    return max(0, min(max(kv4_scalar(b.cu_q + seq + 1), 0), b.tokens) - kv4_first(b, seq));
}

// the page that holds position `at` >= 0 of a sequence, or -1 where its row of
// the table has none of the pool's
__device__ __forceinline__ int kv4_page(const KV4View& c, const KV4Batch& b, int seq, int at) {
    const int i = at >> c.page_shift;
    if (i >= b.max_pages) return -1;
    const int p = b.table[(int64_t)seq * b.max_pages + i];
    return p >= 0 && p < c.num_pages ? p : -1;
}

}  // namespace jh

// The paged cache of keys and values held in 4 bits: where a value's code and scale lie.
//
// A row (one token of one key/value head) is head_dim values in blocks of 32: an fp16 scale d and 32 codes n of 4 bits that
// stand for d * (n - 8).  Rows lie [page][head][token in the page]; codes and scales have planes of their own, so that a
// page's rows of one head are one run of bytes and every load is aligned.  Inside a row
//   values' codes lie in order, two a byte, the first in the low half: sixteen of them are the 8 bytes that a transposing LDS
//     read turns into one value of sixteen tokens;
//   keys' codes lie in words of eight, word w of a row of B blocks holding values 8 * (w / B) .. + 7 of block w % B: the
//     B words that one lane of a matrix instruction multiplies, a block each, are B words in a row.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qproj_device.h"

namespace qproj {

struct KvView {
    uint8_t *k_codes;     // [pages][heads][tokens][dim / 2]
    uint16_t *k_scales;   // [pages][heads][tokens][dim / 32] fp16
    uint8_t *v_codes;
    uint16_t *v_scales;
    int64_t n_pages;
    int32_t page_shift;   // log2 of the tokens of a page
    int32_t n_head;
    int32_t dim;
};

// the row of a token of a head
__device__ __forceinline__ int64_t kv_row(const KvView &kv, int64_t page, int head, int at) {
    return ((page * kv.n_head + head) << kv.page_shift) + at;
}

// the word of a row that holds the codes of 8 values of a block (eighth 0..3)
__device__ __forceinline__ int key_word(int blocks, int block, int eighth) { return eighth * blocks + block; }
__device__ __forceinline__ int value_word(int block, int eighth) { return block * 4 + eighth; }

// bits of the error word that kernels raise (the context's second flag)
constexpr int kKvBadSlot = 1, kKvBadPage = 2, kKvBadRows = 4;

}  // namespace qproj

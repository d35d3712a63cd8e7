// The layout of a KV cache held in 4 bits.
//
// data [blocks, kv_heads, page bytes]: a page of one kv head holds, for its
// `page` tokens, the K codes (D / 2 bytes a token), the V codes, the K words and
// the V words (a 16-bit word for each group of 32 dims), the two word blocks
// filled up to 16 bytes. Of a group's word the low four bits are its zero point
// z, the others a bf16 scale s with four significant bits: x = (c - z) s. A code
// less its zero point has four bits and a sign, so x has at most eight
// significant bits: it is a bf16 value, exactly.
//
// A token's codes are words of 8 dims. V: dims 8 w .. 8 w + 7 in word w, 4 bits a
// dim in order. K: dims 32 a + 8 b .. in word b D / 32 + a, dim 2 i in bits 4 i ..,
// dim 2 i + 1 in bits 16 + 4 i ..: a lane that holds a token's dims 8 b .. of every
// 32 (the matrix cores' operand) reads them at once, and `word >> 4 i & 0x000F000F`
// is a pair of neighbours.
#pragma once

#include <stdint.h>

#if defined(__HIP__) || defined(__HIPCC__)
#define QSA_KV4_HD __host__ __device__
#else
#define QSA_KV4_HD
#endif

namespace qsa {

struct Kv4Page {
  int page, dim;

  QSA_KV4_HD int row() const { return dim / 2; }   // bytes of a token's codes
  QSA_KV4_HD int words() const { return dim / 16; }  // bytes of a token's words
  QSA_KV4_HD int64_t v_codes() const { return (int64_t)page * row(); }
  QSA_KV4_HD int64_t k_words() const { return 2 * v_codes(); }
  QSA_KV4_HD int64_t v_words() const {
    return k_words() + ((int64_t)page * words() + 15) / 16 * 16;
  }
  QSA_KV4_HD int64_t bytes() const {
    return v_words() + ((int64_t)page * words() + 15) / 16 * 16;
  }
};

// The word of a group that holds an infinity, a NaN or a value from 2^126 on (whose
// scale, or the values it stands for, could pass bf16's): its values read as NaN.
constexpr uint32_t kKv4NaN = 0x7FC0;

}  // namespace qsa

// What attention kernels share that stage a paged cache's K and V through LDS
// (tree_attn.hip, paged_attn.hip): the places of rows in a stage, loads into it, the
// transposing read, the output gate, and the host's measure of a cache.
#pragma once

#include "qsa_common.h"

namespace qsa {

constexpr float kNegInf = -__builtin_huge_valf();
constexpr uint32_t kNoToken = 0xFFFFFFFFu;
constexpr float kSlack = 8.0f;  // log2: how far scores may pass the exponents' base
// s_waitcnt for the vector-memory counter alone (gfx9 encoding), at 0.
constexpr int kLoadsDone = (7 << 4) | (15 << 8);

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// sigmoid(g), 0 and 1 at the infinities. The hardware's exponential and reciprocal:
// off by 2^-20 for gates to 10, by 2^-17 for the least: far inside the output's 2^-8.
__device__ __forceinline__ float gate_factor(uint16_t g) {
  return __builtin_amdgcn_rcpf(1.0f + __expf(-bf16_lo(g)));
}

// Byte offset of 16-byte unit `unit` of token `tok`'s row in a K stage: units are
// permuted by the token so that the tokens' same unit (what one pass of the A
// operand's read takes of 8 or 16) lie in different banks.
template <int D>
__device__ __forceinline__ int k_swizzle(int tok) {
  return D == 128 ? tok & 15 : (tok >> 1) & 7;
}
template <int D>
__device__ __forceinline__ int k_at(int tok, int unit) {
  return (tok * (D / 8) + (unit ^ k_swizzle<D>(tok))) * 16;
}
// The same for V, permuted in 32-byte units (what the transposing read takes).
template <int D>
__device__ __forceinline__ int v_swizzle(int tok) {
  return D == 128 ? (tok & 7) << 1 : ((tok >> 1) & 3) << 1;
}
template <int D>
__device__ __forceinline__ int v_at(int tok, int unit) {
  return (tok * (D / 8) + (unit ^ v_swizzle<D>(tok))) * 16;
}

// Lane i of 16 passes the address of 4 dims of token i / 4 and gets dim i of the four.
__device__ __forceinline__ s16x4 read_transposed(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}
__device__ __forceinline__ void load_to_lds(const char* src, char* dst) {  // 16 bytes a lane
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

// max over the two lanes l and l + 32, and over the four 16 apart.
__device__ __forceinline__ float max_over_halves(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float max_over_quarters(float v) {
  v = max_over_halves(v);
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// Elements from a cache's first token row to its last, -1 if a stride is negative or
// the span past 2^62.
inline int64_t cache_span(int64_t blocks, int64_t block_stride, int64_t page, int64_t token_stride) {
  if (block_stride < 0 || token_stride < 0 || block_stride >= INT64_MAX / 4 / (blocks + 1) ||
      token_stride >= INT64_MAX / 4 / page)
    return -1;
  return blocks > 0 ? (blocks - 1) * block_stride + (page - 1) * token_stride : 0;
}

}  // namespace qsa

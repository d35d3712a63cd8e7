// Norm and rotation of query and key heads, K/V into the paged cache, gfx950.
//
// For each (token, head) row of D dims, all in fp32 and rounded once:
//
//   y = x / sqrt(mean(x^2) + eps) * w
//   y_i' = y_i cos - y_{i + R/2} sin,  y_{i + R/2}' = y_{i + R/2} cos + y_i sin   (i < R/2)
//
// with the angle's cosine and sine from the position's table row. V rows are
// copied. K (after that) and V go to their tokens' cache slots as bf16 or as 4-bit
// codes (kv4.h) of the bf16 values, step by step the same as
//
//   s = (max(x, 0) - min(x, 0)) / 15 raised to four significant bits
//   z = round(-min(x, 0) / s), c = round(x / s) + z kept within 0 .. 15
//
// so that the range is covered whatever the rounding of s.
//
// D / 8 lanes share a row, 8 dims a lane: one 16-byte load and store, sums and
// rotation partners by lane exchange. Bound by memory for many tokens (8304 of 20
// heads of 128, 87 MB, in 16.5 us: 5.3 TB/s; 8191 of 48 heads of 64 into 4 bits, 108
// MB, in 22.5: 4.8), by the launch and one chain of loads for few (1 token 2.8 us, 112
// into 4 bits 3.9, of the 7 that the host needs for a call).
#include "qsa_common.h"
#include "../../include/qsa_hip.h"
#include "kv4.h"

#include <algorithm>
#include <climits>

namespace qsa {
namespace {

constexpr int kThreads = 256;
// Rows up to which each has its own group of lanes; past that a group takes four query
// heads or two of K or V of a token, whose position's row is loaded once: 8304 tokens of
// 20 heads 16.5 us for 27, but one token 3.7 for 2.8 and 112 into 4 bits 5.0 for 3.9.
constexpr int kSmall = 4096;

struct Rows {  // [tokens, heads, D] bf16, strides in elements
  uint16_t* p;
  int64_t token, head;
};

struct HeadRopeArgs {
  Rows q, k, v, q_out, k_out, v_out;
  int q_heads, kv_heads;  // 0 query heads without queries
  int kv_parts;           // keys, and values if there are any
  FastDiv q_div, kv_div;  // groups of lanes of a token, of one part
  int q_items, kv_items, q_blocks;  // groups of all tokens, and the queries' workgroups
  const uint16_t* q_weight;
  const uint16_t* k_weight;
  float eps;
  const int64_t* positions;
  const void* cos_sin;
  int cos_sin_fp32;
  int max_positions, rotary;
  const int64_t* slots;
  char* k_cache;  // the 4-bit cache's data, strides in bytes
  char* v_cache;
  int64_t kb, kt, kh, vb, vt, vh;  // bytes
  int64_t num_slots;
  FastDiv page_div;
};

// x / d correctly rounded, for the rounded reciprocal r of d: the quotient's residual is
// exact (Markstein's division step). No operand here is near the type's ends.
__device__ __forceinline__ float divide(float x, float d, float r) {
  const float q = x * r;
  return __builtin_fmaf(__builtin_fmaf(-q, d, x), r, q);
}

// Rows of 8 dims a lane: 4 lanes share a group of 32. The lane's codes go to `codes`,
// and (where `f` is wanted) the values that they stand for to f; returns the group's word.
__device__ __forceinline__ uint32_t quantize4(const u32x4& x, bool wanted, float (&f)[8],
                                              uint32_t (&codes)[8]) {
#pragma clang fp contract(off)
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  unpack8(x, f);
  float low = 0.0f, high = 0.0f;
  u16x2 top = {0, 0};  // largest magnitudes' bits: infinities and NaN are above all others
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    low = fminf(low, fminf(f[2 * i], f[2 * i + 1]));
    high = fmaxf(high, fmaxf(f[2 * i], f[2 * i + 1]));
    top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, x[i] & 0x7FFF7FFFu));
  }
  int bad = top[0] >= 0x7E80 || top[1] >= 0x7E80;
#pragma unroll
  for (int m = 1; m < 4; m *= 2) {
    low = fminf(low, __shfl_xor(low, m, 64));
    high = fmaxf(high, __shfl_xor(high, m, 64));
    bad |= __shfl_xor(bad, m, 64);
  }
  const float step = fmaxf(divide(high - low, 15.0f, 1.0f / 15.0f), 0x1p-100f);
  const uint32_t sbits = (__builtin_bit_cast(uint32_t, step) + 0xFFFFFu) & ~0xFFFFFu;
  const float s = __builtin_bit_cast(float, sbits);
  const float r = __fdiv_rn(1.0f, s);
  const float z = fminf(rintf(divide(-low, s, r)), 15.0f);
  float c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = fminf(fmaxf(rintf(divide(f[i], s, r)) + z, 0.0f), 15.0f);
  if (wanted) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = bad ? __builtin_nanf("") : (c[i] - z) * s;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) codes[i] = bad ? 1u : (uint32_t)c[i];
  return bad ? kKv4NaN : sbits >> 16 | (uint32_t)z;
}

// ROWS heads of one part (0: queries, 1: keys, 2: values) of one token, from head
// `first` on. Everything is loaded before anything is used: one chain of two loads (the
// position, then its row of the table) is all that a call waits for.
template <int D, int BITS, int ROWS>
__device__ __forceinline__ void take_heads(const HeadRopeArgs& a, int part, int token, int first,
                                           int j) {
  constexpr int kLanes = D / 8;
  const Rows& src = part == 0 ? a.q : part == 1 ? a.k : a.v;
  const Rows& dst = part == 0 ? a.q_out : part == 1 ? a.k_out : a.v_out;
  const int heads = part == 0 ? a.q_heads : a.kv_heads;
  const bool store = BITS != 0 && part > 0;
  const bool turn = part < 2 && a.rotary > 0;
  const int64_t pos = turn ? a.positions[token] : 0;
  const int64_t slot = store ? a.slots[token] : -1;
  u32x4 x[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
    x[r] = load_u32x4(src.p + token * src.token + min(first + r, heads - 1) * src.head + 8 * j);
  const uint16_t* const weight = part == 0 ? a.q_weight : part == 1 ? a.k_weight : nullptr;
  const char* const zero = reinterpret_cast<const char*>(g_qsa_zero_rows);
  const u32x4 wr = load_u32x4(weight ? (const char*)(weight + 8 * j) : zero);

  // The table's row: zeros outside it.
  const int half = a.rotary / 2;
  const bool rotated = turn && 8 * j < a.rotary, lower = 8 * j < half;
  const bool in_table = rotated && pos >= 0 && pos < a.max_positions;
  const int64_t entry = in_table ? pos * a.rotary + (lower ? 8 * j : 8 * j - half) : 0;
  float c[8], s[8];
  if (a.cos_sin_fp32) {
    const char* const t = in_table ? (const char*)a.cos_sin + 4 * entry : zero;
    const int64_t apart = in_table ? 4 * half : 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const f32x4 cv = *reinterpret_cast<const f32x4*>(t + 16 * e);
      const f32x4 sv = *reinterpret_cast<const f32x4*>(t + apart + 16 * e);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[4 * e + i] = cv[i];
        s[4 * e + i] = sv[i];
      }
    }
  } else {
    const char* const t = in_table ? (const char*)a.cos_sin + 2 * entry : zero;
    unpack8(load_u32x4(t), c);
    unpack8(load_u32x4(t + (in_table ? 2 * half : 0)), s);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = lower ? -s[i] : s[i];
  // dims i < half turn with i + half: the lane half / 8 further.
  const int lane = threadIdx.x & 63;
  const int partner = rotated ? (lower ? lane + half / 8 : lane - half / 8) : lane;

  int64_t block = -1;
  int place = 0;
  if (slot >= 0 && slot < a.num_slots) {
    block = a.num_slots <= INT_MAX ? a.page_div.div((int)slot) : slot / a.page_div.divisor;
    place = (int)(slot - block * a.page_div.divisor);
  }

#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int head = first + r;
    if (head >= heads) break;
    if (weight || turn) {
      float f[8];
      unpack8(x[r], f);
      if (weight) {
        float w[8], sum = 0.0f;
        unpack8(wr, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += f[i] * f[i];
#pragma unroll
        for (int m = 1; m < kLanes; m *= 2) sum += __shfl_xor(sum, m, 64);
        const float inv = __fdiv_rn(1.0f, __fsqrt_rn(sum * (1.0f / D) + a.eps));
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = f[i] * inv * w[i];
      }
      if (turn) {
        float other[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) other[i] = __shfl(f[i], partner, 64);
        if (rotated) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = f[i] * c[i] + other[i] * s[i];
        }
      }
      x[r] = pack8(f);
    }
    if (store) {
      if constexpr (BITS == 16) {
        char* const to = part == 1 ? a.k_cache + block * a.kb + place * a.kt + head * a.kh
                                   : a.v_cache + block * a.vb + place * a.vt + head * a.vh;
        if (block >= 0) *reinterpret_cast<u32x4*>(to + 16 * j) = x[r];
      } else if constexpr (BITS == 4) {
        float f[8];
        uint32_t code[8];
        const uint32_t word = quantize4(x[r], dst.p != nullptr, f, code);
        const Kv4Page lay{a.page_div.divisor, D};
        char* const to = a.k_cache + block * a.kb + head * a.kh;
        if (block >= 0) {
          uint32_t packed = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            packed |= code[i] << (part == 1 ? 4 * (i / 2) + 16 * (i % 2) : 4 * i);
          *reinterpret_cast<uint32_t*>(
              to + (part == 1 ? 0 : lay.v_codes()) + (int64_t)place * lay.row() +
              4 * (part == 1 ? j % 4 * (D / 32) + j / 4 : j)) = packed;
          if (j % 4 == 0)
            *reinterpret_cast<uint16_t*>(to + (part == 1 ? lay.k_words() : lay.v_words()) +
                                         (int64_t)place * lay.words() + j / 4 * 2) = (uint16_t)word;
        }
        x[r] = pack8(f);
      }
    }
    if (dst.p)
      *reinterpret_cast<u32x4*>(dst.p + token * dst.token + head * dst.head + 8 * j) = x[r];
  }
}

// Groups of lanes: first those of the queries (ROWS heads each), from workgroup q_blocks
// on those of all keys, then of all values, so that a wave's groups have the same to do.
template <int D, int BITS, int ROWS>
__global__ __launch_bounds__(kThreads) void head_rope_kernel(HeadRopeArgs a) {
  constexpr int kLanes = D / 8, kPer = kThreads / kLanes, kKvRows = ROWS > 2 ? 2 : ROWS;
  const int j = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  if ((int)blockIdx.x < a.q_blocks) {
    const int item = blockIdx.x * kPer + group;
    if (item >= a.q_items) return;
    const int token = a.q_div.div(item);
    take_heads<D, BITS, ROWS>(a, 0, token, (item - token * a.q_div.divisor) * ROWS, j);
  } else {
    int item = (blockIdx.x - a.q_blocks) * kPer + group;
    if (item >= a.kv_parts * a.kv_items) return;
    const int part = item < a.kv_items ? 1 : 2;
    item -= (part - 1) * a.kv_items;
    const int token = a.kv_div.div(item);
    take_heads<D, BITS, kKvRows>(a, part, token, (item - token * a.kv_div.divisor) * kKvRows, j);
  }
}

template <int D, int ROWS>
void launch_rows(HeadRopeArgs& a, int tokens, int bits, hipStream_t stream) {
  constexpr int kPer = kThreads / (D / 8), kKvRows = ROWS > 2 ? 2 : ROWS;
  const int q = (a.q_heads + ROWS - 1) / ROWS, kv = (a.kv_heads + kKvRows - 1) / kKvRows;
  a.q_div = FastDiv::make(std::max(q, 1));
  a.kv_div = FastDiv::make(std::max(kv, 1));
  a.q_items = q * tokens;
  a.kv_items = kv * tokens;
  a.q_blocks = (a.q_items + kPer - 1) / kPer;
  const dim3 grid((unsigned)(a.q_blocks + (a.kv_parts * a.kv_items + kPer - 1) / kPer)), block(kThreads);
  if (bits == 0) hipLaunchKernelGGL((head_rope_kernel<D, 0, ROWS>), grid, block, 0, stream, a);
  else if (bits == 16) hipLaunchKernelGGL((head_rope_kernel<D, 16, ROWS>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((head_rope_kernel<D, 4, ROWS>), grid, block, 0, stream, a);
}
template <int D>
void launch_head_rope(HeadRopeArgs& a, int tokens, int bits, hipStream_t stream) {
  const int64_t rows = (int64_t)(a.q_heads + a.kv_parts * a.kv_heads) * tokens;
  if (rows <= kSmall) launch_rows<D, 1>(a, tokens, bits, stream);
  else launch_rows<D, 4>(a, tokens, bits, stream);
}

}  // namespace
}  // namespace qsa

using namespace qsa;

extern "C" int64_t qsa_kv4_page_bytes(int page_size, int head_dim) {
  return page_size > 0 && (head_dim == 64 || head_dim == 128) ? Kv4Page{page_size, head_dim}.bytes()
                                                              : 0;
}

extern "C" int qsa_qk_norm_rope(
    const void* query, int64_t q_token_stride, int64_t q_head_stride, int num_q_heads,
    const void* key, int64_t k_token_stride, int64_t k_head_stride, const void* value,
    int64_t v_token_stride, int64_t v_head_stride, int num_kv_heads, int head_dim, int tokens,
    const void* q_weight, const void* k_weight, float eps, const int64_t* positions,
    const void* cos_sin, int cos_sin_fp32, int max_positions, int rotary_dim, void* q_out,
    int64_t q_out_token_stride, int64_t q_out_head_stride, void* k_out, int64_t k_out_token_stride,
    int64_t k_out_head_stride, void* v_out, int64_t v_out_token_stride, int64_t v_out_head_stride,
    int cache_bits, const int64_t* slot_mapping, void* k_cache, int64_t k_block_stride,
    int64_t k_cache_token_stride, int64_t k_cache_head_stride, void* v_cache,
    int64_t v_block_stride, int64_t v_cache_token_stride, int64_t v_cache_head_stride,
    int num_blocks, int page_size, void* stream) {
  const std::string name = "qsa_qk_norm_rope";
  if (tokens < 0 || num_q_heads < 0 || num_kv_heads < 0 || num_blocks < 0)
    return fail(QSA_ERR_INVALID, name + ": negative size");
  if (tokens == 0) return QSA_OK;
  if (head_dim != 64 && head_dim != 128)
    return fail(QSA_ERR_UNSUPPORTED, name + ": head_dim must be 64 or 128");
  if (cache_bits != 0 && cache_bits != 16 && cache_bits != 4)
    return fail(QSA_ERR_UNSUPPORTED, name + ": a cache holds 16 or 4 bits");
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16)
    return fail(QSA_ERR_UNSUPPORTED, name + ": rotary_dim must be a multiple of 16 up to head_dim");
  if (rotary_dim > 0 && (!positions || !cos_sin || max_positions <= 0))
    return fail(QSA_ERR_INVALID, name + ": a rotation needs positions and a table");
  if ((num_q_heads > 0 && (!query || !q_out)) || (num_kv_heads > 0 && !key))
    return fail(QSA_ERR_INVALID, name + ": null tensor pointer");
  if (v_out && !value) return fail(QSA_ERR_INVALID, name + ": v_out without values");
  if (cache_bits != 0) {
    if (!value || !slot_mapping || ((!k_cache || (cache_bits == 16 && !v_cache)) && num_blocks > 0))
      return fail(QSA_ERR_INVALID, name + ": a cache needs values and slots");
    if (page_size <= 0) return fail(QSA_ERR_INVALID, name + ": page size must be positive");
    if (!aligned16(k_cache) || !aligned16(v_cache))
      return fail(QSA_ERR_INVALID, name + ": caches need 16-byte alignment");
    if (cache_bits == 16 &&
        ((k_block_stride | k_cache_token_stride | k_cache_head_stride | v_block_stride |
          v_cache_token_stride | v_cache_head_stride) & 7))
      return fail(QSA_ERR_INVALID, name + ": cache strides must be multiples of 8 elements");
    if (cache_bits == 4 && ((k_block_stride | k_cache_head_stride) & 15))
      return fail(QSA_ERR_INVALID, name + ": a 4-bit cache's strides must be multiples of 16 bytes");
  }
  if (((q_token_stride | q_head_stride | k_token_stride | k_head_stride | v_token_stride |
        v_head_stride | q_out_token_stride | q_out_head_stride | k_out_token_stride |
        k_out_head_stride | v_out_token_stride | v_out_head_stride) & 7) ||
      !aligned16(query) || !aligned16(key) || !aligned16(value) || !aligned16(q_out) ||
      !aligned16(k_out) || !aligned16(v_out) || !aligned16(q_weight) || !aligned16(k_weight) ||
      !aligned16(cos_sin))
    return fail(QSA_ERR_INVALID, name + ": rows, weights and table need 16-byte alignment and "
                                        "strides of multiples of 8 elements");
  const int64_t rows = (int64_t)num_q_heads + num_kv_heads * (value ? 2 : 1);
  if (rows == 0) return QSA_OK;
  const int64_t groups =
      (num_q_heads + (int64_t)3) / 4 + (num_kv_heads + (int64_t)1) / 2 * (value ? 2 : 1);
  // (32-bit counts of rows, and a launch of less than 2^32 threads)
  if (rows * tokens > INT_MAX - 4096 || groups * tokens * (head_dim / 8) > UINT_MAX - 4096)
    return fail(QSA_ERR_UNSUPPORTED, name + ": too many rows");
  HeadRopeArgs a = {};
  auto view = [](const void* p, int64_t token, int64_t head) {
    return Rows{static_cast<uint16_t*>(const_cast<void*>(p)), token, head};
  };
  a.q = view(query, q_token_stride, q_head_stride);
  a.k = view(key, k_token_stride, k_head_stride);
  a.v = view(value, v_token_stride, v_head_stride);
  a.q_out = view(q_out, q_out_token_stride, q_out_head_stride);
  a.k_out = view(k_out, k_out_token_stride, k_out_head_stride);
  a.v_out = view(v_out, v_out_token_stride, v_out_head_stride);
  a.q_heads = num_q_heads;
  a.kv_heads = num_kv_heads;
  a.kv_parts = value ? 2 : 1;
  a.q_weight = static_cast<const uint16_t*>(q_weight);
  a.k_weight = static_cast<const uint16_t*>(k_weight);
  a.eps = eps;
  a.positions = positions;
  a.cos_sin = cos_sin;
  a.cos_sin_fp32 = cos_sin_fp32;
  a.max_positions = max_positions;
  a.rotary = rotary_dim;
  a.slots = slot_mapping;
  a.k_cache = static_cast<char*>(k_cache);
  a.v_cache = static_cast<char*>(v_cache);
  const int unit = cache_bits == 16 ? 2 : 1;  // bytes of the caches' stride units
  a.kb = unit * k_block_stride;
  a.kt = unit * k_cache_token_stride;
  a.kh = unit * k_cache_head_stride;
  a.vb = unit * v_block_stride;
  a.vt = unit * v_cache_token_stride;
  a.vh = unit * v_cache_head_stride;
  a.num_slots = (int64_t)num_blocks * page_size;
  a.page_div = FastDiv::make(std::max(page_size, 1));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 128) launch_head_rope<128>(a, tokens, cache_bits, s);
  else launch_head_rope<64>(a, tokens, cache_bits, s);
  return check_launch("qsa_qk_norm_rope launch");
}

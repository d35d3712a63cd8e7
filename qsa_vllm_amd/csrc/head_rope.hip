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
// rotation partners by lane exchange. Bound by memory for many tokens, by the
// launch and one chain of loads for few.
#include "qsa_common.h"
#include "../../include/qsa_hip.h"
#include "kv4.h"

#include <climits>

namespace qsa {
namespace {

constexpr int kThreads = 256;

struct Rows {  // [tokens, heads, D] bf16, strides in elements
  uint16_t* p;
  int64_t token, head;
};

struct HeadRopeArgs {
  Rows q, k, v, q_out, k_out, v_out;
  int q_heads, kv_heads;  // of the rows that the launch has: 0 query heads without queries
  FastDiv rows_div;       // rows of a token: query, key and value heads
  int total;              // rows of the launch
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
  int num_blocks, page;
};

__device__ __forceinline__ void unpack8(const u32x4& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = bf16_lo(v[i]);
    f[2 * i + 1] = bf16_hi(v[i]);
  }
}
__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
  return v;
}

// Rows of 8 dims a lane: 4 lanes share a group of 32. Returns the group's word, the
// lane's 8 codes packed (each byte of `lo`: dims 0 .. 3, `hi`: dims 4 .. 7), and puts
// the values that they stand for into f.
__device__ __forceinline__ uint32_t quantize4(const u32x4& x, float (&f)[8], uint32_t (&codes)[8]) {
#pragma clang fp contract(off)
  unpack8(x, f);
  float low = 0.0f, high = 0.0f;
  int bad = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    low = fminf(low, f[i]);
    high = fmaxf(high, f[i]);
    bad |= (__builtin_bit_cast(uint32_t, f[i]) & 0x7FFFFFFFu) >= 0x7E800000u;
  }
#pragma unroll
  for (int m = 1; m < 4; m *= 2) {
    low = fminf(low, __shfl_xor(low, m, 64));
    high = fmaxf(high, __shfl_xor(high, m, 64));
    bad |= __shfl_xor(bad, m, 64);
  }
  if (bad) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      codes[i] = 1;
      f[i] = __builtin_nanf("");
    }
    return kKv4NaN;
  }
  const float step = fmaxf(__fdiv_rn(high - low, 15.0f), 0x1p-100f);
  const uint32_t sbits = (__builtin_bit_cast(uint32_t, step) + 0xFFFFFu) & ~0xFFFFFu;
  const float s = __builtin_bit_cast(float, sbits);
  const float z = fminf(rintf(__fdiv_rn(-low, s)), 15.0f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = fminf(fmaxf(rintf(__fdiv_rn(f[i], s)) + z, 0.0f), 15.0f);
    codes[i] = (uint32_t)c;
    f[i] = (c - z) * s;
  }
  return sbits >> 16 | (uint32_t)z;
}

template <int D, int BITS>
__global__ __launch_bounds__(kThreads) void head_rope_kernel(HeadRopeArgs a) {
  constexpr int kLanes = D / 8;
  const int j = threadIdx.x % kLanes;
  const int64_t item = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  if (item >= a.total) return;  // whole groups of lanes
  const int token = a.rows_div.div((int)item);
  int head = (int)item - token * a.rows_div.divisor;
  const int part = head < a.q_heads ? 0 : head < a.q_heads + a.kv_heads ? 1 : 2;  // q, k, v
  head -= part == 0 ? 0 : a.q_heads + (part - 1) * a.kv_heads;
  const Rows& src = part == 0 ? a.q : part == 1 ? a.k : a.v;
  const Rows& dst = part == 0 ? a.q_out : part == 1 ? a.k_out : a.v_out;

  u32x4 x = load_u32x4(src.p + token * src.token + head * src.head + 8 * j);
  const uint16_t* const weight = part == 0 ? a.q_weight : part == 1 ? a.k_weight : nullptr;
  const bool turn = part < 2 && a.rotary > 0;
  if (weight || turn) {
    float f[8];
    unpack8(x, f);
    if (weight) {
      float w[8], sum = 0.0f;
      unpack8(load_u32x4(weight + 8 * j), w);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += f[i] * f[i];
#pragma unroll
      for (int m = 1; m < kLanes; m *= 2) sum += __shfl_xor(sum, m, 64);
      const float inv = __fdiv_rn(1.0f, __fsqrt_rn(sum * (1.0f / D) + a.eps));
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = f[i] * inv * w[i];
    }
    if (turn) {
      const int half = a.rotary / 2;
      const int64_t pos = a.positions[token];
      float c[8] = {}, s[8] = {};
      if (8 * j < a.rotary && pos >= 0 && pos < a.max_positions) {
        const int64_t at = pos * a.rotary + 8 * j % half;
        if (a.cos_sin_fp32) {
          const float* t = static_cast<const float*>(a.cos_sin) + at;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            c[i] = t[i];
            s[i] = t[half + i];
          }
        } else {
          const uint16_t* t = static_cast<const uint16_t*>(a.cos_sin) + at;
          unpack8(load_u32x4(t), c);
          unpack8(load_u32x4(t + half), s);
        }
      }
      // dims i < half turn with i + half: the lane half / 8 further.
      const int lane = threadIdx.x & 63;
      const bool rotated = 8 * j < a.rotary, first = 8 * j < half;
      const int partner = rotated ? (first ? lane + half / 8 : lane - half / 8) : lane;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float other = __shfl(f[i], partner, 64);
        f[i] = rotated ? f[i] * c[i] + (first ? -other : other) * s[i] : f[i];
      }
    }
    x = pack8(f);
  }

  if (part > 0 && BITS != 0) {
    const int64_t slot = a.slots[token];
    const int64_t block = slot >= 0 ? slot / a.page : -1;
    const bool live = block >= 0 && block < a.num_blocks;
    const int place = live ? (int)(slot - block * a.page) : 0;
    if constexpr (BITS == 16) {
      char* const to = part == 1 ? a.k_cache + block * a.kb + place * a.kt + head * a.kh
                                 : a.v_cache + block * a.vb + place * a.vt + head * a.vh;
      if (live) *reinterpret_cast<u32x4*>(to + 16 * j) = x;
    } else {
      float f[8];
      uint32_t c[8];
      const uint32_t word = quantize4(x, f, c);
      const Kv4Page lay{a.page, D};
      char* const to = a.k_cache + block * a.kb + head * a.kh;
      uint32_t packed = 0;
      if (live) {
        if (part == 1) {
#pragma unroll
          for (int i = 0; i < 8; ++i) packed |= c[i] << (4 * (i / 2) + 16 * (i % 2));
          *reinterpret_cast<uint32_t*>(to + (int64_t)place * lay.row() +
                                       4 * (j % 4 * (D / 32) + j / 4)) = packed;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) packed |= c[i] << (4 * i);
          *reinterpret_cast<uint32_t*>(to + lay.v_codes() + (int64_t)place * lay.row() + 4 * j) =
              packed;
        }
        if (j % 4 == 0)
          *reinterpret_cast<uint16_t*>(to + (part == 1 ? lay.k_words() : lay.v_words()) +
                                       place * lay.words() + j / 4 * 2) = (uint16_t)word;
      }
      x = pack8(f);
    }
  }
  if (dst.p)
    *reinterpret_cast<u32x4*>(dst.p + token * dst.token + head * dst.head + 8 * j) = x;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

template <int D>
void launch_head_rope(const HeadRopeArgs& a, int bits, unsigned blocks, hipStream_t stream) {
  const dim3 grid(blocks), block(kThreads);
  if (bits == 0) hipLaunchKernelGGL((head_rope_kernel<D, 0>), grid, block, 0, stream, a);
  else if (bits == 16) hipLaunchKernelGGL((head_rope_kernel<D, 16>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((head_rope_kernel<D, 4>), grid, block, 0, stream, a);
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
  if (rows * tokens > INT_MAX) return fail(QSA_ERR_UNSUPPORTED, name + ": too many rows");
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
  a.rows_div = FastDiv::make((int)rows);
  a.total = (int)(rows * tokens);
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
  a.num_blocks = num_blocks;
  a.page = page_size;
  const int per = kThreads / (head_dim / 8);
  const unsigned blocks = (unsigned)((rows * tokens + per - 1) / per);
  if (blocks > UINT_MAX / kThreads) return fail(QSA_ERR_UNSUPPORTED, name + ": too many rows");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 128) launch_head_rope<128>(a, cache_bits, blocks, s);
  else launch_head_rope<64>(a, cache_bits, blocks, s);
  return check_launch("qsa_qk_norm_rope launch");
}

// Linear layer with 4-bit weights and group scales on a few activation rows.
//
//   y[m][n] = round(sum_k x[m][k] (c[n][k] - z[n][k / G]) s[n][k / G] + b[n])
//
// c: 4-bit codes; s: one scale per output n and group of G = 32, 64 or 128
// input channels; z: the group's zero point (8 for all if none are given).
//
// Mathematics. A group's scale is a factor of its whole sum, so the codes go
// into the matrix product as small whole numbers and the scale multiplies the
// group's fp32 sum: nothing is rounded before the output. With bf16 the code q
// becomes c0 + q - z by an and and an or (or add), c0 = 192 with zero points
// and 136 without: bf16 holds whole numbers to 256. Then
//   sum x (q - z) = sum x (c0 + q - z) - c0 sum x,
// and the last term, the same for every output, is the accumulator's start: the
// product of x with a constant. Both are summed in fp32, whose step is 2^-16 of
// bf16's; where that gives no finite sum, it is taken again without the constant
// (plain_sum). With fp16 the code becomes 1024 + q (or 1024 + 16 q), a number below
// 2^10 or-ed into the mantissa of 1024 (a common way to make fp16 of small whole
// numbers), and one packed add (or fma) gives q - z exactly.
//
// Layout. Weights are stored in tiles of 16 outputs x 128 inputs, 1 KiB each:
// lane (n, g) of a wave holds output n's codes of inputs 32 j + 8 g .. + 7 as
// word j, the B operand of mfma_f32_16x16x32 after unpacking, element 2 p of a
// word in bits 4 p and element 2 p + 1 in bits 16 + 4 p. So a wave reads a tile
// with one 16-byte load a lane, unpacking is shifts, ands and ors, and a tile's
// scales (zero points) of an output are one load.
//
// Two kernels, by rows:
//  * to 16 rows, bound by streaming the weight: a wave takes whole tiles, its
//    workgroup's waves share the inputs (tile t to wave t mod waves), and
//    activations come straight from L2;
//  * more, where each workgroup's re-reading of the activations is the larger
//    traffic: they go through LDS in whole 256-byte rows, shared by the waves
//    that take different outputs (int4_rows_kernel).
// Waves that share the inputs add their sums through LDS in wave order: no
// atomics, the same bits every time.
//
// Measured (bf16, groups of 128 unless said): 1 row x 49536 x 4096 21.6 us, 4.85 TB/s
// (a large copy 4.8); 61 rows x 11264 x 4096 12.7 us, bound by its few steps in
// series; 250 rows x 22528 x 4096, groups of 64 with zero points, 66 us, 0.70
// PFLOP/s: vector issue, unpacking for each block of 64 rows.
#include "qsa_common.h"
#include "../../include/qsa_hip.h"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace qsa {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kTileN = 16;
constexpr int kTileK = 128;
constexpr int kCUs = 256;  // compute units of an MI355X

// s_waitcnt immediate (gfx9 encoding): no vector-memory, no LDS operation in flight.
constexpr int kMemoryDone = 7 << 4;

struct Int4Args {
  const uint16_t* x;
  int64_t x_row;
  const u32x4* codes;     // [n tiles][k tiles][64 lanes]
  const char* scales;     // [n tiles][k tiles][16][128 / G] 16-bit
  const char* zeros;      // [n tiles][k tiles][16][128 / G] 8-bit, or null
  const uint16_t* bias;   // [n] or null
  uint16_t* y;
  int64_t y_row;
  int rows, n, k;
  int n_tiles, k_tiles;
  int row_blocks;
};

// GROUPS values of 16 (8) bits of a tile's output, loaded at once.
template <int GROUPS>
struct GroupWords;
template <>
struct GroupWords<1> {
  typedef uint16_t scales;
  typedef uint8_t zeros;
};
template <>
struct GroupWords<2> {
  typedef uint32_t scales;
  typedef uint16_t zeros;
};
template <>
struct GroupWords<4> {
  typedef u32x2 scales;
  typedef uint32_t zeros;
};
__device__ __forceinline__ uint16_t scale_of(uint16_t v, int) { return v; }
__device__ __forceinline__ uint16_t scale_of(uint32_t v, int q) { return (uint16_t)(v >> (16 * q)); }
__device__ __forceinline__ uint16_t scale_of(const u32x2& v, int q) {
  return (uint16_t)(v[q >> 1] >> (16 * (q & 1)));
}

// The mask of a word's lowest codes, as a value the compiler cannot see: with
// two known constants it splits (w & mask) | c into two instructions (a VOP3
// instruction takes no literal, and one scalar), with unknown ones it is one.
__device__ __forceinline__ uint32_t code_mask() {
  uint32_t m = 0x000F000Fu;
  asm("" : "+s"(m));
  return m;
}
__device__ __forceinline__ uint32_t hidden(uint32_t c) {
  asm("" : "+v"(c));
  return c;
}

// A type's matrix operand: unpacking a word of codes with a zero point's
// constant, and what the accumulator's start takes off again.
template <bool ZEROS>
struct Bf16 {
  typedef bf16x8 frag;
  static constexpr bool kOffset = true;
  static __device__ __forceinline__ f32x4 mfma(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  // 192 - z in both halves (128, to which a code is or-ed, without zero points).
  static __device__ __forceinline__ uint32_t zero_word(int z) {
    return ZEROS ? 0x43404340u - (uint32_t)z * 0x10001u : hidden(0x43004300u);
  }
  static __device__ __forceinline__ frag unpack(uint32_t w, uint32_t zero) {
    u32x4 r;
    const uint32_t mask = code_mask();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (ZEROS) r[i] = ((w >> (4 * i)) & 0x000F000Fu) + zero;
      else r[i] = ((w >> (4 * i)) & mask) | zero;
    }
    return __builtin_bit_cast(frag, r);
  }
  static __device__ __forceinline__ frag offset() {  // -192 or -136
    const uint32_t c = ZEROS ? 0xC340C340u : 0xC308C308u;
    return __builtin_bit_cast(frag, (u32x4{c, c, c, c}));
  }
  static __device__ __forceinline__ float to_float(uint16_t v) {
    return __builtin_bit_cast(float, (uint32_t)v << 16);
  }
  static __device__ __forceinline__ uint16_t from_float(float v) {
    return (uint16_t)pack_bf16x2(v, v);
  }
};

template <bool ZEROS>
struct Fp16 {
  typedef f16x8 frag;
  static constexpr bool kOffset = false;
  static __device__ __forceinline__ f32x4 mfma(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t zero_word(int z) {  // -1024 - z in both halves
    return 0xE400E400u + (uint32_t)z * 0x10001u;
  }
  static __device__ __forceinline__ frag unpack(uint32_t w, uint32_t zero) {
    const f16x2 low = __builtin_bit_cast(f16x2, zero);
    const f16x2 gap = {(_Float16)960.0f, (_Float16)960.0f};
    const f16x2 high = low + gap;  // -64 - z
    const f16x2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    union {
      f16x2 p[4];
      frag f;
    } r;
    const uint32_t v = w >> 8, mask = code_mask(), magic = hidden(0x64006400u);
    r.p[0] = __builtin_bit_cast(f16x2, (w & mask) | magic) + low;
    r.p[1] = __builtin_elementwise_fma(
        __builtin_bit_cast(f16x2, (w & 0x00F000F0u) | 0x64006400u), sixteenth, high);
    r.p[2] = __builtin_bit_cast(f16x2, (v & mask) | magic) + low;
    r.p[3] = __builtin_elementwise_fma(
        __builtin_bit_cast(f16x2, (v & 0x00F000F0u) | 0x64006400u), sixteenth, high);
    return r.f;
  }
  static __device__ __forceinline__ frag offset() { return frag{}; }  // not used
  static __device__ __forceinline__ float to_float(uint16_t v) {
    return (float)__builtin_bit_cast(_Float16, v);
  }
  static __device__ __forceinline__ uint16_t from_float(float v) {
    return __builtin_bit_cast(uint16_t, (_Float16)v);
  }
};

template <typename V>
__device__ __forceinline__ V load_at(const char* base, uint32_t offset) {
  return *reinterpret_cast<const V*>(base + offset);
}

// A wave's weight tiles of one k tile: NT adjacent n tiles.
template <int GROUP, bool ZEROS, int NT>
struct Tiles {
  static constexpr int kGroups = kTileK / GROUP;
  typedef GroupWords<kGroups> Words;
  u32x4 w[NT];
  typename Words::scales s[NT];
  typename Words::zeros z[NT];
  // Tiles past the last (an odd end) are read as the last one; not stored.
  // tile0 and t are the same in the whole wave: scalar addresses, and a lane's
  // offset from them that never changes.
  __device__ __forceinline__ void load(const Int4Args& a, int tile0, int t, int lane) {
    const uint32_t n = lane & 15;
#pragma unroll
    for (int v = 0; v < NT; ++v) {
      const int64_t at = (int64_t)min(tile0 + v, a.n_tiles - 1) * a.k_tiles + t;
      w[v] = load_at<u32x4>(reinterpret_cast<const char*>(a.codes) + at * 1024, lane * 16u);
      s[v] = load_at<typename Words::scales>(a.scales + at * (32 * kGroups), n * (2 * kGroups));
      if constexpr (ZEROS)
        z[v] = load_at<typename Words::zeros>(a.zeros + at * (16 * kGroups), n * kGroups);
    }
  }
  __device__ __forceinline__ int zero(int v, int q) const {
    return ZEROS ? (int)(((uint32_t)z[v] >> (8 * q)) & 0xFFu) : 8;
  }
};

// acc += x (MT x 16 rows, the k tile's four operands each) times the tiles.
template <typename T, int GROUP, bool ZEROS, int MT, int NT>
__device__ __forceinline__ void multiply(const u32x4 (&x)[MT][4], const Tiles<GROUP, ZEROS, NT>& b,
                                         f32x4 (&acc)[MT][NT]) {
  typedef typename T::frag frag;
  constexpr int kSteps = GROUP / 32;  // matrix instructions per group
#pragma unroll
  for (int q = 0; q < kTileK / GROUP; ++q) {
    f32x4 start[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      start[i] = f32x4{0, 0, 0, 0};
      if constexpr (T::kOffset) {
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
          start[i] = T::mfma(__builtin_bit_cast(frag, x[i][q * kSteps + j]), T::offset(), start[i]);
      }
    }
#pragma unroll
    for (int v = 0; v < NT; ++v) {
      const float scale = T::to_float(scale_of(b.s[v], q));
      const uint32_t zero = T::zero_word(b.zero(v, q));
      f32x4 d[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) d[i] = start[i];
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        const frag f = T::unpack(b.w[v][q * kSteps + j], zero);
#pragma unroll
        for (int i = 0; i < MT; ++i)
          d[i] = T::mfma(__builtin_bit_cast(frag, x[i][q * kSteps + j]), f, d[i]);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][v][r] = __builtin_fmaf(scale, d[i][r], acc[i][v][r]);
    }
  }
}

// A tile's sums (a lane: rows 4 g + r of output n) to y. Returns which of the four
// are not finite, as bits.
template <typename T>
__device__ __forceinline__ uint32_t store(const Int4Args& a, int m0, int tile, int lane,
                                          const f32x4& sum) {
  const int col = tile * kTileN + (lane & 15);
  uint32_t bad = 0;
  if (col >= a.n) return bad;
  const float b = a.bias ? T::to_float(a.bias[col]) : 0.0f;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int m = m0 + 4 * (lane >> 4) + r;
    if (m >= a.rows) continue;
    const float v = sum[r];
    a.y[m * a.y_row + col] = T::from_float(v + b);
    bad |= (uint32_t)((__builtin_bit_cast(uint32_t, v) & 0x7F800000u) == 0x7F800000u) << r;
  }
  return bad;
}

// One result as its formula has it, term by term. Infinities in x, or bf16 values
// past 2^112, make the offset's product and the codes' cancel to NaN, and padded
// inputs repeat the row's first ones, which may be infinite: a sum that is not
// finite is taken again here, a result a lane. A NaN in x ends it at once; an infinity
// at the end of one row, or of each, of 61 rows x 11264 x 4096 takes 0.4 or 2.6 ms.
template <typename T, int GROUP, bool ZEROS>
__device__ __forceinline__ float plain_sum(const Int4Args& a, int m, int col) {
  constexpr int kGroups = kTileK / GROUP;
  const int tile = col / kTileN, n = col % kTileN;
  const uint16_t* const x = a.x + m * a.x_row;
  const uint32_t* const words = reinterpret_cast<const uint32_t*>(a.codes);
  float sum = 0.0f;
  for (int k = 0; k < a.k && sum == sum; k += 8) {
    const int in = k % kTileK, j = in / 32, g = in % 32 / 8;
    const int64_t at = (int64_t)tile * a.k_tiles + k / kTileK;
    const int64_t group = (at * kTileN + n) * kGroups + in / GROUP;
    const uint32_t w = words[(at * 64 + 16 * g + n) * 4 + j];
    const float scale = T::to_float(reinterpret_cast<const uint16_t*>(a.scales)[group]);
    const int zero = ZEROS ? reinterpret_cast<const uint8_t*>(a.zeros)[group] : 8;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < a.k) {
        const int code = (int)(w >> (4 * (i / 2) + 16 * (i % 2))) & 15;
        sum = __builtin_fmaf(T::to_float(x[k + i]), (float)(code - zero) * scale, sum);
      }
  }
  return sum;
}

// Results of a wave's tiles whose sums were not finite: bit 4 u + r of `bad` for row
// 4 g + r of tile u (row block u / NT, output tile u % NT).
template <typename T, int GROUP, bool ZEROS, int NT>
__device__ __forceinline__ void repair(const Int4Args& a, uint64_t bad, int row0, int tile0, int lane) {
  while (bad) {
    const int at = __ffsll((unsigned long long)bad) - 1;
    bad &= bad - 1;
    const int m = row0 + 16 * (at / 4 / NT) + 4 * (lane >> 4) + at % 4;
    const int col = (tile0 + at / 4 % NT) * kTileN + (lane & 15);
    const float b = a.bias ? T::to_float(a.bias[col]) : 0.0f;
    a.y[m * a.y_row + col] = T::from_float(plain_sum<T, GROUP, ZEROS>(a, m, col) + b);
  }
}

// Eight activations from input k on, element by element: rows that 16-byte
// loads cannot take. Inputs past the width are zero and not read.
__device__ __forceinline__ u32x4 gather_x(const uint16_t* row, int k, int width) {
  u32x4 r = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k + i < width) r[i / 2] |= (uint32_t)row[k + i] << (16 * (i & 1));
  return r;
}

// To 16 MT rows a workgroup. VEC: row stride, width and address are multiples of
// 8 elements.
template <typename T, int GROUP, bool ZEROS, int MT, int NT, bool VEC>
__global__ __launch_bounds__(512) void int4_linear_kernel(Int4Args a) {
  typedef Tiles<GROUP, ZEROS, NT> Weights;
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int row0 = (blockIdx.x % a.row_blocks) * (16 * MT);
  const int tile0 = (blockIdx.x / a.row_blocks) * NT;

  f32x4 acc[MT][NT] = {};
  const uint16_t* const xblock = a.x + row0 * a.x_row;
  // Rows past the last repeat it (their results are not stored), and inputs past
  // the width the row's first ones (their codes are the zero point): no load
  // depends on a condition, which would make it wait for the ones before it.
  // The lane's byte offset in the block: rows taken element by element may be any
  // distance apart.
  typename std::conditional<VEC, uint32_t, int64_t>::type at[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int row = min(16 * i + n, a.rows - 1 - row0);
    if constexpr (VEC) at[i] = (uint32_t)row * (uint32_t)(2 * a.x_row);
    else at[i] = row * (2 * a.x_row);
  }
  auto load_rows = [&](int t, u32x4 (&x)[MT][4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = t * kTileK + 32 * j + 8 * g;
#pragma unroll
      for (int i = 0; i < MT; ++i)
        if constexpr (VEC)
          x[i][j] = load_at<u32x4>(reinterpret_cast<const char*>(xblock),
                                   at[i] + (k < a.k ? 2 * k : 0));
        else
          x[i][j] = gather_x(reinterpret_cast<const uint16_t*>(
                                 reinterpret_cast<const char*>(xblock) + at[i]), k, a.k);
    }
  };
  // Two tiles in flight: the next one's loads are issued before this one's
  // product.
  Weights b0, b1;
  u32x4 x0[MT][4], x1[MT][4];
  int t = wave;
  b0.load(a, tile0, t, lane);
  load_rows(t, x0);
  while (true) {
    int next = t + waves;
    if (next < a.k_tiles) {
      b1.load(a, tile0, next, lane);
      load_rows(next, x1);
    }
    multiply<T, GROUP, ZEROS, MT, NT>(x0, b0, acc);
    if (next >= a.k_tiles) break;
    t = next + waves;
    if (t < a.k_tiles) {
      b0.load(a, tile0, t, lane);
      load_rows(t, x0);
    }
    multiply<T, GROUP, ZEROS, MT, NT>(x1, b1, acc);
    if (t >= a.k_tiles) break;
  }

  extern __shared__ f32x4 part[];  // [waves][MT * NT][64]
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int v = 0; v < NT; ++v) part[(wave * MT * NT + i * NT + v) * 64 + lane] = acc[i][v];
  __syncthreads();
  uint64_t bad = 0;
  for (int u = wave; u < MT * NT; u += waves) {
    f32x4 sum = part[u * 64 + lane];
    for (int o = 1; o < waves; ++o) sum += part[(o * MT * NT + u) * 64 + lane];
    bad |= (uint64_t)store<T>(a, row0 + 16 * (u / NT), tile0 + u % NT, lane, sum) << (4 * u);
  }
  repair<T, GROUP, ZEROS, NT>(a, bad, row0, tile0, lane);
}

// More than 16 rows: a workgroup of WN x WK waves takes 16 MT rows and 16 NT WN
// outputs, wave (wn, wk) NT n tiles and one of every WK k tiles. A step's
// activations (WK tiles of 16 MT rows x 256 bytes) go straight into LDS one step
// before they are used, into the other of two buffers; its weights into registers
// (two and three steps ahead measured the same). Unit u (16 bytes) of a row sits at place u ^ (row mod 16),
// so that the A operand's reads (16 rows' same unit) lie in different banks.
template <typename T, int GROUP, bool ZEROS, int MT, int NT, int WN, int WK>
__global__ __launch_bounds__(64 * WN * WK) __attribute__((amdgpu_waves_per_eu(MT > 2 ? 2 : 4))) void
int4_rows_kernel(Int4Args a) {
  typedef Tiles<GROUP, ZEROS, NT> Weights;
  constexpr int kWaves = WN * WK;
  constexpr int kTileBytes = 16 * MT * 256;
  constexpr int kStageBytes = WK * kTileBytes;
  constexpr int kBlocks = WK * 16 * MT / 4;  // 4 rows of 256 bytes an instruction
  static_assert(kBlocks % kWaves == 0, "");
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int wn = wave % WN, wk = wave / WN;
  // Row blocks of the same outputs are 8 blocks apart: one XCD, whose L2 then
  // serves the weight to all but the first.
  const int slot = (int)(blockIdx.x / (8 * a.row_blocks)) * 8 + (int)(blockIdx.x & 7);
  const int row0 = ((int)(blockIdx.x >> 3) % a.row_blocks) * (16 * MT);
  const int tile0 = (slot * WN + wn) * NT;
  if (slot * WN * NT >= a.n_tiles) return;
  const int steps = (a.k_tiles + WK - 1) / WK;

  const char* const zero = reinterpret_cast<const char*>(g_qsa_zero_rows);
  const char* const xbase = reinterpret_cast<const char*>(a.x + row0 * a.x_row);
  // Block i of a step (4 rows of tile i / (4 MT)) is moved by wave i mod waves;
  // the lane's byte offset in its blocks. Rows past the last repeat it (their
  // results are not stored).
  uint32_t at[kBlocks / kWaves];
#pragma unroll
  for (int i = 0; i < kBlocks / kWaves; ++i) {
    const int row = (i * kWaves + wave) % (4 * MT) * 4 + g;
    at[i] = (uint32_t)min(row, a.rows - 1 - row0) * (uint32_t)(2 * a.x_row) +
            (uint32_t)(n ^ (row & 15)) * 16;
  }
  // Loads past the last step repeat it: none depends on a condition.
  auto load_step = [&](int step, char* stage, Weights& b) {
    const int s = min(step, steps - 1);
    auto move = [&](int i, const char* src) {
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)src,
          (__attribute__((address_space(3))) void*)(stage + (i * kWaves + wave) * 1024), 16, 0, 0);
    };
    const char* const base = xbase + (int64_t)s * (2 * WK * kTileK);
    if ((s + 1) * WK * kTileK <= a.k) {
#pragma unroll
      for (int i = 0; i < kBlocks / kWaves; ++i)
        move(i, base + (i * kWaves + wave) / (4 * MT) * (2 * kTileK) + at[i]);
    } else {  // inputs past the width are zero
#pragma unroll
      for (int i = 0; i < kBlocks / kWaves; ++i) {
        const int block = i * kWaves + wave, tile = block / (4 * MT);
        const int k = (s * WK + tile) * kTileK + (n ^ ((block % (4 * MT) * 4 + g) & 15)) * 8;
        move(i, k < a.k ? base + tile * (2 * kTileK) + at[i] : zero);
      }
    }
    b.load(a, tile0, min(s * WK + wk, a.k_tiles - 1), lane);
  };

  f32x4 acc[MT][NT] = {};
  Weights b[2];
  load_step(0, lds, b[0]);
  for (int step = 0;; step += 2) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (step + i >= steps) goto done;
      // This step's loads are done, and the buffer that the next loads go to
      // has been read by all.
      __builtin_amdgcn_s_waitcnt(kMemoryDone);
      __syncthreads();
      load_step(step + i + 1, lds + (1 - i) * kStageBytes, b[1 - i]);
      if ((step + i) * WK + wk >= a.k_tiles) continue;
      const char* const tile = lds + i * kStageBytes + wk * kTileBytes;
      u32x4 x[MT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[m][j] = load_u32x4(tile + (16 * m + n) * 256 + ((4 * j + g) ^ n) * 16);
      multiply<T, GROUP, ZEROS, MT, NT>(x, b[i], acc);
    }
  }
done:
  __builtin_amdgcn_s_waitcnt(kMemoryDone);  // no load into LDS outlives the wave

  static_assert(4 * MT * NT <= 64, "a bit for each of a lane's results");
  uint64_t bad = 0;
  if constexpr (WK > 1) {
    f32x4* const part = reinterpret_cast<f32x4*>(lds);  // [WK][WN][MT * NT][64]
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int v = 0; v < NT; ++v)
        part[((wk * WN + wn) * MT * NT + i * NT + v) * 64 + lane] = acc[i][v];
    __syncthreads();
    for (int u = wk; u < MT * NT; u += WK) {
      f32x4 sum = part[(wn * MT * NT + u) * 64 + lane];
#pragma unroll
      for (int o = 1; o < WK; ++o) sum += part[((o * WN + wn) * MT * NT + u) * 64 + lane];
      if (tile0 + u % NT < a.n_tiles)
        bad |= (uint64_t)store<T>(a, row0 + 16 * (u / NT), tile0 + u % NT, lane, sum) << (4 * u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int v = 0; v < NT; ++v)
        if (tile0 + v < a.n_tiles)
          bad |= (uint64_t)store<T>(a, row0 + 16 * i, tile0 + v, lane, acc[i][v])
                 << (4 * (i * NT + v));
  }
  repair<T, GROUP, ZEROS, NT>(a, bad, row0, tile0, lane);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// What a launch of more than 2^32 - 1 threads is refused with.
constexpr hipError_t kTooLarge = hipErrorInvalidConfiguration;
bool fits(int64_t blocks, int threads) { return blocks <= UINT_MAX / (unsigned)threads; }

template <typename T, int GROUP, bool ZEROS, int MT, int NT, bool VEC>
hipError_t launch_few(Int4Args a, int waves, hipStream_t stream) {
  waves = std::min(waves, a.k_tiles);
  a.row_blocks = (a.rows - 1) / (16 * MT) + 1;
  const int64_t grid = (int64_t)a.row_blocks * ((a.n_tiles - 1) / NT + 1);
  if (!fits(grid, 64 * waves)) return kTooLarge;
  hipLaunchKernelGGL((int4_linear_kernel<T, GROUP, ZEROS, MT, NT, VEC>), dim3((unsigned)grid),
                     dim3(64 * waves), (size_t)waves * MT * NT * 64 * sizeof(f32x4), stream, a);
  return hipGetLastError();
}

template <typename T, int GROUP, bool ZEROS, int MT, int NT, int WN, int WK>
hipError_t launch_many(Int4Args a, hipStream_t stream) {
  constexpr size_t kLds = std::max<size_t>((size_t)2 * WK * 16 * MT * 256,
                                           WK > 1 ? (size_t)WK * WN * MT * NT * 1024 : 0);
  static_assert(kLds <= 65536, "two workgroups a CU, and no attribute to set");
  auto* kernel = &int4_rows_kernel<T, GROUP, ZEROS, MT, NT, WN, WK>;
  a.row_blocks = (a.rows - 1) / (16 * MT) + 1;
  const int64_t n_blocks = (a.n_tiles - 1) / (NT * WN) + 1;
  const int64_t grid = (n_blocks + 7) / 8 * 8 * a.row_blocks;
  if (!fits(grid, 64 * WN * WK)) return kTooLarge;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * WN * WK), kLds, stream, a);
  return hipGetLastError();
}

// More than 16 rows: workgroups of 16 MT rows x 16 NT WN outputs. Time goes by
// how many of them a CU gets: one costs `one`, two at a time `two` (us at 4096
// inputs, in proportion to them otherwise; measured at 17 - 256 rows, 2048 -
// 49536 outputs, groups of 128):
//   rows x outputs     32 x 32   32 x 64   32 x 96   64 x 128   64 x 192
//   one / two a CU    8.3/12.5   10.1/16  12.3/20.5  28.5/45     35/58
// A larger block unpacks each weight for more rows and loads less, a smaller
// one fills the card sooner: the least max(one, two ceil(blocks / CUs) / 2).
// Groups of 128 in fp16 take about the same times. Zero points cost the 32 x 96 blocks
// more than the others (us, 32 x 64 / 32 x 96 / 64 x 128 at 4096 inputs, groups of
// 64: 61 rows x 11264 18.0 / 20.8 / 31.7, 61 x 22528 26.9 / 30.6 / 32.1, 17 x 49536
// 37.3 / 54.4 / 48.6; groups of 32: 61 x 22528 29.3 / 32.0 / 35.9), which this rule
// does not know: it takes 32 x 96 in these four.
enum RowsShape { k32x32, k32x64, k32x96, k64x128, k64x192, kRowsShapes };
RowsShape pick_rows_shape(int rows, int n_tiles) {
  static constexpr struct {
    int rows, tiles;
    float one, two;
  } kShapes[kRowsShapes] = {
      {32, 2, 8.3f, 12.5f}, {32, 4, 10.1f, 16.0f}, {32, 6, 12.3f, 20.5f}, {64, 8, 28.5f, 45.0f},
      {64, 12, 35.0f, 58.0f}};
  int best = 0;
  float least = 0.0f;
  for (int i = 0; i < kRowsShapes; ++i) {
    const int64_t blocks = (int64_t)((rows - 1) / kShapes[i].rows + 1) *
                           ((n_tiles - 1) / kShapes[i].tiles + 1);
    const float us = std::max(kShapes[i].one,
                              kShapes[i].two * 0.5f * (float)((blocks + kCUs - 1) / kCUs));
    if (i == 0 || us < least) {
      best = i;
      least = us;
    }
  }
  return (RowsShape)best;
}

template <typename T, int GROUP, bool ZEROS>
hipError_t launch_rows(const Int4Args& a, bool vec, hipStream_t stream) {
  // Rows that no 16-byte load can take, element by element (11264 x 4095 at 1 / 16 /
  // 61 / 250 rows 21 / 60 / 215 / 829 us; 11264 x 4096 7.5 / 9.9 / 13.7 / 38).
  if (!vec)
    return a.rows <= 16 ? launch_few<T, GROUP, ZEROS, 1, 1, false>(a, 8, stream)
                        : launch_few<T, GROUP, ZEROS, 2, 1, false>(a, 8, stream);
  // To 16 rows: more outputs a wave (and fewer waves) share the activations'
  // loads and the closing sum, once there are enough of them for every CU
  // (K = 4096, us for 1 / 2 / 4 n tiles a wave. 1 row: 11264 outputs 7.1 / 8.0 /
  // 8.4, 22528 11.8 / 10.8 / 12.0, 49536 28.4 / 21.9 / 22.5; 16 rows: 2048
  // 6.7 / 7.0 / 8.3, 8832 14.5 / 11.2 / 9.2, 49536 52 / 35 / 28. In between, groups
  // of 32 with zero points: 7 rows x 11264 11.1 / 10.9 / 12.1, x 22528 18.2 / 14.1 / 16.5).
  if (a.rows <= 4)
    return a.n_tiles < 1024 ? launch_few<T, GROUP, ZEROS, 1, 1, true>(a, 8, stream)
                            : launch_few<T, GROUP, ZEROS, 1, 2, true>(a, 4, stream);
  if (a.rows <= 16)
    return a.n_tiles < 384 ? launch_few<T, GROUP, ZEROS, 1, 1, true>(a, 8, stream)
                           : launch_few<T, GROUP, ZEROS, 1, 4, true>(a, 4, stream);
  switch (pick_rows_shape(a.rows, a.n_tiles)) {
    case k32x32: return launch_many<T, GROUP, ZEROS, 2, 1, 2, 4>(a, stream);
    case k32x64: return launch_many<T, GROUP, ZEROS, 2, 2, 2, 4>(a, stream);
    case k32x96: return launch_many<T, GROUP, ZEROS, 2, 3, 2, 4>(a, stream);
    case k64x128: return launch_many<T, GROUP, ZEROS, 4, 2, 4, 1>(a, stream);
    default: return launch_many<T, GROUP, ZEROS, 4, 3, 4, 1>(a, stream);
  }
}

template <template <bool> class T, int GROUP>
hipError_t launch_zeros(const Int4Args& a, bool vec, hipStream_t stream) {
  return a.zeros ? launch_rows<T<true>, GROUP, true>(a, vec, stream)
                 : launch_rows<T<false>, GROUP, false>(a, vec, stream);
}

template <template <bool> class T>
hipError_t launch(const Int4Args& a, int group, bool vec, hipStream_t stream) {
  if (group == 32) return launch_zeros<T, 32>(a, vec, stream);
  if (group == 64) return launch_zeros<T, 64>(a, vec, stream);
  return launch_zeros<T, 128>(a, vec, stream);
}

bool aligned(const void* p, uintptr_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

}  // namespace
}  // namespace qsa

using namespace qsa;

extern "C" int qsa_int4_linear(const void* x, int64_t x_row_stride, const void* codes,
                               const void* scales, const void* zeros, const void* bias, void* y,
                               int64_t y_row_stride, int rows, int out_features, int in_features,
                               int group_size, int is_fp16, void* stream) {
  const char* name = "qsa_int4_linear";
  if (rows < 0 || out_features < 0 || in_features < 0 || x_row_stride < 0 || y_row_stride < 0)
    return fail(QSA_ERR_INVALID, std::string(name) + ": negative size or stride");
  if (group_size != 32 && group_size != 64 && group_size != 128)
    return fail(QSA_ERR_UNSUPPORTED, std::string(name) + ": group size must be 32, 64 or 128");
  if (rows == 0 || out_features == 0) return QSA_OK;
  if (in_features == 0)
    return fail(QSA_ERR_UNSUPPORTED, std::string(name) + ": no input features");
  if (!x || !codes || !scales || !y)
    return fail(QSA_ERR_INVALID, std::string(name) + ": null tensor pointer");
  if (!aligned(codes, 16) || !aligned(x, 2) || !aligned(scales, 8) || !aligned(zeros, 4) || !aligned(bias, 2) ||
      !aligned(y, 2))
    return fail(QSA_ERR_INVALID, std::string(name) + ": misaligned tensor");
  if (rows > 1 && y_row_stride < out_features)
    return fail(QSA_ERR_INVALID, std::string(name) + ": output rows overlap");
  Int4Args a = {};
  a.x = static_cast<const uint16_t*>(x);
  a.x_row = x_row_stride;
  a.codes = static_cast<const u32x4*>(codes);
  a.scales = static_cast<const char*>(scales);
  a.zeros = static_cast<const char*>(zeros);
  a.bias = static_cast<const uint16_t*>(bias);
  a.y = static_cast<uint16_t*>(y);
  a.y_row = y_row_stride;
  a.rows = rows;
  a.n = out_features;
  a.k = in_features;
  a.n_tiles = (int)(((int64_t)out_features + kTileN - 1) / kTileN);
  a.k_tiles = (int)(((int64_t)in_features + kTileK - 1) / kTileK);
  // The kernels count rows and outputs in 32 bits, to the end of the last block.
  if (rows > INT_MAX - 64 || out_features > INT_MAX - 256)
    return fail(QSA_ERR_UNSUPPORTED, std::string(name) + ": too many rows or outputs");
  if (in_features > (1 << 30) || x_row_stride > INT64_MAX / 4 / rows)
    return fail(QSA_ERR_UNSUPPORTED, std::string(name) + ": at most 2^30 inputs, rows within 2^62");
  // 16-byte loads of whole rows, whose offsets within a block fit 32 bits.
  const bool vec = aligned(x, 16) && x_row_stride % 8 == 0 && in_features % 8 == 0 &&
                   x_row_stride < (1 << 24);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t err = is_fp16 ? launch<Fp16>(a, group_size, vec, s)
                                 : launch<Bf16>(a, group_size, vec, s);
  if (err == kTooLarge)
    return fail(QSA_ERR_UNSUPPORTED, std::string(name) + ": too many rows and outputs");
  if (err != hipSuccess)
    return fail(QSA_ERR_HIP, std::string(name) + " launch: " + hipGetErrorString(err));
  return QSA_OK;
}

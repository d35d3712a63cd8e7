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
// becomes 128 + q by one and-or (bf16 holds whole numbers to 256), and
//   sum x (q - z) = sum x (128 + q) - (128 + z) sum x,
// with sum x from the same matrix instruction against ones; both in fp32, whose
// step is 2^-15 of bf16's. With fp16 the code becomes 1024 + q (or 1024 + 16 q)
// and one packed add (or fma) gives q - z exactly.
//
// Layout. Weights are stored in tiles of 16 outputs x 128 inputs, 1 KiB each:
// lane (n, g) of a wave holds output n's codes of inputs 32 j + 8 g .. + 7 as
// word j, the B operand of mfma_f32_16x16x32 after unpacking, element 2 p of a
// word in bits 4 p and element 2 p + 1 in bits 16 + 4 p. So a wave reads a tile
// with one 16-byte load a lane, and unpacking is shifts and and-ors alone.
//
// Work. A workgroup owns 16 NT outputs and 16 MT rows; its waves share the
// inputs, tile t going to wave t mod waves, and add their sums through LDS in
// wave order (no atomics, the same bits every time). Each weight is read once
// per block of 16 MT rows.
#include "qsa_common.h"
#include "../../include/qsa_hip.h"

#include <algorithm>

namespace qsa {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kTileN = 16;
constexpr int kTileK = 128;

struct Int4Args {
  const uint16_t* x;
  int64_t x_row;
  const u32x4* codes;       // [n tiles][k tiles][64 lanes]
  const uint16_t* scales;   // [n tiles][groups][16]
  const uint8_t* zeros;     // [n tiles][groups][16] or null
  const uint16_t* bias;     // [n] or null
  uint16_t* y;
  int64_t y_row;
  int rows, n, k;
  int n_tiles, k_tiles;
  int row_blocks;
};

struct Bf16 {
  typedef bf16x8 frag;
  static constexpr bool kOffset = true;  // unpacked codes are 128 + q
  static __device__ __forceinline__ f32x4 mfma(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ frag unpack(uint32_t w, int) {
    u32x4 r;
    r[0] = (w & 0x000F000Fu) | 0x43004300u;
    r[1] = ((w >> 4) & 0x000F000Fu) | 0x43004300u;
    r[2] = ((w >> 8) & 0x000F000Fu) | 0x43004300u;
    r[3] = ((w >> 12) & 0x000F000Fu) | 0x43004300u;
    return __builtin_bit_cast(frag, r);
  }
  static __device__ __forceinline__ frag ones() {
    return __builtin_bit_cast(frag, (u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u}));
  }
  static __device__ __forceinline__ float to_float(uint16_t v) {
    return __builtin_bit_cast(float, (uint32_t)v << 16);
  }
  static __device__ __forceinline__ uint16_t from_float(float v) {
    return (uint16_t)pack_bf16x2(v, v);
  }
};

struct Fp16 {
  typedef f16x8 frag;
  static constexpr bool kOffset = false;  // unpacked codes are q - z
  static __device__ __forceinline__ f32x4 mfma(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ frag unpack(uint32_t w, int z) {
    const _Float16 low = (_Float16)(-1024 - z), high = (_Float16)(-64 - z);
    const f16x2 low2 = {low, low}, high2 = {high, high}, sixteenth = {(_Float16)0.0625f,
                                                                      (_Float16)0.0625f};
    union {
      f16x2 p[4];
      frag f;
    } r;
    const uint32_t v = w >> 8;
    r.p[0] = __builtin_bit_cast(f16x2, (w & 0x000F000Fu) | 0x64006400u) + low2;
    r.p[1] = __builtin_elementwise_fma(
        __builtin_bit_cast(f16x2, (w & 0x00F000F0u) | 0x64006400u), sixteenth, high2);
    r.p[2] = __builtin_bit_cast(f16x2, (v & 0x000F000Fu) | 0x64006400u) + low2;
    r.p[3] = __builtin_elementwise_fma(
        __builtin_bit_cast(f16x2, (v & 0x00F000F0u) | 0x64006400u), sixteenth, high2);
    return r.f;
  }
  static __device__ __forceinline__ frag ones() { return frag{}; }  // not used
  static __device__ __forceinline__ float to_float(uint16_t v) {
    return (float)__builtin_bit_cast(_Float16, v);
  }
  static __device__ __forceinline__ uint16_t from_float(float v) {
    return __builtin_bit_cast(uint16_t, (_Float16)v);
  }
};

// Eight activations from input k on: VEC reads 16 bytes (row stride, width and
// address multiples of 8 elements), otherwise element by element. Inputs past
// the width and rows past the last are zero and not read.
template <bool VEC>
__device__ __forceinline__ u32x4 load_x(const uint16_t* row, int k, int width, bool live) {
  if constexpr (VEC) {
    if (live && k < width) return load_u32x4(row + k);
    return u32x4{0, 0, 0, 0};
  } else {
    u32x4 r = {0, 0, 0, 0};
    if (live) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < width) r[i / 2] |= (uint32_t)row[k + i] << (16 * (i & 1));
    }
    return r;
  }
}

template <typename T, int GROUP, bool ZEROS, int MT, int NT, bool VEC>
__global__ __launch_bounds__(512) void int4_linear_kernel(Int4Args a) {
  constexpr int kGroups = kTileK / GROUP;  // per k tile
  constexpr int kSteps = GROUP / 32;       // matrix instructions per group
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int n = lane & 15, g = lane >> 4;
  const int row0 = (blockIdx.x % a.row_blocks) * (16 * MT);
  const int tile0 = (blockIdx.x / a.row_blocks) * NT;

  f32x4 acc[MT][NT] = {};
  const uint16_t* xrow[MT];
  bool live[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = row0 + 16 * i + n;
    live[i] = m < a.rows;
    xrow[i] = a.x + (live[i] ? m : 0) * a.x_row;
  }
  const int64_t groups = (int64_t)a.k_tiles * kGroups;

  for (int t = wave; t < a.k_tiles; t += waves) {
    u32x4 w[NT];
    uint16_t s[NT][kGroups];
    uint8_t z[NT][kGroups];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int64_t tile = min(tile0 + j, a.n_tiles - 1);
      w[j] = a.codes[(tile * a.k_tiles + t) * 64 + lane];
#pragma unroll
      for (int q = 0; q < kGroups; ++q) {
        const int64_t at = (tile * groups + (int64_t)t * kGroups + q) * 16 + n;
        s[j][q] = a.scales[at];
        z[j][q] = ZEROS ? a.zeros[at] : 8;
      }
    }
    u32x4 x[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[i][j] = load_x<VEC>(xrow[i], t * kTileK + 32 * j + 8 * g, a.k, live[i]);

#pragma unroll
    for (int q = 0; q < kGroups; ++q) {
      f32x4 total[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        total[i] = f32x4{0, 0, 0, 0};
        if constexpr (T::kOffset) {
#pragma unroll
          for (int j = 0; j < kSteps; ++j)
            total[i] = T::mfma(__builtin_bit_cast(typename T::frag, x[i][q * kSteps + j]),
                               T::ones(), total[i]);
        }
      }
#pragma unroll
      for (int v = 0; v < NT; ++v) {
        const float scale = T::to_float(s[v][q]);
        const float offset = -(float)(128 + z[v][q]);
        f32x4 d[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          d[i] = f32x4{0, 0, 0, 0};
          if constexpr (T::kOffset) {
#pragma unroll
            for (int r = 0; r < 4; ++r) d[i][r] = offset * total[i][r];
          }
        }
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          const typename T::frag b = T::unpack(w[v][q * kSteps + j], z[v][q]);
#pragma unroll
          for (int i = 0; i < MT; ++i)
            d[i] = T::mfma(__builtin_bit_cast(typename T::frag, x[i][q * kSteps + j]), b, d[i]);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][v][r] = __builtin_fmaf(scale, d[i][r], acc[i][v][r]);
      }
    }
  }

  // The waves' sums, in wave order. A lane's accumulators are rows 4 g + r of
  // output n.
  extern __shared__ f32x4 part[];  // [waves][MT * NT][64]
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int v = 0; v < NT; ++v) part[(wave * MT * NT + i * NT + v) * 64 + lane] = acc[i][v];
  __syncthreads();
  for (int u = wave; u < MT * NT; u += waves) {
    f32x4 sum = part[u * 64 + lane];
    for (int o = 1; o < waves; ++o) sum += part[(o * MT * NT + u) * 64 + lane];
    const int col = (tile0 + u % NT) * kTileN + n;
    if (col < a.n) {
      const float b = a.bias ? T::to_float(a.bias[col]) : 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = row0 + 16 * (u / NT) + 4 * g + r;
        if (m < a.rows) a.y[m * a.y_row + col] = T::from_float(sum[r] + b);
      }
    }
  }
}

template <typename T, int GROUP, bool ZEROS, int MT, int NT>
void launch_vec(const Int4Args& a, bool vec, unsigned grid, int waves, hipStream_t stream) {
  const size_t lds = (size_t)waves * MT * NT * 64 * sizeof(f32x4);
  if (vec)
    hipLaunchKernelGGL((int4_linear_kernel<T, GROUP, ZEROS, MT, NT, true>), dim3(grid),
                       dim3(64 * waves), lds, stream, a);
  else
    hipLaunchKernelGGL((int4_linear_kernel<T, GROUP, ZEROS, MT, NT, false>), dim3(grid),
                       dim3(64 * waves), lds, stream, a);
}

template <typename T, int GROUP, bool ZEROS>
void launch_rows(Int4Args a, bool vec, hipStream_t stream) {
  const int waves = std::min(8, a.k_tiles);
  auto grid = [&](int mt, int nt) {
    a.row_blocks = (a.rows + 16 * mt - 1) / (16 * mt);
    return (unsigned)((int64_t)a.row_blocks * ((a.n_tiles + nt - 1) / nt));
  };
  if (a.rows <= 16)
    launch_vec<T, GROUP, ZEROS, 1, 1>(a, vec, grid(1, 1), waves, stream);
  else if (a.rows <= 32)
    launch_vec<T, GROUP, ZEROS, 2, 1>(a, vec, grid(2, 1), waves, stream);
  else
    launch_vec<T, GROUP, ZEROS, 4, 2>(a, vec, grid(4, 2), waves, stream);
}

template <typename T>
void launch(const Int4Args& a, int group, bool vec, hipStream_t stream) {
  if (group == 32)
    a.zeros ? launch_rows<T, 32, true>(a, vec, stream) : launch_rows<T, 32, false>(a, vec, stream);
  else if (group == 64)
    a.zeros ? launch_rows<T, 64, true>(a, vec, stream) : launch_rows<T, 64, false>(a, vec, stream);
  else
    a.zeros ? launch_rows<T, 128, true>(a, vec, stream) : launch_rows<T, 128, false>(a, vec, stream);
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
  if (!aligned(codes, 16) || !aligned(x, 2) || !aligned(scales, 2) || !aligned(bias, 2) ||
      !aligned(y, 2))
    return fail(QSA_ERR_INVALID, std::string(name) + ": misaligned tensor");
  if (rows > 1 && y_row_stride < out_features)
    return fail(QSA_ERR_INVALID, std::string(name) + ": output rows overlap");
  Int4Args a = {};
  a.x = static_cast<const uint16_t*>(x);
  a.x_row = x_row_stride;
  a.codes = static_cast<const u32x4*>(codes);
  a.scales = static_cast<const uint16_t*>(scales);
  a.zeros = static_cast<const uint8_t*>(zeros);
  a.bias = static_cast<const uint16_t*>(bias);
  a.y = static_cast<uint16_t*>(y);
  a.y_row = y_row_stride;
  a.rows = rows;
  a.n = out_features;
  a.k = in_features;
  a.n_tiles = (int)(((int64_t)out_features + kTileN - 1) / kTileN);
  a.k_tiles = (int)(((int64_t)in_features + kTileK - 1) / kTileK);
  if ((int64_t)a.n_tiles * ((rows + 15) / 16) > 0x7fffffffLL / 2)
    return fail(QSA_ERR_UNSUPPORTED, std::string(name) + ": too many output tiles");
  const bool vec = aligned(x, 16) && x_row_stride % 8 == 0 && in_features % 8 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (is_fp16) launch<Fp16>(a, group_size, vec, s);
  else launch<Bf16>(a, group_size, vec, s);
  return check_launch(name);
}

// Attention of drafted token trees over the paged cache, gfx950.
//
// Request b has c committed tokens (cache positions 0 .. c - 1) and T drafted
// ones (positions c .. c + T - 1, in the order of their query rows). Row i
// attends over every committed position and over drafted position c + j where
// bit j of the row's ancestor words is set:
//
//   o = sum_p e^{s_p - m} v_p / sum_p e^{s_p - m},   s_p = q . k_p / sqrt(D)
//
// in one pass with a running maximum and sum, then sigmoid(gate) if given. A
// row that sees nothing gets zeros.
//
// Unlike the sparse attention, where each row gathers its own slots, the rows
// of a request share their K/V: a workgroup takes a tile of (node, head) rows
// of one kv head and streams a chunk of the request's tokens through LDS once
// for all of them.
//
//   S^T[token][row] = K (A, 16 tokens x 32 dims) Q^T (B, 32 dims x 16 rows)
//   O^T[dim][row]  += V^T (A, 16 dims x 32 tokens) P^T (B, 32 tokens x 16 rows)
//
// on mfma_f32_16x16x32_bf16. P^T is the lane's own exponentials (rounded to
// bf16, the matrix cores' type, as in the sparse attention: 2^-9 of a weight at
// most, of random sign; their sum is taken in fp32 before rounding), so
// it never leaves registers; V^T comes from row-major V rows in LDS by the
// transposing LDS read.
//
// Rows and tokens are shared out over the four waves as WM x WT: with many rows
// each wave has its own 16 NB rows and all tokens of a stage, with few rows the
// waves take different tokens and merge (max, sum, O) through LDS at the end.
//
// A long context is cut into chunks of whole stages, a workgroup each, whose
// normalised fp32 results and log2 sums a second kernel joins in chunk order.
#include "qsa_common.h"
#include "../../include/qsa_hip.h"

#include <algorithm>
#include <climits>

namespace qsa {
namespace {

constexpr int kWaves = 4;
constexpr int kCUs = 256;
constexpr float kNegInf = -__builtin_huge_valf();

typedef short s16x4 __attribute__((ext_vector_type(4)));

struct TreeArgs {
  const uint16_t* q;
  int64_t q_row, q_head;  // elements
  const char* k;
  const char* v;
  int64_t kb, kt, kh, vb, vt, vh;  // bytes
  int num_blocks;
  int page_size;
  FastDiv page_div;
  const int32_t* table;
  int64_t table_row;
  int table_width;
  int requests;
  const int32_t* context_lens;
  const int32_t* query_start_loc;
  const int32_t* ancestors;
  int64_t ancestor_row;
  int words;
  uint16_t* out;
  int64_t out_row, out_head;
  const uint16_t* gate;
  int64_t g_row, g_head, g_dim;
  float* part_out;  // [rows][q heads][splits][D]
  float* part_lse;  // [rows][q heads][splits]
  int rows, num_q_heads, kv_heads, group;
  FastDiv group_div;
  int m_tiles, splits, chunk;
  float scale_log2;
};

// One request's rows and tokens, kept within the query tensor and the page
// table whatever the device arrays say.
struct Request {
  int row0, nodes, context, length;
};
__device__ __forceinline__ Request load_request(const TreeArgs& a, int b) {
  Request r;
  const int first = load_uniform(a.query_start_loc + b);
  const int last = load_uniform(a.query_start_loc + b + 1);
  r.row0 = min(max(first, 0), a.rows);
  r.nodes = min(max(last, r.row0), a.rows) - r.row0;
  const int64_t capacity = min((int64_t)a.table_width * a.page_size, (int64_t)INT_MAX / 2);
  r.context = (int)min((int64_t)max(load_uniform(a.context_lens + b), 0), capacity);
  r.length = (int)min((int64_t)r.context + r.nodes, capacity);
  return r;
}

__device__ __forceinline__ float gate_factor(uint16_t g) {
  return 1.0f / (1.0f + __expf(-__builtin_bit_cast(float, (uint32_t)g << 16)));
}

// Byte offset of 16-byte unit `unit` of token `tok`'s row in a K stage: units
// are permuted by the token so that 16 tokens' same unit (the A operand's
// read) lie in different banks.
template <int D>
__device__ __forceinline__ int k_at(int tok, int unit) {
  constexpr int U = D / 8;
  const int swizzle = D == 128 ? tok & 15 : (tok >> 1) & 7;
  return (tok * U + (unit ^ swizzle)) * 16;
}
// The same for V, permuted in 32-byte units (what the transposing read takes
// of a token).
template <int D>
__device__ __forceinline__ int v_at(int tok, int unit) {
  constexpr int U = D / 8;
  const int swizzle = D == 128 ? (tok & 7) << 1 : ((tok >> 1) & 3) << 1;
  return (tok * U + (unit ^ swizzle)) * 16;
}

template <int D, int NB, int WM, int WT>
struct Shape {
  static constexpr int kRows = 16 * NB * WM;          // query rows of a workgroup
  static constexpr int kTok = 32 * WT < 64 ? 64 : 32 * WT;  // tokens of a stage
  static constexpr int kWaveTok = kTok / WT;
  static constexpr int kSub = kWaveTok / 16;          // 16-token subtiles of a wave
  static constexpr int kLoads = kTok * (D / 8) / (64 * kWaves);  // 16-byte loads of a lane
  static constexpr size_t kStage = (size_t)kTok * D * 2;
  // K and V stages; afterwards the waves' partial results.
  static constexpr size_t kMerge = (size_t)kWaves * 16 * NB * (D + 2) * 4;
  static constexpr size_t kLds = 2 * kStage > kMerge ? 2 * kStage : kMerge;
};

template <int D, int NB, int WM, int WT>
__global__ __launch_bounds__(64 * kWaves) void tree_attn_kernel(TreeArgs a) {
  typedef Shape<D, NB, WM, WT> S;
  constexpr int U = D / 8;       // 16-byte units of a row
  constexpr int kSteps = D / 32;
  constexpr int kDims = D / 16;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char* const k_lds = lds;
  char* const v_lds = lds + S::kStage;

  int block = blockIdx.x;
  const int split = block % a.splits;
  block /= a.splits;
  const int m_tile = block % a.m_tiles;
  block /= a.m_tiles;
  const int kv = block % a.kv_heads;
  const Request rq = load_request(a, block / a.kv_heads);
  const int32_t* const trow = a.table + (block / a.kv_heads) * a.table_row;
  const int rows = rq.nodes * a.group;
  const int m0 = m_tile * S::kRows;
  const int t_begin = split * a.chunk;
  if (m0 >= rows || (split > 0 && t_begin >= rq.length)) return;
  // The last chunk takes whatever is left (a context longer than was said).
  const int t_end = split + 1 == a.splits ? rq.length : min(rq.length, t_begin + a.chunk);

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = lane & 15, g = lane >> 4;
  const int wm = wave / WT, wt = wave % WT;

  // Query rows: lane n's row of each 16-row block, dims 32 s + 8 g .. + 7.
  bf16x8 q[NB][kSteps];
  int node[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int m = min(m0 + (wm * NB + i) * 16 + n, rows - 1);
    node[i] = rq.row0 + a.group_div.div(m);
    const int head = kv * a.group + m - (node[i] - rq.row0) * a.group;
    const uint16_t* src = a.q + node[i] * a.q_row + head * a.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      q[i][s] = __builtin_bit_cast(bf16x8, load_u32x4(src + 32 * s + 8 * g));
  }

  const char* const kbase = a.k + kv * a.kh;
  const char* const vbase = a.v + kv * a.vh;
  const char* const zero = reinterpret_cast<const char*>(g_qsa_zero_rows);

  // A stage's K and V rows, one stage ahead in registers. Tokens past the end
  // or without a page in the cache read zeros and are left out of `valid`.
  u32x4 kr[S::kLoads], vr[S::kLoads];
  uint64_t valid_next[S::kTok / 64], valid[S::kTok / 64];
  auto load_stage = [&](int t) {
    int page[S::kTok / 64];
#pragma unroll
    for (int w = 0; w < S::kTok / 64; ++w) {
      const int pos = t + 64 * w + lane;
      page[w] = pos < t_end ? trow[a.page_div.div(pos)] : -1;
      if (page[w] >= a.num_blocks) page[w] = -1;
      valid_next[w] = __ballot(page[w] >= 0);
    }
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int item = (i * kWaves + wave) * 64 + lane;
      const int tok = item / U, unit = item % U;
      const int pos = t + tok;
      const int mine = __shfl(page[i * kWaves / U], tok & 63, 64);
      const int64_t off = pos - a.page_div.div(pos) * a.page_size;
      const char* ks = mine >= 0 ? kbase + mine * a.kb + off * a.kt + unit * 16 : zero;
      const char* vs = mine >= 0 ? vbase + mine * a.vb + off * a.vt + unit * 16 : zero;
      kr[i] = load_u32x4(ks);
      vr[i] = load_u32x4(vs);
    }
  };

  f32x4 o[NB][kDims];
  float top[NB], sum[NB];  // running maximum (log2 domain) and the lane's share of the sum
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    top[i] = kNegInf;
    sum[i] = 0.0f;
#pragma unroll
    for (int d = 0; d < kDims; ++d) o[i][d] = f32x4{0, 0, 0, 0};
  }

  if (t_begin < t_end) load_stage(t_begin);
  for (int t = t_begin; t < t_end; t += S::kTok) {
    __syncthreads();  // the last stage has been read
    // A drafted token's V may hold infinities or NaN that a row outside its
    // branch must not see (0 times them is NaN): such stages, rare, multiply
    // element by element below.
    bool bad = false;
    const bool drafted = t + S::kTok > rq.context;
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int item = (i * kWaves + wave) * 64 + lane;
      const int tok = item / U, unit = item % U;
      *reinterpret_cast<u32x4*>(k_lds + k_at<D>(tok, unit)) = kr[i];
      *reinterpret_cast<u32x4*>(v_lds + v_at<D>(tok, unit)) = vr[i];
      if (drafted) {
#pragma unroll
        for (int w = 0; w < 4; ++w)
          bad |= (vr[i][w] & 0x7F80u) == 0x7F80u || (vr[i][w] & 0x7F800000u) == 0x7F800000u;
      }
    }
#pragma unroll
    for (int w = 0; w < S::kTok / 64; ++w) valid[w] = valid_next[w];
    if (t + S::kTok < t_end) load_stage(t + S::kTok);
    if (drafted) bad = __syncthreads_or(bad);
    else __syncthreads();

    const int first = wt * S::kWaveTok;  // the wave's tokens of the stage
    f32x4 sc[NB][S::kSub];
#pragma unroll
    for (int u = 0; u < S::kSub; ++u) {
      bf16x8 kf[kSteps];
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        kf[s] = __builtin_bit_cast(
            bf16x8, *reinterpret_cast<const u32x4*>(k_lds + k_at<D>(first + 16 * u + n, 4 * s + g)));
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        sc[i][u] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
          sc[i][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[s], q[i][s], sc[i][u], 0, 0, 0);
      }
    }

    // Scores in the log2 domain; masked ones are replaced, whatever they hold.
    uint32_t seen[NB];
    bool all = !drafted;
#pragma unroll
    for (int w = 0; w < S::kTok / 64; ++w) all = all && valid[w] == ~0ull;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      seen[i] = ~0u;
#pragma unroll
      for (int u = 0; u < S::kSub; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float s = sc[i][u][r] * a.scale_log2;
          if (!all) {
            const int tok = first + 16 * u + 4 * g + r;
            const int j = t + tok - rq.context;
            bool ok = (valid[tok / 64] >> (tok & 63)) & 1;
            if (j >= 0 && ok)
              ok = j < 32 * a.words &&
                   ((uint32_t)a.ancestors[node[i] * a.ancestor_row + (j >> 5)] >> (j & 31)) & 1u;
            if (!ok) {
              s = kNegInf;
              seen[i] &= ~(1u << (4 * u + r));
            }
          }
          sc[i][u][r] = s;
        }
    }

    bf16x8 p[NB][S::kSub / 2];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      float m = top[i];
#pragma unroll
      for (int u = 0; u < S::kSub; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) m = fmaxf(m, sc[i][u][r]);
      m = fmaxf(m, shfl_xor_f(m, 16));
      m = fmaxf(m, shfl_xor_f(m, 32));
      const float base = m == kNegInf ? 0.0f : m;
      const float shrink = fast_exp2(top[i] - base);
      top[i] = m;
      float add = 0.0f;
#pragma unroll
      for (int h = 0; h < S::kSub / 2; ++h) {
        u32x4 packed;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float e[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            e[r] = fast_exp2(sc[i][2 * h + u][r] - base);
            add += e[r];
          }
          packed[2 * u] = pack_bf16x2(e[0], e[1]);
          packed[2 * u + 1] = pack_bf16x2(e[2], e[3]);
        }
        p[i][h] = __builtin_bit_cast(bf16x8, packed);
      }
      sum[i] = sum[i] * shrink + add;
#pragma unroll
      for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[i][d][r] *= shrink;
    }

    if (!(drafted && bad)) {
#pragma unroll
      for (int h = 0; h < S::kSub / 2; ++h)
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          s16x4 part[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int tok = first + 32 * h + 16 * u + 4 * g + (n >> 2);
            part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(
                    v_lds + v_at<D>(tok, 2 * d + ((n & 3) >> 1)) + (n & 1) * 8));
          }
          typedef short s16x8 __attribute__((ext_vector_type(8)));
          const s16x8 joined = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
          for (int i = 0; i < NB; ++i)
            o[i][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8, joined), p[i][h], o[i][d], 0, 0, 0);
        }
    } else {
      for (int c = 0; c < 16 * S::kSub; ++c) {
        // Token c: element (c / 16, c % 4) of the lanes with g = (c % 16) / 4.
        const int tok = first + c;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          float w = 0.0f;
          bool ok = false;
#pragma unroll
          for (int h = 0; h < S::kSub / 2; ++h)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (32 * h + 16 * (e >> 2) + (e & 3) == (c & ~12)) {
                w = (float)p[i][h][e];
                ok = (seen[i] >> (8 * h + e)) & 1u;
              }
          const int from = ((c & 12) << 2) | n;
          w = __shfl(w, from, 64);
          ok = __shfl((int)ok, from, 64);
#pragma unroll
          for (int d = 0; d < kDims; ++d) {
            const u32x2 v = load_u32x2(v_lds + v_at<D>(tok, 2 * d + (g >> 1)) + (g & 1) * 8);
            if (ok) {
              o[i][d][0] += w * bf16_lo(v[0]);
              o[i][d][1] += w * bf16_hi(v[0]);
              o[i][d][2] += w * bf16_lo(v[1]);
              o[i][d][3] += w * bf16_hi(v[1]);
            }
          }
        }
      }
    }
  }

#pragma unroll
  for (int i = 0; i < NB; ++i) {
    sum[i] += shfl_xor_f(sum[i], 16);
    sum[i] += shfl_xor_f(sum[i], 32);
  }

  if constexpr (WT > 1) {
    // The token shares of each row block, joined in wave order by its first wave.
    float* const merge = reinterpret_cast<float*>(lds);
    constexpr int kWave = 16 * NB * (D + 2);
    float* const mine = merge + wave * kWave;
    __syncthreads();
    if (wt > 0) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int d = 0; d < kDims; ++d)
          *reinterpret_cast<f32x4*>(mine + ((i * kDims + d) * 64 + lane) * 4) = o[i][d];
        if (g == 0) {
          mine[16 * NB * D + 16 * i + n] = top[i];
          mine[16 * NB * D + 16 * NB + 16 * i + n] = sum[i];
        }
      }
    }
    __syncthreads();
    if (wt > 0) return;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      float m = top[i];
      for (int w = 1; w < WT; ++w) m = fmaxf(m, mine[w * kWave + 16 * NB * D + 16 * i + n]);
      const float base = m == kNegInf ? 0.0f : m;
      float f = fast_exp2(top[i] - base);
      sum[i] *= f;
#pragma unroll
      for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[i][d][r] *= f;
      for (int w = 1; w < WT; ++w) {
        const float* other = mine + w * kWave;
        f = fast_exp2(other[16 * NB * D + 16 * i + n] - base);
        sum[i] += f * other[16 * NB * D + 16 * NB + 16 * i + n];
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          const f32x4 add = *reinterpret_cast<const f32x4*>(other + ((i * kDims + d) * 64 + lane) * 4);
#pragma unroll
          for (int r = 0; r < 4; ++r) o[i][d][r] += f * add[r];
        }
      }
      top[i] = m;
    }
  }

#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int m = m0 + (wm * NB + i) * 16 + n;
    if (m >= rows) continue;
    const int head = kv * a.group + m - (node[i] - rq.row0) * a.group;
    const float inv = sum[i] == 0.0f ? 0.0f : 1.0f / sum[i];  // a row that sees nothing: zeros
    if (a.splits > 1) {
      const int64_t at = ((int64_t)node[i] * a.num_q_heads + head) * a.splits + split;
#pragma unroll
      for (int d = 0; d < kDims; ++d)
        *reinterpret_cast<f32x4*>(a.part_out + at * D + 16 * d + 4 * g) =
            f32x4{o[i][d][0] * inv, o[i][d][1] * inv, o[i][d][2] * inv, o[i][d][3] * inv};
      if (g == 0) a.part_lse[at] = sum[i] == 0.0f ? kNegInf : top[i] + __log2f(sum[i]);
    } else {
      uint16_t* dst = a.out + node[i] * a.out_row + head * a.out_head;
      const uint16_t* gate = a.gate ? a.gate + node[i] * a.g_row + head * a.g_head : nullptr;
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        float y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          y[r] = o[i][d][r] * inv;
          if (gate) y[r] *= gate_factor(gate[(16 * d + 4 * g + r) * a.g_dim]);
        }
        u32x2 w = {pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
        __builtin_memcpy(dst + 16 * d + 4 * g, &w, 8);
      }
    }
  }
}

// Joins a row's chunks: out = sum_s 2^(lse_s - max) part_s / sum_s 2^(lse_s - max),
// in chunk order. A workgroup per request and group of its rows; D / 4 lanes a
// (row, head).
template <int D>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a, int row_tiles) {
  constexpr int kLanes = D / 4;
  constexpr int kPer = 256 / kLanes;
  const Request rq = load_request(a, blockIdx.x / row_tiles);
  const int64_t item = (int64_t)(blockIdx.x % row_tiles) * kPer + threadIdx.x / kLanes;
  const int64_t node = item / a.num_q_heads;
  if (node >= rq.nodes) return;
  const int head = (int)(item - node * a.num_q_heads);
  const int64_t row = rq.row0 + node;
  const int splits = min(a.splits, max(1, (rq.length + a.chunk - 1) / a.chunk));
  const int lane = threadIdx.x % kLanes;
  const int64_t at = (row * a.num_q_heads + head) * a.splits;
  float top = kNegInf;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, a.part_lse[at + s]);
  const float base = top == kNegInf ? 0.0f : top;
  float sum = 0.0f;
  f32x4 acc = {0, 0, 0, 0};
  for (int s = 0; s < splits; ++s) {
    const float f = fast_exp2(a.part_lse[at + s] - base);
    const f32x4 part = *reinterpret_cast<const f32x4*>(a.part_out + (at + s) * D + 4 * lane);
    sum += f;
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] += f * part[r];
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  float y[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    y[r] = acc[r] * inv;
    if (a.gate)
      y[r] *= gate_factor(a.gate[row * a.g_row + head * a.g_head + (4 * lane + r) * a.g_dim]);
  }
  u32x2 w = {pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
  __builtin_memcpy(a.out + row * a.out_row + head * a.out_head + 4 * lane, &w, 8);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

struct TreePlan {
  int tile_rows;  // (node, head) rows of a workgroup
  int stage;      // tokens of a stage
  int m_tiles, splits, chunk;
};

int tile_rows_for(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

// max_nodes and max_context bound the requests' nodes and committed tokens; the
// results do not depend on the chunks beyond fp32 rounding, and a request longer
// than max_context says is computed whole (its last chunk takes the rest).
TreePlan make_plan(int requests, int num_q_heads, int num_kv_heads, int64_t max_nodes,
                   int64_t max_context) {
  TreePlan p;
  const int64_t rows = max_nodes * (num_q_heads / num_kv_heads);
  p.tile_rows = tile_rows_for(rows);
  p.stage = p.tile_rows <= 32 ? 128 : 64;
  p.m_tiles = (int)((rows + p.tile_rows - 1) / p.tile_rows);
  const int64_t units = (int64_t)requests * num_kv_heads * p.m_tiles;
  const int64_t length = std::min<int64_t>(max_context + max_nodes, INT_MAX / 2);
  const int64_t stages = std::max<int64_t>(1, (length + p.stage - 1) / p.stage);
  int64_t splits = std::min<int64_t>((2 * kCUs + units - 1) / units, (stages + 3) / 4);
  splits = std::max<int64_t>(1, std::min<int64_t>(splits, 256));
  const int64_t per = (stages + splits - 1) / splits;
  p.chunk = (int)std::min<int64_t>(per * p.stage, INT_MAX / 2);
  p.splits = (int)((stages + per - 1) / per);
  return p;
}

template <int D, int NB, int WM, int WT>
hipError_t launch_tile(const TreeArgs& a, unsigned grid, hipStream_t stream) {
  const size_t lds = Shape<D, NB, WM, WT>::kLds;
  auto* kernel = &tree_attn_kernel<D, NB, WM, WT>;
  if (lds > 65536) {
    const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (err != hipSuccess) return err;
  }
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * kWaves), lds, stream, a);
  return hipGetLastError();
}

template <int D>
hipError_t launch_tree(const TreeArgs& a, const TreePlan& plan, int max_nodes, hipStream_t stream) {
  const unsigned grid = (unsigned)((int64_t)a.requests * a.kv_heads * a.m_tiles * a.splits);
  hipError_t err;
  if (plan.tile_rows == 16) err = launch_tile<D, 1, 1, 4>(a, grid, stream);
  else if (plan.tile_rows == 32) err = launch_tile<D, 2, 1, 4>(a, grid, stream);
  else if (plan.tile_rows == 64) err = launch_tile<D, 2, 2, 2>(a, grid, stream);
  else err = launch_tile<D, 2, 4, 1>(a, grid, stream);
  if (err != hipSuccess || a.splits == 1) return err;
  constexpr int kPer = 256 / (D / 4);
  const int row_tiles = (int)(((int64_t)max_nodes * a.num_q_heads + kPer - 1) / kPer);
  hipLaunchKernelGGL((tree_merge_kernel<D>), dim3((unsigned)(a.requests * row_tiles)), dim3(256), 0,
                     stream, a, row_tiles);
  return hipGetLastError();
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace
}  // namespace qsa

using namespace qsa;

extern "C" size_t qsa_tree_attention_workspace_bytes(int rows, int requests, int num_q_heads,
                                                     int num_kv_heads, int head_dim,
                                                     int max_query_len, int max_context_len) {
  if (rows <= 0 || requests <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads ||
      head_dim <= 0 || max_query_len <= 0 || max_context_len < 0)
    return 0;
  const TreePlan p = make_plan(requests, num_q_heads, num_kv_heads, std::min(max_query_len, rows),
                               max_context_len);
  if (p.splits == 1) return 0;
  return (size_t)rows * num_q_heads * p.splits * (head_dim + 1) * sizeof(float);
}

extern "C" int qsa_tree_attention(
    const void* q, int64_t q_row_stride, int64_t q_head_stride, int rows, int num_q_heads,
    int head_dim, const void* k_cache, int64_t k_block_stride, int64_t k_token_stride,
    int64_t k_head_stride, const void* v_cache, int64_t v_block_stride, int64_t v_token_stride,
    int64_t v_head_stride, int num_blocks, int page_size, int num_kv_heads,
    const int32_t* block_table, int64_t table_row_stride, int table_width, int num_requests,
    const int32_t* context_lens, const int32_t* query_start_loc, const int32_t* ancestors,
    int64_t ancestor_row_stride, int ancestor_words, void* out, int64_t out_row_stride,
    int64_t out_head_stride, const void* gate, int64_t gate_row_stride, int64_t gate_head_stride,
    int64_t gate_dim_stride, int max_query_len, int max_context_len, void* workspace,
    size_t workspace_bytes, void* stream) {
  const std::string name = "qsa_tree_attention";
  if (rows < 0 || num_requests < 0 || num_blocks < 0 || table_width < 0 || ancestor_words < 0 ||
      max_query_len < 0 || max_context_len < 0)
    return fail(QSA_ERR_INVALID, name + ": negative size");
  if (rows == 0 || num_requests == 0 || max_query_len == 0) return QSA_OK;
  if (head_dim != 64 && head_dim != 128)
    return fail(QSA_ERR_UNSUPPORTED, name + ": head_dim must be 64 or 128");
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads)
    return fail(QSA_ERR_UNSUPPORTED, name + ": query heads must be a multiple of kv heads");
  if (page_size <= 0) return fail(QSA_ERR_INVALID, name + ": page size must be positive");
  // (an empty cache, table or mask has no address and is not read)
  if (!q || ((!k_cache || !v_cache) && num_blocks > 0) || (!block_table && table_width > 0) ||
      !context_lens || !query_start_loc || (!ancestors && ancestor_words > 0) || !out)
    return fail(QSA_ERR_INVALID, name + ": null tensor pointer");
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || ((uintptr_t)out & 3u) ||
      ((q_row_stride | q_head_stride | k_block_stride | k_token_stride | k_head_stride |
        v_block_stride | v_token_stride | v_head_stride) & 7) ||
      ((out_row_stride | out_head_stride) & 1))
    return fail(QSA_ERR_INVALID, name + ": q and the caches need 16-byte alignment and strides of "
                                        "multiples of 8 elements, out 4-byte alignment");
  max_query_len = std::min(max_query_len, rows);
  const TreePlan plan =
      make_plan(num_requests, num_q_heads, num_kv_heads, max_query_len, max_context_len);
  const int64_t grid = (int64_t)num_requests * num_kv_heads * plan.m_tiles * plan.splits;
  const int64_t merge = (int64_t)num_requests * (((int64_t)max_query_len * num_q_heads + 7) / 8);
  if (grid > INT_MAX || merge > INT_MAX || (int64_t)max_query_len * num_q_heads > INT_MAX / 2)
    return fail(QSA_ERR_UNSUPPORTED, name + ": too many requests, rows or heads");
  TreeArgs a = {};
  if (plan.splits > 1) {
    const size_t need = qsa_tree_attention_workspace_bytes(
        rows, num_requests, num_q_heads, num_kv_heads, head_dim, max_query_len, max_context_len);
    if (!workspace || workspace_bytes < need || !aligned16(workspace))
      return fail(QSA_ERR_WORKSPACE, name + ": needs a 16-byte aligned workspace of " +
                                         std::to_string(need) + " bytes");
    a.part_out = static_cast<float*>(workspace);
    a.part_lse = a.part_out + (size_t)rows * num_q_heads * plan.splits * head_dim;
  }
  a.q = static_cast<const uint16_t*>(q);
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.k = static_cast<const char*>(k_cache);
  a.v = static_cast<const char*>(v_cache);
  a.kb = 2 * k_block_stride;
  a.kt = 2 * k_token_stride;
  a.kh = 2 * k_head_stride;
  a.vb = 2 * v_block_stride;
  a.vt = 2 * v_token_stride;
  a.vh = 2 * v_head_stride;
  a.num_blocks = num_blocks;
  a.page_size = page_size;
  a.page_div = FastDiv::make(page_size);
  a.table = block_table;
  a.table_row = table_row_stride;
  a.table_width = table_width;
  a.requests = num_requests;
  a.context_lens = context_lens;
  a.query_start_loc = query_start_loc;
  a.ancestors = ancestors;
  a.ancestor_row = ancestor_row_stride;
  a.words = ancestor_words;
  a.out = static_cast<uint16_t*>(out);
  a.out_row = out_row_stride;
  a.out_head = out_head_stride;
  a.gate = static_cast<const uint16_t*>(gate);
  a.g_row = gate_row_stride;
  a.g_head = gate_head_stride;
  a.g_dim = gate_dim_stride;
  a.rows = rows;
  a.num_q_heads = num_q_heads;
  a.kv_heads = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.group_div = FastDiv::make(a.group);
  a.m_tiles = plan.m_tiles;
  a.splits = plan.splits;
  a.chunk = plan.chunk;
  a.scale_log2 = 1.4426950408889634f / sqrtf((float)head_dim);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t err = head_dim == 128 ? launch_tree<128>(a, plan, max_query_len, s)
                                         : launch_tree<64>(a, plan, max_query_len, s);
  if (err != hipSuccess)
    return fail(QSA_ERR_HIP, name + " launch: " + hipGetErrorString(err));
  return QSA_OK;
}

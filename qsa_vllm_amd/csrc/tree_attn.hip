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
// of one kv head and streams a stretch of the request's tokens through LDS once
// for all of them, 64 a stage.
//
//   S^T[token][row] = K (A, 16 tokens x 32 dims) Q^T (B, 32 dims x 16 rows)
//   O^T[dim][row]  += V^T (A, 16 dims x 32 tokens) P^T (B, 32 tokens x 16 rows)
//
// on mfma_f32_16x16x32_bf16. P^T is the lane's own exponentials, so it never
// leaves registers; V^T comes from row-major V rows in LDS by the transposing LDS
// read. The exponentials are rounded to bf16, the matrix cores' type (2^-8 of a
// weight at most), and the row's sum is the product of the rounded ones with 1s,
// in fp32: the weights that meet V add up to 1. They are taken from a base that
// follows the row's maximum only when that has passed it by 2^8, so that most
// stages rescale nothing.
//
// Rows and tokens are shared out over the four waves as WM x WT: with many rows
// each wave has its own 16 NB rows and all tokens of a stage, with few rows the
// waves take different tokens and merge (max, sum, O) through LDS at the end.
//
// Work is shared out by stages. A row tile's (request, kv head) units, each of its
// request's stages, lie end to end on that tile's line, and every workgroup takes
// an equal stretch of a line, two workgroups a CU in all. Workgroups at the same
// place of different tiles' lines run on one XCD, whose L2 then serves the K/V to
// all but the first. (Splits of the context by a rule on the launch's sizes, one
// workgroup each, took 234 us when the stretches took 177: 32 trees of 5 - 24 nodes
// on 4096 - 32768 tokens.) Lengths and rows are known on the device only; each
// workgroup adds them up itself. A unit that no one stretch covers leaves
// normalised fp32 pieces and log2 sums, which a second kernel joins in order; the
// others are written at once.
//
// What bounds it (16 query and 2 kv heads of 128, pages of 16): single tokens and
// small trees read HBM (64 single tokens on 1024 - 8192 tokens 69 us, 4.4 TB/s of
// K/V; a large copy 4.8); 32 trees of 5 - 24 nodes on 4096 - 32768 tokens, 174 us,
// a workgroup's stages in series (2.9 us each; the second tiles of requests past
// 16 nodes add to them, though reading K/V once for both measured no faster);
// 64 nodes on 131072 tokens, 103 us, the matrix cores with the softmax between
// them (0.67 PFLOP/s; 1.4 in a large library product). One request of 8 nodes on
// 500 tokens, 14.5 us, is two launches' chains of loads.
#include "paged_stage.h"
#include "../../include/qsa_hip.h"

#include <algorithm>
#include <climits>

namespace qsa {
namespace {

constexpr int kWaves = 4;
constexpr int kCUs = 256;

constexpr int kTok = 64;         // tokens of a stage
constexpr int kTileRows = 128;  // (node, head) rows of a workgroup

struct TreeArgs {
  const uint16_t* q;
  int64_t q_row, q_head;  // elements
  const char* k;
  const char* v;
  uint32_t kb, kt, vb, vt;  // units of 16 bytes
  int64_t kh, vh;  // bytes
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
  // Two pieces a workgroup (the end of a unit it shares with the one before, the
  // start of one it shares with the next): [2 workgroups][slot rows][D], then sums.
  float* part_out;
  float* part_lse;
  int rows, num_q_heads, kv_heads, group;
  FastDiv group_div;
  int workgroups;  // 0: one for each unit (m_tiles a request and kv head)
  int m_tiles, slot_rows, max_nodes;
  float scale_log2;
};

// One request's rows and tokens, kept within the query tensor and the page
// table whatever the device arrays say.
struct Request {
  int row0, nodes, context, length;
};
__device__ __forceinline__ Request make_request(const TreeArgs& a, int first, int last, int context) {
  Request r;
  r.row0 = min(max(first, 0), a.rows);
  r.nodes = min(min(max(last, r.row0), a.rows) - r.row0, a.max_nodes);
  const int64_t capacity = min((int64_t)a.table_width * a.page_size, (int64_t)INT_MAX / 2);
  r.context = (int)min((int64_t)max(context, 0), capacity);
  r.length = (int)min((int64_t)r.context + r.nodes, capacity);
  return r;
}
__device__ __forceinline__ Request load_request(const TreeArgs& a, int b) {  // b: a lane's own
  return make_request(a, a.query_start_loc[b], a.query_start_loc[b + 1], a.context_lens[b]);
}
__device__ __forceinline__ Request uniform_request(const TreeArgs& a, int b) {  // b: the wave's
  return make_request(a, load_uniform(a.query_start_loc + b), load_uniform(a.query_start_loc + b + 1),
                      load_uniform(a.context_lens + b));
}
__device__ __forceinline__ int tiles_of(const TreeArgs& a, const Request& r) {
  return (r.nodes * a.group + kTileRows - 1) / kTileRows;
}
__device__ __forceinline__ int stages_of(const Request& r) {
  return max(1, (r.length + kTok - 1) / kTok);
}
// A request's stages on a tile's line.
__device__ __forceinline__ int stages_on(const TreeArgs& a, const Request& r, int tile) {
  return tile < tiles_of(a, r) ? a.kv_heads * stages_of(r) : 0;
}

// fn(request b), added up over all requests: a wave's 64 lanes take one each.
template <typename F>
__device__ __forceinline__ int sum_requests(const TreeArgs& a, F fn) {
  if (a.requests == 1) return uniform(fn(0, uniform_request(a, 0)));
  int sum = 0;
  for (int b = threadIdx.x & 63; b < a.requests; b += 64) sum += fn(b, load_request(a, b));
#pragma unroll
  for (int w = 32; w > 0; w /= 2) sum += __shfl_xor(sum, w, 64);
  return uniform(sum);
}
__device__ __forceinline__ int line_length(const TreeArgs& a, int tile) {
  return sum_requests(a, [&](int, const Request& r) { return stages_on(a, r, tile); });
}
// Stages of a stretch: as few as keep all workgroups on the card at once. A
// workgroup beyond the 64 that an XCD's CUs hold would run after all the others, so
// the lines' numbers, rounded up to 8, must add up to no more than 512. (One too
// many on one XCD: 24 trees of 1 - 40 nodes on 2048 - 30000 tokens 249 us, else 192.)
__device__ __forceinline__ int stretch(const TreeArgs& a) {
  int lines = 0;
  const int all = sum_requests(a, [&](int, const Request& r) {
    lines = max(lines, tiles_of(a, r));
    return tiles_of(a, r) * a.kv_heads * stages_of(r);
  });
  unsigned n = a.workgroups;
  if (n == 2 * kCUs) {
    if (a.requests == 1) {  // lines of one length
      lines = uniform(lines);
      if (lines <= n / 8) n = lines * (n / (unsigned)max(lines, 1) / 8 * 8);
    } else {
#pragma unroll
      for (int w = 32; w > 0; w /= 2) lines = max(lines, __shfl_xor(lines, w, 64));
      lines = uniform(lines);
      // (lines of unequal lengths; of more than 8 the rounding would cost too much)
      if (lines <= 8) n -= 8 * (max(lines, 1) - 1);
    }
  }
  return max(1u, (all + n - 1) / max(n, 1u));
}
// Workgroups of a line, rounded up so that the next line starts at the first XCD.
__device__ __forceinline__ int line_workgroups(int length, int mine) {
  return ((unsigned)(length + mine - 1) / (unsigned)mine + 7) / 8 * 8;
}
// The request at a place on a tile's line; `place` becomes the place within it.
__device__ __forceinline__ int locate(const TreeArgs& a, int tile, int& place) {
  if (a.requests == 1) return 0;
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < a.requests; b0 += 64) {
    const int n = b0 + lane < a.requests ? stages_on(a, load_request(a, b0 + lane), tile) : 0;
    int end = n;  // inclusive sum over the lanes
#pragma unroll
    for (int w = 1; w < 64; w *= 2) {
      const int below = __shfl_up(end, w, 64);
      end += lane >= w ? below : 0;
    }
    const uint64_t past = __ballot(end > place);
    if (past) {
      const int at = __ffsll((unsigned long long)past) - 1;
      place = uniform(place - __shfl(end - n, at, 64));
      return b0 + at;
    }
    place = uniform(place - __shfl(end, 63, 64));
  }
  return a.requests;
}

// c += A B over 32 tokens (two subtiles' operands) or, when the wave has a
// single subtile, over its 16.
template <int SUB>
__device__ __forceinline__ void add_product(f32x4& c, s16x4 a0, s16x4 a1, const uint32_t (&b0)[2],
                                            const uint32_t (&b1)[2]) {
  if constexpr (SUB > 1) {
    const s16x8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
    const u32x4 b = {b0[0], b0[1], b1[0], b1[1]};
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    c = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(
        a0, __builtin_bit_cast(s16x4, (u32x2{b0[0], b0[1]})), c, 0, 0, 0);
  }
}

template <int D, int NB, int WM, int WT>
struct Shape {
  static constexpr int kRows = 16 * NB * WM;    // query rows of a workgroup
  static constexpr int kWaveTok = kTok / WT;    // tokens of a stage a wave takes
  static constexpr int kSub = kWaveTok / 16;    // 16-token subtiles of them
  static constexpr int kPair = kSub > 1 ? 1 : 0;  // subtiles are multiplied in pairs
  static constexpr int kLoads = kTok * (D / 8) / (64 * kWaves);  // 16-byte K loads of a lane
  static constexpr size_t kStage = (size_t)kTok * D * 2;         // K or V of a stage
  // Two stages of K and V; afterwards the partial results of all but the first
  // wave of each row block.
  static constexpr int kWaveMerge = 16 * NB * (D + 2);
  static constexpr size_t kMerge = (size_t)WM * (WT - 1) * kWaveMerge * 4;
  static constexpr size_t kLds = 4 * kStage > kMerge ? 4 * kStage : kMerge;
};

// Which 16-bit halves hold an infinity or NaN (bf16), as bits; and 0 in their place.
__device__ __forceinline__ uint32_t not_finite(const u32x4& v) {
  uint32_t bits = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    bits |= (uint32_t)((v[w] & 0x7F80u) == 0x7F80u) << (2 * w);
    bits |= (uint32_t)((v[w] & 0x7F800000u) == 0x7F800000u) << (2 * w + 1);
  }
  return bits;
}
__device__ __forceinline__ u32x4 finite_or_zero(u32x4 v) {
  const uint32_t bits = not_finite(v);
#pragma unroll
  for (int w = 0; w < 4; ++w)
    v[w] &= (bits >> (2 * w) & 1 ? 0u : 0xFFFFu) | (bits >> (2 * w + 1) & 1 ? 0u : 0xFFFF0000u);
  return v;
}

// What a row sees of 64 positions: bit i for drafted node j + i, set for the
// committed ones (j + i < 0).
__device__ __forceinline__ uint64_t seen_from(const TreeArgs& a, int row, int j) {
  const int32_t* const words = a.ancestors + row * a.ancestor_row;
  auto word = [&](int w) -> uint64_t {
    return w >= 0 && w < a.words ? (uint32_t)words[w] : 0u;
  };
  if (j <= -64) return ~0ull;
  const int w = j >> 5, shift = j & 31;  // rounded down: w is -2 or -1 where j < 0
  uint64_t bits = (word(w + 1) << 32 | word(w)) >> shift;
  if (shift) bits |= word(w + 2) << (64 - shift);
  return j < 0 ? bits | ((1ull << -j) - 1) : bits;
}

// Tokens t_begin .. t_end of one row tile (rows m0 .. of a request's `rows`), to
// the output or, where others take the rest of them, to piece `piece`.
template <int D, int NB, int WM, int WT>
__device__ __forceinline__ void attend_tile(const TreeArgs& a, const Request& rq,
                                            const int32_t* trow, int kv, int rows, int m0,
                                            int piece, int t_begin, int t_end, char* lds) {
  typedef Shape<D, NB, WM, WT> S;
  constexpr int U = D / 8;  // 16-byte units of a row
  constexpr int kSteps = D / 32;
  constexpr int kDims = D / 16;
  // Not to be known before the tile: what follows from it, for all four shares,
  // would otherwise be kept in registers through the loop over tiles.
  int lane = threadIdx.x & 63;
  asm("" : "+v"(lane));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int wm = wave / WT, wt = wave % WT;
  const bool active = m0 + wm * 16 * NB < rows;  // else the wave only moves K/V

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

  // K/V of a stage go straight into LDS: block i of a stage (64 units) is moved
  // by wave i mod 4, and every lane's unit of a row is the same in all its
  // blocks (a block of 64 / U tokens times the waves is a multiple of the
  // swizzles' periods).
  const char* const zero = reinterpret_cast<const char*>(g_qsa_zero_rows);
  const int tok0 = wave * (64 / U) + lane / U;  // the lane's token of the wave's first block
  const int ku = (lane % U ^ k_swizzle<D>(tok0)) * 16, vu = (lane % U ^ v_swizzle<D>(tok0)) * 16;
  const char* const klane = a.k + kv * a.kh + ku;
  const char* const vlane = a.v + kv * a.vh + vu;

  // Page of token t + lane, -1 past the end or where the table has none.
  auto load_page = [&](int t) {
    const int pos = t + lane;
    return *(pos < t_end ? trow + a.page_div.div(pos) : g_qsa_no_page);
  };
  auto load_stage = [&](int t, int page, char* stage) {
    // Offsets (16-byte units) of token t + lane; blocks without tokens of the
    // cache read zeros in their place.
    const int pos = t + lane;
    const bool ok = page >= 0 && page < a.num_blocks;
    const uint32_t at = pos - a.page_div.div(pos) * a.page_size;
    const uint32_t koff = ok ? page * a.kb + at * a.kt : kNoToken;
    const uint32_t voff = page * a.vb + at * a.vt;
    const uint64_t valid = __ballot(ok);
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int from = (i * kWaves * (64 / U) + tok0) * 4;
      const uint32_t ko = __builtin_amdgcn_ds_bpermute(from, koff);
      const uint32_t vo = __builtin_amdgcn_ds_bpermute(from, voff);
      const char* ks = klane + ((uint64_t)ko << 4);
      const char* vs = vlane + ((uint64_t)vo << 4);
      if (valid != ~0ull) {
        ks = ko != kNoToken ? ks : zero + ku;
        vs = ko != kNoToken ? vs : zero + vu;
      }
      char* const dst = stage + (i * kWaves + wave) * 1024;
      load_to_lds(ks, dst);
      load_to_lds(vs, dst + S::kStage);
    }
    return valid;
  };

  int page_next = -1, buffer = 0;
  uint64_t valid = 0, valid_next = 0;
  if (t_begin < t_end) {
    const int page = load_page(t_begin);
    page_next = load_page(t_begin + kTok);
    valid_next = load_stage(t_begin, page, lds);
  }
  bool poisoned = false;
  // Waits for stage t, starts the next one's loads, and returns stage t's K.
  auto advance = [&](int t) -> const char* {
    char* const stage = lds + buffer * 2 * S::kStage;
    buffer ^= 1;
    __builtin_amdgcn_s_waitcnt(kLoadsDone);
    __syncthreads();  // the stage is in LDS, and the last one has been read by all
    valid = valid_next;
    if (t + kTok < t_end)
      valid_next = load_stage(t + kTok, page_next, lds + buffer * 2 * S::kStage);
    page_next = load_page(t + 2 * kTok);
    if (t + kTok > rq.context) {
      // A drafted token's V may hold infinities or NaN that a row outside its
      // branch must not see (0 times them is NaN). The whole stage's are taken
      // as 0 here, and added at the end to the rows that see them.
      u32x4* const v = reinterpret_cast<u32x4*>(stage + S::kStage);
      bool bad = false;
      for (int i = lane; i < kTok * U; i += 64) bad |= not_finite(v[i]) != 0;
      if (__any(bad)) {  // every wave has looked at the whole stage
        __syncthreads();
        for (int i = threadIdx.x; i < kTok * U; i += 64 * kWaves) v[i] = finite_or_zero(v[i]);
        __syncthreads();
        poisoned = true;
      }
    }
    return stage;
  };

  if (!active) {
    for (int t = t_begin; t < t_end; t += kTok) advance(t);
    if constexpr (WT > 1) {
      __syncthreads();
      __syncthreads();
    }
    return;
  }

  f32x4 o[NB][kDims], sum[NB];  // sum: the row's, in each of the four
  float base[NB];               // what the exponents are taken from: the maximum, or up to kSlack below
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    base[i] = kNegInf;
    sum[i] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int d = 0; d < kDims; ++d) o[i][d] = f32x4{0, 0, 0, 0};
  }
  const float slack = kSlack / a.scale_log2;

  for (int t = t_begin; t < t_end; t += kTok) {
    const char* const k_lds = advance(t);
    const char* const v_lds = k_lds + S::kStage;
    const bool drafted = t + kTok > rq.context;

    const int first = wt * S::kWaveTok;  // the wave's tokens of the stage
    f32x4 sc[NB][S::kSub];
#pragma unroll
    for (int u = 0; u < S::kSub; ++u) {
      bf16x8 kf[kSteps];
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        kf[s] = __builtin_bit_cast(bf16x8, load_u32x4(k_lds + k_at<D>(first + 16 * u + n, 4 * s + g)));
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        sc[i][u] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
          sc[i][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[s], q[i][s], sc[i][u], 0, 0, 0);
      }
    }

    // Masked scores are replaced, whatever they hold.
    if (drafted || valid != ~0ull) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        // bit 16 u + r: the lane's token 16 u + 4 g + r
        const uint64_t seen =
            (valid >> first & seen_from(a, node[i], t + first - rq.context)) >> (4 * g);
#pragma unroll
        for (int u = 0; u < S::kSub; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            sc[i][u][r] = (seen >> (16 * u + r)) & 1 ? sc[i][u][r] : kNegInf;
      }
    }

#pragma unroll
    for (int i = 0; i < NB; ++i) {
      float top = fmaxf(fmaxf(sc[i][0][0], sc[i][0][1]), fmaxf(sc[i][0][2], sc[i][0][3]));
#pragma unroll
      for (int u = 1; u < S::kSub; ++u) {
        top = fmaxf(fmaxf(top, sc[i][u][0]), sc[i][u][1]);
        top = fmaxf(fmaxf(top, sc[i][u][2]), sc[i][u][3]);
      }
      if (__any(top > base[i] + slack)) {
        // Only the rows that passed it: a row's bits are its own. (A row that has
        // seen nothing yet has -inf, and so has one whose scores are NaN.)
        const float row_top = max_over_quarters(top);
        const float m = row_top > base[i] + slack ? row_top : base[i];
        const float shrink =
            m == kNegInf ? 1.0f : fast_exp2((base[i] - m) * a.scale_log2);
        base[i] = m;
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[i][r] *= shrink;
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[i][d][r] *= shrink;
      }
    }

    uint32_t p[NB][S::kSub][2];  // weights of tokens 16 u + 4 g + 0 .. 3, bf16 pairs
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const float from = base[i] == kNegInf ? 0.0f : -base[i] * a.scale_log2;
#pragma unroll
      for (int u = 0; u < S::kSub; ++u) {
        float e[4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          e[r] = fast_exp2(__builtin_fmaf(sc[i][u][r], a.scale_log2, from));
        p[i][u][0] = pack_bf16x2(e[0], e[1]);
        p[i][u][1] = pack_bf16x2(e[2], e[3]);
      }
    }

    const s16x4 ones = {0x3F80, 0x3F80, 0x3F80, 0x3F80};
#pragma unroll
    for (int u = 0; u < S::kSub; u += 2)
#pragma unroll
      for (int i = 0; i < NB; ++i) add_product<S::kSub>(sum[i], ones, ones, p[i][u], p[i][u + S::kPair]);

    const char* const v_lane = v_lds + (first + 4 * g + (n >> 2)) * D * 2 + (n & 1) * 8;
    const int v_unit = (n & 3) >> 1, v_swz = v_swizzle<D>(first + 4 * g + (n >> 2));
#pragma unroll
    for (int u = 0; u < S::kSub; u += 2)
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        const char* const src = v_lane + 16 * u * D * 2 + ((2 * d + v_unit) ^ v_swz) * 16;
        const s16x4 v0 = read_transposed(src);
        const s16x4 v1 = S::kPair ? read_transposed(src + 16 * D * 2) : v0;
#pragma unroll
        for (int i = 0; i < NB; ++i)
          add_product<S::kSub>(o[i][d], v0, v1, p[i][u], p[i][u + S::kPair]);
      }
  }

  float total[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    total[i] = sum[i][0];
    base[i] *= a.scale_log2;  // log2 domain from here on
  }

  if constexpr (WT > 1) {
    // The token shares of each row block, joined in wave order by its first wave.
    float* const merge = reinterpret_cast<float*>(lds) + wm * (WT - 1) * S::kWaveMerge;
    __syncthreads();
    if (wt > 0) {
      float* const mine = merge + (wt - 1) * S::kWaveMerge;
#pragma unroll
      for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int d = 0; d < kDims; ++d)
          *reinterpret_cast<f32x4*>(mine + ((i * kDims + d) * 64 + lane) * 4) = o[i][d];
        if (g == 0) {
          mine[16 * NB * D + 16 * i + n] = base[i];
          mine[16 * NB * D + 16 * NB + 16 * i + n] = total[i];
        }
      }
    }
    __syncthreads();
    if (wt > 0) return;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      float m = base[i];
      for (int w = 0; w < WT - 1; ++w) m = fmaxf(m, merge[w * S::kWaveMerge + 16 * NB * D + 16 * i + n]);
      const float from = m == kNegInf ? 0.0f : m;
      float f = fast_exp2(base[i] - from);
      total[i] *= f;
#pragma unroll
      for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[i][d][r] *= f;
      for (int w = 0; w < WT - 1; ++w) {
        const float* other = merge + w * S::kWaveMerge;
        f = fast_exp2(other[16 * NB * D + 16 * i + n] - from);
        total[i] += f * other[16 * NB * D + 16 * NB + 16 * i + n];
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          const f32x4 add = *reinterpret_cast<const f32x4*>(other + ((i * kDims + d) * 64 + lane) * 4);
#pragma unroll
          for (int r = 0; r < 4; ++r) o[i][d][r] += f * add[r];
        }
      }
      base[i] = m;
    }
  }

  if (poisoned) {
    // From the first stage with a drafted token (stages start at multiples of 64).
    for (int pos = max(t_begin, rq.context / kTok * kTok); pos < t_end; ++pos) {
      const int page = trow[a.page_div.div(pos)];
      if (page < 0 || page >= a.num_blocks) continue;
      const char* const v = a.v + kv * a.vh + ((uint64_t)page * a.vb << 4) +
                            ((uint64_t)(pos - a.page_div.div(pos) * a.page_size) * a.vt << 4);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        if (!(seen_from(a, node[i], pos - rq.context) & 1)) continue;
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          const u32x2 x = load_u32x2(v + (16 * d + 4 * g) * 2);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // (a positive weight times an infinity or NaN is the same)
            const uint32_t bits = r & 1 ? x[r >> 1] & 0xFFFF0000u : x[r >> 1] << 16;
            if ((bits & 0x7F800000u) == 0x7F800000u) o[i][d][r] += __builtin_bit_cast(float, bits);
          }
        }
      }
    }
  }

#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int m = m0 + (wm * NB + i) * 16 + n;
    if (m >= rows) continue;
    const int head = kv * a.group + m - (node[i] - rq.row0) * a.group;
    const float inv = total[i] == 0.0f ? 0.0f : 1.0f / total[i];  // a row that sees nothing: zeros
    if (piece >= 0) {
      const int64_t at = (int64_t)piece * a.slot_rows + m - m0;
#pragma unroll
      for (int d = 0; d < kDims; ++d)
        *reinterpret_cast<f32x4*>(a.part_out + at * D + 16 * d + 4 * g) =
            f32x4{o[i][d][0] * inv, o[i][d][1] * inv, o[i][d][2] * inv, o[i][d][3] * inv};
      if (g == 0) a.part_lse[at] = total[i] == 0.0f ? kNegInf : base[i] + __log2f(total[i]);
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

template <int D>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void
tree_attn_kernel(TreeArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  // The stretch [place, place + left) of a tile's line, place counted from the
  // start of `request`.
  int request, tile, place, left;
  if (a.workgroups) {
    const int mine = stretch(a);
    int id = blockIdx.x, length;
    for (tile = 0;; ++tile) {
      length = line_length(a, tile);
      if (length == 0) return;  // past the last line
      const int n = line_workgroups(length, mine);
      if (id < n) break;
      id -= n;
    }
    place = id * mine;
    left = min(mine, length - place);
    if (left <= 0) return;
    request = locate(a, tile, place);
  } else {
    const int units = a.kv_heads * a.m_tiles;
    request = blockIdx.x / units;
    const int unit = blockIdx.x - request * units;
    tile = unit / a.kv_heads;
    const Request rq = uniform_request(a, request);
    if (tile >= tiles_of(a, rq)) return;
    left = stages_of(rq);
    place = (unit - tile * a.kv_heads) * left;
  }
  const int m0 = tile * kTileRows;
  bool first = true;
  while (left > 0 && request < a.requests) {
    const Request rq = uniform_request(a, request);
    const int stages = stages_of(rq);
    const int units = tile < tiles_of(a, rq) ? a.kv_heads : 0;
    for (int kv = (unsigned)place / (unsigned)stages; kv < units && left > 0; ++kv) {
      const int s0 = place - kv * stages;
      const int s1 = min(stages, s0 + left);
      place += s1 - s0;
      left -= s1 - s0;
      const int rows = rq.nodes * a.group;
      // A unit that starts here and goes on is the stretch's last, one that ends
      // or goes through, its first.
      const int piece = s0 == 0 && s1 == stages ? -1 : 2 * (int)blockIdx.x + (s0 == 0 ? 1 : 0);
      const int t_begin = s0 * kTok, t_end = min(rq.length, s1 * kTok);
      const int32_t* const trow = a.table + request * a.table_row;
      if (!first) __syncthreads();  // LDS has been read by all
      first = false;
      // The wave shares by the tile's own rows: requests of one batch differ.
      const int here = rows - m0;
      if (here > 64) attend_tile<D, 2, 4, 1>(a, rq, trow, kv, rows, m0, piece, t_begin, t_end, lds);
      else if (here > 32) attend_tile<D, 2, 2, 2>(a, rq, trow, kv, rows, m0, piece, t_begin, t_end, lds);
      else if (here > 16) attend_tile<D, 2, 1, 4>(a, rq, trow, kv, rows, m0, piece, t_begin, t_end, lds);
      else attend_tile<D, 1, 1, 4>(a, rq, trow, kv, rows, m0, piece, t_begin, t_end, lds);
    }
    ++request;
    place = 0;
  }
}

// Joins a row's pieces: out = sum_s 2^(lse_s - max) part_s / sum_s 2^(lse_s - max).
// D / 4 lanes hold a (row, head)'s dims; WAYS such groups take its pieces in
// turn (s mod WAYS) and add up in group order, so that a long context's many
// pieces are read side by side. Bound by reading them: 33 MB in 10 us (64 nodes on
// 131072 tokens).
template <int D, int WAYS>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a, int row_tiles) {
  constexpr int kLanes = D / 4;
  constexpr int kGroups = 256 / kLanes;
  constexpr int kPer = kGroups / WAYS;  // (row, head)s of a workgroup
  __shared__ f32x4 acc_lds[WAYS > 1 ? kGroups : 1][kLanes];
  __shared__ float sum_lds[WAYS > 1 ? kGroups : 1];
  const int request = blockIdx.x / row_tiles;
  const Request rq = uniform_request(a, request);
  const int64_t first_item = (int64_t)(blockIdx.x % row_tiles) * kPer;
  if (first_item >= (int64_t)rq.nodes * a.num_q_heads) return;
  const int stages = stages_of(rq);
  // Where the rows' units lie on their tiles' lines, and the first workgroup of each
  // line: found by one wave for all (the sums over the requests by every wave are
  // most of the launch's instructions). Lane i takes (row, head) i mod kPer.
  __shared__ int begin_lds[kPer], id0_lds[kPer], mine_lds;
  if (threadIdx.x < 64) {
    const int64_t item = first_item + threadIdx.x % kPer;
    const int node = (int)(item / a.num_q_heads);
    const int head = (int)(item - (int64_t)node * a.num_q_heads);
    const int kv = head / a.group, my_tile = (node * a.group + head - kv * a.group) / kTileRows;
    const int mine = stretch(a);
    int begin = 0, id0 = 0, ids = 0;
    for (int tile = 0; tile < tiles_of(a, rq); ++tile) {
      const int before = sum_requests(a, [&](int b, const Request& r) {
        return b < request ? stages_on(a, r, tile) : 0;
      });
      if (tile == my_tile) {
        begin = before + kv * stages;
        id0 = ids;
      }
      if (tile + 1 < tiles_of(a, rq)) ids += line_workgroups(line_length(a, tile), mine);
    }
    if (threadIdx.x < kPer) {
      begin_lds[threadIdx.x] = begin;
      id0_lds[threadIdx.x] = id0;
    }
    if (threadIdx.x == 0) mine_lds = mine;
  }
  __syncthreads();
  const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const int way = grp % WAYS;
  const int64_t item = first_item + grp / WAYS;
  const int node = (int)(item / a.num_q_heads);
  const int head = (int)(item - (int64_t)node * a.num_q_heads);
  const int m = node * a.group + head - head / a.group * a.group;
  // The workgroups whose stretches the unit meets: the first one's piece is its
  // second, the others' their first.
  const int mine = mine_lds, begin = begin_lds[grp / WAYS], id0 = id0_lds[grp / WAYS];
  const int w0 = (unsigned)begin / (unsigned)mine;
  const int pieces = (unsigned)(begin + stages - 1) / (unsigned)mine - w0 + 1;
  // One piece: the attention has written the row.
  const bool live = node < rq.nodes && pieces > 1;
  const int64_t row = rq.row0 + node;
  const int splits = live ? pieces : 0;
  auto at = [&](int s) -> int64_t {
    return (int64_t)(2 * (id0 + w0 + s) + (s == 0 ? 1 : 0)) * a.slot_rows + m % kTileRows;
  };
  float top = kNegInf;
  for (int s = lane; s < splits; s += kLanes) top = fmaxf(top, a.part_lse[at(s)]);
#pragma unroll
  for (int w = kLanes / 2; w > 0; w /= 2) top = fmaxf(top, __shfl_xor(top, w, 64));
  const float base = top == kNegInf ? 0.0f : top;
  float sum = 0.0f;
  f32x4 acc = {0, 0, 0, 0};
#pragma unroll 4
  for (int s = way; s < splits; s += WAYS) {
    const float f = fast_exp2(a.part_lse[at(s)] - base);
    const f32x4 part = *reinterpret_cast<const f32x4*>(a.part_out + at(s) * D + 4 * lane);
    sum += f;
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] += f * part[r];
  }
  if constexpr (WAYS > 1) {
    acc_lds[grp][lane] = acc;
    if (lane == 0) sum_lds[grp] = sum;
    __syncthreads();
    if (way > 0) return;
#pragma unroll
    for (int w = 1; w < WAYS; ++w) {
      acc += acc_lds[grp + w][lane];
      sum += sum_lds[grp + w];
    }
  }
  if (!live) return;
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
  int workgroups, m_tiles, slot_rows;
};

// Workgroups of a launch at most: each line's last stretch may be short, and its
// number is rounded up to 8.
int grid_of(const TreePlan& p) { return p.workgroups + 8 * p.m_tiles; }

// max_nodes and max_context bound the requests' nodes and committed tokens. They
// shape the launch: a longer context is computed whole all the same.
TreePlan make_plan(int requests, int num_q_heads, int num_kv_heads, int64_t max_nodes,
                   int64_t max_context) {
  TreePlan p;
  const int64_t rows = max_nodes * (num_q_heads / num_kv_heads);
  p.m_tiles = (int)((rows + kTileRows - 1) / kTileRows);
  p.slot_rows = (int)std::min<int64_t>(kTileRows, (rows + 15) / 16 * 16);
  const int64_t units = (int64_t)requests * num_kv_heads * p.m_tiles;
  const int64_t stages = (std::min<int64_t>(max_context + max_nodes, INT_MAX / 2) + kTok - 1) / kTok;
  p.workgroups = stages > 1 ? (int)std::min<int64_t>(2 * kCUs, units * stages) : 0;
  return p;
}

// What a launch of more than 2^32 - 1 threads (256 a workgroup) is refused with.
constexpr hipError_t kTooLarge = hipErrorInvalidConfiguration;
bool fits(int64_t blocks) { return blocks <= UINT_MAX / 256; }

// Workgroups of the joining launch for each request.
template <int D, int WAYS>
int64_t merge_tiles(int64_t pairs) {
  constexpr int kPer = 256 / (D / 4) / WAYS;
  return (pairs + kPer - 1) / kPer;
}
template <int D, int WAYS>
hipError_t launch_merge(const TreeArgs& a, int64_t pairs, hipStream_t stream) {
  const int64_t row_tiles = merge_tiles<D, WAYS>(pairs);
  hipLaunchKernelGGL((tree_merge_kernel<D, WAYS>), dim3((unsigned)(a.requests * row_tiles)),
                     dim3(256), 0, stream, a, (int)row_tiles);
  return hipGetLastError();
}

template <int D>
hipError_t launch_tree(const TreeArgs& a, const TreePlan& plan, int max_nodes, hipStream_t stream) {
  const int64_t grid =
      a.workgroups ? grid_of(plan) : (int64_t)a.requests * a.kv_heads * a.m_tiles;
  // Both launches' sizes before the first: a call that is refused has written nothing.
  // (Only few (row, head)s are joined 8 ways.)
  const int64_t pairs = (int64_t)max_nodes * a.num_q_heads;
  if (!fits(grid) || (a.workgroups && !fits(a.requests * merge_tiles<D, 1>(pairs)))) return kTooLarge;
  constexpr size_t kLds = std::max({Shape<D, 2, 4, 1>::kLds, Shape<D, 2, 2, 2>::kLds,
                                    Shape<D, 2, 1, 4>::kLds, Shape<D, 1, 1, 4>::kLds});
  static_assert(kLds <= 65536, "two workgroups a CU, and no attribute to set");
  hipLaunchKernelGGL((tree_attn_kernel<D>), dim3((unsigned)grid), dim3(64 * kWaves), kLds, stream, a);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess || !a.workgroups) return err;
  // Many (row, head)s have few pieces each and need no more workgroups. In all, us,
  // WAYS 8 / 4 / 2 / 1, by (row, head)s at most:
  //   1024   64 nodes on 131072 tokens          100.3 / 100.0 / 100.5 / 103.0
  //   1024   8 trees of 8 nodes on 8000          33.1 / 33.0 / 33.5 / 33.7
  //   2048   2 trees of 64 nodes on 65536       109.9 / 109.0 / 109.2 / 109.8
  //   4096   4 trees of 64 nodes on 32768       118.4 / 110.0 / 109.3 / 108.4
  //   4096   256 single tokens on 1024 - 4096   146.4 / 140.6 / 138.8 / 138.7
  //   8192   8 trees of 64 nodes on 16384       135.5 / 117.9 / 110.7 / 109.7
  //   12288  32 trees of 5 - 24 nodes           186.9 / 177.6 / 175.7 / 172.3
  return pairs * a.requests <= 2048 ? launch_merge<D, 8>(a, pairs, stream)
                                    : launch_merge<D, 1>(a, pairs, stream);
}

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
  if (!p.workgroups) return 0;
  return (size_t)2 * grid_of(p) * p.slot_rows * (head_dim + 1) * sizeof(float);
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
  // The kernel's offsets are 32-bit counts of 16 bytes.
  const int64_t k_span = cache_span(num_blocks, k_block_stride, page_size, k_token_stride);
  const int64_t v_span = cache_span(num_blocks, v_block_stride, page_size, v_token_stride);
  if (k_span < 0 || v_span < 0 || std::max(k_span, v_span) / 8 >= kNoToken)
    return fail(QSA_ERR_UNSUPPORTED, name + ": the cache must span under 64 GiB");
  max_query_len = std::min(max_query_len, rows);
  const TreePlan plan =
      make_plan(num_requests, num_q_heads, num_kv_heads, max_query_len, max_context_len);
  const int64_t units = (int64_t)num_requests * num_kv_heads * plan.m_tiles;
  const int64_t merge = (int64_t)num_requests * max_query_len * num_q_heads;
  const int64_t capacity = (int64_t)table_width * page_size / kTok + 1;
  if (units > INT_MAX / 2 / capacity || merge > INT_MAX ||
      (int64_t)max_query_len * num_q_heads > INT_MAX / 2)
    return fail(QSA_ERR_UNSUPPORTED, name + ": too many requests, rows or heads for the page table");
  TreeArgs a = {};
  if (plan.workgroups) {
    const size_t need = qsa_tree_attention_workspace_bytes(
        rows, num_requests, num_q_heads, num_kv_heads, head_dim, max_query_len, max_context_len);
    if (!workspace || workspace_bytes < need || !aligned16(workspace))
      return fail(QSA_ERR_WORKSPACE, name + ": needs a 16-byte aligned workspace of " +
                                         std::to_string(need) + " bytes");
    a.part_out = static_cast<float*>(workspace);
    a.part_lse = a.part_out +
                 (size_t)2 * grid_of(plan) * plan.slot_rows * head_dim;
  }
  a.q = static_cast<const uint16_t*>(q);
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.k = static_cast<const char*>(k_cache);
  a.v = static_cast<const char*>(v_cache);
  a.kb = (uint32_t)(k_block_stride / 8);
  a.kt = (uint32_t)(k_token_stride / 8);
  a.kh = 2 * k_head_stride;
  a.vb = (uint32_t)(v_block_stride / 8);
  a.vt = (uint32_t)(v_token_stride / 8);
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
  a.workgroups = plan.workgroups;
  a.slot_rows = plan.slot_rows;
  a.max_nodes = max_query_len;
  a.scale_log2 = 1.4426950408889634f / sqrtf((float)head_dim);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t err = head_dim == 128 ? launch_tree<128>(a, plan, max_query_len, s)
                                         : launch_tree<64>(a, plan, max_query_len, s);
  if (err == kTooLarge)
    return fail(QSA_ERR_UNSUPPORTED, name + ": too many requests, rows or heads");
  if (err != hipSuccess)
    return fail(QSA_ERR_HIP, name + " launch: " + hipGetErrorString(err));
  return QSA_OK;
}

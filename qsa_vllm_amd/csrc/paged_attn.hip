// Causal attention over the paged cache, whole or windowed, bf16 or 4 bits, gfx950.
//
// Request b's rows of this step are its last tokens: row i of n has position
// p = length - n + i, and attends over the positions j <= p with j > p - window or
// j < sinks (all of them without a window):
//
//   o = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m},   s_j = q . k_j / sqrt(D)
//
// in one pass with a running maximum and sum, then sigmoid(gate) if given. A row
// that sees nothing gets zeros.
//
// A workgroup takes a tile of 32 W (token, head) rows of one kv head, 32 a wave, and
// streams the positions that any of them sees through LDS, 64 a stage:
//
//   S^T[token][row] = K (A, 32 tokens x 16 dims) Q^T (B, 16 dims x 32 rows)
//   O^T[dim][row]  += V^T (A, 32 dims x 16 tokens) P^T (B, 16 tokens x 32 rows)
//
// on mfma_f32_32x32x16_bf16. P^T is the lane's own exponentials, so it never leaves
// registers; V^T comes from row-major V rows in LDS by the transposing LDS read. The
// exponentials are rounded to bf16, the matrix cores' type (2^-8 of a weight at
// most), and the rounded ones are what is summed, in fp32: the weights that meet V
// add up to 1 (but not those of few rows from 4 bits, below). They are taken from a
// base that follows the row's maximum only when that has passed it by 2^8, so that
// most stages rescale nothing.
//
// A 4-bit cache (kv4.h) is taken apart on the way into LDS: its values are bf16
// values, exactly, and the rest is the same.
//
// 8192 rows of 16 heads of 128 in a window of 4096 are 206 Gflop and take 256 us, 0.80
// Pflop/s (the card's large bf16 product reaches 1.2). No unit is full: by the counters
// the matrix cores are busy for 0.44 of the waves' time and the vector unit for 0.47 (from
// 4 bits, in tiles of 256 rows, 0.33 and 0.51). A stage is 32 products of a wave and 210
// vector instructions (masks, exponentials, packing, addresses), which follow each other
// in a wave; two waves a SIMD, of workgroups of their own, overlap them in part. Tried and
// slower: two groups of four waves in turns in one workgroup (313 us), 64 rows a wave
// (380: too few registers), raised priority around the products (274), maxima and sums in
// four chains each (268).
#include "paged_stage.h"
#include "../../include/qsa_hip.h"
#include "kv4.h"

#include <algorithm>
#include <climits>

namespace qsa {
namespace {

constexpr int kCUs = 256;
constexpr int kTok = 64;  // tokens of a stage
constexpr int kNoWindow = INT_MAX / 2;  // past every position

struct PagedArgs {
  const uint16_t* q;
  int64_t q_row, q_head;  // elements
  // bf16: both caches, strides in units of 16 bytes, heads in bytes. 4 bits: k is the
  // data, kb its block stride in units of 16 bytes and kh its head stride.
  const char* k;
  const char* v;
  uint32_t kb, kt, vb, vt;
  int64_t kh, vh;
  int num_blocks, page_size;
  FastDiv page_div;
  const int32_t* table;
  int64_t table_row;
  int table_width;
  int requests;
  const int32_t* seq_lens;
  const int32_t* query_start_loc;
  int window, sinks;  // window: kNoWindow for none
  uint16_t* out;
  int64_t out_row, out_head;
  const uint16_t* gate;
  int64_t g_row, g_head, g_dim;
  float* part_out;  // tiles' pieces [pieces][tile rows][D], normalised
  float* part_lse;  // [pieces][tile rows], log2
  float* row_out;   // the same of requests of few rows, [pieces][16][D]
  float* row_lse;
  int32_t* row_pieces;  // [requests]: first piece, pieces of a kv head
  int rows, num_q_heads, kv_heads, group;
  FastDiv group_div;
  int max_rows;   // a request's rows at most
  int splits;     // pieces of a tile's positions
  int tiles;      // of the launch
  int few;        // (row, head)s of a kv head up to which a request is one of few rows; 0: none is
  int few_groups;  // workgroups of the launch for those, 0: one for each request and kv head
  int few_waves;   // of such a workgroup
  float scale_log2;
};

// One request's rows and tokens, kept within the query tensor and the page table
// whatever the device arrays say.
struct Request {
  int row0, rows;   // rows that are computed
  int first;        // position of row 0, negative where the length is too short
  int length;       // tokens within the table
};
__device__ __forceinline__ Request make_request(const PagedArgs& a, int first, int last, int length) {
  Request r;
  r.row0 = min(max(first, 0), a.rows);
  const int rows = min(max(last, r.row0), a.rows) - r.row0;
  r.rows = min(rows, a.max_rows);
  const int len = min(max(length, 0), kNoWindow);
  r.first = len - rows;
  r.length = (int)min((int64_t)len, (int64_t)a.table_width * a.page_size);
  return r;
}
__device__ __forceinline__ Request load_request(const PagedArgs& a, int b) {  // b: a lane's own
  return make_request(a, a.query_start_loc[b], a.query_start_loc[b + 1], a.seq_lens[b]);
}
__device__ __forceinline__ Request uniform_request(const PagedArgs& a, int b) {  // b: the wave's
  return make_request(a, load_uniform(a.query_start_loc + b), load_uniform(a.query_start_loc + b + 1),
                      load_uniform(a.seq_lens + b));
}
__device__ __forceinline__ bool is_few(const PagedArgs& a, const Request& r) {
  return r.rows * a.group <= a.few;
}
template <int R>
__device__ __forceinline__ int tiles_of(const PagedArgs& a, const Request& r) {
  return is_few(a, r) ? 0 : (r.rows * a.group + R - 1) / R;
}

// The request that holds item `place` where request b has count(b) of them; `place`
// becomes the place within it. a.requests if there are fewer.
template <typename F>
__device__ __forceinline__ int locate(const PagedArgs& a, int& place, F count) {
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < a.requests; b0 += 64) {
    const int n = b0 + lane < a.requests ? count(load_request(a, b0 + lane)) : 0;
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

// The positions that rows at p_lo .. p_hi see, as stages of T.
template <int T>
struct Span {
  int p_lo, p_hi, end;           // end: past the last position that a row may see
  int sink_stages, main, count;  // main: the first stage of the window
  __device__ __forceinline__ int base(int stage) const {
    return (stage < sink_stages ? stage : main + stage - sink_stages) * T;
  }
  // Whether the rows see the stage differently.
  __device__ __forceinline__ bool mixed(const PagedArgs& a, int base) const {
    return base + T - 1 > p_lo || (base <= p_hi - a.window && base + T > a.sinks);
  }
};
template <int T>
__device__ __forceinline__ Span<T> make_span(const PagedArgs& a, const Request& r, int i_lo, int i_hi) {
  Span<T> s;
  s.p_lo = r.first + i_lo;
  s.p_hi = r.first + i_hi;
  s.end = max(0, min(s.p_hi + 1, r.length));
  const int begin = max(0, min(s.p_lo - a.window + 1, s.end));
  s.main = begin / T;
  const int sink_end = min(a.sinks, s.end);
  s.sink_stages = min((sink_end + T - 1) / T, s.main);
  s.count = s.sink_stages + max(0, (s.end + T - 1) / T - s.main);
  return s;
}
// Bits 0 .. n - 1.
__device__ __forceinline__ uint64_t below(int n) {
  return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1;
}
// What the row at position p sees of base .. base + 63.
__device__ __forceinline__ uint64_t seen_from(const PagedArgs& a, int p, int base) {
  return below(p + 1 - base) & (~below(p - a.window + 1 - base) | below(a.sinks - base));
}
// Whether any of eight bf16 values is an infinity or NaN; and 0 in their place.
__device__ __forceinline__ bool not_finite(const u32x4& v) {
  bool bad = false;
#pragma unroll
  for (int w = 0; w < 4; ++w)
    bad |= (v[w] & 0x7F80u) == 0x7F80u || (v[w] & 0x7F800000u) == 0x7F800000u;
  return bad;
}
__device__ __forceinline__ u32x4 finite_or_zero(u32x4 v) {
#pragma unroll
  for (int w = 0; w < 4; ++w)
    v[w] &= ((v[w] & 0x7F80u) == 0x7F80u ? 0u : 0xFFFFu) |
            ((v[w] & 0x7F800000u) == 0x7F800000u ? 0u : 0xFFFF0000u);
  return v;
}

// c + both halves of a pair of bf16 values.
__device__ __forceinline__ float add_pair(uint32_t pair, float c) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair),
                                         __builtin_bit_cast(bf16x2, 0x3F803F80u), c, false);
}

// 8 codes (a word of kv4.h) as bf16 values in dim order.
template <bool K>
__device__ __forceinline__ u32x4 values4(uint32_t codes, uint32_t word) {
  const float s = __builtin_bit_cast(float, (word & 0xFFF0u) << 16);
  const float zs = -(float)(word & 15u) * s;
  const uint32_t even = codes & 0x0F0F0F0Fu, odd = codes >> 4 & 0x0F0F0F0Fu;  // a code a byte
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b0 = K ? (i % 2 ? odd : even) >> 8 * (i / 2) : even >> 8 * i;
    const uint32_t b1 = K ? b0 >> 16 : odd >> 8 * i;
    // (All exact, and exact in bf16, so the packing truncates nothing.)
    r[i] = perm_b32(__builtin_bit_cast(uint32_t, __builtin_fmaf((float)(b1 & 255u), s, zs)),
                    __builtin_bit_cast(uint32_t, __builtin_fmaf((float)(b0 & 255u), s, zs)),
                    0x07060302u);
  }
  return r;
}

// Workgroup `block` of a tiles' launch.
template <int D, int W, bool KV4>
__device__ __forceinline__ void paged_tile(const PagedArgs& a, int block) {
  constexpr int R = 32 * W;          // rows of the tile
  constexpr int U = D / 8;           // 16-byte units of a row
  constexpr int kSteps = D / 16;     // products of a score
  constexpr int kDims = D / 32;
  constexpr int kStage = kTok * D * 2;                    // bytes of K or V of a stage
  constexpr int kLoads = 2 * kTok * U / (64 * W);         // 16-byte loads of a lane, K then V
  constexpr int kCodes = kLoads / 2;                      // pairs of code words of a lane, K then V
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;

  // Which tile: kv heads innermost, then the pieces, then the tiles.
  const int kv = block % a.kv_heads;
  const int split = block / a.kv_heads % a.splits;
  const int tile_id = block / a.kv_heads / a.splits;
  int tile = tile_id;
  const int b = locate(a, tile, [&](const Request& r) { return tiles_of<R>(a, r); });
  if (b >= a.requests) return;
  const Request rq = uniform_request(a, b);
  // The last rows see most: they come first.
  tile = tiles_of<R>(a, rq) - 1 - tile;
  const int rows = rq.rows * a.group, m0 = tile * R;
  const Span<kTok> span = make_span<kTok>(a, rq, a.group_div.div(m0), a.group_div.div(min(m0 + R, rows) - 1));
  const int s_begin = (int)((int64_t)span.count * split / a.splits);
  const int s_end = (int)((int64_t)span.count * (split + 1) / a.splits);
  const int32_t* const trow = a.table + b * a.table_row;

  // The lane's query row, dims 16 s + 8 h .. + 7.
  const int m = min(m0 + wave * 32 + n, rows - 1);
  const int node = a.group_div.div(m);
  const int head = kv * a.group + m - node * a.group;
  const int pos = rq.first + node;
  bf16x8 q[kSteps];
  {
    const uint16_t* src = a.q + (int64_t)(rq.row0 + node) * a.q_row + head * a.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      q[s] = __builtin_bit_cast(bf16x8, load_u32x4(src + 16 * s + 8 * h));
  }

  // Page of token base + lane; past the end some other's. (Without a token there is no
  // stage, and any address does.)
  auto load_page = [&](int stage) {
    return *(span.end > 0 ? trow + a.page_div.div(min(span.base(stage) + lane, span.end - 1))
                          : a.seq_lens);
  };
  // Offsets (16-byte units) of token base + lane. In place of what is no token the last
  // one is loaded, or the cache's first rows where a page is missing: those scores are masked.
  struct Places {
    uint32_t k, v;
    int at;
    uint64_t valid;
  };
  auto places = [&](int stage, int page) __attribute__((always_inline)) {
    Places p;
    const int t = min(span.base(stage) + lane, span.end - 1);
    const bool paged = page >= 0 && page < a.num_blocks;
    const bool ok = paged && span.base(stage) + lane < span.end && stage < s_end;
    const int live = paged ? -1 : 0;
    p.at = (t - a.page_div.div(t) * a.page_size) & live;
    const uint32_t block = page & live;
    p.k = block * a.kb + (KV4 ? 0 : p.at * a.kt);
    p.v = KV4 ? p.k : block * a.vb + p.at * a.vt;
    p.valid = __ballot(ok);
    return p;
  };
  const char* const zero = reinterpret_cast<const char*>(g_qsa_zero_rows);
  const char* const k_rows = a.num_blocks > 0 ? a.k + kv * a.kh : zero;  // (no cache: zeros)
  const char* const v_rows = a.num_blocks > 0 && !KV4 ? a.v + kv * a.vh : zero;

  // bf16: straight into LDS. Block i of a stage (64 units) is moved by wave i mod W.
  auto start_loads = [&](const Places& p, char* stage) __attribute__((always_inline)) {
    uint32_t o[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const bool is_v = i >= kLoads / 2;
      const int tok = ((i % (kLoads / 2)) * W + wave) * (64 / U) + lane / U;
      o[i] = __builtin_amdgcn_ds_bpermute(4 * tok, is_v ? p.v : p.k);
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const bool is_v = i >= kLoads / 2;
      const int block = (i % (kLoads / 2)) * W + wave;
      const int tok = block * (64 / U) + lane / U;
      const int unit = lane % U ^ (is_v ? v_swizzle<D>(tok) : k_swizzle<D>(tok));
      load_to_lds((is_v ? v_rows : k_rows) + unit * 16 + ((uint64_t)o[i] << 4),
                  stage + (is_v ? kStage : 0) + block * 1024);
    }
  };
  // 4 bits: codes and words into registers, values into LDS a stage later. Pair i of a
  // lane is two words of a token's K (first half of the pairs) or V codes.
  u32x2 codes[KV4 ? kCodes : 1];
  uint32_t words[KV4 ? kCodes : 1];
  const Kv4Page lay{a.page_size, D};
  const int64_t v_codes = a.num_blocks > 0 ? lay.v_codes() : 0;
  const int64_t k_words = a.num_blocks > 0 ? lay.k_words() : 0;
  const int64_t v_words = a.num_blocks > 0 ? lay.v_words() : 0;
  constexpr int kPairs = kTok * (D / 16);  // of K, and of V
  auto load_codes = [&](const Places& p) {
#pragma unroll
    for (int i = 0; i < kCodes; ++i) {
      const int pair = i * 64 * W + threadIdx.x;
      const bool is_v = pair >= kPairs;
      const int at = pair % kPairs, tok = at / (D / 16), part = at % (D / 16);
      const uint32_t o = __builtin_amdgcn_ds_bpermute(4 * tok, p.k);
      const int place = __builtin_amdgcn_ds_bpermute(4 * tok, p.at);
      const char* const src = k_rows + ((uint64_t)o << 4);
      codes[i] = load_u32x2(src + (is_v ? v_codes : 0) + (int64_t)place * lay.row() + part * 8);
      // K: words of groups 2 (part % (D / 64)) and the next. V: both of one group.
      const char* const w = src + (is_v ? v_words : k_words) + (int64_t)place * lay.words();
      if (is_v) words[i] = reinterpret_cast<const uint16_t*>(w)[part / 2] * 0x10001u;
      else words[i] = reinterpret_cast<const uint32_t*>(w)[part % (D / 64)];
    }
  };
  auto store_values = [&](char* stage) {
#pragma unroll
    for (int i = 0; i < kCodes; ++i) {
      const int pair = i * 64 * W + threadIdx.x;
      const bool is_v = pair >= kPairs;
      const int at = pair % kPairs, tok = at / (D / 16), part = at % (D / 16);
      if (!is_v) {
        // word 2 part of b D / 32 + a: group a, dims 8 b ..
        const int first = 2 * part % (D / 32), b8 = 2 * part / (D / 32);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<u32x4*>(stage + k_at<D>(tok, 4 * (first + e) + b8)) =
              values4<true>(codes[i][e], words[i] >> (16 * e));
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<u32x4*>(stage + kStage + v_at<D>(tok, 2 * part + e)) =
              values4<false>(codes[i][e], words[i] >> (16 * e));
      }
    }
  };

  f32x16 o[kDims];
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
  float sum = 0.0f, base = kNegInf;  // base: what the exponents are taken from
  const float slack = kSlack / a.scale_log2;
  bool poisoned = false;

  int buffer = 0;
  uint64_t valid = 0, valid_next = 0;
  if (s_begin < s_end) {
    const Places p = places(s_begin, load_page(s_begin));
    valid_next = p.valid;
    if constexpr (KV4) {
      load_codes(p);
      store_values(lds);
    } else {
      start_loads(p, lds);
    }
  }
  int page_next = load_page(s_begin + 1);

  // (The pointers are said to be apart: the compiler would otherwise wait for the loads
  // into `next` before it reads V from `here`.)
  auto step = [&](int stage, char* __restrict here, char* __restrict next) {
    __builtin_amdgcn_s_waitcnt(kLoadsDone);
    __syncthreads();  // the stage is in LDS, and the one before has been read by all
    valid = valid_next;
    if (stage + 1 < s_end) {
      const Places p = places(stage + 1, page_next);
      valid_next = p.valid;
      if constexpr (KV4) load_codes(p);
      else start_loads(p, next);
    }
    page_next = load_page(stage + 2);
    const int t0 = span.base(stage);
    const bool mixed = valid != ~0ull || span.mixed(a, t0);
    if (mixed) {
      // V may hold infinities or NaN that a row must not see (0 times them is NaN). The
      // whole stage's are taken as 0 here, and added at the end to the rows that see them.
      u32x4* const v = reinterpret_cast<u32x4*>(here + kStage);
      bool bad = false;
      for (int i = lane; i < kTok * U; i += 64) bad |= not_finite(v[i]);
      if (__any(bad)) {  // every wave has looked at the whole stage
        __syncthreads();
        for (int i = threadIdx.x; i < kTok * U; i += 64 * W) v[i] = finite_or_zero(v[i]);
        __syncthreads();
        poisoned = true;
      }
    }

    f32x16 sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[u][r] = 0.0f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const bf16x8 kf =
            __builtin_bit_cast(bf16x8, load_u32x4(here + k_at<D>(32 * u + n, 2 * s + h)));
        sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, q[s], sc[u], 0, 0, 0);
      }
    }
    if (mixed) {
      // bit 8 (r / 4) + r % 4 of each subtile's: the lane's token 8 (r / 4) + 4 h + r % 4
      const uint64_t seen = (valid & seen_from(a, pos, t0)) >> (4 * h);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          sc[u][r] = (seen >> (32 * u + 8 * (r / 4) + r % 4)) & 1 ? sc[u][r] : kNegInf;
    }

    float top = kNegInf;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, sc[u][r]);
    if (__any(top > base + slack)) {
      // Only the rows that passed it: a row's bits are its own. (A row that has seen
      // nothing yet has -inf, and so has one whose scores are NaN.)
      const float row_top = max_over_halves(top);
      const float to = row_top > base + slack ? row_top : base;
      const float shrink = to == kNegInf ? 1.0f : fast_exp2((base - to) * a.scale_log2);
      base = to;
      sum *= shrink;
#pragma unroll
      for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= shrink;
    }

    const float from = base == kNegInf ? 0.0f : -base * a.scale_log2;
    const int vt = 4 * h + (lane & 15) / 4;  // the lane's token of a transposing read
    const char* const v_lane = here + kStage + vt * D * 2 + (lane & 1) * 8;
    const int v_unit = (lane >> 4 & 1) * 2 + (lane >> 1 & 1), v_swz = v_swizzle<D>(vt);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t p[8];  // weights of tokens 8 (i / 2) + 4 h + 2 (i % 2) .., bf16 pairs
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = pack_bf16x2(fast_exp2(__builtin_fmaf(sc[u][2 * i], a.scale_log2, from)),
                           fast_exp2(__builtin_fmaf(sc[u][2 * i + 1], a.scale_log2, from)));
        sum = add_pair(p[i], sum);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const bf16x8 pb = __builtin_bit_cast(
            bf16x8, (u32x4{p[4 * half], p[4 * half + 1], p[4 * half + 2], p[4 * half + 3]}));
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          const char* const src =
              v_lane + (32 * u + 16 * half) * D * 2 + ((4 * d + v_unit) ^ v_swz) * 16;
          const s16x4 v0 = read_transposed(src);
          const s16x4 v1 = read_transposed(src + 8 * D * 2);
          const s16x8 vf = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, vf), pb, o[d],
                                                         0, 0, 0);
        }
      }
    }
    if constexpr (KV4) {
      if (stage + 1 < s_end) store_values(next);
    }
  };
  for (int stage = s_begin; stage < s_end; ++stage) {
    step(stage, lds + buffer * 2 * kStage, lds + (buffer ^ 1) * 2 * kStage);
    buffer ^= 1;
  }
  sum = sum_wave_halves(sum);

  if (poisoned) {
    for (int stage = s_begin; stage < s_end; ++stage) {
      const int t0 = span.base(stage);
      for (int i = 0; i < kTok && t0 + i < span.end; ++i) {
        const int page = trow[a.page_div.div(t0 + i)];
        if (page < 0 || page >= a.num_blocks) continue;
        const int at = t0 + i - a.page_div.div(t0 + i) * a.page_size;
        // A stage with a page missing is one that was looked at, as all mixed ones are.
        if (!(span.mixed(a, t0) || t0 + kTok > span.end)) {
          bool whole = true;
          for (int k = 0; k < kTok; ++k) {
            const int other = trow[a.page_div.div(t0 + k)];
            whole &= other >= 0 && other < a.num_blocks;
          }
          if (whole) break;
        }
        if (!(seen_from(a, pos, t0) >> i & 1)) continue;
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int dim = 32 * d + 8 * j + 4 * h;
            if constexpr (KV4) {
              const char* const src = a.k + kv * a.kh + ((uint64_t)((uint32_t)page * a.kb) << 4);
              const uint32_t word = *reinterpret_cast<const uint16_t*>(
                  src + lay.v_words() + (int64_t)at * lay.words() + d * 2);
              if ((word & 0x7F80u) == 0x7F80u)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[d][4 * j + r] = __builtin_nanf("");
            } else {
              const char* const src = a.v + kv * a.vh +
                                      ((uint64_t)((uint32_t)page * a.vb + (uint32_t)at * a.vt) << 4);
              const u32x2 x = load_u32x2(src + dim * 2);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                // (a positive weight times an infinity or NaN is the same)
                const uint32_t bits = r & 1 ? x[r >> 1] & 0xFFFF0000u : x[r >> 1] << 16;
                if ((bits & 0x7F800000u) == 0x7F800000u)
                  o[d][4 * j + r] += __builtin_bit_cast(float, bits);
              }
            }
          }
      }
    }
  }

  if (m0 + wave * 32 + n >= rows) return;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // a row that sees nothing: zeros
  if (a.splits > 1) {
    const int64_t at =
        (((int64_t)tile_id * a.kv_heads + kv) * a.splits + split) * R + wave * 32 + n;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(a.part_out + at * D + 32 * d + 8 * j + 4 * h) =
            f32x4{o[d][4 * j] * inv, o[d][4 * j + 1] * inv, o[d][4 * j + 2] * inv,
                  o[d][4 * j + 3] * inv};
    if (h == 0)
      a.part_lse[at] = sum == 0.0f ? kNegInf : base * a.scale_log2 + __log2f(sum);
    return;
  }
  uint16_t* const dst = a.out + (int64_t)(rq.row0 + node) * a.out_row + head * a.out_head;
  const uint16_t* const gate =
      a.gate ? a.gate + (int64_t)(rq.row0 + node) * a.g_row + head * a.g_head : nullptr;
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float y[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        y[r] = o[d][4 * j + r] * inv;
        if (gate) y[r] *= gate_factor(gate[(32 * d + 8 * j + 4 * h + r) * a.g_dim]);
      }
      u32x2 w = {pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
      __builtin_memcpy(dst + 32 * d + 8 * j + 4 * h, &w, 8);
    }
}

template <int D, int W, bool KV4>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2, 2))) void
paged_tile_kernel(PagedArgs a) {
  paged_tile<D, W, KV4>(a, blockIdx.x);
}

// Joining of pieces in a fixed order, D / 4 lanes a (row, head) and WAYS times as many
// that take every WAYS-th piece, some of them in flight together.
template <int WAYS>
constexpr int kMergeThreads = WAYS == 32 ? 1024 : 256;
template <int D, int WAYS>
constexpr int kMergeHeads = kMergeThreads<WAYS> / (D / 4) / WAYS;  // of a workgroup

// `pieces` of a (row, head), `stride` rows apart from `first` on, times the gate, to dst.
// All of a workgroup's threads come here; `write`: whether the head is one of the row's.
template <int D, int WAYS>
__device__ __forceinline__ void join_pieces(const float* out, const float* lses, int64_t first,
                                            int64_t stride, int pieces, bool write, uint16_t* dst,
                                            const uint16_t* gate, int64_t gate_dim) {
  constexpr int kLanes = D / 4, kAhead = WAYS == 1 ? 4 : 8, kGroups = kMergeThreads<WAYS> / kLanes;
  __shared__ f32x4 acc_lds[kGroups][kLanes];
  __shared__ float top_lds[kGroups], sum_lds[kGroups];
  const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes, way = grp % WAYS;
  // Running maximum and sum over the way's pieces.
  float top = kNegInf, sum = 0.0f;
  f32x4 acc = {0, 0, 0, 0};
  for (int s = way; s < pieces; s += WAYS * kAhead) {
    float lse[kAhead];
    f32x4 part[kAhead];
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const int64_t at = first + min(s + e * WAYS, pieces - 1) * stride;
      lse[e] = lses[at];
      part[e] = *reinterpret_cast<const f32x4*>(out + at * D + 4 * lane);
    }
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      if (s + e * WAYS >= pieces) break;
      const float to = fmaxf(top, lse[e]);
      const float from = to == kNegInf ? 0.0f : to;
      const float old = fast_exp2(top - from), f = fast_exp2(lse[e] - from);
      top = to;
      sum = sum * old + f;
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] = acc[r] * old + f * part[e][r];
    }
  }
  if constexpr (WAYS > 1) {
    acc_lds[grp][lane] = acc;
    if (lane == 0) {
      top_lds[grp] = top;
      sum_lds[grp] = sum;
    }
    __syncthreads();
    if (way > 0) return;
    float all = top;
#pragma unroll
    for (int w = 1; w < WAYS; ++w) all = fmaxf(all, top_lds[grp + w]);
    const float from = all == kNegInf ? 0.0f : all;
    const float own = fast_exp2(top - from);
    sum *= own;
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] *= own;
#pragma unroll
    for (int w = 1; w < WAYS; ++w) {
      const float f = fast_exp2(top_lds[grp + w] - from);
      sum += f * sum_lds[grp + w];
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] += f * acc_lds[grp + w][lane][r];
    }
  }
  if (!write) return;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  float y[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    y[r] = acc[r] * inv;
    if (gate) y[r] *= gate_factor(gate[(4 * lane + r) * gate_dim]);
  }
  u32x2 w = {pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
  __builtin_memcpy(dst + 4 * lane, &w, 8);
}

// A tile's pieces: a workgroup for some heads of a row.
template <int D, int W, int WAYS>
__global__ __launch_bounds__(kMergeThreads<WAYS>) void paged_merge_kernel(PagedArgs a, int head_groups) {
  constexpr int R = 32 * W, kHeads = kMergeHeads<D, WAYS>;
  // The row's request: rows past the last one are of none.
  const int hg = blockIdx.x % head_groups, row = blockIdx.x / head_groups;
  const int wave_lane = threadIdx.x & 63;
  int tiles = 0, b = -1;
  for (int b0 = 0; b0 < a.requests; b0 += 64) {
    Request r = {0, 0, 0, 0};
    if (b0 + wave_lane < a.requests) r = load_request(a, b0 + wave_lane);
    const uint64_t mine = __ballot(row >= r.row0 && row < r.row0 + r.rows);
    const int at = mine ? __ffsll((unsigned long long)mine) - 1 : 64;
    int before = wave_lane < at ? tiles_of<R>(a, r) : 0;
#pragma unroll
    for (int w = 32; w > 0; w /= 2) before += __shfl_xor(before, w, 64);
    tiles += uniform(before);
    if (mine) {
      b = b0 + at;
      break;
    }
  }
  if (b < 0) return;
  const Request rq = uniform_request(a, b);
  if (is_few(a, rq)) return;
  const int of_group = threadIdx.x / (D / 4) / WAYS;
  const int head = min(hg * kHeads + of_group, a.num_q_heads - 1);
  const int kv = a.group_div.div(head);
  const int m = (row - rq.row0) * a.group + head - kv * a.group;
  // (Requests whose rows overlap may have more tiles than the launch.)
  const int tile = tiles + tiles_of<R>(a, rq) - 1 - m / R;
  const int64_t first = ((int64_t)min(tile, a.tiles - 1) * a.kv_heads + kv) * a.splits * R + m % R;
  join_pieces<D, WAYS>(a.part_out, a.part_lse, first, R, a.splits,
                       tile < a.tiles && hg * kHeads + of_group < a.num_q_heads,
                       a.out + row * a.out_row + head * a.out_head,
                       a.gate ? a.gate + row * a.g_row + head * a.g_head : nullptr, a.g_dim);
}

// ---------------------------------------------------------------------------
// Few rows
// ---------------------------------------------------------------------------
//
// A request of at most 16 (row, head)s a kv head (single tokens, a few drafted ones)
// is bound by its K/V, which one workgroup reads for all of its rows. The four waves
// of a workgroup take blocks of positions in turn, each on its own: K goes from memory
// into the matrix cores' operand registers, V through the wave's own LDS, so that no
// wave waits for another until they join their results at the end. The scores are the
// transposed products of 16 rows, mfma_f32_16x16x32_bf16, weights and sums as above
// from a bf16 cache.
//
// Work is shared out by blocks: requests of more blocks than an equal share of the
// whole launch are cut into pieces, found on the device, which a second kernel joins.
// 112 tokens in windows of 4096 of a bf16 cache take 98 us with the joining, 472 MB at
// the rate of a large copy. A wave has its next block on the way in registers; a second
// one behind it made all cases slower (130 us here: registers spilled, and short pieces
// load blocks that they do not have).
//
// From a 4-bit cache the codes themselves are the matrix cores' operands, as the bf16
// numbers 16 + c (a code's bits in the fraction of 16.0), and the groups' scales and
// zero points come in afterwards, by 32 dims (one product):
//
//   s_t  = sum_G s_tG sum_d (16 + c_td) q_d  -  sum_G (16 s_tG + s_tG z_tG) sum_d q_d
//   o_d += sum_t (p_t s_tG) (16 + c_td)  -  sum_t (p_t s_tG) (16 + z_tG)
//
// the last sums by one more product each: 16 s and s z are bf16 numbers (of 4 and 8
// bits), the sums of q are split in three. p_t s_tG is rounded to bf16 for both (2^-8 of
// a weight at most); the weights p_t that are summed are not, as a group's scale is not
// theirs. Over n tokens the sums reach 2^8 n 31 s, where s is at most 0.15 of V's largest
// magnitude: under 2^128 for magnitudes of 2^117 / n, which is the range that the interface
// states. 64 tokens on 1024 .. 8192, 82 MB, take 30 us with the joining, one on 131071 24
// us (values of fp32 taken apart first: 208 and 330). 64 positions are 860 vector
// instructions (the codes' bits 256, scales of K and V 128, exponentials 50), and the vector
// unit is busy for 0.59 of the waves' time, the matrix cores for 0.13: the rest is waiting,
// with two waves a SIMD (206 registers) and one block on its way for each.

constexpr int kFew = 16;

template <int D, bool KV4, int W>
struct RowShape {
  static constexpr int kBlock = KV4 ? 64 : 32;    // positions of a wave's block
  static constexpr int kSub = kBlock / 16;
  static constexpr int kGroups = D / 32;
  static constexpr int kVRow = KV4 ? D / 2 : 2 * D;  // bytes of a V row in LDS
  static constexpr int kV = kBlock * kVRow;
  // 4 bits: K's scales (fp32), its 16 s and s z (bf16), V's scales (fp32), V's 16 + z (bf16)
  static constexpr int kWords = KV4 ? kGroups * kBlock * 14 : 0;
  static constexpr int kWave = kV + kWords;
  static constexpr int kMerge = 16 * (D + 2) * 4;  // a wave's result
  static constexpr int kLds = W * (kWave > kMerge ? kWave : kMerge);
};

template <int T>
__device__ __forceinline__ int blocks_of(const PagedArgs& a, const Request& r) {
  return r.rows > 0 && is_few(a, r) ? make_span<T>(a, r, 0, r.rows - 1).count : 0;
}
// What a workgroup of the launch takes: a piece of a request and kv head.
struct Share {
  Request rq;
  int request, kv, piece, pieces;
  int first;  // the request's first piece of the launch
};
__device__ __forceinline__ int pieces_of(int blocks, int per) {
  return max(1, (int)(((unsigned)blocks + (unsigned)per - 1u) / (unsigned)per));
}
// Blocks of a piece, such that all pieces are at most a.few_groups: a request's last
// piece may be short, so that there are up to blocks / per + requests for a kv head.
__device__ __forceinline__ int piece_blocks(const PagedArgs& a, int blocks, int requests) {
  if (!a.few_groups) return INT_MAX;
  const unsigned spare = max(a.few_groups / a.kv_heads - requests, 1);
  return max(a.few_waves, (int)(((unsigned)blocks + spare - 1u) / spare));
}
// False where the launch has no such workgroup.
template <int T>
__device__ __forceinline__ bool find_share(const PagedArgs& a, int place, Share& s) {
  if (a.requests == 1) {
    s.rq = uniform_request(a, 0);
    if (s.rq.rows <= 0 || !is_few(a, s.rq)) return false;
    const int blocks = uniform(blocks_of<T>(a, s.rq));
    s.request = s.first = 0;
    s.pieces = pieces_of(blocks, piece_blocks(a, blocks, 1));
  } else {
    // A lane for each request, the first 64 kept.
    const int lane = threadIdx.x & 63;
    const Request none = {0, 0, 0, 0};
    const Request own = lane < a.requests ? load_request(a, lane) : none;
    auto request = [&](int b0) {
      return b0 == 0 ? own : b0 + lane < a.requests ? load_request(a, b0 + lane) : none;
    };
    int blocks = 0, live = 0;
    for (int b0 = 0; b0 < a.requests; b0 += 64) {
      const Request r = request(b0);
      blocks += blocks_of<T>(a, r);
      live += r.rows > 0 && is_few(a, r);
    }
#pragma unroll
    for (int w = 32; w > 0; w /= 2) {
      blocks += __shfl_xor(blocks, w, 64);
      live += __shfl_xor(live, w, 64);
    }
    const int per = piece_blocks(a, uniform(blocks), uniform(live));
    s.request = -1;
    s.first = 0;
    for (int b0 = 0; b0 < a.requests; b0 += 64) {
      const Request r = request(b0);
      const int n = r.rows > 0 && is_few(a, r) ? pieces_of(blocks_of<T>(a, r), per) * a.kv_heads : 0;
      int end = n;  // inclusive sum over the lanes
#pragma unroll
      for (int w = 1; w < 64; w *= 2) {
        const int below = __shfl_up(end, w, 64);
        end += lane >= w ? below : 0;
      }
      const uint64_t past = __ballot(end > place);
      if (past) {
        const int at = __ffsll((unsigned long long)past) - 1;
        const int before = __builtin_amdgcn_readlane(end - n, at);
        s.request = b0 + at;
        s.pieces = __builtin_amdgcn_readlane(n, at) / a.kv_heads;
        s.rq.row0 = __builtin_amdgcn_readlane(r.row0, at);
        s.rq.rows = __builtin_amdgcn_readlane(r.rows, at);
        s.rq.first = __builtin_amdgcn_readlane(r.first, at);
        s.rq.length = __builtin_amdgcn_readlane(r.length, at);
        s.first += before;
        place -= before;
        break;
      }
      const int all = __builtin_amdgcn_readlane(end, 63);
      s.first += all;
      place -= all;
    }
    if (s.request < 0) return false;
  }
  s.kv = place / s.pieces;
  s.piece = place - s.kv * s.pieces;
  return s.kv < a.kv_heads;
}

__device__ __forceinline__ float sum_over_quarters(float v) {
  v = sum_wave_halves(v);
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// Codes of nibbles i and i + 4 of a word, i = 0 .. 3, as bf16 pairs of 16 + c.
// `bits` is 0x00780078, in a vector register: two constants do not fit one instruction.
__device__ __forceinline__ u32x4 codes_of(uint32_t w, uint32_t bits) {
  u32x4 r;
  r[0] = ((w << 3) & bits) | 0x41804180u;
  r[1] = ((w >> 1) & bits) | 0x41804180u;
  r[2] = ((w >> 5) & bits) | 0x41804180u;
  r[3] = ((w >> 9) & bits) | 0x41804180u;
  return r;
}
__device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// Lane i of 16 passes the address of 16 codes (8 bytes) and gets code i of all 16.
__device__ __forceinline__ u32x2 read_transposed4(const char* p) {
  typedef int v2i __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) v2i*)p));
}
// Where 16-byte unit `unit` of a token's V codes lies: the units of 64 tokens' same
// place are spread over the banks.
template <int D>
__device__ __forceinline__ int v4_at(int tok, int unit) {
  return tok * (D / 2) + (unit ^ (D == 128 ? tok >> 2 & 3 : tok >> 3 & 1)) * 16;
}

// Workgroup `place` of a launch for requests of few rows.
template <int D, bool KV4, int W>
__device__ __forceinline__ void paged_rows(const PagedArgs& a, int place) {
  typedef RowShape<D, KV4, W> S;
  constexpr int T = S::kBlock;
  constexpr int U = D / 8;
  constexpr int kGroups = S::kGroups;  // of 32 dims: products of a score
  constexpr int kDims = D / 16;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;

  Share share;
  if (!find_share<T>(a, place, share)) return;
  const Request rq = share.rq;
  const int kv = share.kv, pieces = share.pieces;
  if (a.few_groups && kv == 0 && share.piece == 0 && threadIdx.x == 0) {
    a.row_pieces[2 * share.request] = share.first;
    a.row_pieces[2 * share.request + 1] = pieces;
  }
  const int rows = rq.rows * a.group;
  const Span<T> span = make_span<T>(a, rq, 0, rq.rows - 1);
  const int s_begin = (int)((int64_t)span.count * share.piece / pieces);
  const int s_end = (int)((int64_t)span.count * (share.piece + 1) / pieces);
  const int32_t* const trow = a.table + share.request * a.table_row;

  // The lane's query row, dims 32 s + 8 g .. + 7.
  const int m = min(n, rows - 1);
  const int node = a.group_div.div(m);
  const int head = kv * a.group + m - node * a.group;
  const int pos = rq.first + node;
  u32x4 q[kGroups];
  {
    const uint16_t* src = a.q + (int64_t)(rq.row0 + node) * a.q_row + head * a.q_head;
#pragma unroll
    for (int s = 0; s < kGroups; ++s) q[s] = load_u32x4(src + 32 * s + 8 * g);
  }
  // 4 bits: minus the sums of q over the groups, in three bf16 parts (all 24 bits), part g
  // in quarter g, as the operand that meets 16 s and s z.
  u32x4 q_sums = {0, 0, 0, 0};
  if constexpr (KV4) {
#pragma unroll
    for (int s = 0; s < kGroups; ++s) {
      float v = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) v += bf16_lo(q[s][i]) + bf16_hi(q[s][i]);
      float rest = -sum_over_quarters(v);
#pragma unroll
      for (int part = 0; part < 3; ++part) {
        const uint32_t top = __builtin_bit_cast(uint32_t, rest) & 0xFFFF0000u;
        q_sums[s] = g == part ? top | top >> 16 : q_sums[s];
        rest -= __builtin_bit_cast(float, top);
      }
    }
  }

  char* const mine = lds + wave * S::kWave;  // V, then a 4-bit cache's words
  char* const words = mine + S::kV;
  const char* const zero = reinterpret_cast<const char*>(g_qsa_zero_rows);
  const Kv4Page lay{a.page_size, D};
  const bool any = a.num_blocks > 0;  // (no cache: zeros)
  const char* const k_rows = any ? a.k + kv * a.kh : zero;
  const char* const v_rows = !any ? zero : KV4 ? k_rows + lay.v_codes() : a.v + kv * a.vh;
  const char* const k_words = k_rows + (any ? lay.k_words() : 0);
  const char* const v_words = k_rows + (any ? lay.v_words() : 0);

  // Page of token base + lane, past the end the last one's. (Without a token any address does.)
  auto load_page = [&](int block) __attribute__((always_inline)) {
    return *(span.end > 0 ? trow + a.page_div.div(min(span.base(block) + lane % T, span.end - 1))
                          : a.seq_lens);
  };
  // A block on its way, all of it in registers.
  struct Block {
    u32x4 k[S::kSub][KV4 ? 1 : kGroups];
    u32x4 v[S::kV / 1024];
    u32x2 kw, vw;  // 4 bits: the lane's token's words
    uint64_t valid;
  };
  // In place of what is no token the last one is loaded, or the cache's first rows where
  // a page is missing: those scores are masked.
  auto start = [&](int block, int page, Block& r) __attribute__((always_inline)) {
    const int own = span.base(block) + lane % T;
    const int t = min(own, span.end - 1);
    const bool paged = page >= 0 && page < a.num_blocks && span.end > 0;
    const uint32_t at = paged ? t - a.page_div.div(t) * a.page_size : 0;
    const uint32_t in = paged ? page : 0;
    r.valid = __ballot(paged && own < span.end && block < s_end);
    // (units of 16 bytes)
    const uint32_t k_at = in * a.kb + at * (KV4 ? D / 32 : a.kt);
    const uint32_t v_at = KV4 ? k_at : in * a.vb + at * a.vt;
#pragma unroll
    for (int u = 0; u < S::kSub; ++u) {
      const uint32_t o = __builtin_amdgcn_ds_bpermute(4 * (16 * u + n), k_at);
      const char* const src = k_rows + ((uint64_t)o << 4) + (KV4 ? g * (D / 8) : 16 * g);
      if constexpr (KV4 && D == 64) {
        const u32x2 x = load_u32x2(src);
        r.k[u][0] = u32x4{x[0], x[1], 0, 0};
      } else {
#pragma unroll
        for (int s = 0; s < (KV4 ? 1 : kGroups); ++s) r.k[u][s] = load_u32x4(src + 64 * s);
      }
    }
    constexpr int kUnits = S::kVRow / 16;
#pragma unroll
    for (int i = 0; i < S::kV / 1024; ++i) {
      const int tok = i * (64 / kUnits) + lane / kUnits;
      const uint32_t o = __builtin_amdgcn_ds_bpermute(4 * tok, v_at);
      r.v[i] = load_u32x4(v_rows + ((uint64_t)o << 4) + lane % kUnits * 16);
    }
    if constexpr (KV4) {
      const uint64_t from = ((uint64_t)(in * a.kb) << 4) + at * (D / 16);
      if constexpr (D == 128) {
        r.kw = load_u32x2(k_words + from);
        r.vw = load_u32x2(v_words + from);
      } else {
        r.kw = u32x2{*reinterpret_cast<const uint32_t*>(k_words + from), 0};
        r.vw = u32x2{*reinterpret_cast<const uint32_t*>(v_words + from), 0};
      }
    }
  };

  f32x4 o[kDims], oz[KV4 ? kGroups : 1];
#pragma unroll
  for (int d = 0; d < kDims; ++d) o[d] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < (KV4 ? kGroups : 1); ++s) oz[s] = f32x4{0, 0, 0, 0};
  float sum = 0.0f, base = kNegInf;
  const float slack = kSlack / a.scale_log2;
  bool poisoned = false;

  uint32_t bits = 0x00780078u;
  asm volatile("" : "+v"(bits));
  Block now;  // the wave's next block
  start(s_begin + wave, load_page(s_begin + wave), now);
  int page = load_page(s_begin + wave + W);  // of the one behind it

  for (int block = s_begin + wave; block < s_end; block += W) {
    char* const v_lds = mine;
    const uint64_t valid = now.valid;
#pragma unroll
    for (int i = 0; i < S::kV / 1024; ++i) {
      constexpr int kUnits = S::kVRow / 16;
      const int tok = i * (64 / kUnits) + lane / kUnits, unit = lane % kUnits;
      *reinterpret_cast<u32x4*>(mine + (KV4 ? v4_at<D>(tok, unit) : v_at<D>(tok, unit))) = now.v[i];
    }
    const int t0 = span.base(block);
    constexpr uint64_t kAll = T == 64 ? ~0ull : (1ull << (T % 64)) - 1;
    const bool mixed = (valid & kAll) != kAll || span.mixed(a, t0);
    const uint64_t seen = mixed ? valid & seen_from(a, pos, t0) : 0;  // of the lane's row

    f32x4 sc[S::kSub];
    if constexpr (KV4) {
      // The lane's token's words, taken apart for all.
      float* const ks = reinterpret_cast<float*>(words);
      uint32_t* const kz = reinterpret_cast<uint32_t*>(ks + kGroups * T);
      float* const vs = reinterpret_cast<float*>(kz + kGroups * T);
      uint16_t* const vz = reinterpret_cast<uint16_t*>(vs + kGroups * T);
      u32x4 zero_at = {0, 0, 0, 0};
      bool bad = false;
#pragma unroll
      for (int s = 0; s < kGroups; ++s) {
        const uint32_t kw = now.kw[s / 2] >> (16 * (s % 2)), vw = now.vw[s / 2] >> (16 * (s % 2));
        const float scale = __builtin_bit_cast(float, (kw & 0xFFF0u) << 16);
        ks[s * T + lane] = scale;
        zero_at[s] = perm_b32(__builtin_bit_cast(uint32_t, scale * (float)(kw & 15u)),
                              __builtin_bit_cast(uint32_t, scale * 16.0f), 0x07060302u);
        bad |= (vw & 0x7F80u) == 0x7F80u;  // no finite scale, of either sign
        vs[s * T + lane] = __builtin_bit_cast(float, (vw & 0xFFF0u) << 16);
        // Token 16 u + 4 g' + r at the place of its code in the other operand.
        const int u = lane >> 4, gt = lane >> 2 & 3, r = lane & 3;
        vz[((s * 2 + u / 2) * 4 + gt) * 8 + r * 2 + u % 2] = (uint16_t)(0x4180u | (vw & 15u) << 3);
      }
      if constexpr (D == 128)
        *reinterpret_cast<u32x4*>(kz + 4 * lane) = zero_at;
      else
        *reinterpret_cast<u32x2*>(kz + 2 * lane) = u32x2{zero_at[0], zero_at[1]};
      if (mixed && __any(bad)) {
        // V may be NaN where a row must not see it: as in the tiles' kernel.
#pragma unroll
        for (int s = 0; s < kGroups; ++s)
          if ((__builtin_bit_cast(uint32_t, vs[s * T + lane]) & 0x7F800000u) == 0x7F800000u)
            vs[s * T + lane] = 0.0f;
        poisoned = true;
      }
      asm volatile("" ::: "memory");  // other lanes read it: a wave's LDS accesses stay in order
#pragma unroll
      for (int u = 0; u < S::kSub; ++u) {
        if constexpr (D == 128) {
          zero_at = load_u32x4(kz + 4 * (16 * u + n));
        } else {
          const u32x2 x = load_u32x2(kz + 2 * (16 * u + n));
          zero_at = u32x4{x[0], x[1], 0, 0};
        }
        sc[u] = product(zero_at, q_sums, f32x4{0, 0, 0, 0});
#pragma unroll
        for (int s = 0; s < kGroups; ++s) {
          const f32x4 x = product(codes_of(now.k[u][0][s], bits), q[s], f32x4{0, 0, 0, 0});
          const f32x4 scale = *reinterpret_cast<const f32x4*>(ks + s * T + 16 * u + 4 * g);
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[u][r] = __builtin_fmaf(scale[r], x[r], sc[u][r]);
        }
        // (Pinned: the compiler would move the sums behind the branch, and spill.)
        asm volatile("" : "+v"(sc[u]));
      }
    } else {
      if (mixed) {
        // V may hold infinities or NaN that a row must not see: as in the tiles' kernel.
        u32x4* const v = reinterpret_cast<u32x4*>(v_lds);
        bool bad = false;
        for (int i = lane; i < T * U; i += 64) bad |= not_finite(v[i]);
        if (__any(bad)) {
          for (int i = lane; i < T * U; i += 64) v[i] = finite_or_zero(v[i]);
          poisoned = true;
        }
      }
#pragma unroll
      for (int u = 0; u < S::kSub; ++u) {
        sc[u] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < kGroups; ++s) sc[u] = product(now.k[u][s], q[s], sc[u]);
      }
    }
    start(block + W, page, now);
    page = load_page(block + 2 * W);
    if (mixed) {
#pragma unroll
      for (int u = 0; u < S::kSub; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          sc[u][r] = seen >> (16 * u + 4 * g + r) & 1 ? sc[u][r] : kNegInf;
    }

    float top = kNegInf;
#pragma unroll
    for (int u = 0; u < S::kSub; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, sc[u][r]);
    if (__any(top > base + slack)) {
      const float row_top = max_over_quarters(top);
      const float to = row_top > base + slack ? row_top : base;
      const float shrink = to == kNegInf ? 1.0f : fast_exp2((base - to) * a.scale_log2);
      base = to;
      sum *= shrink;
#pragma unroll
      for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[d][r] *= shrink;
      if constexpr (KV4)
#pragma unroll
        for (int s = 0; s < kGroups; ++s)
#pragma unroll
          for (int r = 0; r < 4; ++r) oz[s][r] *= shrink;
    }
    const float from = base == kNegInf ? 0.0f : -base * a.scale_log2;
#pragma unroll
    for (int u = 0; u < S::kSub; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        sc[u][r] = fast_exp2(__builtin_fmaf(sc[u][r], a.scale_log2, from));

    if constexpr (KV4) {
      const float* const vs = reinterpret_cast<const float*>(words) + 2 * kGroups * T;
      const uint16_t* const vz = reinterpret_cast<const uint16_t*>(vs + kGroups * T);
#pragma unroll
      for (int u = 0; u < S::kSub; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += sc[u][r];
      // The lane's V row of a transposing read: code i of its token, in the weights' order.
      const int tok = 16 * (n >> 2) + 4 * g + (n & 3);
#pragma unroll
      for (int s = 0; s < kGroups; ++s) {
        u32x4 p[2];  // weights times scales of subtiles 2 i and 2 i + 1, pairs by token
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f32x4 w[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int u = 2 * i + e;
            w[e] = *reinterpret_cast<const f32x4*>(vs + s * T + 16 * u + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) w[e][r] *= sc[u][r];
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) p[i][r] = pack_bf16x2(w[0][r], w[1][r]);
          oz[s] = product(load_u32x4(vz + ((s * 2 + i) * 4 + g) * 8), p[i], oz[s]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int d = 2 * s + e;
          const u32x2 c = read_transposed4(v_lds + v4_at<D>(tok, d / 2) + d % 2 * 8);
          o[d] = product(codes_of(c[0], bits), p[0], o[d]);
          o[d] = product(codes_of(c[1], bits), p[1], o[d]);
        }
      }
    } else {
      u32x4 p;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = pack_bf16x2(sc[i / 2][2 * (i % 2)], sc[i / 2][2 * (i % 2) + 1]);
        sum = add_pair(p[i], sum);
      }
      const int vt = 4 * g + (n >> 2);
      const char* const v_lane = v_lds + vt * D * 2 + (n & 1) * 8;
      const int v_unit = (n & 3) >> 1, v_swz = v_swizzle<D>(vt);
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        const char* const src = v_lane + ((2 * d + v_unit) ^ v_swz) * 16;
        const s16x4 v0 = read_transposed(src), v1 = read_transposed(src + 16 * D * 2);
        o[d] = product(__builtin_bit_cast(
                           u32x4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7)),
                       p, o[d]);
      }
    }
  }
  sum = sum_over_quarters(sum);
  if constexpr (KV4) {
#pragma unroll
    for (int d = 0; d < kDims; ++d) o[d] -= oz[d / 2];
  }

  if (poisoned) {
    for (int block = s_begin + wave; block < s_end; block += W) {
      const int t0 = span.base(block);
      bool whole = t0 + T <= span.end;  // a page missing: a block that was looked at
      for (int i = 0; i < T && t0 + i < span.end; ++i) {
        const int page = trow[a.page_div.div(t0 + i)];
        whole &= page >= 0 && page < a.num_blocks;
      }
      if (whole && !span.mixed(a, t0)) continue;
      for (int i = 0; i < T && t0 + i < span.end; ++i) {
        const int page = trow[a.page_div.div(t0 + i)];
        if (page < 0 || page >= a.num_blocks || !(seen_from(a, pos, t0) >> i & 1)) continue;
        const int at = t0 + i - a.page_div.div(t0 + i) * a.page_size;
        if constexpr (KV4) {
          const char* const from =
              v_words + ((uint64_t)((uint32_t)page * a.kb) << 4) + (int64_t)at * (D / 16);
#pragma unroll
          for (int d = 0; d < kDims; ++d)
            if ((reinterpret_cast<const uint16_t*>(from)[d / 2] & 0x7F80u) == 0x7F80u)
              o[d] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
          continue;
        }
        const char* const v = a.v + kv * a.vh +
                              ((uint64_t)((uint32_t)page * a.vb + (uint32_t)at * a.vt) << 4);
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          const u32x2 x = load_u32x2(v + (16 * d + 4 * g) * 2);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t bits = r & 1 ? x[r >> 1] & 0xFFFF0000u : x[r >> 1] << 16;
            if ((bits & 0x7F800000u) == 0x7F800000u) o[d][r] += __builtin_bit_cast(float, bits);
          }
        }
      }
    }
  }

  // The waves' shares, joined in wave order by D / 4 lanes a row.
  __syncthreads();  // (all have read their V)
  float* const merge = reinterpret_cast<float*>(lds);
  {
    float* const to = merge + wave * (S::kMerge / 4);
#pragma unroll
    for (int d = 0; d < kDims; ++d)
      *reinterpret_cast<f32x4*>(to + n * D + ((16 * d + 4 * g) ^ ((n & 7) << 2))) = o[d];
    if (g == 0) {
      to[16 * D + n] = base == kNegInf ? kNegInf : base * a.scale_log2;
      to[16 * D + 16 + n] = sum;
    }
  }
  __syncthreads();
  constexpr int kLanes = D / 4;
  const int at = threadIdx.x % kLanes;
  for (int row = threadIdx.x / kLanes; row < rows; row += 64 * W / kLanes) {
    float top = kNegInf;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, merge[w * (S::kMerge / 4) + 16 * D + row]);
    const float from = top == kNegInf ? 0.0f : top;
    f32x4 acc = {0, 0, 0, 0};
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float* const part = merge + w * (S::kMerge / 4);
      const float f = fast_exp2(part[16 * D + row] - from);
      total += f * part[16 * D + 16 + row];
      const f32x4 x = *reinterpret_cast<const f32x4*>(part + row * D + ((4 * at) ^ ((row & 7) << 2)));
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] += f * x[r];
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;  // a row that sees nothing: zeros
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] *= inv;
    if (pieces > 1) {
      const int64_t slot = (int64_t)place * kFew + row;
      *reinterpret_cast<f32x4*>(a.row_out + slot * D + 4 * at) = acc;
      if (at == 0) a.row_lse[slot] = total == 0.0f ? kNegInf : top + __log2f(total);
      continue;
    }
    const int own = a.group_div.div(row);
    const int h = kv * a.group + row - own * a.group;
    const int64_t r0 = rq.row0 + own;
    if (a.gate)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc[r] *= gate_factor(a.gate[r0 * a.g_row + h * a.g_head + (4 * at + r) * a.g_dim]);
    u32x2 w = {pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3])};
    __builtin_memcpy(a.out + r0 * a.out_row + h * a.out_head + 4 * at, &w, 8);
  }
}

template <int D, bool KV4, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2, 3))) void
paged_rows_kernel(PagedArgs a) {
  paged_rows<D, KV4, W>(a, blockIdx.x);
}

// Both in one launch, for a step of prompt chunks and single tokens: the tiles first, as
// they take longest, and few rows on the CUs that they leave.
template <int D, bool KV4>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void
paged_both_kernel(PagedArgs a, int tiles) {
  const int i = blockIdx.x;
  if (i < tiles) paged_tile<D, 4, KV4>(a, i);
  else paged_rows<D, KV4, 4>(a, i - tiles);
}

// The pieces of requests of few rows: a workgroup for some heads of a row.
template <int D, int WAYS>
__global__ __launch_bounds__(kMergeThreads<WAYS>) void paged_rows_merge_kernel(PagedArgs a, int rows_each,
                                                                               int head_groups) {
  constexpr int kHeads = kMergeHeads<D, WAYS>;
  const int hg = blockIdx.x % head_groups;
  const int bi = blockIdx.x / head_groups, b = bi / rows_each, i = bi - b * rows_each;
  const int first_piece = a.row_pieces[2 * b], pieces = a.row_pieces[2 * b + 1];
  const Request rq = uniform_request(a, b);
  // (Only requests of few rows have their pieces written.)
  if (i >= rq.rows || !is_few(a, rq) || pieces <= 1) return;
  if (first_piece < 0 || first_piece + (int64_t)pieces * a.kv_heads > a.few_groups)
    return;  // (requests whose rows overlap: some have no workgroup)
  const int row = rq.row0 + i, of_group = threadIdx.x / (D / 4) / WAYS;
  const int head = min(hg * kHeads + of_group, a.num_q_heads - 1);
  const int kv = a.group_div.div(head);
  const int m = i * a.group + head - kv * a.group;
  join_pieces<D, WAYS>(a.row_out, a.row_lse, ((int64_t)first_piece + (int64_t)kv * pieces) * kFew + m,
                       kFew, pieces, hg * kHeads + of_group < a.num_q_heads,
                       a.out + row * a.out_row + head * a.out_head,
                       a.gate ? a.gate + row * a.g_row + head * a.g_head : nullptr, a.g_dim);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

struct PagedPlan {
  int waves, splits;   // of the tiles
  int64_t tiles;       // of all requests, at most; 0: no launch
  int requests, few, few_groups, few_waves;
  int64_t few_units;   // requests of few rows and kv heads, at most; 0: no launch
};

// The bounds shape the launch: a longer context is computed whole all the same.
PagedPlan make_plan(bool kv4, int rows, int requests, int num_q_heads, int num_kv_heads,
                    int max_query_len, int max_seq_len, int window, int sinks) {
  PagedPlan p = {};
  const int64_t group = num_q_heads / num_kv_heads;
  const int64_t most = std::min(max_query_len, rows) * group;
  p.requests = requests;
  const int64_t all = (int64_t)requests * max_query_len;
  requests = std::min(requests, rows);
  // Positions that n rows see, in whole blocks.
  auto seen = [&](int64_t n) {
    int64_t s = std::min<int64_t>(max_seq_len, (int64_t)window + n);
    return window < max_seq_len ? s + std::min(sinks, max_seq_len) + 2 * kTok : s;
  };
  // Where all requests have as many rows, more than a few, the tiles do for them all
  // (whatever their numbers turn out to be).
  if (group <= kFew && (most <= kFew || rows < all)) {
    p.few = kFew;
    p.few_units = (int64_t)requests * num_kv_heads;
    const int64_t blocks = seen(kFew / group) / (kv4 ? 64 : 32) + 1;
    // Workgroups of 4 waves, pieces of a block a wave at least: 11.4 us for one request of
    // 700 .. 4000 tokens, 12.4 from 4 bits. Where 8 waves have 3 blocks each at most (2 from
    // 4 bits) they are the whole launch: 8.3 us on 300 tokens, 10.3 on 500, 11.7 on 1000
    // from 4 bits, 14.6 and 17.4 at twice that.
    const bool whole = most <= kFew && p.few_units <= kCUs && blocks <= (kv4 ? 16 : 24);
    p.few_waves = whole ? 8 : 4;
    // As many pieces as two workgroups a CU take (one: 2 us less for a single request, but
    // 51 us for 31 for 64 on 1024 .. 8192 of 4 bits), and more than the units, so that long
    // ones are cut: four each up to one a CU (128 requests 130 us for 147 with two, 60 for
    // 68 from 4 bits), two past that (512 requests on 512 .. 2048 145 us for 175 with four).
    if (!whole && blocks > p.few_waves && p.few_units <= 16 * kCUs)
      p.few_groups =
          (int)std::max<int64_t>(2 * kCUs, (p.few_units <= kCUs ? 4 : 2) * p.few_units);
  }
  if (most > p.few) {
    // Tiles of 128 rows, two workgroups a CU; of fewer where requests have no more. Tiles
    // of 256 read K/V half as often and wait for their longest longer: 286 us for 259 on
    // 8192 rows of 16 heads and a window of 4096. From a 4-bit cache, whose values are made
    // once a tile, they are 256: 288 us for 343 on 4 x 500 rows of 16 heads on 8k .. 16k.
    // Beside requests of few rows, in one launch, both have 4 waves; so have chunks of unlike
    // lengths, which may hold such requests (500, 500, 500 and 499 rows 330 us, 4 x 500 275).
    // More than 16 heads a kv head are tiles of 64 rows for single tokens too: 64 tokens of 24
    // heads of one kv head on 1024 .. 8192 48 us, where memory takes 30.
    p.waves = p.few_units || most > 64 ? 4 : 2;
    if (kv4 && !p.few_units && most > 128) p.waves = 8;
    const int64_t tile_rows = 32 * p.waves;
    p.tiles = std::min<int64_t>((rows * group) / tile_rows + requests,
                                requests * ((most + tile_rows - 1) / tile_rows));
    const int64_t stages = (seen(tile_rows / group + 1) + kTok - 1) / kTok;
    // The tiles that there likely are: beside requests of few rows those of the longest
    // allowed, the others being single tokens (64 tokens on 1000 .. 8000 and 4 chunks of 512
    // 161 us, 212 with the bound's pieces; from 4 bits 203 and 338). Many more would fit the
    // bounds, whose workgroups end at once; their pieces' room is kept to 2048 tiles.
    int64_t likely = p.tiles;
    if (p.few_units) {
      const int64_t more = rows - requests;  // rows past the first of each request
      const int64_t chunks = std::max<int64_t>(more / std::max(max_query_len - 1, 1), 1);
      likely = std::min(likely, chunks * (((more / chunks + 1) * group + tile_rows - 1) / tile_rows));
    }
    const int64_t room = std::max<int64_t>(8 * kCUs / std::max<int64_t>(p.tiles * num_kv_heads, 1), 1);
    const int64_t units = std::max<int64_t>(likely * num_kv_heads, 1);
    // Pieces of four stages at least, for two workgroups a CU; of two for one a CU (32 rows
    // on 2000 15.2 us for 17.4, but 1000 on themselves from 4 bits 44 for 31, in two rounds).
    // A workgroup of 8 waves fills a CU: two in turn even out tiles of unlike lengths (four
    // requests on 8k .. 16k 278 us for 341, a prompt of 4096 121 for 167), alike ones need
    // one (500 rows on 8192 69 us for 86; measured for one request, as the rule has it).
    const bool alike = p.waves == 8 && requests == 1 && 4 * (int64_t)max_query_len <= max_seq_len;
    const int64_t most_pieces = std::max(stages / 4, std::min(kCUs / units, stages / 2));
    p.splits = (int)std::max<int64_t>(
        1, std::min({(alike ? kCUs : 2 * kCUs) / units, most_pieces, room}));
  }
  return p;
}

// Floats of the pieces' rows: the tiles', then those of few rows.
size_t tile_rows_of(const PagedPlan& p, int num_kv_heads) {
  return p.splits <= 1 ? 0 : (size_t)p.tiles * num_kv_heads * p.splits * 32 * p.waves;
}
size_t workspace_of(const PagedPlan& p, int num_kv_heads, int head_dim) {
  const size_t rows = tile_rows_of(p, num_kv_heads) + (size_t)p.few_groups * kFew;
  return (rows * (head_dim + 1) + (p.few_groups ? 2 * (size_t)p.requests : 0)) * sizeof(float);
}

// A launch of more than 2^32 - 1 threads is refused.
constexpr hipError_t kTooLarge = hipErrorInvalidConfiguration;
bool fits(int64_t blocks, int threads) { return blocks <= UINT_MAX / threads; }

template <int D>
constexpr int kTileLds = 4 * kTok * D * 2;

// Workgroups of a row of a joining launch.
template <int D, int WAYS>
int head_groups_of(const PagedArgs& a) {
  return (a.num_q_heads + kMergeHeads<D, WAYS> - 1) / kMergeHeads<D, WAYS>;
}
template <int D, int W, int WAYS>
hipError_t launch_tile_merge_ways(const PagedArgs& a, hipStream_t stream) {
  const int head_groups = head_groups_of<D, WAYS>(a);
  hipLaunchKernelGGL((paged_merge_kernel<D, W, WAYS>), dim3((unsigned)((int64_t)a.rows * head_groups)),
                     dim3(kMergeThreads<WAYS>), 0, stream, a, head_groups);
  return hipGetLastError();
}
template <int D, int W>
hipError_t launch_tile_merge(const PagedArgs& a, hipStream_t stream) {
  if (a.splits <= 1) return hipSuccess;
  return (int64_t)a.rows * a.num_q_heads <= 2048 ? launch_tile_merge_ways<D, W, 8>(a, stream)
                                                 : launch_tile_merge_ways<D, W, 1>(a, stream);
}
template <int D, int W, bool KV4>
hipError_t launch_tiles(const PagedArgs& a, int64_t grid, hipStream_t stream) {
  hipLaunchKernelGGL((paged_tile_kernel<D, W, KV4>), dim3((unsigned)grid), dim3(64 * W), kTileLds<D>,
                     stream, a);
  const hipError_t err = hipGetLastError();
  return err != hipSuccess ? err : launch_tile_merge<D, W>(a, stream);
}
template <int D, int WAYS>
hipError_t launch_rows_merge_ways(const PagedArgs& a, int rows_each, hipStream_t stream) {
  const int head_groups = head_groups_of<D, WAYS>(a);
  hipLaunchKernelGGL((paged_rows_merge_kernel<D, WAYS>),
                     dim3((unsigned)((int64_t)a.requests * rows_each * head_groups)),
                     dim3(kMergeThreads<WAYS>), 0, stream, a, rows_each, head_groups);
  return hipGetLastError();
}
template <int D>
hipError_t launch_rows_merge(const PagedArgs& a, int rows_each, hipStream_t stream) {
  if (!a.few_groups) return hipSuccess;
  // The fewer (row, head)s, the more pieces have each: a call of one token on 131071 takes
  // 24 us with 32 ways, 30 with 8, 100 with one; of 64 tokens on 1024 .. 8192 43, 31 and 32;
  // of 512 on 512 .. 2048 143, 85 and 81. (With 32 ways the last sum spills 19 registers of
  // 128, 30 at dim 64, and a launch is few workgroups.)
  const int64_t heads = (int64_t)a.requests * rows_each * a.num_q_heads;
  return heads <= 256    ? launch_rows_merge_ways<D, 32>(a, rows_each, stream)
         : heads <= 2048 ? launch_rows_merge_ways<D, 8>(a, rows_each, stream)
                         : launch_rows_merge_ways<D, 1>(a, rows_each, stream);
}
template <int D, bool KV4, int W>
hipError_t launch_rows(const PagedArgs& a, int64_t grid, int rows_each, hipStream_t stream) {
  constexpr int kLds = RowShape<D, KV4, W>::kLds;
  static_assert(kLds <= 163840, "of a CU");
  hipLaunchKernelGGL((paged_rows_kernel<D, KV4, W>), dim3((unsigned)grid), dim3(64 * W), kLds, stream, a);
  const hipError_t err = hipGetLastError();
  return err != hipSuccess ? err : launch_rows_merge<D>(a, rows_each, stream);
}
template <int D, bool KV4>
hipError_t launch_both(const PagedArgs& a, int64_t tiles, int64_t few, int rows_each, hipStream_t stream) {
  constexpr int kLds = std::max(kTileLds<D>, RowShape<D, KV4, 4>::kLds);
  hipLaunchKernelGGL((paged_both_kernel<D, KV4>), dim3((unsigned)(tiles + few)), dim3(256), kLds, stream,
                     a, (int)tiles);
  hipError_t err = hipGetLastError();
  if (err == hipSuccess) err = launch_tile_merge<D, 4>(a, stream);
  return err != hipSuccess ? err : launch_rows_merge<D>(a, rows_each, stream);
}
template <int D, bool KV4>
hipError_t launch_paged(const PagedArgs& a, const PagedPlan& p, hipStream_t stream) {
  // All launches' sizes before the first: a call that is refused has written nothing. (Only
  // few (row, head)s are joined more than one way.)
  const int64_t few = p.few_groups ? p.few_groups : p.few_units;
  const int64_t tiles = p.tiles * std::max(p.splits, 1) * a.kv_heads;
  const int rows_each = std::min(a.max_rows, kFew / std::min(a.group, kFew));
  const int64_t head_groups = head_groups_of<D, 1>(a);
  if (!fits(tiles + few, 64 * std::max(p.waves, p.few_waves)) ||
      (p.splits > 1 && !fits(a.rows * head_groups, kMergeThreads<1>)) ||
      (p.few_groups && !fits((int64_t)a.requests * rows_each * head_groups, kMergeThreads<1>)))
    return kTooLarge;
  if (tiles && few) return launch_both<D, KV4>(a, tiles, few, rows_each, stream);
  if (few)
    return p.few_waves == 4 ? launch_rows<D, KV4, 4>(a, few, rows_each, stream)
                            : launch_rows<D, KV4, 8>(a, few, rows_each, stream);
  return p.waves == 2   ? launch_tiles<D, 2, KV4>(a, tiles, stream)
         : p.waves == 4 ? launch_tiles<D, 4, KV4>(a, tiles, stream)
                        : launch_tiles<D, KV4 ? 8 : 4, KV4>(a, tiles, stream);
}

// What both entry points check and set; the caches are theirs.
int run_paged(const std::string& name, PagedArgs a, bool kv4, const void* q, int64_t q_row_stride,
              int64_t q_head_stride, int rows, int num_q_heads, int head_dim, int num_blocks,
              int page_size, int num_kv_heads, const int32_t* block_table, int64_t table_row_stride,
              int table_width, int num_requests, const int32_t* seq_lens,
              const int32_t* query_start_loc, int window, int sink_tokens, void* out,
              int64_t out_row_stride, int64_t out_head_stride, const void* gate,
              int64_t gate_row_stride, int64_t gate_head_stride, int64_t gate_dim_stride,
              int max_query_len, int max_seq_len, void* workspace, size_t workspace_bytes,
              void* stream) {
  if ((!block_table && table_width > 0) || !q || !seq_lens || !query_start_loc || !out)
    return fail(QSA_ERR_INVALID, name + ": null tensor pointer");
  if (!aligned16(q) || ((uintptr_t)out & 3u) || ((q_row_stride | q_head_stride) & 7) ||
      ((out_row_stride | out_head_stride) & 1))
    return fail(QSA_ERR_INVALID, name + ": q needs 16-byte alignment and strides of multiples of 8 "
                                        "elements, out 4-byte alignment");
  max_query_len = std::min(max_query_len, rows);
  a.window = window > 0 ? std::min(window, kNoWindow) : kNoWindow;
  if ((int64_t)rows * num_q_heads > INT_MAX / 2)
    return fail(QSA_ERR_UNSUPPORTED, name + ": too many rows or heads");
  const PagedPlan plan = make_plan(kv4, rows, num_requests, num_q_heads, num_kv_heads,
                                   max_query_len, max_seq_len, a.window, sink_tokens);
  const size_t need = workspace_of(plan, num_kv_heads, head_dim);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(QSA_ERR_WORKSPACE, name + ": needs a 16-byte aligned workspace of " +
                                       std::to_string(need) + " bytes");
  if (need) {
    const size_t tile_rows = tile_rows_of(plan, num_kv_heads);
    a.part_out = static_cast<float*>(workspace);
    a.row_out = a.part_out + tile_rows * head_dim;
    a.part_lse = a.row_out + (size_t)plan.few_groups * kFew * head_dim;
    a.row_lse = a.part_lse + tile_rows;
    a.row_pieces = reinterpret_cast<int32_t*>(a.row_lse + (size_t)plan.few_groups * kFew);
  }
  a.q = static_cast<const uint16_t*>(q);
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.num_blocks = num_blocks;
  a.page_size = page_size;
  a.page_div = FastDiv::make(page_size);
  a.table = block_table;
  a.table_row = table_row_stride;
  a.table_width = table_width;
  a.requests = num_requests;
  a.seq_lens = seq_lens;
  a.query_start_loc = query_start_loc;
  a.sinks = sink_tokens;
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
  a.max_rows = max_query_len;
  a.splits = plan.splits;
  a.tiles = (int)plan.tiles;
  a.few = plan.few;
  a.few_groups = plan.few_groups;
  a.few_waves = plan.few_waves;
  a.scale_log2 = 1.4426950408889634f / sqrtf((float)head_dim);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t err = head_dim == 128 ? (kv4 ? launch_paged<128, true>(a, plan, s)
                                                : launch_paged<128, false>(a, plan, s))
                                         : (kv4 ? launch_paged<64, true>(a, plan, s)
                                                : launch_paged<64, false>(a, plan, s));
  if (err == kTooLarge)
    return fail(QSA_ERR_UNSUPPORTED, name + ": too many requests, rows or heads");
  if (err != hipSuccess) return fail(QSA_ERR_HIP, name + " launch: " + hipGetErrorString(err));
  return QSA_OK;
}

// QSA_OK: go on; 1: nothing to do.
int check_sizes(const std::string& name, int rows, int num_q_heads, int num_kv_heads, int head_dim,
                int num_blocks, int page_size, int table_width, int num_requests, int window,
                int sink_tokens, int max_query_len, int max_seq_len) {
  if (rows < 0 || num_requests < 0 || num_blocks < 0 || table_width < 0 || max_query_len < 0 ||
      max_seq_len < 0 || window < 0 || sink_tokens < 0)
    return fail(QSA_ERR_INVALID, name + ": negative size");
  if (rows == 0 || num_requests == 0 || max_query_len == 0) return 1;
  if (head_dim != 64 && head_dim != 128)
    return fail(QSA_ERR_UNSUPPORTED, name + ": head_dim must be 64 or 128");
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads)
    return fail(QSA_ERR_UNSUPPORTED, name + ": query heads must be a multiple of kv heads");
  if (page_size <= 0) return fail(QSA_ERR_INVALID, name + ": page size must be positive");
  return QSA_OK;
}

}  // namespace
}  // namespace qsa

using namespace qsa;

extern "C" size_t qsa_paged_attention_workspace_bytes(int rows, int requests, int num_q_heads,
                                                      int num_kv_heads, int head_dim, int window,
                                                      int sink_tokens, int max_query_len,
                                                      int max_seq_len) {
  if (rows <= 0 || requests <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads ||
      head_dim <= 0 || max_query_len <= 0 || max_seq_len < 0 || window < 0 || sink_tokens < 0)
    return 0;
  size_t need = 0;  // for either cache
  for (const bool kv4 : {false, true})
    need = std::max(need, workspace_of(make_plan(kv4, rows, requests, num_q_heads, num_kv_heads,
                                                 std::min(max_query_len, rows), max_seq_len,
                                                 window > 0 ? std::min(window, kNoWindow) : kNoWindow,
                                                 sink_tokens),
                                       num_kv_heads, head_dim));
  return need;
}

extern "C" int qsa_window_attention(
    const void* q, int64_t q_row_stride, int64_t q_head_stride, int rows, int num_q_heads,
    int head_dim, const void* k_cache, int64_t k_block_stride, int64_t k_token_stride,
    int64_t k_head_stride, const void* v_cache, int64_t v_block_stride, int64_t v_token_stride,
    int64_t v_head_stride, int num_blocks, int page_size, int num_kv_heads,
    const int32_t* block_table, int64_t table_row_stride, int table_width, int num_requests,
    const int32_t* seq_lens, const int32_t* query_start_loc, int window, int sink_tokens, void* out,
    int64_t out_row_stride, int64_t out_head_stride, const void* gate, int64_t gate_row_stride,
    int64_t gate_head_stride, int64_t gate_dim_stride, int max_query_len, int max_seq_len,
    void* workspace, size_t workspace_bytes, void* stream) {
  const std::string name = "qsa_window_attention";
  const int st = check_sizes(name, rows, num_q_heads, num_kv_heads, head_dim, num_blocks, page_size,
                             table_width, num_requests, window, sink_tokens, max_query_len,
                             max_seq_len);
  if (st) return st > 0 ? QSA_OK : st;
  // (an empty cache has no address and is not read)
  if ((!k_cache || !v_cache) && num_blocks > 0)
    return fail(QSA_ERR_INVALID, name + ": null tensor pointer");
  if (!aligned16(k_cache) || !aligned16(v_cache) ||
      ((k_block_stride | k_token_stride | k_head_stride | v_block_stride | v_token_stride |
        v_head_stride) & 7))
    return fail(QSA_ERR_INVALID, name + ": the caches need 16-byte alignment and strides of "
                                        "multiples of 8 elements");
  // The kernel's offsets are 32-bit counts of 16 bytes.
  const int64_t k_span = cache_span(num_blocks, k_block_stride, page_size, k_token_stride);
  const int64_t v_span = cache_span(num_blocks, v_block_stride, page_size, v_token_stride);
  if (k_span < 0 || v_span < 0 || std::max(k_span, v_span) / 8 >= kNoToken)
    return fail(QSA_ERR_UNSUPPORTED, name + ": the cache must span under 64 GiB");
  PagedArgs a = {};
  a.k = static_cast<const char*>(k_cache);
  a.v = static_cast<const char*>(v_cache);
  a.kb = (uint32_t)(k_block_stride / 8);
  a.kt = (uint32_t)(k_token_stride / 8);
  a.kh = 2 * k_head_stride;
  a.vb = (uint32_t)(v_block_stride / 8);
  a.vt = (uint32_t)(v_token_stride / 8);
  a.vh = 2 * v_head_stride;
  return run_paged(name, a, false, q, q_row_stride, q_head_stride, rows, num_q_heads, head_dim,
                   num_blocks, page_size, num_kv_heads, block_table, table_row_stride, table_width,
                   num_requests, seq_lens, query_start_loc, window, sink_tokens, out,
                   out_row_stride, out_head_stride, gate, gate_row_stride, gate_head_stride,
                   gate_dim_stride, max_query_len, max_seq_len, workspace, workspace_bytes, stream);
}

extern "C" int qsa_int4_kv_attention(
    const void* q, int64_t q_row_stride, int64_t q_head_stride, int rows, int num_q_heads,
    int head_dim, const void* cache, int64_t block_stride, int64_t head_stride, int num_blocks,
    int page_size, int num_kv_heads, const int32_t* block_table, int64_t table_row_stride,
    int table_width, int num_requests, const int32_t* seq_lens, const int32_t* query_start_loc,
    int window, int sink_tokens, void* out, int64_t out_row_stride, int64_t out_head_stride,
    const void* gate, int64_t gate_row_stride, int64_t gate_head_stride, int64_t gate_dim_stride,
    int max_query_len, int max_seq_len, void* workspace, size_t workspace_bytes, void* stream) {
  const std::string name = "qsa_int4_kv_attention";
  const int st = check_sizes(name, rows, num_q_heads, num_kv_heads, head_dim, num_blocks, page_size,
                             table_width, num_requests, window, sink_tokens, max_query_len,
                             max_seq_len);
  if (st) return st > 0 ? QSA_OK : st;
  if (!cache && num_blocks > 0) return fail(QSA_ERR_INVALID, name + ": null tensor pointer");
  if (!aligned16(cache) || block_stride < 0 || head_stride < 0 || ((block_stride | head_stride) & 15))
    return fail(QSA_ERR_INVALID, name + ": the cache needs 16-byte alignment and strides of "
                                        "multiples of 16 bytes");
  // The kernel's offsets are 32-bit counts of 16 bytes.
  const int64_t page_units = Kv4Page{page_size, head_dim}.bytes() / 16, stride = block_stride / 16;
  if (stride >= kNoToken || std::max(num_blocks - 1, 0) * stride + page_units >= kNoToken)
    return fail(QSA_ERR_UNSUPPORTED, name + ": the cache must span under 64 GiB");
  PagedArgs a = {};
  a.k = static_cast<const char*>(cache);
  a.kb = (uint32_t)(block_stride / 16);
  a.kh = head_stride;
  return run_paged(name, a, true, q, q_row_stride, q_head_stride, rows, num_q_heads, head_dim,
                   num_blocks, page_size, num_kv_heads, block_table, table_row_stride, table_width,
                   num_requests, seq_lens, query_start_loc, window, sink_tokens, out,
                   out_row_stride, out_head_stride, gate, gate_row_stride, gate_head_stride,
                   gate_dim_stride, max_query_len, max_seq_len, workspace, workspace_bytes, stream);
}

// Rules on logits before sampling: penalties for repeated tokens, biases and
// grammar masks, one pass over each row.
//
// Row r of request b, token v (its count among the spoken tokens c, in the
// prompt or spoken: seen):
//
//   y = x;  seen: y = x > 0 ? x / repetition : x * repetition
//   y -= frequency c;  c > 0: y -= presence;  y += sum of b's biases on v
//   y = -inf where the row's grammar bit v is 0
//
// all in fp32. Spoken tokens are the request's history past its prompt and, for
// a drafted node, its visible ancestors' tokens (itself among them).
//
// The pass is bound by memory: a logit read (2 or 4 bytes), its result written
// (4), a grammar bit. A workgroup takes a chunk of the vocabulary for one row, or
// for several rows of one request (a drafted tree's):
//
//   1. it counts the request's history within the chunk in LDS, with LDS atomics
//      (whole numbers: any order gives the same counts);
//   2. it lists the chunk's special columns, those of biases and of drafted
//      tokens, whose values differ by row or need a sum, sorts the list by column
//      and marks them in the table;
//   3. it streams its rows, four vectors of a thread in flight, each logit by its
//      count alone, and leaves the special columns;
//   4. it computes those, one (row, column) a thread: the visible nodes' tokens
//      on top of the count, the biases in list order.
//
// A history is scanned once per chunk, so chunks are as large as LDS allows for
// two workgroups a CU, unless there would be too few workgroups.
//
// Measured: 128 rows x 99072 fp32, histories of 512 - 32768 tokens, 35 us (2.9 TB/s
// of the logits, results and masks); 8 x 61 drafted nodes x 49536 bf16 51 us (2.9
// TB/s); one row of 49536 6.5 us, the chain of loads before the stream. A history of
// one repeated token serialises its LDS atomics: 128 such rows take 92 us.
#include "qsa_common.h"
#include "../../include/qsa_hip.h"

#include <algorithm>
#include <climits>

namespace qsa {
namespace {

constexpr int kThreads = 512;
constexpr int kCUs = 256;
constexpr int kMinChunk = 2048;   // vocabulary entries of a workgroup, at least; at most
constexpr int kMaxChunk = 25344;  // what fits 64 KiB of LDS (two workgroups a CU) with 16-bit
constexpr int kMaxChunkWide = 13440;  // counts, and with 32-bit ones
constexpr int kRounds = 2;            // workgroups wanted for each CU
constexpr int kMaxNarrow = 65535;     // history tokens that 16 bits count
constexpr int kTreeRows = 8;          // rows of a workgroup with drafted trees
constexpr int kMaxNodes = 1024;       // a request's nodes and biases: what the list holds
constexpr int kMaxBiases = 1024;
constexpr int kBatch = 4;             // vectors of a thread in flight
constexpr float kNegInf = -__builtin_huge_valf();

enum LogitType { kFp32 = 0, kBf16 = 1, kFp16 = 2 };

struct LogitsArgs {
  const void* logits;
  int64_t in_row;
  float* out;
  int64_t out_row;
  int rows, vocab;
  int64_t vocab_start;
  const int32_t* token_to_req;
  int requests;
  const int32_t* history;
  int64_t history_row;
  int history_width;
  const int32_t* history_lens;
  const int32_t* prompt_lens;
  const float* repetition;
  const float* frequency;
  const float* presence;
  const int32_t* bias_ids;
  const float* bias_values;
  int64_t bias_id_row, bias_value_row;
  int biases;
  const int32_t* allowed;
  int64_t allowed_row;
  const int32_t* draft_tokens;
  const int32_t* ancestors;
  int64_t ancestor_row;
  int words;
  const int32_t* query_start_loc;
  int chunks, chunk, group_rows;
};

template <int TYPE>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
  if constexpr (TYPE == kFp32) return static_cast<const float*>(p)[i];
  else if constexpr (TYPE == kBf16)
    return __builtin_bit_cast(float, (uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
  else return (float)static_cast<const _Float16*>(p)[i];
}

// 16 bytes of logits (4 or 8) as they lie in memory, 4-byte aligned; and one of them.
template <int TYPE>
constexpr int kVec = TYPE == kFp32 ? 4 : 8;
__device__ __forceinline__ u32x4 load_16(const void* p) {
  u32x4 v;
  __builtin_memcpy(&v, __builtin_assume_aligned(p, 4), 16);
  return v;
}
template <int TYPE>
__device__ __forceinline__ float logit_of(const u32x4& v, int e) {
  if constexpr (TYPE == kFp32) {
    return __builtin_bit_cast(float, (uint32_t)v[e]);
  } else {
    const uint32_t pair = v[e >> 1];
    if constexpr (TYPE == kBf16) return e & 1 ? bf16_hi(pair) : bf16_lo(pair);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(pair >> (16 * (e & 1))));
  }
}

struct RowRules {
  float repetition, frequency, presence;
};

// A logit of a token said `spoken` times (and seen: in the prompt or spoken).
__device__ __forceinline__ float penalised(float x, bool seen, uint32_t spoken, const RowRules& r) {
  if (seen) x = x > 0.0f ? x / r.repetition : x * r.repetition;
  if (spoken) x = x - r.frequency * (float)spoken - r.presence;
  return x;
}

// Special columns of a chunk. An entry is a column, whether it is a bias (else a
// drafted node's token), and which of the request's. Sorted, a column's entries
// lie side by side, its nodes first, then its biases in list order.
constexpr int kMaxSpecials = kMaxNodes + kMaxBiases;
constexpr uint32_t kBias = 0x8000u;
static_assert(kMaxNodes <= kBias && kMaxBiases <= kBias && kMaxChunk <= 65536, "16 bits each");
struct Specials {
  __attribute__((aligned(16))) uint32_t entry[kMaxSpecials];
  int wave[kThreads / 64];
};

// Appends the threads' entries in thread order; returns the list's new length.
__device__ __forceinline__ int append(Specials& list, int length, uint32_t column, uint32_t size,
                                      uint32_t source) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool take = column < size;
  const uint64_t mask = __ballot(take);
  if (lane == 0) list.wave[wave] = __popcll(mask);
  __syncthreads();
  int at = length;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    const int n = list.wave[w];
    at += w < wave ? n : 0;
    length += n;
  }
  if (take) {
    at += __popcll(mask & ((1ull << lane) - 1));
    list.entry[at] = column << 16 | source;
  }
  __syncthreads();
  return length;
}

// Sorts the list: no two entries are alike, so an entry's place is how many are
// smaller. Every thread compares its entries with all, 16 at a time from one
// address for the whole wave. (A list of 300 entries takes about 1 us, of 1000
// 18. 8 x 64 rows, 2000 columns, 1024 biases a request: 63 us in all; 2.2 ms with a
// pass over the list for every row and entry instead. One column listed 1024 times
// is added up by one thread a row: 200 us.)
__device__ __forceinline__ void sort(Specials& list, int length) {
  constexpr int kOwn = kMaxSpecials / kThreads, kStep = 16;
  const int padded = (length + kStep - 1) / kStep * kStep;
  if ((int)threadIdx.x < padded - length) list.entry[length + threadIdx.x] = ~0u;
  uint32_t mine[kOwn];
  int place[kOwn];
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const int e = threadIdx.x + o * kThreads;
    mine[o] = e < length ? list.entry[e] : 0u;
    place[o] = 0;
  }
  __syncthreads();
  for (int j = 0; j < padded; j += kStep) {
    u32x4 other[kStep / 4];
#pragma unroll
    for (int i = 0; i < kStep / 4; ++i)
      other[i] = *reinterpret_cast<const u32x4*>(list.entry + j + 4 * i);
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
      if (o * kThreads >= length) break;
#pragma unroll
      for (int i = 0; i < kStep; ++i) place[o] += other[i / 4][i % 4] < mine[o];
    }
  }
  __syncthreads();
#pragma unroll
  for (int o = 0; o < kOwn; ++o)
    if ((int)threadIdx.x + o * kThreads < length) list.entry[place[o]] = mine[o];
  __syncthreads();
}

// The chunk's table in LDS: how often each token was said (WIDE: 32 bits, else
// 16), which were in the prompt, and which columns are special.
template <bool WIDE>
struct Table {
  uint32_t *counts, *prompt, *special;
  static __host__ __device__ __forceinline__ int words(int chunk) {
    return (WIDE ? chunk : chunk / 2) + 2 * (chunk / 32);
  }
  __device__ __forceinline__ Table(uint32_t* lds, int chunk)
      : counts(lds), prompt(lds + (WIDE ? chunk : chunk / 2)), special(prompt + chunk / 32) {}
  __device__ __forceinline__ void say(uint32_t at) {
    if constexpr (WIDE) atomicAdd(&counts[at], 1u);
    else atomicAdd(&counts[at >> 1], at & 1 ? 0x10000u : 1u);
  }
  __device__ __forceinline__ void see(uint32_t at) { atomicOr(&prompt[at >> 5], 1u << (at & 31)); }
  __device__ __forceinline__ void mark(uint32_t at) { atomicOr(&special[at >> 5], 1u << (at & 31)); }
  __device__ __forceinline__ uint32_t said(int at) const {
    return WIDE ? counts[at] : (counts[at >> 1] >> (16 * (at & 1))) & 0xFFFFu;
  }
  __device__ __forceinline__ u32x4 said4(int at) const {  // at a multiple of 4
    if constexpr (WIDE) {
      return *reinterpret_cast<const u32x4*>(counts + at);
    } else {
      const u32x2 c = *reinterpret_cast<const u32x2*>(counts + at / 2);
      return u32x4{c[0] & 0xFFFFu, c[0] >> 16, c[1] & 0xFFFFu, c[1] >> 16};
    }
  }
};

template <int TYPE, bool VEC, bool WIDE>
__global__ __launch_bounds__(kThreads) void logits_kernel(LogitsArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  __shared__ Specials list;
  Table<WIDE> table(lds, a.chunk);
  const bool penalise = a.repetition || a.frequency || a.presence;
  const bool ruled = penalise || a.biases > 0;
  const int base = (blockIdx.x % a.chunks) * a.chunk;
  const int size = min(a.chunk, a.vocab - base);
  // The chunk's first token id. Ids lie below 2^31 (checked on the host), so that
  // a negative one's distance from it, taken without sign, is past any chunk.
  const uint32_t first = (uint32_t)a.vocab_start + (uint32_t)base;
  int row = (int)(blockIdx.x / a.chunks) * a.group_rows;
  const int row_end = min(a.rows, row + a.group_rows);

  // The rows of one request at a time.
  while (row < row_end) {
    const int req = a.token_to_req ? load_uniform(a.token_to_req + row) : row;
    int rows = 1;
    if (a.token_to_req)
      while (row + rows < row_end && load_uniform(a.token_to_req + row + rows) == req) ++rows;
    // A thread's next vectors of the rows, and their grammar bits. The first are
    // asked for before the table is built.
    constexpr int V = kVec<TYPE>;
    const int vec_end = VEC ? size / V * V : 0;
    const int per_row = vec_end / V, items = rows * per_row;
    const uint32_t* const allowed = reinterpret_cast<const uint32_t*>(a.allowed) + base / 32;
    auto bits_at = [&](int m, int i) -> uint32_t {
      return a.allowed ? allowed[m * a.allowed_row + i / 32] >> (i & 31) : ~0u;
    };
    u32x4 x[kBatch];
    uint32_t bits[kBatch];
    int m[kBatch], i[kBatch];
    auto fetch = [&](int k) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int item = min(k + b * kThreads, items - 1);
        m[b] = row + (rows > 1 ? item / per_row : 0);
        i[b] = V * (item - (m[b] - row) * per_row);
        x[b] = load_16(static_cast<const char*>(a.logits) +
                       (m[b] * a.in_row + base + i[b]) * (TYPE == kFp32 ? 4 : 2));
        bits[b] = bits_at(m[b], i[b]);
      }
    };
    if (items > 0) fetch(threadIdx.x);

    const bool live = ruled && req >= 0 && req < a.requests;  // else the grammar mask alone
    int specials = 0;
    if (live) {
      // The first drafted tokens and biases: asked for before the rest.
      int node0 = 0, all_nodes = 0;
      if (penalise && a.ancestors) {
        node0 = max(load_uniform(a.query_start_loc + req), 0);
        const int end = max(min(load_uniform(a.query_start_loc + req + 1), a.rows), 0);
        all_nodes = min(end - node0, 32 * a.words);
      }
      auto draft = [&](int j) {
        return j < all_nodes ? (uint32_t)a.draft_tokens[node0 + j] - first : ~0u;
      };
      auto bias_id = [&](int j) {
        return j < a.biases ? (uint32_t)a.bias_ids[req * a.bias_id_row + j] - first : ~0u;
      };
      const uint32_t draft0 = draft(threadIdx.x);
      const uint32_t id0 = bias_id(threadIdx.x);

      __syncthreads();  // the last request's table has been read
      for (int w = threadIdx.x; w < (Table<WIDE>::words(a.chunk) + 3) / 4; w += kThreads)
        reinterpret_cast<u32x4*>(lds)[w] = u32x4{0, 0, 0, 0};
      __syncthreads();
      if (penalise && a.history) {
        const int len = min(max(load_uniform(a.history_lens + req), 0), a.history_width);
        const int prompt = a.prompt_lens ? load_uniform(a.prompt_lens + req) : 0;
        const int32_t* const h = a.history + req * a.history_row;
        // Prompt tokens set a bit, the later ones add up.
        auto see = [&](int token) {
          const uint32_t at = (uint32_t)token - first;
          if (at < (uint32_t)size) table.see(at);
        };
        auto say = [&](int token) {
          const uint32_t at = (uint32_t)token - first;
          if (at < (uint32_t)size) table.say(at);
        };
        int done = 0;
        if (((uintptr_t)h & 15u) == 0) {
          done = len & ~3;
          for (int i = 4 * threadIdx.x; i < done; i += 4 * kBatch * kThreads) {
            i32x4 t[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
              t[b] = *reinterpret_cast<const i32x4*>(h + min(i + 4 * b * kThreads, done - 4));
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
              const int j = i + 4 * b * kThreads;
              if (j >= done) break;
              if (j >= prompt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) say(t[b][e]);
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  if (j + e < prompt) see(t[b][e]);
                  else say(t[b][e]);
                }
              }
            }
          }
        }
        for (int i = done + threadIdx.x; i < len; i += kThreads) {
          if (i < prompt) see(h[i]);
          else say(h[i]);
        }
      }
      for (int j = 0; j < all_nodes; j += kThreads)
        specials = append(list, specials, j ? draft(j + threadIdx.x) : draft0, size, j + threadIdx.x);
      for (int j = 0; j < a.biases; j += kThreads)
        specials = append(list, specials, j ? bias_id(j + threadIdx.x) : id0, size,
                          kBias | (j + threadIdx.x));
      for (int e = threadIdx.x; e < specials; e += kThreads) table.mark(list.entry[e] >> 16);
      if (specials > 1) sort(list, specials);
      else __syncthreads();
    }

    RowRules r = {1.0f, 0.0f, 0.0f};
    if (live && a.repetition) r.repetition = load_uniform(a.repetition + req);
    if (live && a.frequency) r.frequency = load_uniform(a.frequency + req);
    if (live && a.presence) r.presence = load_uniform(a.presence + req);
    // The ordinary columns.
    if constexpr (VEC) {
      for (int k = threadIdx.x; k < items; k += kBatch * kThreads) {
        if (k >= kBatch * kThreads) fetch(k);
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          if (k + b * kThreads >= items) break;
          float* const out = a.out + m[b] * a.out_row + base + i[b];
#pragma unroll
          for (int h = 0; h < V; h += 4) {
            f32x4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = logit_of<TYPE>(x[b], h + e);
            const int at = i[b] + h;
            uint32_t skip = 0;
            if (live) {
              const u32x4 c = table.said4(at);
              const uint32_t seen = table.prompt[at / 32] >> (at & 31) & 15u;
              skip = table.special[at / 32] >> (at & 31) & 15u;
              if (c[0] | c[1] | c[2] | c[3] | seen) {
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = penalised(y[e], c[e] || seen >> e & 1u, c[e], r);
              }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!((bits[b] >> (h + e)) & 1u)) y[e] = kNegInf;
            if (skip) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!(skip >> e & 1u)) out[h + e] = y[e];
            } else {
              *reinterpret_cast<f32x4*>(out + h) = y;
            }
          }
        }
      }
    }
    for (int m = row; m < row + rows; ++m)
      for (int i = vec_end + threadIdx.x; i < size; i += kThreads) {
        float y = load_logit<TYPE>(a.logits, m * a.in_row + base + i);
        if (live) {
          if (table.special[i / 32] >> (i & 31) & 1u) continue;
          const uint32_t c = table.said(i);
          y = penalised(y, c || table.prompt[i / 32] >> (i & 31) & 1u, c, r);
        }
        if (!(bits_at(m, i) & 1u)) y = kNegInf;
        a.out[m * a.out_row + base + i] = y;
      }

    // The special ones, each by its column's first entry.
    for (int k = threadIdx.x; k < rows * specials; k += kThreads) {
      const int m = row + k / specials, e = k % specials;
      const int column = list.entry[e] >> 16;
      if (e > 0 && (int)(list.entry[e - 1] >> 16) == column) continue;
      const float x = load_logit<TYPE>(a.logits, m * a.in_row + base + column);
      const uint32_t bits = bits_at(m, column);
      uint32_t spoken = table.said(column);
      float bias = 0.0f;
      bool biased = false;
      for (int j = e; j < specials; ++j) {
        const uint32_t entry = list.entry[j];
        if ((int)(entry >> 16) != column) break;
        const int source = entry & (kBias - 1);
        if (entry & kBias) {
          const float value = a.bias_values[req * a.bias_value_row + source];
          bias = biased ? bias + value : value;
          biased = true;
        } else {
          const uint32_t word = (uint32_t)a.ancestors[m * a.ancestor_row + (source >> 5)];
          spoken += (word >> (source & 31)) & 1u;
        }
      }
      float y = penalised(x, spoken || table.prompt[column / 32] >> (column & 31) & 1u, spoken, r);
      if (biased) y += bias;
      a.out[m * a.out_row + base + column] = bits & 1u ? y : kNegInf;
    }
    row += rows;
  }
}

template <int TYPE, bool WIDE>
void launch_table(const LogitsArgs& a, bool vec, unsigned grid, size_t lds, hipStream_t stream) {
  if (vec)
    hipLaunchKernelGGL((logits_kernel<TYPE, true, WIDE>), dim3(grid), dim3(kThreads), lds, stream, a);
  else
    hipLaunchKernelGGL((logits_kernel<TYPE, false, WIDE>), dim3(grid), dim3(kThreads), lds, stream, a);
}

template <int TYPE>
void launch(const LogitsArgs& a, bool vec, bool wide, unsigned grid, bool ruled, hipStream_t stream) {
  const size_t words = wide ? Table<true>::words(a.chunk) : Table<false>::words(a.chunk);
  const size_t lds = ruled ? (words + 3) / 4 * 16 : 0;
  if (wide) launch_table<TYPE, true>(a, vec, grid, lds, stream);
  else launch_table<TYPE, false>(a, vec, grid, lds, stream);
}

}  // namespace
}  // namespace qsa

using namespace qsa;

extern "C" int qsa_process_logits(
    const void* logits, int logits_type, int64_t logits_row_stride, float* out,
    int64_t out_row_stride, int rows, int vocab, int64_t vocab_start, const int32_t* token_to_req,
    int num_requests, const int32_t* history, int64_t history_row_stride, int history_width,
    const int32_t* history_lens, const int32_t* prompt_lens, const float* repetition,
    const float* frequency, const float* presence, const int32_t* bias_ids,
    int64_t bias_id_row_stride, const float* bias_values, int64_t bias_value_row_stride,
    int num_biases, const int32_t* allowed, int64_t allowed_row_stride,
    const int32_t* draft_tokens, const int32_t* ancestors, int64_t ancestor_row_stride,
    int ancestor_words, const int32_t* query_start_loc, void* stream) {
  const std::string name = "qsa_process_logits";
  if (rows < 0 || vocab < 0 || num_requests < 0 || history_width < 0 || num_biases < 0 ||
      ancestor_words < 0 || vocab_start < 0)
    return fail(QSA_ERR_INVALID, name + ": negative size");
  if (logits_type != kFp32 && logits_type != kBf16 && logits_type != kFp16)
    return fail(QSA_ERR_UNSUPPORTED, name + ": logits must be fp32, bf16 or fp16");
  if (vocab_start > INT_MAX - vocab)
    return fail(QSA_ERR_INVALID, name + ": token ids must lie below 2^31");
  if (rows == 0 || vocab == 0) return QSA_OK;
  if (!logits || !out) return fail(QSA_ERR_INVALID, name + ": null tensor pointer");
  if (history && !history_lens)
    return fail(QSA_ERR_INVALID, name + ": a history needs its lengths");
  if (num_biases > 0 && (!bias_ids || !bias_values))
    return fail(QSA_ERR_INVALID, name + ": biases need ids and values");
  if (num_biases > kMaxBiases)
    return fail(QSA_ERR_UNSUPPORTED,
                name + ": at most " + std::to_string(kMaxBiases) + " biases a request");
  if (ancestors && ancestor_words > kMaxNodes / 32)
    return fail(QSA_ERR_UNSUPPORTED, name + ": at most " + std::to_string(kMaxNodes) +
                                         " nodes a request (" + std::to_string(kMaxNodes / 32) +
                                         " ancestor words)");
  if (ancestors && (!draft_tokens || !query_start_loc))
    return fail(QSA_ERR_INVALID, name + ": ancestors need draft tokens and query_start_loc");
  const size_t item = logits_type == kFp32 ? 4 : 2;
  if (((uintptr_t)logits % item) || ((uintptr_t)out & 3u))
    return fail(QSA_ERR_INVALID, name + ": misaligned logits or output");
  LogitsArgs a = {};
  a.logits = logits;
  a.in_row = logits_row_stride;
  a.out = out;
  a.out_row = out_row_stride;
  a.rows = rows;
  a.vocab = vocab;
  a.vocab_start = vocab_start;
  a.token_to_req = token_to_req;
  a.requests = num_requests;
  a.history = history;
  a.history_row = history_row_stride;
  a.history_width = history_width;
  a.history_lens = history_lens;
  a.prompt_lens = prompt_lens;
  a.repetition = repetition;
  a.frequency = frequency;
  a.presence = presence;
  a.bias_ids = bias_ids;
  a.bias_id_row = bias_id_row_stride;
  a.bias_values = bias_values;
  a.bias_value_row = bias_value_row_stride;
  a.biases = num_biases;
  a.allowed = allowed;
  a.allowed_row = allowed_row_stride;
  a.draft_tokens = draft_tokens;
  a.ancestors = ancestors;
  a.ancestor_row = ancestor_row_stride;
  a.words = ancestor_words;
  a.query_start_loc = query_start_loc;
  a.group_rows = ancestors ? kTreeRows : 1;
  const bool ruled = repetition || frequency || presence || num_biases > 0;
  const bool wide = history_width > kMaxNarrow;
  const int64_t groups = (rows - 1) / a.group_rows + 1;
  const int64_t most = (vocab - 1) / kMinChunk + 1;
  const int64_t least = (vocab - 1) / (wide ? kMaxChunkWide : kMaxChunk) + 1;
  const int64_t chunks = std::max(least, std::min(most, kRounds * kCUs / groups));
  a.chunk = (int)(((vocab + chunks - 1) / chunks + 31) / 32 * 32);  // whole mask words
  a.chunks = (vocab - 1) / a.chunk + 1;
  const int64_t grid = (int64_t)a.chunks * groups;
  if (grid > UINT_MAX / kThreads)  // what a launch holds
    return fail(QSA_ERR_UNSUPPORTED, name + ": too many rows");
  const bool vec = ((uintptr_t)logits & 3u) == 0 && logits_row_stride * item % 4 == 0 &&
                   ((uintptr_t)out & 15u) == 0 && out_row_stride % 4 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (logits_type == kFp32) launch<kFp32>(a, vec, wide, (unsigned)grid, ruled, s);
  else if (logits_type == kBf16) launch<kBf16>(a, vec, wide, (unsigned)grid, ruled, s);
  else launch<kFp16>(a, vec, wide, (unsigned)grid, ruled, s);
  return check_launch(name.c_str());
}

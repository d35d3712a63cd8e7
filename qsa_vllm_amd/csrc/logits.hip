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
// (4), a grammar bit. What a token's penalties need is kept in LDS for a chunk
// of the vocabulary: a workgroup counts its request's history within its chunk
// with LDS atomics (whole numbers: any order gives the same counts), sums the
// biases in list order, then streams the chunk of its rows. The rows of a
// request that share a workgroup (a drafted tree's) share the table: a node's
// ancestors are added to it before its row and taken off after.
#include "qsa_common.h"
#include "../../include/qsa_hip.h"

#include <algorithm>
#include <climits>

namespace qsa {
namespace {

constexpr int kThreads = 512;
constexpr int kChunk = 8192;            // vocabulary entries of a workgroup
constexpr int kTreeRows = 8;            // rows of a workgroup with drafted trees
constexpr uint32_t kPrompt = 1u << 31;  // count table: in the prompt
constexpr uint32_t kNoBias = 0xFFFFFFFFu;
constexpr uint32_t kTwice = 1u << 30;   // bias table, while it is built: an id listed twice
constexpr int kMaxBiases = 64 * kThreads;
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
  int chunks, group_rows;
};

template <int TYPE>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
  if constexpr (TYPE == kFp32) return static_cast<const float*>(p)[i];
  else if constexpr (TYPE == kBf16)
    return __builtin_bit_cast(float, (uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
  else return (float)static_cast<const _Float16*>(p)[i];
}

template <int TYPE>
__device__ __forceinline__ f32x4 load_logit4(const void* p, int64_t i) {
  if constexpr (TYPE == kFp32) {
    return *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
  } else if constexpr (TYPE == kBf16) {
    const u32x2 v = load_u32x2(static_cast<const uint16_t*>(p) + i);
    return f32x4{bf16_lo(v[0]), bf16_hi(v[0]), bf16_lo(v[1]), bf16_hi(v[1])};
  } else {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    const f16x4 v = *reinterpret_cast<const f16x4*>(static_cast<const _Float16*>(p) + i);
    return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
  }
}

struct RowRules {
  float repetition, frequency, presence;
  bool count, bias;
};

__device__ __forceinline__ float apply(float x, uint32_t c, uint32_t b, const RowRules& r) {
  if (r.count && c) {
    const uint32_t spoken = c & ~kPrompt;
    x = x > 0.0f ? x / r.repetition : x * r.repetition;
    if (spoken) x = x - r.frequency * (float)spoken - r.presence;
  }
  if (r.bias && b != kNoBias) x += __builtin_bit_cast(float, b);
  return x;
}

template <int TYPE, bool VEC>
__global__ __launch_bounds__(kThreads) void logits_kernel(LogitsArgs a) {
  extern __shared__ uint32_t table[];  // [kChunk] counts, [kChunk] biases (whichever are used)
  const bool penalise = a.repetition || a.frequency || a.presence;
  const bool biased = a.biases > 0;
  uint32_t* const counts = table;
  uint32_t* const bias = table + (penalise ? kChunk : 0);
  const int base = (blockIdx.x % a.chunks) * kChunk;
  const int size = min(kChunk, a.vocab - base);
  const int64_t first = a.vocab_start + base;  // the chunk's first token id
  const int row_begin = (blockIdx.x / a.chunks) * a.group_rows;
  const int row_end = min(a.rows, row_begin + a.group_rows);

  int held = -1;  // the request whose tokens and biases the tables hold
  for (int row = row_begin; row < row_end; ++row) {
    const int req = a.token_to_req ? load_uniform(a.token_to_req + row) : row;
    const bool live = req >= 0 && req < a.requests;  // a padding row: no penalties, no biases
    if (live && req != held && (penalise || biased)) {
      __syncthreads();
      for (int i = threadIdx.x; i < kChunk; i += kThreads) {
        if (penalise) counts[i] = 0;
        if (biased) bias[i] = kNoBias;
      }
      __syncthreads();
      if (penalise && a.history) {
        const int len = min(max(load_uniform(a.history_lens + req), 0), a.history_width);
        const int prompt = a.prompt_lens ? load_uniform(a.prompt_lens + req) : 0;
        const int32_t* const h = a.history + req * a.history_row;
        for (int i = threadIdx.x; i < len; i += kThreads) {
          const int64_t at = h[i] - first;
          if (at >= 0 && at < size) {
            if (i < prompt) atomicOr(&counts[at], kPrompt);
            else atomicAdd(&counts[at], 1u);
          }
        }
      }
      if (biased) {
        const int32_t* const ids = a.bias_ids + req * a.bias_id_row;
        const float* const values = a.bias_values + req * a.bias_value_row;
        auto slot = [&](int i) -> int64_t { return ids[i] - first; };
        // The first entry of an id owns its slot and adds up the later ones.
        // Bit k of `owned`: the thread's k-th entry does.
        uint64_t owned = 0;
        for (int i = threadIdx.x; i < a.biases; i += kThreads) {
          const int64_t at = slot(i);
          if (at >= 0 && at < size) atomicMin(&bias[at], (uint32_t)i);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < a.biases; i += kThreads) {
          const int64_t at = slot(i);
          if (at < 0 || at >= size) continue;
          if ((bias[at] & ~kTwice) == (uint32_t)i) owned |= 1ull << (i / kThreads);
          else atomicOr(&bias[at], kTwice);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < a.biases; i += kThreads) {
          if (!((owned >> (i / kThreads)) & 1)) continue;
          const int64_t at = slot(i);
          float sum = values[i];
          if (bias[at] & kTwice)
            for (int j = i + 1; j < a.biases; ++j)
              if (slot(j) == at) sum += values[j];
          if (sum != sum) sum = __builtin_nanf("");  // no NaN with the bits of kNoBias
          bias[at] = __builtin_bit_cast(uint32_t, sum);
        }
      }
      __syncthreads();
      held = req;
    }

    // A drafted node's own path: its visible ancestors' tokens.
    int node0 = 0, nodes = 0;
    if (live && penalise && a.ancestors) {
      node0 = max(load_uniform(a.query_start_loc + req), 0);
      nodes = min(min(load_uniform(a.query_start_loc + req + 1), a.rows) - node0, 32 * a.words);
    }
    auto path = [&](uint32_t step) {
      for (int j = threadIdx.x; j < nodes; j += kThreads) {
        const uint32_t word = (uint32_t)a.ancestors[row * a.ancestor_row + (j >> 5)];
        const int64_t at = a.draft_tokens[node0 + j] - first;
        if ((word >> (j & 31)) & 1u && at >= 0 && at < size) atomicAdd(&counts[at], step);
      }
    };
    if (nodes > 0) {
      path(1u);
      __syncthreads();
    }

    RowRules r;
    r.count = live && penalise;
    r.bias = live && biased;
    r.repetition = live && a.repetition ? load_uniform(a.repetition + req) : 1.0f;
    r.frequency = live && a.frequency ? load_uniform(a.frequency + req) : 0.0f;
    r.presence = live && a.presence ? load_uniform(a.presence + req) : 0.0f;
    const uint32_t* const allowed =
        a.allowed ? reinterpret_cast<const uint32_t*>(a.allowed) + row * a.allowed_row + base / 32
                  : nullptr;
    const int64_t in = row * a.in_row + base;
    float* const out = a.out + row * a.out_row + base;
    const int vec_end = VEC ? size & ~3 : 0;
    if constexpr (VEC) {
      for (int i = 4 * threadIdx.x; i < vec_end; i += 4 * kThreads) {
        f32x4 y = load_logit4<TYPE>(a.logits, in + i);
        const uint32_t bits = allowed ? allowed[i / 32] >> (i & 31) : 15u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[e] = apply(y[e], r.count ? counts[i + e] : 0, r.bias ? bias[i + e] : kNoBias, r);
          if (!((bits >> e) & 1u)) y[e] = kNegInf;
        }
        *reinterpret_cast<f32x4*>(out + i) = y;
      }
    }
    for (int i = vec_end + threadIdx.x; i < size; i += kThreads) {
      float y = apply(load_logit<TYPE>(a.logits, in + i), r.count ? counts[i] : 0,
                      r.bias ? bias[i] : kNoBias, r);
      if (allowed && !((allowed[i / 32] >> (i & 31)) & 1u)) y = kNegInf;
      out[i] = y;
    }
    if (nodes > 0) {
      __syncthreads();
      path(~0u);  // - 1
      __syncthreads();
    }
  }
}

template <int TYPE>
void launch(const LogitsArgs& a, bool vec, unsigned grid, size_t lds, hipStream_t stream) {
  if (vec)
    hipLaunchKernelGGL((logits_kernel<TYPE, true>), dim3(grid), dim3(kThreads), lds, stream, a);
  else
    hipLaunchKernelGGL((logits_kernel<TYPE, false>), dim3(grid), dim3(kThreads), lds, stream, a);
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
  if (rows == 0 || vocab == 0) return QSA_OK;
  if (!logits || !out) return fail(QSA_ERR_INVALID, name + ": null tensor pointer");
  if (history && !history_lens)
    return fail(QSA_ERR_INVALID, name + ": a history needs its lengths");
  if (num_biases > 0 && (!bias_ids || !bias_values))
    return fail(QSA_ERR_INVALID, name + ": biases need ids and values");
  if (num_biases > kMaxBiases)
    return fail(QSA_ERR_UNSUPPORTED,
                name + ": at most " + std::to_string(kMaxBiases) + " biases a request");
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
  a.chunks = (vocab - 1) / kChunk + 1;
  a.group_rows = ancestors ? kTreeRows : 1;
  const int64_t grid = (int64_t)a.chunks * ((rows - 1) / a.group_rows + 1);
  if (grid > INT_MAX) return fail(QSA_ERR_UNSUPPORTED, name + ": too many rows");
  const bool vec = ((uintptr_t)logits % (4 * item)) == 0 && logits_row_stride % 4 == 0 &&
                   ((uintptr_t)out & 15u) == 0 && out_row_stride % 4 == 0;
  const bool penalise = repetition || frequency || presence;
  const size_t lds = ((penalise ? 1 : 0) + (num_biases > 0 ? 1 : 0)) * kChunk * sizeof(uint32_t);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (logits_type == kFp32) launch<kFp32>(a, vec, (unsigned)grid, lds, s);
  else if (logits_type == kBf16) launch<kBf16>(a, vec, (unsigned)grid, lds, s);
  else launch<kFp16>(a, vec, (unsigned)grid, lds, s);
  return check_launch(name.c_str());
}

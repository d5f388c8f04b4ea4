// What a server does to a row of logits before it draws a token from it: penalties
// for tokens that its history holds, biases of single tokens, and the tokens
// that a grammar allows:
//   x > 0 ? x / repetition : x repetition     where the token occurs in the history
//   x - frequency count - presence [count > 0]     count: its times behind the prompt
//   x + the sum of the token's biases
//   -inf                                      where the token is not allowed
// in float32, rounded once.
//
// HBM-bound for batches (a row is read and written once: [512, 65536] bf16 under a grammar 27 us, 5.0 TB/s), latency for single
// rows ([1, 32000], a history of 700: 4.3 us), and with long histories bound by reading them ([512, 128256] float32,
// histories of 32768: 136 us).  All figures here are of launches in a row, three sets of
// inputs in turn.  A workgroup takes a range of a row's columns.  It counts the range's tokens in LDS: it
// reads the row's whole history (from the L2, which the row's other workgroups
// share) and keeps what falls into its range, so no counts go through memory and there is
// one launch; integer counts do not depend on the order of the additions.  Counts
// are 16 bits where the history is short enough for them, so that a range is long
// and the history is read few times; what the prompt holds and which tokens have a
// bias are bits.  The biases' sums are in LDS, in a hash table of the range's tokens or, of many, one for each
// of its columns; the entries of a token add theirs in turn, in their order, so that the sum does not
// depend on which thread comes first.  The range's first logits are requested before
// the history is read.
#include "row_group.h"

namespace sa {

constexpr int kAdjApart = 8;                 // XCDs
constexpr int kAdjVecs = 4;                  // vectors of logits that a thread has in flight
constexpr int kAdjUnroll = 2;                // 16-byte loads of the history in flight a thread: with 1 the long histories took 146 us, with 2 136
constexpr int kAdjMaxRange = 32768;          // histories of 32768 tokens: 136 us, with 16384 166, with 65536, one workgroup a CU, 150
constexpr int kAdjHash = 1024;               // most biases that go into a hash table
constexpr int kAdjDense = 8192;              // columns of a range where there are more: 64 KiB of sums and turns
constexpr int64_t kAdjNarrow = 65535;        // the longest history that 16 bits count

constexpr int kAdjNobody = 0x7fffffff;

struct AdjustArgs {
  const void* in;
  void* out;
  int64_t in_stride, out_stride;
  const void* tokens;
  const void* lengths;
  const void* prompts;
  const float *repetition, *presence, *frequency;
  const void* bias_tokens;
  const float* bias;
  const uint32_t* allowed;
  int64_t tokens_stride, bias_tokens_stride, bias_stride, allowed_stride;
  int64_t vocab, history;
  int32_t biases, range;
  FastDiv ranges;   // of a row
  int32_t apart;    // a row's workgroups are kAdjApart of the launch apart; else `rows` of it
  int32_t hash;     // slots of the biases' hash table, a power of two >= 2 biases; 0: a slot for each column
  int32_t tok64, len64, prompt64, bias_tok64;
  float repetition_value, presence_value, frequency_value;
};

__device__ __forceinline__ int64_t adj_int(const void* p, int is64, int64_t at) {
  return is64 ? static_cast<const int64_t*>(p)[at] : (int64_t)static_cast<const int32_t*>(p)[at];
}

// LDS of a workgroup, in words: counts, bits of the prompt's tokens (PEN), bits of the tokens with a
// bias, and of each slot of the biases' table its column (of a hash table), sum and whose turn it is (BIAS).
inline __host__ __device__ int adj_count_words(int range, bool wide) { return wide ? range : range / 2; }
inline size_t adj_lds_bytes(int range, bool pen, bool wide, bool biased, int hash) {
  return (pen ? 4 * (size_t)(adj_count_words(range, wide) + range / 32) : 0) +
         (biased ? 4 * (size_t)(range / 32) + (hash != 0 ? 12 * (size_t)hash : 8 * (size_t)range) : 0);
}

// A token's column from c0 on; one far outside is not in any range.
__device__ __forceinline__ int64_t adj_column(const void* p, int is64, int64_t at, int64_t c0) {
  return (int64_t)((uint64_t)adj_int(p, is64, at) - (uint64_t)c0);
}

// WIDE: counts of 32 bits.
template <typename T, bool PEN, bool WIDE, bool BIAS>
__global__ void __launch_bounds__(1024) k_adjust(AdjustArgs g, int64_t row0, int64_t rows) {
  constexpr int V = VecOf<T>::V;
  extern __shared__ uint4 lds[];
  uint32_t* const count = reinterpret_cast<uint32_t*>(lds);
  uint32_t* const prompt_bits = count + adj_count_words(g.range, WIDE);
  uint32_t* const bias_bits = PEN ? prompt_bits + g.range / 32 : count;
  int32_t* const hash_at = reinterpret_cast<int32_t*>(bias_bits + g.range / 32);
  const int slots = g.hash != 0 ? g.hash : g.range;
  float* const slot_sum = reinterpret_cast<float*>(hash_at + g.hash);
  int32_t* const turn = hash_at + g.hash + slots;
  uint32_t row_at = blockIdx.x, range = blockIdx.y;
  if (g.apart) {  // in runs of as many rows with all their ranges
    uint32_t run;
    g.ranges.divmod(blockIdx.x / (uint32_t)kAdjApart, run, range);
    row_at = run * kAdjApart + blockIdx.x % (uint32_t)kAdjApart;
    if (row_at >= rows) return;
  }
  const int64_t row = row0 + row_at, c0 = (int64_t)range * g.range;
  const int width = (int)(g.vocab - c0 < g.range ? g.vocab - c0 : g.range), nt = blockDim.x;
  const T* in = static_cast<const T*>(g.in) + (row * g.in_stride + c0);
  T* out = static_cast<T*>(g.out) + (row * g.out_stride + c0);
  float rho = 1.0f, presence = 0.0f, frequency = 0.0f;
  int64_t n = g.history, prompt = 0;
  if constexpr (PEN) {
    rho = g.repetition ? g.repetition[row] : g.repetition_value;
    presence = g.presence ? g.presence[row] : g.presence_value;
    frequency = g.frequency ? g.frequency[row] : g.frequency_value;
    if (g.lengths) {
      const int64_t v = adj_int(g.lengths, g.len64, row);
      n = v < 0 ? 0 : (v < n ? v : n);
    }
    if (g.prompts) prompt = adj_int(g.prompts, g.prompt64, row);
  }
  RowVec<T, V> w[kAdjVecs];
  auto request = [&](int base) {
#pragma unroll
    for (int i = 0; i < kAdjVecs; ++i) {
      const int col = base + (threadIdx.x + i * nt) * V;
      if (col < width) w[i] = row_load<true, V>(in, col, width);
    }
  };
  request(0);
  if (PEN || BIAS) {
    const int words = (PEN ? adj_count_words(g.range, WIDE) + g.range / 32 : 0) + (BIAS ? g.range / 32 : 0);
    for (int i = threadIdx.x; i < words / 4; i += nt) lds[i] = make_uint4(0u, 0u, 0u, 0u);
    for (int i = words / 4 * 4 + threadIdx.x; i < words; i += nt) count[i] = 0u;
    if (BIAS) {
      for (int i = threadIdx.x; i < g.hash; i += nt) hash_at[i] = -1;
      for (int i = threadIdx.x; i < slots; i += nt) {
        slot_sum[i] = 0.0f;
        turn[i] = kAdjNobody;
      }
    }
    __syncthreads();
  }
  if constexpr (PEN) {
    // n is below 2^31, and so are tokens that count: those with a higher half are in no range.  Whole loads need no check
    // of each token's place: one token a load, each checked, took 152 us for 136.
    auto scan = [&](auto* history) {
      using Token = std::remove_cv_t<std::remove_pointer_t<decltype(history)>>;
      const Token* at = history + row * g.tokens_stride;
      const uint32_t end = (uint32_t)n, start = prompt < 0 ? 0u : (uint32_t)(prompt < n ? prompt : n), base = (uint32_t)c0;
      auto take = [&](Token token, uint32_t t) {
        const uint32_t c = (uint32_t)token - base;
        if (c >= (uint32_t)width || (sizeof(Token) == 8 && (uint64_t)token >> 32 != 0)) return;
        if (t < start) atomicOr(&prompt_bits[c / 32], 1u << (c % 32));
        else if (WIDE) atomicAdd(&count[c], 1u);
        else atomicAdd(&count[c / 2], c & 1 ? 0x10000u : 1u);
      };
      constexpr int N = 16 / (int)sizeof(Token);  // tokens of a load; it needs their alignment alone
      struct alignas(sizeof(Token)) Tokens { Token v[N]; };
      const uint32_t step = (uint32_t)nt * N;
      uint32_t t = threadIdx.x * N;
      auto batch = [&](auto size) {
        constexpr int U = decltype(size)::value;
        Tokens tokens[U];
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(&tokens[u], at + t + u * step, sizeof(Tokens));
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int k = 0; k < N; ++k) take(tokens[u].v[k], t + u * step + k);
        }
        t += step * U;
      };
      while (t + step * (kAdjUnroll - 1) + N <= end) batch(std::integral_constant<int, kAdjUnroll>{});
      while (t + N <= end) batch(std::integral_constant<int, 1>{});
      for (; t < end; ++t) take(at[t], t);  // fewer than N, of one thread
    };
    if (g.tok64) scan(static_cast<const int64_t*>(g.tokens));
    else scan(static_cast<const int32_t*>(g.tokens));
  }
  // the slot that holds a column, or the free one that it would get: at most half of them are taken, so one is met
  auto slot_of = [&](int col, auto&& step) {
    uint32_t h = ((uint32_t)col * 0x9E3779B1u) >> 16 & (uint32_t)(g.hash - 1);
    while (!step(h)) h = (h + 1) & (uint32_t)(g.hash - 1);
    return (int)h;
  };
  if constexpr (BIAS) {
    const int64_t at = row * g.bias_tokens_stride, bt = row * g.bias_stride;
    for (int64_t j0 = 0; j0 < g.biases; j0 += nt) {
      const int64_t j = j0 + threadIdx.x, col = j < g.biases ? adj_column(g.bias_tokens, g.bias_tok64, at + j, c0) : -1;
      bool waits = (uint64_t)col < (uint64_t)width;
      int slot = (int)col;
      float b = 0.0f;
      if (waits) {
        b = g.bias[bt + j];
        atomicOr(&bias_bits[col / 32], 1u << (col % 32));
        if (g.hash != 0) slot = slot_of((int)col, [&](uint32_t h) {
          const int was = atomicCAS(&hash_at[h], -1, (int)col);
          return was == -1 || was == (int)col;
        });
      }
      do {  // the first of a slot's entries that wait takes its turn: each round ends with fewer
        if (waits) atomicMin(&turn[slot], (int)j);
        __syncthreads();
        const bool now = waits && turn[slot] == (int)j;
        __syncthreads();
        if (now) {
          slot_sum[slot] += b;
          turn[slot] = kAdjNobody;
          waits = false;
        }
      } while (__syncthreads_or(waits));
    }
  }
  if (PEN || BIAS) __syncthreads();
  auto bias_of = [&](int col) {
    return slot_sum[g.hash != 0 ? slot_of(col, [&](uint32_t h) { return hash_at[h] == col || hash_at[h] == -1; }) : col];
  };
  const uint32_t* allowed = g.allowed ? g.allowed + row * g.allowed_stride : nullptr;
  for (int base = 0; base < width; base += nt * V * kAdjVecs) {
    if (base > 0) request(base);
#pragma unroll
    for (int i = 0; i < kAdjVecs; ++i) {
      const int col = base + (threadIdx.x + i * nt) * V;  // the tables reach to the range's end, which is whole vectors
      if (col >= width) continue;
      float f[V];
#pragma unroll
      for (int k = 0; k < V; ++k) f[k] = row_elem<T, V>(w[i], k);
      constexpr uint32_t all = (1u << V) - 1u;
      if constexpr (PEN) {
        uint32_t c[WIDE ? V : V / 2], any = 0u;
        __builtin_memcpy(c, count + (WIDE ? col : col / 2), sizeof(c));
#pragma unroll
        for (int k = 0; k < (WIDE ? V : V / 2); ++k) any |= c[k];
        const uint32_t said = prompt_bits[col / 32] >> (col % 32) & all;
        if (any | said) {
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const uint32_t n = WIDE ? c[k] : (c[k / 2] >> (k % 2 * 16) & 0xffffu);
            if (n == 0u && !(said >> k & 1u)) continue;
            f[k] = f[k] > 0.0f ? f[k] / rho : f[k] * rho;
            f[k] = f[k] - frequency * (float)n;
            f[k] = f[k] - (n > 0u ? presence : 0.0f);
          }
        }
      }
      if constexpr (BIAS) {
        const uint32_t biased = bias_bits[col / 32] >> (col % 32) & all;
        if (biased) {
#pragma unroll 1
          for (int k = 0; k < V; ++k)
            if (biased >> k & 1u) {
              const float b = bias_of(col + k);
#pragma unroll
              for (int e = 0; e < V; ++e) f[e] = e == k ? f[e] + b : f[e];
            }
        }
      }
      if (allowed) {
        const int64_t v = c0 + col;
        const uint32_t bits = allowed[v / 32] >> (v % 32);
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (!(bits >> k & 1u)) f[k] = -__builtin_inff();
      }
      row_store<T, V>(out, col, width, f);
    }
  }
}

}  // namespace sa

using namespace sa;

extern "C" int supa_amd_adjust_logits(const supa_amd_adjust_desc* d, void* stream) {
  if (!d || d->rows < 0 || d->vocab < 1 || d->history < 0 || d->biases < 0) return SUPA_AMD_EINVAL;
  if (d->rows >= (int64_t(1) << 31) || d->vocab >= (int64_t(1) << 29) || d->history >= (int64_t(1) << 31) ||
      d->biases >= (int64_t(1) << 31) - 1)
    return SUPA_AMD_ELAYOUT;
  const auto is_int = [](int32_t t) { return t == SUPA_AMD_I64 || t == SUPA_AMD_I32; };
  if (d->dtype != SUPA_AMD_F32 && d->dtype != SUPA_AMD_BF16 && d->dtype != SUPA_AMD_F16) return SUPA_AMD_EDTYPE;
  const bool pen = d->tokens && d->history > 0, biased = d->bias_tokens && d->biases > 0;
  if ((d->history > 0 && !d->tokens) || (d->biases > 0 && (!d->bias_tokens || !d->bias))) return SUPA_AMD_EINVAL;
  if ((pen && !is_int(d->token_dtype)) || (d->lengths && !is_int(d->length_dtype)) ||
      (d->prompt_lengths && !is_int(d->prompt_dtype)) || (biased && !is_int(d->bias_token_dtype)))
    return SUPA_AMD_EDTYPE;
  if (d->rows == 0) return SUPA_AMD_OK;
  if (!d->in || !d->out) return SUPA_AMD_EINVAL;
  AdjustArgs a{};
  a.in = d->in;
  a.out = d->out;
  a.in_stride = d->in_stride;
  a.out_stride = d->out_stride;
  a.tokens = d->tokens;
  a.lengths = d->lengths;
  a.prompts = d->prompt_lengths;
  a.repetition = d->repetition;
  a.presence = d->presence;
  a.frequency = d->frequency;
  a.bias_tokens = d->bias_tokens;
  a.bias = d->bias;
  a.allowed = d->allowed;
  a.tokens_stride = d->tokens_stride;
  a.bias_tokens_stride = d->bias_tokens_stride;
  a.bias_stride = d->bias_stride;
  a.allowed_stride = d->allowed_stride;
  a.vocab = d->vocab;
  a.history = d->history;
  a.biases = (int32_t)d->biases;
  a.tok64 = d->token_dtype == SUPA_AMD_I64;
  a.len64 = d->length_dtype == SUPA_AMD_I64;
  a.prompt64 = d->prompt_dtype == SUPA_AMD_I64;
  a.bias_tok64 = d->bias_token_dtype == SUPA_AMD_I64;
  a.repetition_value = (float)d->repetition_value;
  a.presence_value = (float)d->presence_value;
  a.frequency_value = (float)d->frequency_value;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_float_storage(d->dtype, [&](auto* tag) -> int {
    using T = std::remove_pointer_t<decltype(tag)>;
    constexpr int V = VecOf<T>::V;
    const bool wide = pen && d->history > kAdjNarrow;
    // 512 workgroups, two a CU, if the rows are long enough for them; no shorter ranges than 1024
    // columns, and none whose counts pass 64 KiB of LDS: two workgroups a CU
    if (biased && a.biases <= kAdjHash) {
      a.hash = 64;
      while (a.hash < 2 * a.biases) a.hash *= 2;
    }
    const int most_range = biased && a.hash == 0 ? kAdjDense : (wide || a.hash > 512 ? 16384 : kAdjMaxRange);
    a.range = 1024;
    while (a.range < most_range && (a.vocab + a.range - 1) / a.range * d->rows > 512) a.range *= 2;
    const unsigned ranges = (unsigned)((a.vocab + a.range - 1) / a.range);
    a.range = (int32_t)(((a.vocab + ranges - 1) / ranges + 255) / 256 * 256);  // evenly
    // a vector of the range for each thread, and of a history 8 tokens at most, up to 1024 threads
    const int64_t threads = std::max<int64_t>(a.range / V, pen ? d->history / 8 : 0);
    const int block = (int)std::min<int64_t>(1024, (threads + 63) / 64 * 64);
    const size_t lds = adj_lds_bytes(a.range, pen, wide, biased, a.hash);
    // Workgroups go to the eight XCDs in turn.  Where the histories pass what the eight L2s hold, those of a row are
    // eight apart and next to each other in time, so that its history comes from memory once and from one XCD's L2 for
    // the others ([512, 128256] float32, histories of 32768: 147 us with all rows' first ranges first, 136 so); else
    // rows come first, which spreads a number of rows that is no multiple of eight evenly ([37, 50257]: 6.8 and 9.1).
    a.ranges = FastDiv(ranges);
    a.apart = (pen && d->rows >= 64 && d->rows * d->history * 8 > (int64_t(32) << 20)) || ranges > 65535;
    const int64_t most = ((int64_t(1) << 32) - 1) / block / ranges;  // HIP: fewer than 2^32 threads a launch
    const int64_t slab = std::max<int64_t>(kAdjApart, most / kAdjApart * kAdjApart);
    for (int64_t r0 = 0; r0 < d->rows; r0 += slab) {
      const int64_t n = std::min(slab, d->rows - r0);
      const dim3 grid = a.apart ? dim3((unsigned)((n + kAdjApart - 1) / kAdjApart * kAdjApart * ranges)) : dim3((unsigned)n, ranges);
      auto go = [&](auto p, auto w, auto b) {
        auto kernel = k_adjust<T, p.value, w.value, b.value>;
        if (lds > 65536) {
          const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
          if (e != hipSuccess) return (int)e;
        }
        kernel<<<grid, block, lds, st>>>(a, r0, n);
        return launch_status();
      };
      auto with_bias = [&](auto p, auto w) { return biased ? go(p, w, std::true_type{}) : go(p, w, std::false_type{}); };
      const int rc = !pen ? with_bias(std::false_type{}, std::false_type{})
                          : (wide ? with_bias(std::true_type{}, std::true_type{}) : with_bias(std::true_type{}, std::false_type{}));
      if (rc) return rc;
    }
    return SUPA_AMD_OK;
  });
}

// What a server does to a row of logits before it draws a token from it: penalties
// for tokens that its history holds, biases of single tokens, and the tokens
// that a grammar allows:
//   x > 0 ? x / repetition : x repetition     where the token occurs in the history
//   x - frequency count - presence [count > 0]     count: its times behind the prompt
//   x + the sum of the token's biases
//   -inf                                      where the token is not allowed
// in float32, rounded once.
//
// HBM-bound for batches (a row is read and written once), latency for single
// rows.  A workgroup takes a range of a row's columns.  It counts the range's tokens in LDS: it
// reads the row's whole history (from the L2, which the row's other workgroups
// share) and keeps what falls into its range, so no counts go through memory and there is
// one launch; integer counts do not depend on the order of the additions.
// Biases are put into a second table by one owner per token.  The range's
// logits are requested before the history is read.
#include "row_group.h"

namespace sa {

constexpr int kAdjVecs = 4;                  // most vectors of logits a thread holds
constexpr uint32_t kAdjSeen = 0x80000000u;   // in the prompt
constexpr int kAdjUnroll = 4;                // tokens of the history in flight a thread

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
  int32_t tok64, len64, prompt64, bias_tok64;
  float repetition_value, presence_value, frequency_value;
};

__device__ __forceinline__ int64_t adj_int(const void* p, int is64, int64_t at) {
  return is64 ? static_cast<const int64_t*>(p)[at] : (int64_t)static_cast<const int32_t*>(p)[at];
}

template <typename T, bool PEN, bool BIAS> __global__ void __launch_bounds__(1024) k_adjust(AdjustArgs g, int64_t row0) {
  constexpr int V = VecOf<T>::V;
  extern __shared__ uint32_t lds[];  // PEN: counts of the range's tokens; BIAS: their biases
  __shared__ int twice;
  uint32_t* count = lds;
  float* bias = reinterpret_cast<float*>(lds + (PEN ? g.range : 0));
  const int64_t row = row0 + blockIdx.x, c0 = (int64_t)blockIdx.y * g.range;
  const int width = (int)(g.vocab - c0 < g.range ? g.vocab - c0 : g.range), nt = blockDim.x;
  const T* in = static_cast<const T*>(g.in) + (row * g.in_stride + c0);
  T* out = static_cast<T*>(g.out) + (row * g.out_stride + c0);
  RowVec<T, V> w[kAdjVecs];
#pragma unroll
  for (int i = 0; i < kAdjVecs; ++i) {
    const int col = (threadIdx.x + i * nt) * V;
    if (col < width) w[i] = row_load<true, V>(in, col, width);
  }
  if (PEN) {
    for (int i = threadIdx.x; i < g.range; i += nt) count[i] = 0u;
  }
  if (BIAS) {
    for (int i = threadIdx.x; i < g.range; i += nt) reinterpret_cast<int32_t*>(bias)[i] = 0;
    if (threadIdx.x == 0) twice = 0;
  }
  if (PEN || BIAS) __syncthreads();
  float rho = 1.0f, presence = 0.0f, frequency = 0.0f;
  if constexpr (PEN) {
    rho = g.repetition ? g.repetition[row] : g.repetition_value;
    presence = g.presence ? g.presence[row] : g.presence_value;
    frequency = g.frequency ? g.frequency[row] : g.frequency_value;
    int64_t n = g.history, prompt = 0;
    if (g.lengths) {
      const int64_t v = adj_int(g.lengths, g.len64, row);
      n = v < 0 ? 0 : (v < n ? v : n);
    }
    if (g.prompts) prompt = adj_int(g.prompts, g.prompt64, row);
    const int64_t at = row * g.tokens_stride;
    for (int64_t t0 = threadIdx.x; t0 < n; t0 += (int64_t)nt * kAdjUnroll) {
      int64_t tok[kAdjUnroll];
#pragma unroll
      for (int u = 0; u < kAdjUnroll; ++u) {
        const int64_t t = t0 + u * nt;
        tok[u] = t < n ? adj_int(g.tokens, g.tok64, at + t) - c0 : -1;
      }
#pragma unroll
      for (int u = 0; u < kAdjUnroll; ++u) {
        if ((uint64_t)tok[u] >= (uint64_t)width) continue;
        if (t0 + u * nt < prompt) atomicOr(&count[tok[u]], kAdjSeen);
        else atomicAdd(&count[tok[u]], 1u);
      }
    }
  }
  if constexpr (BIAS) {
    // the last entry of a token owns its place: first by number, then with the sum
    int32_t* owner = reinterpret_cast<int32_t*>(bias);
    const int64_t at = row * g.bias_tokens_stride, bt = row * g.bias_stride;
    for (int j = threadIdx.x; j < g.biases; j += nt) {
      const int64_t tok = adj_int(g.bias_tokens, g.bias_tok64, at + j) - c0;
      if ((uint64_t)tok < (uint64_t)width) atomicMax(&owner[tok], j + 1);
    }
    __syncthreads();
    for (int j = threadIdx.x; j < g.biases; j += nt) {
      const int64_t tok = adj_int(g.bias_tokens, g.bias_tok64, at + j) - c0;
      if ((uint64_t)tok < (uint64_t)width && owner[tok] != j + 1) twice = 1;
    }
    __syncthreads();
    for (int j0 = 0; j0 < g.biases; j0 += nt) {
      const int j = j0 + threadIdx.x;
      int64_t tok = -1;
      float b = 0.0f;
      bool own = false;
      if (j < g.biases) {
        tok = adj_int(g.bias_tokens, g.bias_tok64, at + j) - c0;
        own = (uint64_t)tok < (uint64_t)width && owner[tok] == j + 1;
        if (own && twice) {
          for (int i = 0; i < j; ++i)
            if (adj_int(g.bias_tokens, g.bias_tok64, at + i) - c0 == tok) b += g.bias[bt + i];
        }
        if (own) b += g.bias[bt + j];
      }
      __syncthreads();  // a sum's bits must not pass for an entry's number
      if (own) bias[tok] = b;
    }
  }
  if (PEN || BIAS) __syncthreads();
  const uint32_t* allowed = g.allowed ? g.allowed + row * g.allowed_stride : nullptr;
#pragma unroll
  for (int i = 0; i < kAdjVecs; ++i) {
    const int col = (threadIdx.x + i * nt) * V;
    if (col >= width) continue;
    float f[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      f[k] = row_elem<T, V>(w[i], k);
      const int at = col + k;  // tables reach to the end of the range, which is whole vectors
      if constexpr (PEN) {
        const uint32_t c = count[at];
        if (c) {
          f[k] = f[k] > 0.0f ? f[k] / rho : f[k] * rho;
          const float times = (float)(c & ~kAdjSeen);
          f[k] = f[k] - frequency * times;
          f[k] = f[k] - (times > 0.0f ? presence : 0.0f);
        }
      }
      if constexpr (BIAS) f[k] = f[k] + bias[at];
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
    // a thread holds up to kAdjVecs vectors; 8192 columns' two tables are 64 KiB of LDS
    const int block = 1024;
    a.range = 8192;
    const unsigned ranges = (unsigned)((a.vocab + a.range - 1) / a.range);
    static_assert(1024 * kAdjVecs * V >= 8192);
    const size_t lds = (size_t)a.range * 4 * ((pen ? 1 : 0) + (biased ? 1 : 0));
    const int64_t slab = std::max<int64_t>(1, ((int64_t(1) << 32) - 1) / block / ranges);
    for (int64_t r0 = 0; r0 < d->rows; r0 += slab) {
      const dim3 grid((unsigned)std::min(slab, d->rows - r0), ranges);
      if (pen && biased) k_adjust<T, true, true><<<grid, block, lds, st>>>(a, r0);
      else if (pen) k_adjust<T, true, false><<<grid, block, lds, st>>>(a, r0);
      else if (biased) k_adjust<T, false, true><<<grid, block, lds, st>>>(a, r0);
      else k_adjust<T, false, false><<<grid, block, lds, st>>>(a, r0);
      const int rc = launch_status();
      if (rc) return rc;
    }
    return SUPA_AMD_OK;
  });
}

// The balance loss of a mixture's router, and how often it took each expert.
// Per sequence of n counted tokens (all tokens together count as one sequence, or
// each sequence for itself):
//   p_te = softmax_e(x_te), or sigmoid(x_te) / sum_e sigmoid(x_te)
//   c_e  = counted tokens' choices of expert e,  a_e = E c_e / (k n) - 1
//   loss = sum_e (a_e + 1) sum_t p_te / n,  the mean of it over sequences with n > 0
//   dloss/dx_te = p_te (a_e - sum_e p_te a_e) / n    (sigmoid: times 1 - sigmoid(x_te))
// Exponents are (x - max) log2(e) in float32, as in this library's softmax: the product's rounding adds |x - max| 2^-24 of
// itself to a share's error, as much as the difference's own.
// The - 1 changes nothing, as the shares of a token sum to 1; near balance it keeps
// the difference in the last line from cancelling.
//
// HBM-bound where there are many tokens (the logits are read by both passes, the
// gradient written), launches where there are few: [262144, 256] float32 58 us (4.9 TB/s with the choices), 9 for
// the second launch and 87 for the backward (6.2 TB/s); [512, 8] 4.6, 6.2 and 3.5.  G threads share a token's
// logits, as one or more 16-byte vectors each, and keep their columns' sums of
// p in registers over their tokens; choices are counted in LDS.  A second launch
// adds the workgroups' partials in a fixed order, in float64, and forms a, counts and,
// in its last workgroup, the loss; the backward forms p again.
#include "row_group.h"

namespace sa {

constexpr int kBalFwdBlock = 512, kBalBwdBlock = 256;
constexpr int kBalMaxExperts = 1024;
constexpr int kBalCols = 16;      // columns a workgroup of the second launch adds
constexpr int kBalSumBlock = 1024;

struct BalanceArgs {
  const void* x;
  const void* chosen;
  const uint8_t* mask;
  int64_t tokens;          // of a sequence
  int32_t experts, k, idx64;
  int32_t blocks;          // workgroups a sequence
  int64_t sequences;
};

// Maximum or sum over the G threads of a token (4, 8, 16 or 64), in every one of them.
template <int G, typename F> __device__ __forceinline__ float token_join(float v, F&& f) {
  auto perm = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v = f(v, perm(v, std::integral_constant<int, 0xB1>{}));                           // quad_perm [1, 0, 3, 2]
  v = f(v, perm(v, std::integral_constant<int, 0x4E>{}));                           // quad_perm [2, 3, 0, 1]
  if constexpr (G >= 8) v = f(v, perm(v, std::integral_constant<int, 0x141>{}));    // row_half_mirror
  if constexpr (G >= 16) v = f(v, perm(v, std::integral_constant<int, 0x140>{}));   // row_mirror
  if constexpr (G == 64) {
    auto lane = [&](int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); };
    v = f(f(lane(0), lane(16)), f(lane(32), lane(48)));
  }
  return v;
}
template <int G> __device__ __forceinline__ float token_max(float v) {
  return token_join<G>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int G> __device__ __forceinline__ float token_sum(float v) {
  return token_join<G>(v, [](float a, float b) { return a + b; });
}

// The thread's columns of a token: NV vectors of V, the one that would run past the end moved back to
// it.  Its first elements are another vector's too: they have the same values, and are left out of sums.
// Element k of vector j is the thread's own where bit j V + k of `own` is set.  Fewer than V experts go element
// by element.
template <typename T, int G, int NV> struct BalCols {
  static constexpr int V = 16 / (int)sizeof(T);
  int col[NV];
  uint32_t own;
  int experts;
  bool ragged;  // some vector is not all its thread's own
  __device__ __forceinline__ BalCols(int l, int e) : own(0u), experts(e), ragged(e % V != 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (l + j * G) * V;
      col[j] = e >= V && c + V > e ? e - V : c;
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (col[j] + k >= c && col[j] + k < e) own |= 1u << (j * V + k);
    }
  }
  __device__ __forceinline__ bool is_own(int i) const { return own >> i & 1u; }
  __device__ __forceinline__ bool live(int j) const { return own >> (j * V) & ((1u << V) - 1u); }
  // Vector j of a token; -inf in the vectors that are not there, zeros for a token that does not count.
  __device__ __forceinline__ RowVec<T, V> load(const T* row, int j, bool on) const {
    constexpr uint32_t ninf = std::is_same<T, float>::value ? 0xff800000u : (std::is_same<T, bf16>::value ? 0xff80ff80u : 0xfc00fc00u);
    RowVec<T, V> r;
    const uint32_t fill = live(j) ? 0u : ninf;
    r.q[0] = make_uint4(fill, fill, fill, fill);
    if (!on || !live(j)) return r;
    if (experts >= V) {
      r.q[0] = ld_any_stream(row + col[j]);
    } else {
      const uint16_t half = (uint16_t)(ninf & 0xffffu);
      T e[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if constexpr (std::is_same<T, float>::value) e[k] = k < experts ? row[k] : -__builtin_inff();
        else e[k] = k < experts ? row[k] : __builtin_bit_cast(T, half);
      }
      __builtin_memcpy(&r, e, sizeof(r));
    }
    return r;
  }
  // The sum of f(i) over the thread's own elements.
  template <typename F> __device__ __forceinline__ float own_sum(F&& f) const {
    float s = 0.0f;
    if (!ragged) {  // the whole launch's threads
#pragma unroll
      for (int i = 0; i < NV * V; ++i) s += f(i);
    } else {
#pragma unroll
      for (int i = 0; i < NV * V; ++i) s += is_own(i) ? f(i) : 0.0f;
    }
    return s;
  }
  // e of a token's shares e / (sum of e): the reciprocal of the sum; 1 - sigmoid in `rest` (SIG).
  template <bool SIG>
  __device__ __forceinline__ float shares(const RowVec<T, V> (&w)[NV], float (&e)[NV * V], float (&rest)[NV * V]) const {
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < NV * V; ++i) {
      e[i] = row_elem<T, V>(w[i / V], i % V);
      // sigmoid(x) = e^min(x, 0) / (1 + e^-|x|): the largest is scaled to at least 1/2, so none is lost to underflow
      m = fmaxf(m, SIG ? fminf(e[i], 0.0f) : e[i]);
    }
    m = token_max<G>(m);  // subtracted before the scale: the type's lowest value times log2(e) is no float
#pragma unroll
    for (int i = 0; i < NV * V; ++i) {
      if constexpr (SIG) {
        const float x = e[i], u = __builtin_amdgcn_exp2f(-fabsf(x) * kLog2e), r = 1.0f / (1.0f + u);
        rest[i] = x > 0.0f ? u * r : r;
        e[i] = __builtin_amdgcn_exp2f((fminf(x, 0.0f) - m) * kLog2e) * r;  // a NaN is in r
      } else {
        e[i] = __builtin_amdgcn_exp2f((e[i] - m) * kLog2e);
      }
    }
    return 1.0f / token_sum<G>(own_sum([&](int i) { return e[i]; }));
  }
};

// Tokens that a thread's group has on their way at once in the backward.  In the forward it is one: a second one's
// registers cost more than they gave, and requesting the next one early gained at [262144, 256] alone (65 us for 68; [131072, 300] 43 for 40).
constexpr int kBalUnroll = 2;

template <typename T, int G, int NV, bool SIG>
__global__ void __launch_bounds__(kBalFwdBlock)
k_balance_fwd(BalanceArgs g, int64_t seq0, float* __restrict__ part_p, int32_t* __restrict__ part_c,
              int32_t* __restrict__ part_n, int32_t* __restrict__ arrived, int32_t* error_flag) {
  using Cols = BalCols<T, G, NV>;
  constexpr int V = Cols::V, TEAMS = kBalFwdBlock / G, WAVES = kBalFwdBlock / 64;
  extern __shared__ float lds[];  // [WAVES][experts] sums, then [experts] counts
  int32_t* hist = reinterpret_cast<int32_t*>(lds + WAVES * g.experts);
  __shared__ int32_t lds_n;
  const int team = threadIdx.x / G, l = threadIdx.x % G;
  const int64_t seq = seq0 + blockIdx.y;
  if (seq0 == 0 && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *arrived = 0;  // for the second launch
  for (int i = threadIdx.x; i < g.experts; i += kBalFwdBlock) hist[i] = 0;
  if (threadIdx.x == 0) lds_n = 0;
  __syncthreads();
  const Cols cols(l, g.experts);
  float acc[NV * V];
#pragma unroll
  for (int i = 0; i < NV * V; ++i) acc[i] = 0.0f;
  int32_t n = 0;
  const int64_t step = (int64_t)g.blocks * TEAMS;
  // the same number of rounds for every group: exchanges among threads of a wavefront need all of them
  for (int64_t t0 = (int64_t)blockIdx.x * TEAMS; t0 < g.tokens; t0 += step) {
    const int64_t t = t0 + team, row = seq * g.tokens + t;
    const bool on = t < g.tokens && (!g.mask || g.mask[row]);
    RowVec<T, V> w[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) w[j] = cols.load(static_cast<const T*>(g.x) + row * g.experts, j, on);
    for (int i = l; on && i < g.k; i += G) {
      const int64_t at = row * g.k + i;
      const int64_t e = g.idx64 ? static_cast<const int64_t*>(g.chosen)[at]
                                : (int64_t)static_cast<const int32_t*>(g.chosen)[at];
      if (e >= g.experts && error_flag) *error_flag = 3;
      if (e >= 0 && e < g.experts) atomicAdd(&hist[e], 1);
    }
    float e[NV * V], rest[NV * V];
    const float inv = cols.template shares<SIG>(w, e, rest), scale = on ? inv : 0.0f;
#pragma unroll
    for (int i = 0; i < NV * V; ++i) acc[i] = fmaf(e[i], scale, acc[i]);
    n += on && l == 0 ? 1 : 0;
  }
  // the groups of a wavefront, then the wavefronts
#pragma unroll
  for (int off = G; off < 64; off *= 2) {
#pragma unroll
    for (int i = 0; i < NV * V; ++i) acc[i] += __shfl_xor(acc[i], off, 64);
  }
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) < G) {
#pragma unroll
    for (int i = 0; i < NV * V; ++i)
      if (cols.is_own(i)) lds[wave * g.experts + cols.col[i / V] + i % V] = acc[i];
  }
  if (n > 0) atomicAdd(&lds_n, n);
  __syncthreads();
  const int64_t at = seq * g.blocks + blockIdx.x;
  for (int i = threadIdx.x; i < g.experts; i += kBalFwdBlock) {
    float s = lds[i];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) s += lds[v * g.experts + i];
    part_p[at * g.experts + i] = s;
    part_c[at * g.experts + i] = hist[i];
  }
  if (threadIdx.x == 0) part_n[at] = lds_n;
}

// Columns kBalCols blockIdx.x ... of sequence blockIdx.y: counts, loads (a) and their share of the loss; the
// workgroup that ends last adds the shares up.  scale: 1 / n of each sequence, and behind them 1 / sequences that count.
__global__ void __launch_bounds__(kBalSumBlock)
k_balance_sum(BalanceArgs g, int64_t seq0, int64_t all_blocks, const float* __restrict__ part_p,
              const int32_t* __restrict__ part_c, const int32_t* __restrict__ part_n, int32_t* arrived,
              double* shares, int64_t* __restrict__ counts, float* __restrict__ load, float* scale,
              float* __restrict__ loss) {
  constexpr int SLICES = kBalSumBlock / kBalCols, WAVES = kBalSumBlock / 64;
  __shared__ double lds_p[WAVES][kBalCols];
  __shared__ int64_t lds_c[WAVES][kBalCols], lds_n[WAVES];
  __shared__ int last;
  __shared__ double lds_t[2][WAVES];
  const int64_t seq = seq0 + blockIdx.y;
  const int c = threadIdx.x % kBalCols, slice = threadIdx.x / kBalCols, wave = threadIdx.x >> 6;
  const int e = blockIdx.x * kBalCols + c;
  double p = 0.0;
  int64_t count = 0, tokens = 0;
  if (e < g.experts) {
    constexpr int U = 4;
    for (int b0 = slice; b0 < g.blocks; b0 += SLICES * U) {
      float v[U];
      int32_t k[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool on = b0 + u * SLICES < g.blocks;
        const int64_t at = (seq * g.blocks + b0 + u * SLICES) * g.experts + e;
        v[u] = on ? part_p[at] : 0.0f;
        k[u] = on ? part_c[at] : 0;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        p += (double)v[u];
        count += k[u];
      }
    }
  }
  for (int b = threadIdx.x; b < g.blocks; b += kBalSumBlock) tokens += part_n[seq * g.blocks + b];
#pragma unroll
  for (int off = 32; off >= kBalCols; off >>= 1) {  // the wavefront's slices
    p += __shfl_xor(p, off, 64);
    count += __shfl_xor(count, off, 64);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) tokens += __shfl_xor(tokens, off, 64);
  if ((threadIdx.x & 63) < kBalCols) {
    lds_p[wave][c] = p;
    lds_c[wave][c] = count;
  }
  if ((threadIdx.x & 63) == 0) lds_n[wave] = tokens;
  __syncthreads();
  int64_t n = 0;
  p = 0.0;
  count = 0;
  if (threadIdx.x < kBalCols) {
    for (int w = 0; w < WAVES; ++w) {
      p += lds_p[w][c];
      count += lds_c[w][c];
      n += lds_n[w];
    }
  }
  double share = 0.0;
  if (threadIdx.x < kBalCols && e < g.experts) {
    const double a = n > 0 ? (double)g.experts * (double)count / ((double)g.k * (double)n) : 0.0;
    counts[seq * g.experts + e] = count;
    load[seq * g.experts + e] = (float)(a - 1.0);
    share = n > 0 ? a * p / (double)n : 0.0;
  }
#pragma unroll
  for (int off = kBalCols / 2; off > 0; off >>= 1) share += __shfl_xor(share, off, 64);
  if (threadIdx.x == 0) {
    const int64_t at = seq * gridDim.x + blockIdx.x;
    __hip_atomic_store(&shares[at], share, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (blockIdx.x == 0) __hip_atomic_store(&scale[seq], n > 0 ? (float)(1.0 / (double)n) : 0.0f, __ATOMIC_RELAXED,
                                            __HIP_MEMORY_SCOPE_AGENT);
    last = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == all_blocks - 1;
  }
  __syncthreads();
  if (!last) return;
  double v[2] = {0.0, 0.0};  // the shares, and the sequences that count
  for (int64_t i = threadIdx.x; i < all_blocks; i += kBalSumBlock)
    v[0] += __hip_atomic_load(&shares[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (int64_t i = threadIdx.x; i < g.sequences; i += kBalSumBlock)
    v[1] += __hip_atomic_load(&scale[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) > 0.0f ? 1.0 : 0.0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v[i] += __shfl_xor(v[i], off, 64);
    if ((threadIdx.x & 63) == 0) lds_t[i][threadIdx.x >> 6] = v[i];
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  double s = 0.0, q = 0.0;
  for (int w = 0; w < kBalSumBlock / 64; ++w) {
    s += lds_t[0][w];
    q += lds_t[1][w];
  }
  loss[0] = q > 0.0 ? (float)(s / q) : 0.0f;
  scale[g.sequences] = q > 0.0 ? (float)(1.0 / q) : 0.0f;
}

template <typename T, int G, int NV, bool SIG>
__global__ void __launch_bounds__(kBalBwdBlock)
k_balance_bwd(BalanceArgs g, int64_t seq0, const float* __restrict__ load, const float* __restrict__ scale,
              const float* __restrict__ grad_out, T* __restrict__ grad) {
  using Cols = BalCols<T, G, NV>;
  constexpr int V = Cols::V, TEAMS = kBalBwdBlock / G, U = kBalUnroll;
  const int team = threadIdx.x / G, l = threadIdx.x % G;
  const int64_t seq = seq0 + blockIdx.y;
  const Cols cols(l, g.experts);
  float a[NV * V];
#pragma unroll
  for (int i = 0; i < NV * V; ++i)
    a[i] = cols.live(i / V) && cols.col[i / V] + i % V < g.experts ? load[seq * g.experts + cols.col[i / V] + i % V] : 0.0f;
  const float gs = grad_out[0] * scale[seq] * scale[g.sequences];
  const int64_t step = (int64_t)g.blocks * TEAMS;
  for (int64_t t0 = (int64_t)blockIdx.x * TEAMS; t0 < g.tokens; t0 += step * U) {
    RowVec<T, V> w[U][NV];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = t0 + u * step + team;
      on[u] = t < g.tokens && (!g.mask || g.mask[seq * g.tokens + t]);
#pragma unroll
      for (int j = 0; j < NV; ++j) w[u][j] = cols.load(static_cast<const T*>(g.x) + (seq * g.tokens + t) * g.experts, j, on[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = t0 + u * step + team;
      float e[NV * V], rest[NV * V];
      const float inv = cols.template shares<SIG>(w[u], e, rest);
      const float d = token_sum<G>(cols.own_sum([&](int i) { return e[i] * a[i]; })) * inv;
      if (t >= g.tokens) continue;
      const float k0 = on[u] ? inv * gs : 0.0f;
      T* dst = grad + (seq * g.tokens + t) * g.experts;
#pragma unroll
      for (int i = 0; i < NV * V; ++i) {
        e[i] = e[i] * (a[i] - d) * k0;
        if (SIG) e[i] *= rest[i];
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!cols.live(j)) continue;
        float f[V];
#pragma unroll
        for (int k = 0; k < V; ++k) f[k] = e[j * V + k];
        if (g.experts >= V) {
          store_any<T, V>(dst + cols.col[j], f);
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (k < g.experts) dst[k] = from_arith<T>(f[k]);
        }
      }
    }
  }
}

int balance_args(const supa_amd_balance_desc* d, BalanceArgs& g) {
  if (!d || d->sequences < 0 || d->tokens < 0 || d->experts < 1 || d->k < 1) return SUPA_AMD_EINVAL;
  if (d->experts > kBalMaxExperts || d->k > d->experts || d->sequences >= (int64_t(1) << 31) ||
      d->tokens >= (int64_t(1) << 31) || (d->sequences > 0 && d->tokens > ((int64_t(1) << 31) - 1) / d->sequences))
    return SUPA_AMD_ELAYOUT;
  if (d->scores != SUPA_AMD_SCORES_SOFTMAX && d->scores != SUPA_AMD_SCORES_SIGMOID) return SUPA_AMD_EINVAL;
  if (d->dtype != SUPA_AMD_F32 && d->dtype != SUPA_AMD_BF16 && d->dtype != SUPA_AMD_F16) return SUPA_AMD_EDTYPE;
  if (d->index_dtype != SUPA_AMD_I64 && d->index_dtype != SUPA_AMD_I32) return SUPA_AMD_EDTYPE;
  g = BalanceArgs{};
  g.x = d->logits;
  g.chosen = d->chosen;
  g.mask = static_cast<const uint8_t*>(d->mask);
  g.sequences = d->sequences;
  g.tokens = d->tokens;
  g.experts = (int32_t)d->experts;
  g.k = (int32_t)d->k;
  g.idx64 = d->index_dtype == SUPA_AMD_I64;
  return SUPA_AMD_OK;
}

// f(type, threads a token, vectors a thread).  Few threads with up to 16 elements each: what a token's threads
// exchange, its maximum and sum, is then a few steps for many tokens at once.  32 elements of 16 bits where 64 threads would
// idle ([131072, 300] bf16: 40 us and 57 backward, 72 and 68 with 64 threads).
template <typename F> int with_balance(const supa_amd_balance_desc* d, F&& f) {
  return with_float_storage(d->dtype, [&](auto* tag) -> int {
    using T = std::remove_pointer_t<decltype(tag)>;
    constexpr int V = 16 / (int)sizeof(T), N = 16 / V;
    auto scores = [&](auto threads, auto vecs) -> int {
      return d->scores == SUPA_AMD_SCORES_SIGMOID ? f(tag, threads, vecs, std::true_type{})
                                                  : f(tag, threads, vecs, std::false_type{});
    };
    using std::integral_constant;
    const int64_t vecs = (d->experts + V - 1) / V;
    if (vecs <= 4) return scores(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    if (vecs <= 4 * N) return scores(integral_constant<int, 4>{}, integral_constant<int, N>{});
    if (vecs <= 8 * N) return scores(integral_constant<int, 8>{}, integral_constant<int, N>{});
    if (vecs <= 16 * N) return scores(integral_constant<int, 16>{}, integral_constant<int, N>{});
    if (N == 2 && vecs <= 64) return scores(integral_constant<int, 16>{}, integral_constant<int, 4>{});
    if (vecs <= 128) return scores(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    if constexpr (N == 4) return scores(integral_constant<int, 64>{}, integral_constant<int, 4>{});
    return SUPA_AMD_ELAYOUT;
  });
}

// Threads that share a token, as with_balance chooses them.
int balance_threads(int64_t experts, int dtype) {
  const int64_t vecs = (experts * dtype_size(dtype) + 15) / 16;
  const int n = dtype == SUPA_AMD_F32 ? 4 : 2;
  return vecs <= 4 * n ? 4 : (vecs <= 8 * n ? 8 : (vecs <= 64 ? 16 : 64));
}

// Workgroups a sequence: `most` in all, each with a round of its groups at least.
int32_t balance_blocks(const supa_amd_balance_desc* d, int64_t most, int threads) {
  const int64_t round = threads / balance_threads(d->experts, d->dtype);
  const int64_t want = (d->tokens + round - 1) / round, each = std::max<int64_t>(1, most / std::max<int64_t>(1, d->sequences));
  return (int32_t)std::max<int64_t>(1, std::min(want, each));
}
// Two workgroups of 512 threads a CU for the forward: more have more partials, which the second launch adds
// ([262144, 256] float32, both launches: 68 us; 1024 of 256 threads 73, 2048 84; [262144, 64] bf16 24, 28 and 40).
constexpr int64_t kBalFwdBlocks = 512;
constexpr int64_t kBalBwdBlocks = 1 << 14;

// Workspace: the shares of the loss, then the partials: sums, counts, tokens; the arrivals.
struct BalanceSpace {
  int64_t shares, p, c, n, arrived, bytes;
};
BalanceSpace balance_space(const BalanceArgs& g) {
  const int64_t slices = (g.experts + kBalCols - 1) / kBalCols, blocks = g.sequences * g.blocks;
  BalanceSpace s{};
  s.p = 8 * g.sequences * slices;
  s.c = s.p + 4 * blocks * g.experts;
  s.n = s.c + 4 * blocks * g.experts;
  s.arrived = s.n + 4 * blocks;
  s.bytes = s.arrived + 4;
  return s;
}

}  // namespace sa

using namespace sa;

extern "C" {

int64_t supa_amd_balance_workspace_bytes(const supa_amd_balance_desc* d) {
  BalanceArgs g;
  const int rc = balance_args(d, g);
  if (rc) return rc;
  g.blocks = balance_blocks(d, kBalFwdBlocks, kBalFwdBlock);
  return balance_space(g).bytes;
}

int supa_amd_balance_forward(const supa_amd_balance_desc* d, float* loss, int64_t* counts, float* load, float* scale,
                             void* workspace, int64_t ws_bytes, int32_t* error_flag, void* stream) {
  BalanceArgs g;
  const int rc = balance_args(d, g);
  if (rc) return rc;
  if (d->sequences == 0) return SUPA_AMD_EINVAL;
  if (!loss || !counts || !load || !scale || (d->tokens > 0 && (!d->logits || !d->chosen))) return SUPA_AMD_EINVAL;
  g.blocks = balance_blocks(d, kBalFwdBlocks, kBalFwdBlock);
  const BalanceSpace s = balance_space(g);
  if (!workspace || ws_bytes < s.bytes) return SUPA_AMD_EWORKSPACE;
  if (!aligned(workspace, 8)) return SUPA_AMD_EINVAL;
  char* ws = static_cast<char*>(workspace);
  double* shares = reinterpret_cast<double*>(ws);
  float* part_p = reinterpret_cast<float*>(ws + s.p);
  int32_t *part_c = reinterpret_cast<int32_t*>(ws + s.c), *part_n = reinterpret_cast<int32_t*>(ws + s.n),
          *arrived = reinterpret_cast<int32_t*>(ws + s.arrived);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t lds = (size_t)g.experts * 4 * (kBalFwdBlock / 64 + 1);
  for (int64_t s0 = 0; s0 < g.sequences; s0 += 65535) {
    const unsigned n = (unsigned)std::min<int64_t>(65535, g.sequences - s0);
    const int rc = with_balance(d, [&](auto* tag, auto threads, auto vecs, auto sig) -> int {
      using T = std::remove_pointer_t<decltype(tag)>;
      k_balance_fwd<T, threads.value, vecs.value, sig.value><<<dim3(g.blocks, n), kBalFwdBlock, lds, st>>>(
          g, s0, part_p, part_c, part_n, arrived, error_flag);
      return launch_status();
    });
    if (rc) return rc;
  }
  const unsigned slices = (unsigned)((g.experts + kBalCols - 1) / kBalCols);
  for (int64_t s0 = 0; s0 < g.sequences; s0 += 65535) {
    const unsigned n = (unsigned)std::min<int64_t>(65535, g.sequences - s0);
    k_balance_sum<<<dim3(slices, n), kBalSumBlock, 0, st>>>(g, s0, (int64_t)slices * g.sequences, part_p, part_c, part_n,
                                                            arrived, shares, counts, load, scale, loss);
    const int rc = launch_status();
    if (rc) return rc;
  }
  return SUPA_AMD_OK;
}

int supa_amd_balance_backward(const supa_amd_balance_desc* d, const float* grad_loss, const float* load,
                              const float* scale, void* grad_logits, void* stream) {
  BalanceArgs g;
  const int rc = balance_args(d, g);
  if (rc) return rc;
  if (d->sequences == 0 || d->tokens == 0) return SUPA_AMD_OK;
  if (!grad_loss || !load || !scale || !grad_logits || !d->logits) return SUPA_AMD_EINVAL;
  g.blocks = balance_blocks(d, kBalBwdBlocks, kBalBwdBlock * kBalUnroll);
  hipStream_t st = static_cast<hipStream_t>(stream);
  for (int64_t s0 = 0; s0 < g.sequences; s0 += 65535) {
    const unsigned n = (unsigned)std::min<int64_t>(65535, g.sequences - s0);
    const int rc = with_balance(d, [&](auto* tag, auto threads, auto vecs, auto sig) -> int {
      using T = std::remove_pointer_t<decltype(tag)>;
      k_balance_bwd<T, threads.value, vecs.value, sig.value><<<dim3(g.blocks, n), kBalBwdBlock, 0, st>>>(
          g, s0, load, scale, grad_loss, static_cast<T*>(grad_logits));
      return launch_status();
    });
    if (rc) return rc;
  }
  return SUPA_AMD_OK;
}

}  // extern "C"

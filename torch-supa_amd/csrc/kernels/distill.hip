// Distillation from a teacher's top logits: per row of student logits x and K
// stored (token, teacher logit) pairs, with z = x / temperature,
//   p_k = exp(t_k / temperature - lt),  lt the pairs' own log-sum-exp or a given one
//   loss = sum_k p_k (log p_k - log q_{i_k}),  q = softmax(z)
// and, where lt is given, the rest of both as one more class: with r = 1 - sum p
// and q_R the student's mass outside the listed tokens, + r (log r - log q_R).
// The gradient of z is w q_j - p_j at a listed token and
// (w q_R - r) exp(z_j - lse_R) elsewhere (w = sum p + r; without rest: q_j).
//
// HBM-bound: the forward reads the logits once, the backward reads them and
// writes the gradient; the pairs are a few hundred bytes a row.  The forward
// keeps an online (max, sum of exp2) pair a thread, float32; what depends on the
// pairs alone (K exponentials, their sums, logarithms) is float64: r and small
// losses are differences of near values.  q_R is summed over its own elements,
// not as 1 minus the listed ones: a bitmap of the listed tokens, in LDS, tells
// them apart.  A workgroup of the backward puts the listed tokens among its columns into LDS
// (a bit, and the pair's number in a table by column) while its logits are on their way; an
// element whose bit is set takes its p from there.
//
// A token listed twice has the sum of its p: the row's first such pair carries it.
// Twice-listed tokens are found by a hash table in LDS; only rows that have one
// compare all pairs.
#include <cmath>

#include "softmax_common.h"

namespace sa {

constexpr int kDisBlock = 256;
constexpr int kDisEntries = 4;            // pairs a thread holds in the forward
constexpr int kDisMaxEntries = kDisBlock * kDisEntries;
static_assert(kDisMaxEntries == SUPA_AMD_DISTILL_MAX_ENTRIES);
constexpr int kDisUnroll = 4;             // 16-byte vectors in flight per thread
constexpr int kDisWaveVecs = 2048;        // most vectors of a row that a wavefront takes alone
constexpr int kDisSegment = 1 << 17;      // columns whose bitmap is in LDS at a time: 16 KiB
constexpr int kDisStats = 8;              // floats a row keeps for the backward
constexpr double kLn2 = 0.69314718055994530942;
constexpr double kLog2eD = 1.44269504088896340736;

struct DistillArgs {
  const void* x;
  const void* idx;
  const void* teacher;
  const float* teacher_lse;
  int64_t xs[2];     // distance of rows: outer, inner
  FastDiv inner;     // row -> (outer, inner)
  int64_t vocab;
  int32_t entries, hash;  // pairs a row; slots of its hash table, a power of two >= 2 entries
  int32_t idx64, teacher_dtype;
  int32_t segment;   // columns of a bitmap
  double c;          // log2(e) / temperature
  float c_near;      // c rounded
  float c_hi, c_lo;  // c in two parts, both above 0: -inf stays -inf through their products
  double inv_t;
};

template <typename T> __device__ __forceinline__ const T* dis_row(const DistillArgs& g, int64_t row) {
  uint32_t o, i;
  g.inner.divmod((uint32_t)row, o, i);
  return static_cast<const T*>(g.x) + ((int64_t)o * g.xs[0] + (int64_t)i * g.xs[1]);
}
__device__ __forceinline__ int64_t dis_index(const DistillArgs& g, int64_t at) {
  return g.idx64 ? static_cast<const int64_t*>(g.idx)[at] : (int64_t)static_cast<const int32_t*>(g.idx)[at];
}

// Exchange among the G threads of a row through LDS.
template <int G> __device__ __forceinline__ void team_sync() {
  if constexpr (G == 64) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}
// Maxima / sums of N values over the G threads, in every one of them, in a fixed order.  lds: N values
// a wavefront of the row, used by no other exchange.
template <int G, int N> __device__ __forceinline__ void team_max(float (&v)[N], float* lds) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v[i] = fmaxf(v[i], __shfl_xor(v[i], off, 64));
  }
  if constexpr (G > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) lds[wave * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int w = 0; w < G / 64; ++w) v[i] = fmaxf(v[i], lds[w * N + i]);
    }
  }
}
template <int G, int N> __device__ __forceinline__ void team_sum(double (&v)[N], double* lds) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v[i] += __shfl_xor(v[i], off, 64);
  }
  if constexpr (G > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) lds[wave * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = lds[i];
#pragma unroll
      for (int w = 1; w < G / 64; ++w) v[i] += lds[w * N + i];
    }
  }
}

// A row's pairs: thread l of G holds pairs l, l + G, ...
struct DistillEntries {
  int32_t at[kDisEntries];  // token, or -1: none there
  float t[kDisEntries], x[kDisEntries];  // teacher's and student's logits
};

// A pair as the backward reads it: the token, or -1 where another pair carries it or none is there, and the bits of its p.
struct DistillPair {
  int32_t at;
  float p;
};

// LDS of a row, in this order: the slow path's p (float64), the pairs' tokens, the hash table, the bitmap.
struct DistillLds {
  double* p;
  int32_t* at;
  int32_t* hash;
  uint32_t* bits;
};
inline __host__ __device__ size_t dis_lds_bytes(int entries, int hash, int64_t segment) {
  return (size_t)((entries + 1) / 2 * 2) * 12 + (size_t)hash * 4 + (size_t)((segment + 63) / 64) * 8;
}
__device__ __forceinline__ DistillLds dis_lds(char* p, int entries, int hash) {
  const int n = (entries + 1) / 2 * 2;
  DistillLds s;
  s.p = reinterpret_cast<double*>(p);
  s.at = reinterpret_cast<int32_t*>(s.p + n);
  s.hash = s.at + n;
  s.bits = reinterpret_cast<uint32_t*>(s.hash + hash);
  return s;
}

// Loads a row's pairs, and finds tokens that are listed twice (*dup, zero before).  A pair is there if its
// token is in [0, vocab) and its teacher logit is not -inf.  Not HASH: the tokens alone.  Ends without an exchange.
template <typename T, int G, bool HASH>
__device__ __forceinline__ DistillEntries dis_entries(const DistillArgs& g, const T* xr, int64_t row, int l,
                                                      const DistillLds& s, int* dup, int32_t* error_flag) {
  DistillEntries e;
#pragma unroll
  for (int i = 0; i < kDisEntries; ++i) {
    e.at[i] = -1;
    e.t[i] = -__builtin_inff();
    e.x[i] = -__builtin_inff();
    const int k = l + i * G;
    if (k >= g.entries) continue;
    const int64_t at = dis_index(g, row * g.entries + k);
    e.t[i] = load_dyn<float>(g.teacher, row * g.entries + k, g.teacher_dtype);
    if (HASH && at >= g.vocab && error_flag) *error_flag = 3;
    if (at >= 0 && at < g.vocab && e.t[i] != -__builtin_inff()) e.at[i] = (int32_t)at;
    if (!HASH) continue;
    if (e.at[i] >= 0) e.x[i] = (float)to_arith(xr[at]);
    s.at[k] = e.at[i];
    if (e.at[i] >= 0) {  // at most half of the slots are taken: the search ends
      uint32_t h = ((uint32_t)at * 0x9E3779B1u) >> 16;
      for (;; ++h) {
        const int old = atomicCAS(&s.hash[h & (uint32_t)(g.hash - 1)], -1, e.at[i]);
        if (old == -1) break;
        if (old == e.at[i]) {
          *dup = 1;
          break;
        }
      }
    }
  }
  return e;
}

__device__ __forceinline__ void dis_split(double v, float* out) {
  out[0] = (float)v;
  out[1] = (float)(v - (double)out[0]);
}

// What a row's finish writes: its loss, alone or with whether it counts, its statistics and its pairs (may be null).
struct DistillOut {
  float* loss;
  float2* loss_count;
  float* stats;
  DistillPair* pairs;
  __device__ __forceinline__ void row(int64_t row, float v, bool counted) const {
    if (loss) loss[row] = v;
    else loss_count[row] = make_float2(v, counted ? 1.0f : 0.0f);
  }
};

// A row without a pair: nothing is read of its logits.
template <int G>
__device__ __forceinline__ void dis_nothing(const DistillArgs& g, int64_t row, int l, const DistillOut& out) {
  if (out.pairs) {
    for (int k = l; k < g.entries; k += G) out.pairs[row * g.entries + k] = DistillPair{-1, 0.0f};
  }
  if (l < kDisStats) out.stats[row * kDisStats + l] = 0.0f;
  if (l == 0) out.row(row, 0.0f, false);
}

// From the stream's pair (m, s) -- the largest of its raw logits and the sum of exp2((x - m) c) -- and
// the row's pairs to the row's loss, its statistics and the pairs' weights.  Every thread of the row; exchanged before.
template <int G, bool REST>
__device__ __forceinline__ void dis_finish(const DistillArgs& g, int64_t row, int l, float m, float s,
                                           const DistillEntries& e, const DistillLds& lds, const int* dup, float* lds_f,
                                           double* lds_d, const DistillOut& out) {
  float top[2] = {-__builtin_inff(), m};
#pragma unroll
  for (int i = 0; i < kDisEntries; ++i) {
    if (e.at[i] < 0) continue;
    top[0] = fmaxf(top[0], e.t[i]);
    if (REST) top[1] = fmaxf(top[1], e.x[i]);
  }
  team_max<G, 2>(top, lds_f);
  const bool twice = *dup != 0;
  const double M = top[1] == -__builtin_inff() ? 0.0 : (double)top[1];
  const double lt = REST ? (double)g.teacher_lse[row] * kLog2eD : (double)top[0] * g.c;
  double p[kDisEntries];
  bool first[kDisEntries];  // no pair before lists the token
  double sum[5] = {0.0, 0.0, 0.0, 0.0, 0.0};  // p, p log2 p, p (z - M), listed tokens' exp2(z - M) and their number
#pragma unroll
  for (int i = 0; i < kDisEntries; ++i) {
    p[i] = 0.0;
    first[i] = e.at[i] >= 0;
    if (e.at[i] < 0) continue;
    const double log_p = (double)e.t[i] * g.c - lt;
    p[i] = exp2(log_p);
    if (p[i] != 0.0) {
      sum[0] += p[i];
      sum[1] += p[i] * log_p;
      sum[2] += p[i] * (((double)e.x[i] - M) * g.c);
    }
    if (twice) {
      const int k = l + i * G;
      for (int j = 0; j < k && first[i]; ++j) first[i] = lds.at[j] != e.at[i];
      lds.p[k] = p[i];
    }
    if (REST && first[i]) {
      sum[3] += exp2(((double)e.x[i] - M) * g.c);
      sum[4] += 1.0;
    }
  }
  team_sum<G, 5>(sum, lds_d);
  if (twice) {
    if constexpr (G == 64) team_sync<G>();  // the sums have exchanged otherwise
#pragma unroll
    for (int i = 0; i < kDisEntries; ++i) {
      const int k = l + i * G;
      if (!first[i]) continue;
      for (int j = k + 1; j < g.entries; ++j)
        if (lds.at[j] == e.at[i]) p[i] += lds.p[j];
    }
  }
  const double norm = REST ? 1.0 : 1.0 / sum[0];
#pragma unroll
  for (int i = 0; i < kDisEntries; ++i) {
    const int k = l + i * G;
    if (out.pairs && k < g.entries)
      out.pairs[row * g.entries + k] = DistillPair{first[i] ? e.at[i] : -1, (float)(p[i] * norm)};
  }
  if (l != 0) return;
  float st[kDisStats] = {};
  double total = (double)s;  // of exp2(z - M)
  if (REST) total = (s != 0.0f ? (double)s * exp2(((double)m - M) * g.c) : 0.0) + sum[3];
  const double lse = M * g.c + log2(total);
  double weight = 1.0, L;
  if constexpr (REST) {
    weight = sum[0];
    L = sum[1] - sum[2] + weight * log2(total);
    const bool empty = sum[4] == (double)g.vocab;  // every token is listed
    const double r = empty ? 0.0 : fmax(0.0, 1.0 - sum[0]);
    const double rest = (m == -__builtin_inff() ? 0.0 : (double)m * g.c) + log2((double)s);  // -inf: no mass outside
    if (r > 0.0) L += r * (log2(r) - (rest - lse));
    weight += r;
    const bool mass = rest != -__builtin_inf() && !empty;
    dis_split(mass ? rest : 0.0, st);
    st[2] = mass ? (float)(weight * exp2(rest - lse) - r) : 0.0f;
  } else {
    L = (sum[1] - sum[2]) * norm - log2(sum[0]) + log2(total);
    dis_split(lse, st);
    st[2] = 1.0f;
  }
  st[3] = (float)weight;
  dis_split(lse, st + 4);
  st[6] = 1.0f;  // the row counts
  out.row(row, (float)(L * kLn2), true);
#pragma unroll
  for (int i = 0; i < kDisStats; ++i) out.stats[row * kDisStats + i] = st[i];
}

// One online step over a batch of values: (m, s) with those of f.
template <int N> __device__ __forceinline__ void dis_online(float& m, float& s, const float (&f)[N], float c) {
  float mb = f[0];
#pragma unroll
  for (int k = 1; k < N; ++k) mb = fmaxf(mb, f[k]);
  // fmaxf passes over a NaN, so M says nothing of them: the sum is always taken, and is then NaN
  const float M = fmaxf(m, mb), base = M == -__builtin_inff() ? 0.0f : M;
  float sb = 0.0f;
#pragma unroll
  for (int k = 0; k < N; ++k) sb += __builtin_amdgcn_exp2f((f[k] - base) * c);
  s = (M != -__builtin_inff() ? s * __builtin_amdgcn_exp2f((m - M) * c) : s) + sb;
  m = M;
}

// (m, s) of the columns [c0, c1) of a row for one of G threads; c0 is a multiple of a vector.  REST: the
// listed tokens, whose bits are set from column c0 on, count as -inf.
template <typename T, int G, bool REST>
__device__ __forceinline__ void dis_stream(const T* xr, int64_t c0, int64_t c1, int l, float c, const uint32_t* bits,
                                           float& m, float& s) {
  constexpr int V = VecOf<T>::V;
  const T* p = xr + c0;
  const int n = (int)(c1 - c0), nvec = n / V;
  for (int v0 = l; v0 < nvec; v0 += G * kDisUnroll) {
    uint4 w[kDisUnroll];
#pragma unroll
    for (int u = 0; u < kDisUnroll; ++u)
      if (v0 + u * G < nvec) w[u] = ld_any_stream(p + (int64_t)(v0 + u * G) * V);
    float f[kDisUnroll * V];
#pragma unroll
    for (int u = 0; u < kDisUnroll; ++u) {
      const int v = v0 + u * G;
      if (v < nvec) {
#pragma unroll
        for (int k = 0; k < V; ++k) f[u * V + k] = elem_f<T>(w[u], k);
        if constexpr (REST) {
          const uint32_t b = bits[v * V / 32] >> (v * V % 32) & ((1u << V) - 1u);
          if (b) {
#pragma unroll
            for (int k = 0; k < V; ++k)
              if (b >> k & 1u) f[u * V + k] = -__builtin_inff();
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) f[u * V + k] = -__builtin_inff();
      }
    }
    dis_online(m, s, f, c);
  }
  for (int j = nvec * V + l; j < n; j += G) {  // after the whole vectors
    float f[1] = {(float)to_arith(p[j])};
    if (REST && (bits[j / 32] >> (j % 32) & 1u)) f[0] = -__builtin_inff();
    dis_online(m, s, f, c);
  }
}

// (m, s) of all G threads, in every one of them.
template <int G> __device__ __forceinline__ void dis_join(float& m, float& s, float c, float* lds_m, float* lds_s) {
  float M = m;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
  if constexpr (G > 64) {
    if ((threadIdx.x & 63) == 0) lds_m[threadIdx.x >> 6] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < G / 64; ++w) M = fmaxf(M, lds_m[w]);
  }
  if (M != -__builtin_inff()) s *= __builtin_amdgcn_exp2f((m - M) * c);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if constexpr (G > 64) {
    if ((threadIdx.x & 63) == 0) lds_s[threadIdx.x >> 6] = s;
    __syncthreads();
    s = lds_s[0];
#pragma unroll
    for (int w = 1; w < G / 64; ++w) s += lds_s[w];
  }
  m = M;
}

// Sets the bits of the listed tokens in [c0, c0 + segment); exchanges before and after.
template <int G>
__device__ __forceinline__ void dis_mark(const DistillArgs& g, const DistillEntries& e, int64_t c0, int l, uint32_t* bits) {
  team_sync<G>();
  for (int i = l; i < (g.segment + 31) / 32; i += G) bits[i] = 0u;
  team_sync<G>();
#pragma unroll
  for (int i = 0; i < kDisEntries; ++i) {
    const int64_t at = (int64_t)e.at[i] - c0;
    if (e.at[i] >= 0 && at >= 0 && at < g.segment) atomicOr(&bits[at / 32], 1u << (at % 32));
  }
  team_sync<G>();
}

// Whether any of the row's pairs is there, in every thread of the row.
template <int G> __device__ __forceinline__ bool dis_any(const DistillEntries& e) {
  bool any = false;
#pragma unroll
  for (int i = 0; i < kDisEntries; ++i) any = any || e.at[i] >= 0;
  if constexpr (G == 64) {
    team_sync<G>();
    return __any(any);
  } else {
    return __syncthreads_or(any);
  }
}

// Exchanges of a row's finish.
template <int G> struct DistillJoin {
  float f[2 * G / 64], m[G / 64], s[G / 64];
  double d[5 * G / 64];
  int dup;
};

// G threads a row.
template <typename T, int G, bool REST>
__global__ void __launch_bounds__(kDisBlock)
k_distill_fwd(DistillArgs g, int64_t row0, int64_t rows, DistillOut out, int32_t* error_flag) {
  constexpr int TEAMS = kDisBlock / G;
  extern __shared__ double lds_dyn[];
  __shared__ DistillJoin<G> join[TEAMS];
  const int team = threadIdx.x / G, l = threadIdx.x % G;
  const int64_t row = row0 + (int64_t)blockIdx.x * TEAMS + team;
  if (row >= row0 + rows) return;  // whole rows: no exchange is left waiting
  DistillJoin<G>& j = join[team];
  const T* xr = dis_row<T>(g, row);
  const DistillLds s = dis_lds(
      reinterpret_cast<char*>(lds_dyn) + team * dis_lds_bytes(g.entries, g.hash, REST ? g.segment : 0), g.entries, g.hash);
  for (int i = l; i < g.hash; i += G) s.hash[i] = -1;
  if (l == 0) j.dup = 0;
  team_sync<G>();
  const DistillEntries e = dis_entries<T, G, true>(g, xr, row, l, s, &j.dup, error_flag);
  if (!dis_any<G>(e)) return dis_nothing<G>(g, row, l, out);
  float m = -__builtin_inff(), sum = 0.0f;
  for (int64_t c0 = 0; c0 < g.vocab; c0 += g.segment) {
    if (REST) dis_mark<G>(g, e, c0, l, s.bits);
    dis_stream<T, G, REST>(xr, c0, c0 + g.segment < g.vocab ? c0 + g.segment : g.vocab, l, g.c_near, s.bits, m, sum);
  }
  dis_join<G>(m, sum, g.c_near, j.m, j.s);
  dis_finish<G, REST>(g, row, l, m, sum, e, s, &j.dup, j.f, j.d, out);
}

// Few rows: parts of a row (of `columns` columns, a multiple of 32) to a workgroup each; (m, s) of each part ...
template <typename T, bool REST>
__global__ void __launch_bounds__(kDisBlock)
k_distill_part(DistillArgs g, int64_t columns, float2* __restrict__ parts) {
  constexpr int G = kDisBlock;
  extern __shared__ double lds_dyn[];
  __shared__ float lds_m[G / 64], lds_s[G / 64];
  const int64_t row = blockIdx.y, c0 = blockIdx.x * columns, c1 = c0 + columns < g.vocab ? c0 + columns : g.vocab;
  const T* xr = dis_row<T>(g, row);
  uint32_t* bits = reinterpret_cast<uint32_t*>(lds_dyn);
  DistillEntries e;
  if constexpr (REST) e = dis_entries<T, G, false>(g, xr, row, threadIdx.x, DistillLds{}, nullptr, nullptr);
  float m = -__builtin_inff(), sum = 0.0f;
  for (int64_t s0 = c0; s0 < c1; s0 += g.segment) {
    if (REST) dis_mark<G>(g, e, s0, threadIdx.x, bits);
    dis_stream<T, G, REST>(xr, s0, s0 + g.segment < c1 ? s0 + g.segment : c1, threadIdx.x, g.c_near, bits, m, sum);
  }
  dis_join<G>(m, sum, g.c_near, lds_m, lds_s);
  if (threadIdx.x == 0) parts[row * gridDim.x + blockIdx.x] = make_float2(m, sum);
}
// ... and the rows from their parts, G threads a row.
template <typename T, int G, bool REST>
__global__ void __launch_bounds__(G)
k_distill_rows(DistillArgs g, int nparts, const float2* __restrict__ parts, DistillOut out, int32_t* error_flag) {
  extern __shared__ double lds_dyn[];
  __shared__ DistillJoin<G> j;
  const int64_t row = blockIdx.x;
  const int l = threadIdx.x;
  const DistillLds s = dis_lds(reinterpret_cast<char*>(lds_dyn), g.entries, g.hash);
  for (int i = l; i < g.hash; i += G) s.hash[i] = -1;
  if (l == 0) j.dup = 0;
  team_sync<G>();
  const DistillEntries e = dis_entries<T, G, true>(g, dis_row<T>(g, row), row, l, s, &j.dup, error_flag);
  if (!dis_any<G>(e)) return dis_nothing<G>(g, row, l, out);
  const float2 part = l < nparts ? parts[row * nparts + l] : make_float2(-__builtin_inff(), 0.0f);
  float m = part.x, sum = part.y;
  dis_join<G>(m, sum, g.c_near, j.m, j.s);
  dis_finish<G, REST>(g, row, l, m, sum, e, s, &j.dup, j.f, j.d, out);
}

// The sum (or mean) of the rows' losses and the number of rows that count, in float64 and a fixed order.  More
// rows than kDisSumRows: a first launch (PART) leaves the sums of runs of rows.
constexpr int kDisSumBlock = 1024;
constexpr int64_t kDisSumRows = 8 * kDisSumBlock;

template <bool PART>
__global__ void __launch_bounds__(kDisSumBlock)
k_distill_total(const float2* __restrict__ rows, const double* __restrict__ parts, int64_t n, int mean,
                double* __restrict__ parts_out, float* __restrict__ loss, float* __restrict__ count) {
  __shared__ double lds[2 * kDisSumBlock / 64];
  double v[2] = {0.0, 0.0};
  if (parts) {
    for (int64_t i = threadIdx.x; i < n; i += kDisSumBlock) {
      v[0] += parts[2 * i];
      v[1] += parts[2 * i + 1];
    }
  } else {
    const int64_t i0 = (int64_t)blockIdx.x * kDisSumRows + threadIdx.x;
    float2 r[kDisSumRows / kDisSumBlock];
#pragma unroll
    for (int u = 0; u < (int)(kDisSumRows / kDisSumBlock); ++u)
      r[u] = i0 + u * kDisSumBlock < n ? rows[i0 + u * kDisSumBlock] : make_float2(0.0f, 0.0f);
#pragma unroll
    for (int u = 0; u < (int)(kDisSumRows / kDisSumBlock); ++u) {
      v[0] += (double)r[u].x;
      v[1] += (double)r[u].y;
    }
  }
  team_sum<kDisSumBlock, 2>(v, lds);
  if (threadIdx.x != 0) return;
  if constexpr (PART) {
    parts_out[2 * blockIdx.x] = v[0];
    parts_out[2 * blockIdx.x + 1] = v[1];
  } else {
    loss[0] = (float)(mean ? v[0] / v[1] : v[0]);  // 0 / 0 = NaN: a mean over no rows
    count[0] = (float)v[1];
  }
}

// Vectors per thread of a backward workgroup.
constexpr int kDisBwdUnroll = 4;

// grad[row, columns of the workgroup].  The exponent x c - base is formed with c and base in two
// floats each: next to 0, where the probabilities are large, it has 24 bits.
template <typename T>
__global__ void __launch_bounds__(kDisBlock)
k_distill_bwd(DistillArgs g, int64_t row0, const float* __restrict__ stats, const DistillPair* __restrict__ pairs,
              const float* __restrict__ count, const float* __restrict__ grad_out, int reduction, T* __restrict__ grad) {
  constexpr int V = VecOf<T>::V, U = kDisBwdUnroll;
  extern __shared__ float listed[];  // p of the row's pairs
  __shared__ uint32_t bits[kDisBlock * U * V / 32];
  __shared__ uint16_t number[kDisBlock * U * V];  // of a column's pair, where its bit is set
  const int64_t row = row0 + blockIdx.y;
  const T* xr = dis_row<T>(g, row);
  T* dst = grad + row * g.vocab;
  const int64_t off = grid_off<T, V>(dst, g.vocab);
  const int64_t c0 = (int64_t)blockIdx.x * blockDim.x * U * V - off;
  const float* st = stats + row * kDisStats;
  const bool counted = st[6] != 0.0f;
  auto at = [&](int u) { return (int)(threadIdx.x + u * blockDim.x) * V; };  // a vector's first column from c0 on
  if (!counted) {
    float zero[V] = {};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t col = c0 + at(u);
      if (col >= 0 && col + V <= g.vocab) {
        store_any<T, V>(dst + col, zero);
      } else {
        for (int k = col < 0 ? (int)-col : 0; k < V && col + k < g.vocab; ++k) dst[col + k] = from_arith<T>(0.0f);
      }
    }
    return;
  }
  uint4 w[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t col = c0 + at(u);
    if (col >= 0 && col + V <= g.vocab) {
      w[u] = ld_any_stream(xr + col);
    } else {
      T e[V];
#pragma unroll
      for (int k = 0; k < V; ++k) e[k] = col + k >= 0 && col + k < g.vocab ? xr[col + k] : T{};
      __builtin_memcpy(&w[u], e, 16);
    }
  }
  const int reach = (int)blockDim.x * U * V;
  for (int i = threadIdx.x; i < reach / 32; i += blockDim.x) bits[i] = 0u;
  __syncthreads();
  for (int k = threadIdx.x; k < g.entries; k += blockDim.x) {
    const DistillPair e = pairs[row * g.entries + k];
    const int64_t col = e.at - c0;
    if (e.at < 0 || col < 0 || col >= reach) continue;
    atomicOr(&bits[col / 32], 1u << (col % 32));
    number[col] = (uint16_t)k;  // the one pair that carries the token
    listed[k] = e.p;
  }
  const float base_hi = st[0], base_lo = st[1], lse_hi = st[4], lse_lo = st[5], weight = st[3];
  float gs = reduction == SUPA_AMD_REDUCTION_NONE ? grad_out[row] : grad_out[0];
  if (reduction == SUPA_AMD_REDUCTION_MEAN) gs /= count[0];
  gs = (float)((double)gs * g.inv_t);
  const float k0 = st[2] * gs;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t col = c0 + at(u);
    float f[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float x = elem_f<T>(w[u], k);
      f[k] = __builtin_amdgcn_exp2f(fmaf(x, g.c_hi, -base_hi) + fmaf(x, g.c_lo, -base_lo)) * k0;
    }
    const uint32_t here = bits[at(u) / 32] >> (at(u) % 32) & ((1u << V) - 1u);
    if (here) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (!(here >> k & 1u)) continue;
        const float x = elem_f<T>(w[u], k);
        const float q = __builtin_amdgcn_exp2f(fmaf(x, g.c_hi, -lse_hi) + fmaf(x, g.c_lo, -lse_lo));
        f[k] = (q * weight - listed[number[at(u) + k]]) * gs;
      }
    }
    if (col >= 0 && col + V <= g.vocab) {
      store_any<T, V>(dst + col, f);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (col + k >= 0 && col + k < g.vocab) dst[col + k] = from_arith<T>(f[k]);
    }
  }
}

inline int64_t dis_parts(int64_t rows) { return rows > kDisSumRows ? (rows + kDisSumRows - 1) / kDisSumRows : 0; }

// Checks a descriptor and fills the arguments; 0, or a status.
int dis_args(const supa_amd_distill_desc* d, DistillArgs& g) {
  if (!d || d->rows < 0 || d->vocab < 1 || d->entries < 1 || d->inner < 1) return SUPA_AMD_EINVAL;
  if (d->rows >= (int64_t(1) << 31) || d->vocab >= (int64_t(1) << 31) || d->entries > kDisMaxEntries ||
      d->inner >= (int64_t(1) << 31))
    return SUPA_AMD_ELAYOUT;
  if (!(d->temperature >= 1e-30 && d->temperature <= 1e30)) return SUPA_AMD_EINVAL;
  if (d->reduction != SUPA_AMD_REDUCTION_NONE && d->reduction != SUPA_AMD_REDUCTION_MEAN &&
      d->reduction != SUPA_AMD_REDUCTION_SUM)
    return SUPA_AMD_EINVAL;
  for (int t : {d->dtype, d->teacher_dtype})
    if (t != SUPA_AMD_F32 && t != SUPA_AMD_BF16 && t != SUPA_AMD_F16) return SUPA_AMD_EDTYPE;
  if (d->index_dtype != SUPA_AMD_I64 && d->index_dtype != SUPA_AMD_I32) return SUPA_AMD_EDTYPE;
  g = DistillArgs{};
  g.x = d->logits;
  g.idx = d->indices;
  g.teacher = d->teacher;
  g.teacher_lse = d->teacher_lse;
  g.xs[0] = d->logits_strides[0];
  g.xs[1] = d->logits_strides[1];
  g.inner = FastDiv((uint32_t)d->inner);
  g.vocab = d->vocab;
  g.entries = (int32_t)d->entries;
  g.hash = 64;
  while (g.hash < 2 * g.entries) g.hash *= 2;
  g.idx64 = d->index_dtype == SUPA_AMD_I64;
  g.teacher_dtype = d->teacher_dtype;
  g.segment = (int32_t)std::min<int64_t>(kDisSegment, (d->vocab + 31) / 32 * 32);
  g.c = kLog2eD / d->temperature;
  g.c_near = (float)g.c;
  g.c_hi = (double)g.c_near < g.c ? g.c_near : std::nextafterf(g.c_near, 0.0f);
  g.c_lo = std::max((float)(g.c - (double)g.c_hi), 1.2e-38f);
  g.inv_t = 1.0 / d->temperature;
  return SUPA_AMD_OK;
}

// Parts of a row's columns for each of `rows` rows; 1: whole rows.
int64_t dis_splits(int64_t rows, int64_t vocab, int dtype) {
  const int64_t vecs = vocab * dtype_size(dtype) / 16;
  return std::max<int64_t>(1, std::min<int64_t>({64, 768 / std::max<int64_t>(1, rows), vecs / (2 * kDisBlock * kDisUnroll)}));
}

template <typename T, bool REST>
int dis_forward(const DistillArgs& g, int64_t rows, int dtype, const DistillOut& out, float2* parts, int32_t* error_flag,
                hipStream_t st) {
  const int64_t splits = dis_splits(rows, g.vocab, dtype);
  if (splits > 1) {
    DistillArgs p = g;
    const int64_t columns = ((g.vocab + splits - 1) / splits + 255) / 256 * 256;
    const int64_t n = (g.vocab + columns - 1) / columns;
    p.segment = (int32_t)std::min<int64_t>(columns, kDisSegment);
    const size_t bitmap = REST ? (size_t)p.segment / 8 : 0;
    k_distill_part<T, REST><<<dim3((unsigned)n, (unsigned)rows), kDisBlock, bitmap, st>>>(p, columns, parts);
    const int rc = launch_status();
    if (rc) return rc;
    const size_t lds = dis_lds_bytes(g.entries, g.hash, 0);
    if (g.entries <= 64 * kDisEntries)
      k_distill_rows<T, 64, REST><<<(unsigned)rows, 64, lds, st>>>(g, (int)n, parts, out, error_flag);
    else
      k_distill_rows<T, kDisBlock, REST><<<(unsigned)rows, kDisBlock, lds, st>>>(g, (int)n, parts, out, error_flag);
    return launch_status();
  }
  auto go = [&](auto threads) -> int {
    constexpr int G = decltype(threads)::value, per = kDisBlock / G;
    const size_t lds = per * dis_lds_bytes(g.entries, g.hash, REST ? g.segment : 0);
    const int64_t slab = ((int64_t(1) << 32) - 1) / kDisBlock * per;  // HIP: fewer than 2^32 threads a launch
    for (int64_t r0 = 0; r0 < rows; r0 += slab) {
      const int64_t n = std::min(slab, rows - r0);
      k_distill_fwd<T, G, REST><<<(unsigned)((n + per - 1) / per), kDisBlock, lds, st>>>(g, r0, n, out, error_flag);
      const int rc = launch_status();
      if (rc) return rc;
    }
    return SUPA_AMD_OK;
  };
  // a wavefront a row where rows are short
  if (g.entries <= 64 * kDisEntries && g.vocab * dtype_size(dtype) <= 16 * kDisWaveVecs)
    return go(std::integral_constant<int, 64>{});
  return go(std::integral_constant<int, kDisBlock>{});
}

// Workspace: partial sums, the rows' losses and counts, the rows' parts.
struct DistillSpace {
  int64_t rows, parts, bytes;
};
DistillSpace distill_space(const supa_amd_distill_desc* d) {
  DistillSpace s{};
  const int64_t splits = dis_splits(d->rows, d->vocab, d->dtype);
  s.rows = 16 * dis_parts(d->rows);
  s.parts = s.rows + (d->reduction == SUPA_AMD_REDUCTION_NONE ? 0 : 8 * d->rows);
  s.bytes = s.parts + (splits > 1 ? 8 * splits * d->rows : 0);
  return s;
}

}  // namespace sa

using namespace sa;

extern "C" {

int64_t supa_amd_distill_workspace_bytes(const supa_amd_distill_desc* d) {
  DistillArgs g;
  const int rc = dis_args(d, g);
  if (rc) return rc;
  return distill_space(d).bytes;
}

int supa_amd_distill_forward(const supa_amd_distill_desc* d, float* loss, float* count, float* stats, void* pairs,
                             void* workspace, int64_t ws_bytes, int32_t* error_flag, void* stream) {
  DistillArgs g;
  int rc = dis_args(d, g);
  if (rc) return rc;
  const bool total = d->reduction != SUPA_AMD_REDUCTION_NONE;
  if (d->rows == 0 && !total) return SUPA_AMD_OK;
  if (!loss || (total && !count)) return SUPA_AMD_EINVAL;
  if (d->rows > 0 && (!d->logits || !d->indices || !d->teacher || !stats)) return SUPA_AMD_EINVAL;
  const DistillSpace space = distill_space(d);
  if (space.bytes > 0 && (!workspace || ws_bytes < space.bytes)) return SUPA_AMD_EWORKSPACE;
  if (!aligned(workspace, 8) || !aligned(pairs, 8)) return SUPA_AMD_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t nparts = dis_parts(d->rows);
  char* ws = static_cast<char*>(workspace);
  double* sums = reinterpret_cast<double*>(ws);
  float2 *rows = reinterpret_cast<float2*>(ws + space.rows), *parts = reinterpret_cast<float2*>(ws + space.parts);
  const DistillOut out{total ? nullptr : loss, rows, stats, static_cast<DistillPair*>(pairs)};
  if (d->rows > 0) {
    rc = with_float_storage(d->dtype, [&](auto* tag) -> int {
      using T = std::remove_pointer_t<decltype(tag)>;
      return d->teacher_lse ? dis_forward<T, true>(g, d->rows, d->dtype, out, parts, error_flag, st)
                            : dis_forward<T, false>(g, d->rows, d->dtype, out, parts, error_flag, st);
    });
  }
  if (rc || !total) return rc;
  if (nparts > 0) {
    k_distill_total<true><<<(unsigned)nparts, kDisSumBlock, 0, st>>>(rows, nullptr, d->rows, 0, sums, nullptr, nullptr);
    rc = launch_status();
    if (rc) return rc;
  }
  k_distill_total<false><<<1, kDisSumBlock, 0, st>>>(rows, nparts > 0 ? sums : nullptr, nparts > 0 ? nparts : d->rows,
                                                    d->reduction == SUPA_AMD_REDUCTION_MEAN, nullptr, loss, count);
  return launch_status();
}

int supa_amd_distill_backward(const supa_amd_distill_desc* d, const float* grad_loss, const float* count,
                              const float* stats, const void* pairs, void* grad_logits, void* stream) {
  DistillArgs g;
  const int rc = dis_args(d, g);
  if (rc) return rc;
  if (d->rows == 0) return SUPA_AMD_OK;
  if (!grad_loss || !stats || !pairs || !grad_logits || !d->logits) return SUPA_AMD_EINVAL;
  if (!aligned(pairs, 8)) return SUPA_AMD_EINVAL;
  if (d->reduction == SUPA_AMD_REDUCTION_MEAN && !count) return SUPA_AMD_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_float_storage(d->dtype, [&](auto* tag) -> int {
    using T = std::remove_pointer_t<decltype(tag)>;
    constexpr int V = VecOf<T>::V;
    T* gx = static_cast<T*>(grad_logits);
    const int64_t vecs = grid_vecs<T, V>(gx, g.vocab);
    // rows shorter than a workgroup's reach get fewer threads
    const int64_t each = (vecs + kDisBwdUnroll - 1) / kDisBwdUnroll;
    const int block = (int)std::min<int64_t>(kDisBlock, (each + 63) / 64 * 64);
    const unsigned blocks = (unsigned)((each + block - 1) / block);
    const int64_t slab = std::min<int64_t>(65535, ((int64_t(1) << 32) - 1) / block / blocks);
    for (int64_t r0 = 0; r0 < d->rows; r0 += slab) {
      const unsigned n = (unsigned)std::min(slab, d->rows - r0);
      k_distill_bwd<T><<<dim3(blocks, n), block, sizeof(float) * g.entries, st>>>(
          g, r0, stats, static_cast<const DistillPair*>(pairs), count, grad_loss, d->reduction, gx);
      const int rc = launch_status();
      if (rc) return rc;
    }
    return SUPA_AMD_OK;
  });
}

}  // extern "C"

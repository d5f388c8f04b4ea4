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
// writes the gradient; the pairs are a few hundred bytes a row.  [3700, 128256] bf16 with 64 pairs: forward 155 us
// (6.1 TB/s of a read stream's 6.8), backward 304 (6.2 of 6.7).  Rows of a few hundred tokens are bound by the instructions of a
// row's finish ([65536, 256]: 99 us, 781 a row).  The forward
// keeps an online (max, sum of exp2) pair a thread, float32 (the exponent (x - max) c too, whose product is off by 2^-24 of
// itself, as in this library's softmax); what depends on the
// pairs alone (K exponentials, their sums, logarithms) is float64: r and small
// losses are differences of near values.  q_R is summed over its own elements,
// not as 1 minus the listed ones: a bitmap of the listed tokens, in LDS, tells
// them apart.  A workgroup of the backward puts the listed tokens among its columns into LDS
// (a bit, and the pair's number in a table by column) while its logits are on their way; an
// element whose bit is set takes its p from there.
//
// A token listed twice has the sum of its p in the gradient, and counts once for the listed tokens' mass: the row's first
// such pair carries it.  The loss is the sum over the pairs as they are, each with its own log p; merged they would have
// p1 log(P / p1) + p2 log(P / p2) more, P = p1 + p2, which does not depend on the student.  Such tokens,
// and their first pairs, are found by a hash table in LDS; the others add their p to the first's in turn, in the order of the pairs.
#include "row_group.h"

namespace sa {

constexpr int kDisBlock = 256;  // threads a row; 512 and 1024 gained 1 to 4 us below 256 rows, and lost 12 to 45 % with the rest or many pairs
constexpr int kDisMaxEntries = 1024;
static_assert(kDisMaxEntries == SUPA_AMD_DISTILL_MAX_ENTRIES);
constexpr int kDisUnroll = 2;             // 16-byte vectors in flight per thread; 4 and 8 cost registers, and so rows on a CU
constexpr int kDisSegment = 1 << 17;      // columns whose bitmap is in LDS at a time: 16 KiB
constexpr int kDisStats = 8;              // floats a row keeps for the backward
constexpr double kLn2 = 0.69314718055994530942;
constexpr double kLog2eD = 1.44269504088896340736;

struct DistillArgs {
  const void* x;
  const void* idx;
  const void* teacher;
  const void* teacher_lse;  // float32, or float64 (lse64)
  int64_t xs[2], is[2], ts[2], ls[2];  // distances of rows, outer and inner: of logits, indices, teacher, teacher_lse
  FastDiv inner;     // row -> (outer, inner)
  int64_t vocab;
  int32_t entries, hash;  // pairs a row; slots of its hash table, a power of two >= 2 entries
  int32_t idx64, lse64, teacher_dtype;
  int32_t segment;   // columns of a bitmap
  double teacher_c;  // log2(e) / temperature
  float c;           // that rounded, for all that is the student's: a temperature off by 2^-25 of itself
  double inv_t;
};

template <typename T> __device__ __forceinline__ const T* dis_row(const DistillArgs& g, int64_t row) {
  uint32_t o, i;
  g.inner.divmod((uint32_t)row, o, i);
  return static_cast<const T*>(g.x) + ((int64_t)o * g.xs[0] + (int64_t)i * g.xs[1]);
}
// Where a row of one of the others starts.
__device__ __forceinline__ int64_t dis_at(const DistillArgs& g, int64_t row, const int64_t (&strides)[2]) {
  uint32_t o, i;
  g.inner.divmod((uint32_t)row, o, i);
  return (int64_t)o * strides[0] + (int64_t)i * strides[1];
}
__device__ __forceinline__ int64_t dis_index(const DistillArgs& g, int64_t at) {
  return g.idx64 ? static_cast<const int64_t*>(g.idx)[at] : (int64_t)static_cast<const int32_t*>(g.idx)[at];
}

// A row's teacher_lse.  A float64 one stays so: r = 1 - sum p is a difference of near values, and of a log-sum-exp of 20 float32
// leaves out up to 1e-6.
__device__ __forceinline__ double dis_lse(const DistillArgs& g, int64_t row) {
  const int64_t at = dis_at(g, row, g.ls);
  return g.lse64 ? static_cast<const double*>(g.teacher_lse)[at] : (double)static_cast<const float*>(g.teacher_lse)[at];
}

// Exchange among the threads of a wavefront through LDS.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  return v;
}
template <typename F> __device__ __forceinline__ double wave_halves(double x, F&& f) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)f((int)(uint32_t)u), hi = (uint32_t)f((int)(uint32_t)(u >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// The value of one lane.
__device__ __forceinline__ double wave_lane(double v, int l) {
  return wave_halves(v, [&](int h) { return __builtin_amdgcn_readlane(h, l); });
}
// The sum of a wavefront, in every lane: four lane permutations within 16 lanes, then the four rows of 16.
__device__ __forceinline__ double wave_sum(double v) {
  auto perm = [&](double x, auto ctrl) {
    return wave_halves(x, [](int h) { return __builtin_amdgcn_update_dpp(0, h, decltype(ctrl)::value, 0xf, 0xf, true); });
  };
  v += perm(v, std::integral_constant<int, 0xB1>{});   // quad_perm [1, 0, 3, 2]
  v += perm(v, std::integral_constant<int, 0x4E>{});   // quad_perm [2, 3, 0, 1]
  v += perm(v, std::integral_constant<int, 0x141>{});  // row_half_mirror
  v += perm(v, std::integral_constant<int, 0x140>{});  // row_mirror
  return (wave_lane(v, 0) + wave_lane(v, 16)) + (wave_lane(v, 32) + wave_lane(v, 48));
}

// A row's pairs in a wavefront: lane l holds pairs l, l + 64, ... NE of them.
template <int NE> struct DistillEntries {
  int32_t at[NE];          // token, or -1: none there
  float t[NE], x[NE];      // teacher's and student's logits
};

// A pair as the backward reads it: the token, or -1 where another pair carries it or none is there, and the bits of its p.
struct DistillPair {
  int32_t at;
  float p;
};

// LDS of a row, in this order: the pairs' p (float64) and whose turn it is to add to it, both of rows that list a token
// twice alone; the hash table's tokens and their first pairs; the bitmap.
struct DistillLds {
  double* p;
  int32_t *turn, *hash, *first;
  uint32_t* bits;
};
// Words of a bitmap: a segment, which may begin some places into a vector and end in one.
inline __host__ __device__ int dis_bit_words(int segment) { return (segment + 16 + 63) / 64 * 2; }
inline __host__ __device__ size_t dis_lds_bytes(int entries, int hash, int segment) {
  return (size_t)((entries + 1) / 2 * 2) * 12 + (size_t)hash * 8 + (segment > 0 ? 4 * (size_t)dis_bit_words(segment) : 0);
}
__device__ __forceinline__ DistillLds dis_lds(char* p, int entries, int hash) {
  const int n = (entries + 1) / 2 * 2;
  DistillLds s;
  s.p = reinterpret_cast<double*>(p);
  s.turn = reinterpret_cast<int32_t*>(s.p + n);
  s.hash = s.turn + n;
  s.first = s.hash + hash;
  s.bits = reinterpret_cast<uint32_t*>(s.first + hash);
  return s;
}

// The token of pair k of a row, or -1: a pair is there if its token is not negative and its teacher logit is not -inf.
// One that is there and lists a token of vocab or more is an error.
__device__ __forceinline__ int32_t dis_token(const DistillArgs& g, int64_t indices, int64_t teacher, int k, float* t,
                                             int32_t* error_flag) {
  const int64_t at = dis_index(g, indices + k);
  *t = load_dyn<float>(g.teacher, teacher + k, g.teacher_dtype);
  if (at < 0 || *t == -__builtin_inff()) return -1;
  if (at < g.vocab) return (int32_t)at;
  if (error_flag) *error_flag = 3;
  return -1;
}

// Loads a row's pairs; whether any is there, in every lane.
template <int NE>
__device__ __forceinline__ bool dis_entries(const DistillArgs& g, int64_t row, int lane, DistillEntries<NE>& e,
                                            int32_t* error_flag) {
  const int64_t indices = dis_at(g, row, g.is), teacher = dis_at(g, row, g.ts);
  bool any = false;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int k = lane + i * 64;
    e.at[i] = -1;
    e.t[i] = -__builtin_inff();
    if (k < g.entries) e.at[i] = dis_token(g, indices, teacher, k, &e.t[i], error_flag);
    any = any || e.at[i] >= 0;
  }
  return __any(any);
}

// The slot of a token in the hash table, of which at most half are taken: step says whether this is it.
template <typename F> __device__ __forceinline__ int dis_slot(const DistillArgs& g, int32_t token, F&& step) {
  uint32_t h = ((uint32_t)token * 0x9E3779B1u) >> 16 & (uint32_t)(g.hash - 1);
  while (!step(h)) h = (h + 1) & (uint32_t)(g.hash - 1);
  return (int)h;
}

// The student's logits of the pairs, and whether a token is listed twice, in every lane.  One wavefront a row.
template <typename T, int NE>
__device__ __forceinline__ bool dis_listed(const DistillArgs& g, const T* xr, int lane, DistillEntries<NE>& e,
                                           const DistillLds& s) {
#pragma unroll
  for (int i = 0; i < NE; ++i) e.x[i] = e.at[i] >= 0 ? (float)to_arith(xr[e.at[i]]) : -__builtin_inff();
  for (int i = lane; i < g.hash; i += 64) {
    s.hash[i] = -1;
    s.first[i] = kDisMaxEntries;
  }
  wave_sync();
  bool twice = false;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    if (e.at[i] < 0) continue;
    const int h = dis_slot(g, e.at[i], [&](uint32_t h) {
      const int old = atomicCAS(&s.hash[h], -1, e.at[i]);
      twice = twice || old == e.at[i];
      return old == -1 || old == e.at[i];
    });
    atomicMin(&s.first[h], lane + i * 64);
  }
  wave_sync();
  return __any(twice);
}

// Gives the p of pairs whose token an earlier one lists to the first that does; `first` says which pairs are.
template <int NE>
__device__ __forceinline__ void dis_share(const DistillArgs& g, int lane, const DistillEntries<NE>& e, double (&p)[NE],
                                          bool (&first)[NE], const DistillLds& s) {
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    if (e.at[i] < 0) continue;
    s.p[lane + i * 64] = p[i];
    s.turn[lane + i * 64] = 64;
  }
  wave_sync();
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    int to = lane + i * 64;
    if (e.at[i] >= 0) to = s.first[dis_slot(g, e.at[i], [&](uint32_t h) { return s.hash[h] == e.at[i]; })];
    bool waits = to != lane + i * 64;
    first[i] = first[i] && !waits;
    while (__any(waits)) {  // the lowest lane that waits for a pair takes its turn: each round ends with fewer
      if (waits) atomicMin(&s.turn[to], lane);
      wave_sync();
      const bool now = waits && s.turn[to] == lane;
      wave_sync();
      if (now) {
        s.p[to] += p[i];
        s.turn[to] = 64;
        waits = false;
      }
      wave_sync();
    }
  }
#pragma unroll
  for (int i = 0; i < NE; ++i)
    if (first[i]) p[i] = s.p[lane + i * 64];
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

// A row without a pair: nothing is read of its logits.  One wavefront.
__device__ __forceinline__ void dis_nothing(const DistillArgs& g, int64_t row, int lane, const DistillOut& out) {
  if (out.pairs) {
    for (int k = lane; k < g.entries; k += 64) out.pairs[row * g.entries + k] = DistillPair{-1, 0.0f};
  }
  if (lane < kDisStats) out.stats[row * kDisStats + lane] = 0.0f;
  if (lane == 0) out.row(row, 0.0f, false);
}

// What a row keeps for the backward, as floats in this order.
enum { kStatRestMax, kStatRest, kStatMax, kStatListed, kStatCounts };

// From the stream's pair (m, s) -- the largest x, and the sum of exp2((x - m) c) -- and
// the row's pairs to the row's loss, its statistics and the pairs' weights.  One wavefront.
template <int NE, bool REST>
__device__ __forceinline__ void dis_finish(const DistillArgs& g, int64_t row, int lane, float m, float s,
                                           const DistillEntries<NE>& e, double teacher_lse, bool twice,
                                           const DistillLds& lds, const DistillOut& out) {
  float top_t = -__builtin_inff(), top = m;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    if (e.at[i] < 0) continue;
    top_t = fmaxf(top_t, e.t[i]);
    if (REST) top = fmaxf(top, e.x[i]);
  }
  if (REST) top = wave_max(top);
  else top_t = wave_max(top_t);
  const float M = top == -__builtin_inff() ? 0.0f : top;
  const double lt = REST ? teacher_lse * kLog2eD : (double)top_t * g.teacher_c;
  double p[NE];
  bool first[NE];  // no pair before lists the token
  double sum[3] = {0.0, 0.0, 0.0};  // p, p log2 p, p z with z = (x - M) c
  float mass = 0.0f;                // the listed tokens' exp2(z)
  int distinct = 0;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    p[i] = 0.0;
    first[i] = e.at[i] >= 0;
    if (!first[i]) continue;
    const double log_p = (double)e.t[i] * g.teacher_c - lt, z = ((double)e.x[i] - (double)M) * (double)g.c;
    p[i] = exp2(log_p);
    if (p[i] != 0.0) {
      sum[0] += p[i];
      sum[1] += p[i] * log_p;
      sum[2] += p[i] * z;
    }
  }
  if (twice) dis_share(g, lane, e, p, first, lds);
  if (REST) {
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      if (!first[i]) continue;
      mass += __builtin_amdgcn_exp2f((e.x[i] - M) * g.c);
      ++distinct;
    }
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) sum[i] = wave_sum(sum[i]);
  if (REST) {
    mass = sum64(mass);
    distinct = (int)sum64((float)distinct);  // at most 1024
  }
  const double norm = REST ? 1.0 : 1.0 / sum[0];
  if (out.pairs) {
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int k = lane + i * 64;
      if (k < g.entries) out.pairs[row * g.entries + k] = DistillPair{first[i] ? e.at[i] : -1, (float)(p[i] * norm)};
    }
  }
  // the same in all lanes from here on, but for the logarithms: a float64 one costs about 60 instructions, so each
  // lane takes one
  double weight = 1.0, r = 0.0, total = (double)s, rest_scale = 1.0;  // total: of exp2((x - M) c) over the row
  bool rest = true;
  const double down = ((double)m - (double)M) * (double)g.c;
  if constexpr (REST) {
    rest = (int64_t)distinct != g.vocab && s != 0.0f;  // some token is not listed, and has mass
    r = (int64_t)distinct == g.vocab ? 0.0 : fmax(0.0, 1.0 - sum[0]);
    weight = sum[0] + r;
    const double whole = rint(fmax(down, -2000.0));
    rest_scale = ldexp((double)__builtin_amdgcn_exp2f((float)(fmax(down, -2000.0) - whole)), (int)whole);
    total = (double)s * rest_scale + (double)mass;
  }
  const double lg = log2(lane == 0 ? total : (lane == 1 ? (REST ? (double)s : sum[0]) : r));
  const double log_total = wave_lane(lg, 0);
  double L;
  if constexpr (REST) {
    L = sum[1] - sum[2] + sum[0] * log_total;
    if (r > 0.0) L += r * (wave_lane(lg, 2) - (down + wave_lane(lg, 1) - log_total));  // log2 of r and of q_R
  } else {
    L = (sum[1] - sum[2]) * norm - wave_lane(lg, 1) + log_total;
  }
  if (lane != 0) return;
  const double scale = weight / total;
  float st[kDisStats] = {};
  st[kStatRestMax] = s == 0.0f ? 0.0f : m;  // no mass: of logits of -inf, whose gradient is 0, not -inf - -inf
  st[kStatRest] = !rest ? 0.0f : (float)(scale * rest_scale - (REST ? r / (double)s : 0.0));
  st[kStatMax] = top;
  st[kStatListed] = (float)scale;
  st[kStatCounts] = 1.0f;
  out.row(row, (float)(L * kLn2), true);
#pragma unroll
  for (int i = 0; i < kDisStats; ++i) out.stats[row * kDisStats + i] = st[i];
}

// One online step over a batch of logits: (m, s) with those of f.  m is the largest x itself, subtracted before the scale:
// a row whose logits are all the type's lowest value, whose product with c is no float, is as even as any other.
template <int N> __device__ __forceinline__ void dis_online(float& m, float& s, const float (&f)[N], float c) {
  float M = m;
#pragma unroll
  for (int k = 0; k < N; ++k) M = fmaxf(M, f[k]);
  // fmaxf passes over a NaN, so M says nothing of them: the sum is always taken, and is then NaN
  const float base = M == -__builtin_inff() ? 0.0f : M;
  float sb = 0.0f;
#pragma unroll
  for (int k = 0; k < N; ++k) sb += __builtin_amdgcn_exp2f((f[k] - base) * c);
  s = s * __builtin_amdgcn_exp2f((m - base) * c) + sb;
  m = M;
}

// The columns [c0, c1) of a row for one of G threads, in vectors at multiples of 16 bytes, whatever the row's
// address; the few elements before and behind them go one to a thread.  The first batch is requested when it
// is made.
template <typename T, int G, bool REST> struct DistillStream {
  static constexpr int V = VecOf<T>::V, U = kDisUnroll;
  const T* p;        // the first whole vector
  int head, tail;    // elements before and behind the vectors
  int nvec, l;
  uint4 w[U];
  T edge;

  __device__ __forceinline__ DistillStream(const T* xr, int64_t c0, int64_t c1, int thread) : l(thread) {
    const int n = (int)(c1 - c0), at = (int)(reinterpret_cast<uintptr_t>(xr + c0) % 16 / sizeof(T));
    head = at == 0 ? 0 : (V - at < n ? V - at : n);
    p = xr + c0 + head;
    nvec = (n - head) / V;
    tail = n - head - nvec * V;
    request(l);
    if (l < head + tail) edge = p[edge_at()];
  }
  __device__ __forceinline__ int64_t edge_at() const { return l < head ? l - head : (int64_t)nvec * V + (l - head); }
  // Where the bitmap has column c0: the first vector's bits begin at bit V.
  __device__ __forceinline__ int shift() const { return V - head; }
  __device__ __forceinline__ void request(int v0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v0 + u * G < nvec) w[u] = ld_any_stream(p + (int64_t)(v0 + u * G) * V);
  }
  // Adds them to (m, s).  REST: the listed tokens, whose bits are set, count as -inf.
  __device__ __forceinline__ void run(float c, const uint32_t* bits, float& m, float& s) {
    for (int v0 = l; v0 < nvec; v0 += G * U) {
      float f[U * V];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int v = v0 + u * G;
        if (v < nvec) {
#pragma unroll
          for (int k = 0; k < V; ++k) f[u * V + k] = elem_f<T>(w[u], k);
          if constexpr (REST) {
            const int bit = (v + 1) * V;
            const uint32_t b = bits[bit / 32] >> (bit % 32) & ((1u << V) - 1u);
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
      request(v0 + G * U);
      dis_online(m, s, f, c);
    }
    if (l < head + tail) {
      float f[1] = {(float)to_arith(edge)};
      if constexpr (REST) {
        const int bit = (int)edge_at() + V;
        if (bits[bit / 32] >> (bit % 32) & 1u) f[0] = -__builtin_inff();
      }
      dis_online(m, s, f, c);
    }
  }
};

// (m, s) of a wavefront, in every lane.
__device__ __forceinline__ void dis_join(float& m, float& s, float c) {
  const float M = wave_max(m);
  if (M != -__builtin_inff()) s *= __builtin_amdgcn_exp2f((m - M) * c);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  m = M;
}

// Sets the bits of the listed tokens in [c0, c0 + segment), `shift` places on, by all G threads of a row; exchanged at its end.
template <int G>
__device__ __forceinline__ void dis_mark(const DistillArgs& g, int64_t row, int64_t c0, int shift, int l, uint32_t* bits) {
  auto sync = [] {
    if constexpr (G == 64) wave_sync();
    else __syncthreads();
  };
  sync();
  for (int i = l; i < dis_bit_words(g.segment); i += G) bits[i] = 0u;
  sync();
  const int64_t indices = dis_at(g, row, g.is), teacher = dis_at(g, row, g.ts);
  for (int k = l; k < g.entries; k += G) {
    float t;
    const int32_t token = dis_token(g, indices, teacher, k, &t, nullptr);
    const int64_t at = token - c0;
    if (token < 0 || at < 0 || at >= g.segment) continue;
    const int bit = (int)at + shift;
    atomicOr(&bits[bit / 32], 1u << (bit % 32));
  }
  sync();
}

// G threads a row; the first wavefront knows the pairs and finishes the row.  Short rows: several to a workgroup.
template <typename T, int G, int NE, bool REST>
__global__ void __launch_bounds__(G < kDisBlock ? kDisBlock : G)
k_distill_fwd(DistillArgs g, int64_t row0, int64_t rows, DistillOut out, int32_t* error_flag) {
  constexpr int TEAMS = G < kDisBlock ? kDisBlock / G : 1, W = G / 64;
  extern __shared__ double lds_dyn[];
  __shared__ float2 lds_join[W];
  // the same in a wavefront, and known to be: a row's addresses are scalar then
  const int team = TEAMS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / G);
  const int l = TEAMS == 1 ? threadIdx.x : threadIdx.x & 63, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(l >> 6);
  const int64_t row = row0 + (int64_t)blockIdx.x * TEAMS + team;
  if (row >= row0 + rows) return;  // whole rows: no exchange is left waiting
  const T* xr = dis_row<T>(g, row);
  const DistillLds s = dis_lds(
      reinterpret_cast<char*>(lds_dyn) + team * dis_lds_bytes(g.entries, g.hash, REST ? g.segment : 0), g.entries, g.hash);
  auto end = [&](int64_t c0) { return c0 + g.segment < g.vocab ? c0 + g.segment : g.vocab; };
  DistillStream<T, G, REST> first(xr, 0, end(0), l);
  DistillEntries<NE> e;
  const double teacher_lse = REST ? dis_lse(g, row) : 0.0;
  const bool any = dis_entries(g, row, lane, e, wave == 0 ? error_flag : nullptr);  // in every wavefront: all know without a barrier
  if (!any) {
    if (wave == 0) dis_nothing(g, row, lane, out);
    return;
  }
  bool twice = false;
  if (wave == 0) twice = dis_listed(g, xr, lane, e, s);
  float m = -__builtin_inff(), sum = 0.0f;
  if (REST) dis_mark<G>(g, row, 0, first.shift(), l, s.bits);
  first.run(g.c, s.bits, m, sum);
  for (int64_t c0 = g.segment; c0 < g.vocab; c0 += g.segment) {
    DistillStream<T, G, REST> next(xr, c0, end(c0), l);
    if (REST) dis_mark<G>(g, row, c0, next.shift(), l, s.bits);
    next.run(g.c, s.bits, m, sum);
  }
  dis_join(m, sum, g.c);
  if constexpr (W > 1) {
    if (lane == 0) lds_join[wave] = make_float2(m, sum);
    __syncthreads();
    if (wave != 0) return;
    const float2 part = lane < W ? lds_join[lane] : make_float2(-__builtin_inff(), 0.0f);
    m = part.x;
    sum = part.y;
    dis_join(m, sum, g.c);
  }
  dis_finish<NE, REST>(g, row, lane, m, sum, e, teacher_lse, twice, s, out);
}

// Few rows: parts of a row (of `columns` columns, a multiple of 32) to a workgroup each; (m, s) of each part ...
template <typename T, bool REST>
__global__ void __launch_bounds__(kDisBlock)
k_distill_part(DistillArgs g, int64_t columns, float2* __restrict__ parts) {
  constexpr int G = kDisBlock, W = G / 64;
  extern __shared__ double lds_dyn[];
  __shared__ float2 lds_join[W];
  const int64_t row = blockIdx.y, c0 = blockIdx.x * columns, c1 = c0 + columns < g.vocab ? c0 + columns : g.vocab;
  const T* xr = dis_row<T>(g, row);
  uint32_t* bits = reinterpret_cast<uint32_t*>(lds_dyn);
  float m = -__builtin_inff(), sum = 0.0f;
  for (int64_t s0 = c0; s0 < c1; s0 += g.segment) {
    DistillStream<T, G, REST> stream(xr, s0, s0 + g.segment < c1 ? s0 + g.segment : c1, threadIdx.x);
    if (REST) dis_mark<G>(g, row, s0, stream.shift(), threadIdx.x, bits);
    stream.run(g.c, bits, m, sum);
  }
  dis_join(m, sum, g.c);
  if ((threadIdx.x & 63) == 0) lds_join[threadIdx.x >> 6] = make_float2(m, sum);
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const float2 part = threadIdx.x < W ? lds_join[threadIdx.x] : make_float2(-__builtin_inff(), 0.0f);
  m = part.x;
  sum = part.y;
  dis_join(m, sum, g.c);
  if (threadIdx.x == 0) parts[row * gridDim.x + blockIdx.x] = make_float2(m, sum);
}
// ... and the rows from their parts, a wavefront each.
template <typename T, int NE, bool REST>
__global__ void __launch_bounds__(64)
k_distill_rows(DistillArgs g, int nparts, const float2* __restrict__ parts, DistillOut out, int32_t* error_flag) {
  extern __shared__ double lds_dyn[];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const float2 part = lane < nparts ? parts[row * nparts + lane] : make_float2(-__builtin_inff(), 0.0f);
  const DistillLds s = dis_lds(reinterpret_cast<char*>(lds_dyn), g.entries, g.hash);
  DistillEntries<NE> e;
  const double teacher_lse = REST ? dis_lse(g, row) : 0.0;
  if (!dis_entries(g, row, lane, e, error_flag)) return dis_nothing(g, row, lane, out);
  const bool twice = dis_listed(g, dis_row<T>(g, row), lane, e, s);
  float m = part.x, sum = part.y;
  dis_join(m, sum, g.c);
  dis_finish<NE, REST>(g, row, lane, m, sum, e, teacher_lse, twice, s, out);
}

// The sum (or mean) of the rows' losses and the number of rows that count, in float64 and a fixed order.  More
// rows than kDisSumRows: a first launch (PART) leaves the sums of runs of rows.
constexpr int kDisSumBlock = 1024;
constexpr int64_t kDisSumRows = 8 * kDisSumBlock;

template <bool PART>
__global__ void __launch_bounds__(kDisSumBlock)
k_distill_total(const float2* __restrict__ rows, const double* __restrict__ parts, int64_t n, int mean,
                double* __restrict__ parts_out, float* __restrict__ loss, float* __restrict__ count) {
  __shared__ double lds[2][kDisSumBlock / 64];
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
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[i] = wave_sum(v[i]);
    if ((threadIdx.x & 63) == 0) lds[i][threadIdx.x >> 6] = v[i];
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) v[i] = wave_sum(threadIdx.x < kDisSumBlock / 64 ? lds[i][threadIdx.x] : 0.0);
  if (threadIdx.x != 0) return;
  if constexpr (PART) {
    parts_out[2 * blockIdx.x] = v[0];
    parts_out[2 * blockIdx.x + 1] = v[1];
  } else {
    loss[0] = (float)(mean ? v[0] / v[1] : v[0]);  // 0 / 0 = NaN: a mean over no rows
    count[0] = (float)v[1];
  }
}

// grad[row, columns of the G threads]: one vector a thread, as memory takes a read and a
// write stream best ([3700, 128256] bf16, reading and writing alone: 287 us so, 310 to 335 with four
// vectors a thread, 64 to 1024 threads).  Everything is requested before anything is waited for.
// The probabilities are exp2((x - largest x) c) times a factor of the row: the exponent is exact next to 0, where
// they are large.
// EDGES: rows that do not consist of whole vectors at multiples of 16 bytes.  The elements before a row's first and
// behind its last then go one to a thread.
template <typename T, int G, bool EDGES>
__global__ void __launch_bounds__(G < kDisBlock ? kDisBlock : G)
k_distill_bwd(DistillArgs g, int64_t row0, int64_t rows, const float* __restrict__ stats,
              const DistillPair* __restrict__ pairs, const float* __restrict__ count,
              const float* __restrict__ grad_out, int reduction, T* __restrict__ grad) {
  constexpr int V = VecOf<T>::V, TEAMS = G < kDisBlock ? kDisBlock / G : 1, reach = G * V;
  __shared__ uint32_t lds_bits[TEAMS][reach / 32];
  __shared__ float lds_p[TEAMS][reach];
  const int team = TEAMS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / G);  // scalar, as the row's addresses then
  const int l = TEAMS == 1 ? threadIdx.x : threadIdx.x & 63;
  uint32_t* bits = lds_bits[team];
  float* listed = lds_p[team];  // p of a column whose bit is set
  const int64_t row = row0 + (int64_t)blockIdx.y * TEAMS + team;
  if (row >= row0 + rows) return;  // whole rows: no exchange is left waiting
  const T* xr = dis_row<T>(g, row);
  T* dst = grad + row * g.vocab;
  const int shift = EDGES ? grid_off<T, V>(dst, g.vocab) : 0;
  const int64_t c0 = (int64_t)blockIdx.x * reach - shift, col = c0 + l * V;
  const bool whole = (!EDGES || col >= 0) && col + V <= g.vocab;
  uint4 w{};
  if (whole) w = ld_any_stream(xr + col);
  int64_t lone = 0;
  bool edge = false;
  T alone{};
  if constexpr (EDGES) {
    const int head = (V - shift % V) % V;
    const int64_t tail = head < g.vocab ? g.vocab - (g.vocab - head) % V : g.vocab;
    lone = l < V ? l : tail + (l - V);
    edge = lone >= c0 && lone < c0 + reach && (l < V ? l < head && lone < g.vocab : lone < g.vocab);
    if (edge) alone = xr[lone];
  }
  const DistillPair* pr = pairs + row * g.entries;
  DistillPair pair{-1, 0.0f};
  if (l < g.entries) pair = pr[l];
  const float* st = stats + row * kDisStats;
  const float rest_max = st[kStatRestMax], rest = st[kStatRest], max = st[kStatMax], mass = st[kStatListed];
  const bool counted = st[kStatCounts] != 0.0f;
  float gs = reduction == SUPA_AMD_REDUCTION_NONE ? grad_out[row] : grad_out[0];
  if (reduction == SUPA_AMD_REDUCTION_MEAN) gs /= count[0];
  gs = (float)((double)gs * g.inv_t);
  for (int i = l; i < reach / 32; i += G) bits[i] = 0u;
  auto sync = [] {
    if constexpr (G == 64) wave_sync();
    else __syncthreads();
  };
  sync();
  for (int k = l; k < g.entries; k += G) {
    if (k != l) pair = pr[k];
    const int64_t at = pair.at - c0;
    if (pair.at < 0 || at < 0 || at >= reach) continue;
    atomicOr(&bits[at / 32], 1u << (at % 32));
    listed[at] = pair.p;  // the one pair that carries the token
  }
  const float k0 = rest * gs;
  sync();
  auto other = [&](float x) {  // the gradient at a token that is not listed, and at one that is
    const float v = __builtin_amdgcn_exp2f((x - rest_max) * g.c) * k0;
    return counted ? v : 0.0f;
  };
  auto of_listed = [&](float x, float p) {
    return (__builtin_amdgcn_exp2f((x - max) * g.c) * mass - p) * gs;
  };
  if (whole) {
    float f[V];
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = other(elem_f<T>(w, k));
    const uint32_t here = bits[l * V / 32] >> (l * V % 32) & ((1u << V) - 1u);
    if (here) {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (here >> k & 1u) f[k] = of_listed(elem_f<T>(w, k), listed[l * V + k]);
    }
    store_any<T, V>(dst + col, f);
  }
  if (edge) {
    const int at = (int)(lone - c0);
    const float x = (float)to_arith(alone);
    dst[lone] = from_arith<T>(bits[at / 32] >> (at % 32) & 1u ? of_listed(x, listed[at]) : other(x));
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
  for (int i = 0; i < 2; ++i) {
    g.xs[i] = d->logits_strides[i];
    g.is[i] = d->indices_strides[i];
    g.ts[i] = d->teacher_strides[i];
    g.ls[i] = d->lse_strides[i];
  }
  g.inner = FastDiv((uint32_t)d->inner);
  g.vocab = d->vocab;
  g.entries = (int32_t)d->entries;
  g.hash = 64;
  while (g.hash < 2 * g.entries) g.hash *= 2;
  g.idx64 = d->index_dtype == SUPA_AMD_I64;
  g.teacher_dtype = d->teacher_dtype;
  g.segment = (int32_t)std::min<int64_t>(kDisSegment, (d->vocab + 31) / 32 * 32);
  g.teacher_c = kLog2eD / d->temperature;
  g.c = (float)g.teacher_c;
  g.inv_t = 1.0 / d->temperature;
  return SUPA_AMD_OK;
}

// Parts of a row's columns for each of `rows` rows; 1: whole rows.  With two launches more than 500 rows
// gain nothing ([700, 128256] bf16 35 us whole, 39 in parts), nor do parts of under 32 KiB ([500, 32000] bf16 13
// and 15); few long rows do ([100, 128256] bf16 22 us whole, 14 in parts; [16, 262144] float32 32 and 11).
int64_t dis_splits(int64_t rows, int64_t vocab, int dtype) {
  const int64_t vecs = vocab * dtype_size(dtype) / 16;
  if (rows >= 512) return 1;
  return std::max<int64_t>(1, std::min<int64_t>({64, 1536 / std::max<int64_t>(1, rows), vecs / 2048}));
}

template <typename T, int NE, bool REST>
int dis_forward(const DistillArgs& g, int64_t rows, int dtype, const DistillOut& out, float2* parts, int32_t* error_flag,
                hipStream_t st) {
  const int64_t splits = dis_splits(rows, g.vocab, dtype);
  if (splits > 1) {
    DistillArgs p = g;
    const int64_t columns = ((g.vocab + splits - 1) / splits + 255) / 256 * 256;
    const int64_t n = (g.vocab + columns - 1) / columns;
    p.segment = (int32_t)std::min<int64_t>(columns, kDisSegment);
    const size_t bitmap = REST ? 4 * (size_t)dis_bit_words(p.segment) : 0;
    k_distill_part<T, REST><<<dim3((unsigned)n, (unsigned)rows), kDisBlock, bitmap, st>>>(p, columns, parts);
    const int rc = launch_status();
    if (rc) return rc;
    const size_t lds = dis_lds_bytes(g.entries, g.hash, 0);
    k_distill_rows<T, NE, REST><<<(unsigned)rows, 64, lds, st>>>(g, (int)n, parts, out, error_flag);
    return launch_status();
  }
  auto go = [&](auto threads) -> int {
    constexpr int G = decltype(threads)::value, block = G < kDisBlock ? kDisBlock : G, per = block / G;
    const size_t lds = per * dis_lds_bytes(g.entries, g.hash, REST ? g.segment : 0);
    const int64_t slab = ((int64_t(1) << 32) - 1) / block * per;  // HIP: fewer than 2^32 threads a launch
    for (int64_t r0 = 0; r0 < rows; r0 += slab) {
      const int64_t n = std::min(slab, rows - r0);
      k_distill_fwd<T, G, NE, REST><<<(unsigned)((n + per - 1) / per), block, lds, st>>>(g, r0, n, out, error_flag);
      const int rc = launch_status();
      if (rc) return rc;
    }
    return SUPA_AMD_OK;
  };
  // A wavefront a row, where there are enough for four a SIMD, up to 16 KiB a row ([65536, 1000] bf16 76 us, 149 with 256
  // threads; [16384, 8192] 63 and 65; [8192, 12000] 51 and 46), with the rest, whose bitmap then needs no barrier, up to 64 KiB
  // ([5000, 20000] 46 and 55); of fewer rows, up to 8 KiB ([600, 4000] 8.2 and 8.5, [600, 8000] 9.8 and 8.7).
  const int64_t wave_bytes = rows >= 4096 ? (REST ? 64 << 10 : 16 << 10) : 8 << 10;
  if (NE == 4 && g.vocab * dtype_size(dtype) <= wave_bytes) return go(std::integral_constant<int, 64>{});
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

// g: what dis_args made of d, with the teacher_lse that counts.
int distill_forward(const supa_amd_distill_desc* d, const DistillArgs& g, float* loss, float* count, float* stats, void* pairs,
                    void* workspace, int64_t ws_bytes, int32_t* error_flag, void* stream) {
  int rc = SUPA_AMD_OK;
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
      auto forward = [&](auto entries, auto rest) {
        return dis_forward<T, entries.value, rest.value>(g, d->rows, d->dtype, out, parts, error_flag, st);
      };
      auto lists = [&](auto rest) {
        return g.entries <= 256 ? forward(std::integral_constant<int, 4>{}, rest)
                                : forward(std::integral_constant<int, kDisMaxEntries / 64>{}, rest);
      };
      return g.teacher_lse ? lists(std::true_type{}) : lists(std::false_type{});
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
  const int rc = dis_args(d, g);
  return rc ? rc : distill_forward(d, g, loss, count, stats, pairs, workspace, ws_bytes, error_flag, stream);
}

int supa_amd_distill_forward_lse64(const supa_amd_distill_desc* d, const double* teacher_lse, float* loss, float* count,
                                   float* stats, void* pairs, void* workspace, int64_t ws_bytes, int32_t* error_flag,
                                   void* stream) {
  DistillArgs g;
  const int rc = dis_args(d, g);
  if (rc) return rc;
  if (d->rows > 0 && !teacher_lse) return SUPA_AMD_EINVAL;
  g.teacher_lse = teacher_lse;
  g.lse64 = 1;
  return distill_forward(d, g, loss, count, stats, pairs, workspace, ws_bytes, error_flag, stream);
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
    const bool edges = g.vocab % V != 0 || !aligned(gx, 16);
    auto go = [&](auto threads, auto with_edges) -> int {
      constexpr int G = decltype(threads)::value, block = G < kDisBlock ? kDisBlock : G, teams = block / G;
      unsigned blocks = (unsigned)((vecs + G - 1) / G);
      // Workgroups go to the eight XCDs in turn.  Where a row takes a multiple of eight, its first and last one, which have
      // the lone elements, would fall to the same two throughout; one more, which has nothing to do, moves them on from
      // row to row ([2047, 64001] float16, 32 a row: 100 us, with 33 87).
      if (decltype(with_edges)::value && blocks % 8 == 0) ++blocks;
      const int64_t slab = teams * std::max<int64_t>(1, std::min<int64_t>(65535, ((int64_t(1) << 32) - 1) / block / blocks));
      for (int64_t r0 = 0; r0 < d->rows; r0 += slab) {
        const int64_t n = std::min(slab, d->rows - r0);
        k_distill_bwd<T, G, decltype(with_edges)::value><<<dim3(blocks, (unsigned)((n + teams - 1) / teams)), block, 0, st>>>(
            g, r0, n, stats, static_cast<const DistillPair*>(pairs), count, grad_loss, d->reduction, gx);
        const int rc = launch_status();
        if (rc) return rc;
      }
      return SUPA_AMD_OK;
    };
    auto size = [&](auto threads) { return edges ? go(threads, std::true_type{}) : go(threads, std::false_type{}); };
    // Every workgroup looks all pairs through: more of them, and more columns a workgroup ([2000, 50257] bf16 with 1000 pairs
    // 92 us, 109 with 256 threads).  Short rows: a wavefront each ([65536, 1024] bf16 49 us, 63 with 256 threads).
    if (vecs <= 128) return size(std::integral_constant<int, 64>{});
    if (g.entries <= 256 || vecs <= 256) return size(std::integral_constant<int, 256>{});
    return size(std::integral_constant<int, 1024>{});
  });
}

}  // extern "C"

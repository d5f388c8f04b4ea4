// The gated residual with the norms around it: of each row
//   u = N_post(x),  h = s r + g u,  y = N(h)
// (N an RMS or layer norm, or absent), and its gradients.
//
// HBM-bound: the forward reads x and r and writes h and y, once each; the
// backward reads x, r (or a float32 h alone where neither gate nor post norm needs x), dh
// and dy and writes dx and dr.  A row stays in the registers of the G threads
// that share it (row_group.h), as float32, so that its statistics are taken in
// two passes over registers: the mean, then the deviations from it.
//
// Backward, with n = (h - mean) rstd, a = dy w and the row means [.]:
//   dH = dh + rstd (a - [a] - n [a n])     ([a] for LAYER alone)
//   dr = s dH,  dg = sum u dH,  du = g dH
//   dx likewise from du, x's normalised value and the post norm's weight
//   dw = sum dy n, db = sum dy, dw_post = sum du xn, db_post = sum du
// The statistics come from the forward (four floats a row); h is formed again
// from x and r, not taken rounded.  The sums run down the columns: a
// workgroup stays for many rows and keeps its columns' sums in registers,
// writes them as one row of partials, and a second launch adds the partials in
// a fixed order.
//
// Measured on MI355X (this library's copy: 6.2 TB/s): bf16 [8192, 4096] with
// both norms and a gate 47 us forward (5.7 TB/s), 75 + 5 backward (5.4 of its own
// bytes, 0.43 GB with the partials); float32 [6006, 2047], layer norms, a gate a
// sample: 40 us (4.9; rows at 4-byte alignment) and 65 + 5; bf16 on a float32 stream
// [16384, 8192], no gate: 288 us (5.6) and 385 + 5 (5.6); bf16 [8192, 4096], one RMS norm and
// no gate: 44 us (6.1) and 70 + 5 (4.8); [4096, 16384], both norms and a gate: 107 us (5.0).
// Rows of more than 8192 elements with layer norms on both sides spill registers in
// the backward ([4096, 16384] bf16 525 us, RMS norms 226).
#pragma once

#include <atomic>

#include "row_group.h"

namespace sa {

constexpr int kNone = SUPA_AMD_NORM_NONE, kLayer = SUPA_AMD_NORM_LAYER;
// Threads of a backward workgroup.  Where 128 registers a thread are enough
// (`light`), four wavefronts a SIMD hide more of the loads' time ([8192, 4096] bf16,
// RMS norms: 84 us with 512 threads, 81 with 1024; [32768, 1024] 94, 81); where not,
// two, with 256 registers (they would spill: [6006, 2047] float32, layer norms:
// 72 us, 113 with 1024).
constexpr int rn_bwd_block(int g, bool light) { return light || g > 512 ? 1024 : 512; }
// For x of esize bytes an element, ept of them a thread, and the kernel's flags.
constexpr bool rn_light(int esize, int ept, bool post, bool layer, bool own) {
  return esize * ept <= 16 && (esize == 4 || !(own || (post && layer)));
}
constexpr int kRnParts = 256;  // workgroups of the backward: one for each of the chip's CUs

struct RnArgs {
  const void *x, *res, *gate, *pw, *pb, *w, *b;
  int64_t x_stride, res_stride;
  int64_t row0, rows;  // the rows [row0, rows)
  int32_t width;
  uint32_t period;  // rows that share a row of the gate
  int32_t post, norm;
  int32_t pf32;  // the parameters are float32
  float scale, eps, inv_width;
};

// A vector of a parameter (the row at p + at); `fill` where there is none.
template <typename T, int G, int NV, int VW>
__device__ __forceinline__ void rn_param(const RowSlots<G, NV, VW>& c, const void* p, int pf32, int64_t at, int j,
                                         float fill, float (&f)[VW], bool on = true) {
  if (p == nullptr) {
#pragma unroll
    for (int k = 0; k < VW; ++k) f[k] = fill;
  } else if (std::is_same<T, float>::value || pf32) {
    const auto r = c.template load<false>(static_cast<const float*>(p) + at, j, on);
#pragma unroll
    for (int k = 0; k < VW; ++k) f[k] = row_elem<float, VW>(r, k);
  } else {
    const auto r = c.template load<false>(static_cast<const T*>(p) + at, j, on);
#pragma unroll
    for (int k = 0; k < VW; ++k) f[k] = row_elem<T, VW>(r, k);
  }
}
template <typename T, int G, int NV, int VW>
__device__ __forceinline__ void rn_param_store(const RowSlots<G, NV, VW>& c, void* p, int pf32, int64_t at, int j,
                                               const float (&f)[VW], bool on = true) {
  if (std::is_same<T, float>::value || pf32) c.store(static_cast<float*>(p) + at, j, f, on);
  else c.store(static_cast<T*>(p) + at, j, f, on);
}

// Mean and reciprocal deviation of a row's values.
template <bool LAYER, int G, int NV, int VW>
__device__ __forceinline__ float2 rn_stats(const float (&v)[NV][VW], const RowSlots<G, NV, VW>& c, const RnArgs& a,
                                           bool layer, float* lds0, float* lds1) {
  float mean = 0.f;
  if (LAYER && layer) {
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) c.each(j, [&](int k) { s[0] += v[j][k]; });
    group_sum<G>(s, lds0);
    mean = s[0] * a.inv_width;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int j = 0; j < NV; ++j)
    c.each(j, [&](int k) {
      const float d = LAYER ? v[j][k] - mean : v[j][k];
      q[0] = fmaf(d, d, q[0]);
    });
  group_sum<G>(q, lds1);
  return make_float2(mean, rsqrtf(fmaf(q[0], a.inv_width, a.eps)));
}

// The group of a row in the workgroup, as a scalar where a wavefront has one row.
template <int G> __device__ __forceinline__ int rn_group() {
  const int g = threadIdx.x / G;
  return G >= 64 ? __builtin_amdgcn_readfirstlane(g) : g;
}

// P is the parameters' type, LAYER as in the backward.  Parameters are asked for
// before the row's sums, which hide their time ([8192, 8192] bf16 101 -> 96 us,
// [12000, 2560] 53 -> 46); not where float32 ones would cost a workgroup its
// place on the CU ([8192, 6144] bf16 on a float32 stream, layer norm: 115 us, 133
// with them early; [16384, 8192] 287, 294).
template <typename T, typename R, typename P, int G, int EPT, bool LAYER>
__global__ void __launch_bounds__(G > 256 ? G : 256)
k_residual_norm(RnArgs a, R* __restrict__ h_out, T* __restrict__ y_out, float4* __restrict__ stats) {
  constexpr int BS = G > 256 ? G : 256;
  constexpr int VW = 16 / (int)sizeof(T), NV = EPT / VW;
  __shared__ float lds[4][BS / 64];
  const int l = threadIdx.x & (G - 1);
  const int64_t row = a.row0 + (int64_t)blockIdx.x * (BS / G) + rn_group<G>();
  const bool on = row < a.rows;
  if (G <= 64 && !on) return;  // above 64, every thread joins the barriers
  const RowSlots<G, NV, VW> c(l, a.width);
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const R* res = static_cast<const R*>(a.res) + row * a.res_stride;
  RowVec<T, VW> xq[NV];
  RowVec<R, VW> rq[NV];
  constexpr bool kEarly = !(sizeof(P) == 4 && (LAYER || G == 1024));
  RowVec<P, VW> pwq[NV], pbq[NV], gq[NV], wq[NV], bq[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) xq[j] = c.template load<true>(x, j, on);
#pragma unroll
  for (int j = 0; j < NV; ++j) rq[j] = c.template load<true>(res, j, on);
  const int64_t gate_at = a.gate ? (int64_t)((uint32_t)row / a.period) * a.width : 0;
  auto ask = [&](RowVec<P, VW> (&to)[NV], const void* p, int64_t at) {
    if (!p) return;
#pragma unroll
    for (int j = 0; j < NV; ++j) to[j] = c.template load<false>(static_cast<const P*>(p) + at, j, on);
  };
  auto ask_post = [&]() {
    ask(pwq, a.pw, 0);
    if (LAYER) ask(pbq, a.pb, 0);
    ask(gq, a.gate, gate_at);
  };
  auto ask_norm = [&]() {
    ask(wq, a.w, 0);
    if (LAYER) ask(bq, a.b, 0);
  };
  if (kEarly) ask_post(), ask_norm();
  float v[NV][VW];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < VW; ++k) v[j][k] = row_elem<T, VW>(xq[j], k);
  // v from its row's mean and deviation
  auto normalise = [&](float2 m, const void* w, const RowVec<P, VW> (&wv)[NV], const void* b,
                       const RowVec<P, VW> (&bv)[NV]) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < VW; ++k) v[j][k] = (LAYER ? v[j][k] - m.x : v[j][k]) * m.y;
    if (w) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VW; ++k) v[j][k] *= row_elem<P, VW>(wv[j], k);
    }
    if (LAYER && b) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VW; ++k) v[j][k] += row_elem<P, VW>(bv[j], k);
    }
  };
  float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
  if (a.post != kNone) {
    const float2 m = rn_stats<LAYER>(v, c, a, a.post == kLayer, lds[0], lds[1]);
    st.x = m.x;
    st.y = m.y;
    if (!kEarly) ask_post();
    normalise(m, a.pw, pwq, a.pb, pbq);
  }
  if (!kEarly && a.post == kNone) ask_post();
  if (a.gate) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < VW; ++k) v[j][k] *= row_elem<P, VW>(gq[j], k);
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int k = 0; k < VW; ++k) v[j][k] = fmaf(a.scale, row_elem<R, VW>(rq[j], k), v[j][k]);
    c.store(h_out + row * a.width, j, v[j], on);
  }
  if (a.norm != kNone) {
    const float2 m = rn_stats<LAYER>(v, c, a, a.norm == kLayer, lds[2], lds[3]);
    st.z = m.x;
    st.w = m.y;
    if (!kEarly) ask_norm();
    normalise(m, a.w, wq, a.b, bq);
#pragma unroll
    for (int j = 0; j < NV; ++j) c.store(y_out + row * a.width, j, v[j], on);
  }
  if (stats && l == 0 && on) stats[row] = st;
}

// The backward's outputs and how its rows are shared out: `sections` of
// `section` rows (the rows of one row of the gate, or all), each of them
// shared by `cuts` workgroups, or (cuts 1) `per` sections a workgroup.  Of a
// section, workgroup i begins at row i `first` and takes rows `step` apart,
// `span` in all.
struct RnGrads {
  const void *h, *gh, *gy;
  const float4* stats;
  void *gx, *gres, *ggate;
  float* part;      // [workgroups][sums][width]
  int64_t section, sections, first, step, span;
  int32_t cuts, per;
  int32_t sums;     // column sums written: those of the flags below, in their order
  int32_t want_gate, want_pw, want_pb, want_w, want_b;  // want_gate 1: a sum a section, 2: a value an element
};

// A row's operands of the backward as loaded.
template <typename T, typename R, int NV, int VW, bool OWN> struct RnRaw {
  static constexpr int kGate = OWN ? NV : 1;
  RowVec<T, VW> x[NV], gy[NV], gt[kGate];
  RowVec<R, VW> r[NV], gh[NV];
  RowVec<float, VW> gf[kGate];  // the gate's row: gf where it is float32, else gt
  float4 st;
  // keeps the compiler from holding on to floats formed before this
  __device__ __forceinline__ void hide() {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      opaque(x[j].q);
      opaque(gy[j].q);
      opaque(r[j].q);
      opaque(gh[j].q);
    }
  }
};

// Where the backward keeps what a column needs for all rows: the norm's weight
// w, the factor p = w_post g and the offset b_post g that lead from x's
// normalised value xn to g u, and the sums over rows.  One sum of dH xn serves
// the gate and the post norm's weight: over rows of one gate
//   dg = w_post sum dH xn + b_post sum dH,  dw_post = g sum dH xn,  db_post = g sum dH.
// Up to 8 elements a thread (float32: 4), factors and sums fit the registers beside a row and
// the next one's operands.  With 16, the factors lie in LDS (in global memory
// their loads, which return in order, would wait for the row requested before
// them); and a workgroup of 1024 threads, with half the registers each, has two
// of the sums in LDS instead and those of the post norm's parameters with its
// partials, requests a row when it begins, and reads the factors again.
template <int G, int EPT> struct RnKeep {
  static constexpr bool kRegs = EPT <= 8;
  static constexpr bool kLdsFactors = EPT == 16 && G <= 512;
  static constexpr bool kLdsSums = EPT == 16 && G == 1024;
  static constexpr bool kAhead = !kLdsSums;
  // bytes of LDS beside the static ones
  static constexpr int bytes(bool layer) {
    return kLdsSums ? 2 * G * EPT * 4 : kLdsFactors ? (2 + layer) * G * EPT * 4 : 0;
  }
};

// A vector of a thread in LDS: its groups of four floats lie G NV vectors
// apart, so that neighbouring threads read neighbouring 16 bytes.
template <int G, int NV, int VW> struct RnLds {
  float4* p;
  __device__ __forceinline__ void get(int l, int j, float (&f)[VW]) const {
#pragma unroll
    for (int i = 0; i < VW / 4; ++i) {
      const float4 v = p[i * (G * NV) + l + j * G];
      f[4 * i] = v.x;
      f[4 * i + 1] = v.y;
      f[4 * i + 2] = v.z;
      f[4 * i + 3] = v.w;
    }
  }
  __device__ __forceinline__ void put(int l, int j, const float (&f)[VW]) const {
#pragma unroll
    for (int i = 0; i < VW / 4; ++i)
      p[i * (G * NV) + l + j * G] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
  }
};

// The operands of the next row are requested as soon as this row's are
// widened, before its sums are joined.  LAYER: a norm subtracts its mean, or
// there is a bias.  OWN: every row has a row of the gate to itself.
template <typename T, typename R, int G, int EPT, bool POST, bool LAYER, bool OWN>
__global__ void __launch_bounds__(rn_bwd_block(G, rn_light(sizeof(T), EPT, POST, LAYER, OWN)))
k_residual_norm_backward(RnArgs a, RnGrads o) {
  constexpr int BS = rn_bwd_block(G, rn_light(sizeof(T), EPT, POST, LAYER, OWN)), ROWS = BS / G;
  constexpr int VW = 16 / (int)sizeof(T), NV = EPT / VW;
  using Keep = RnKeep<G, EPT>;
  using Lds = RnLds<G, NV, VW>;
  constexpr int kReg = Keep::kRegs ? NV : 1, kSums = Keep::kLdsSums ? 1 : NV;
  constexpr bool kTotals = POST && !Keep::kLdsSums;  // else kept with the partials, section by section
  constexpr int kPost = kTotals ? NV : 1, kPostBias = kTotals && LAYER ? NV : 1, kBias = LAYER ? NV : 1;
  constexpr int NS = LAYER ? 2 : 1;  // sums along a row: a n (and a)
  __shared__ float lds[2][2][NS * BS / 64];
  __shared__ float fold[ROWS > 1 ? BS * EPT : 1];
  extern __shared__ float4 keep[];
  // the factors (kLdsFactors), or the sums of dw and dH xn (kLdsSums)
  const Lds lw{keep}, lp{keep + G * EPT / 4}, lq{keep + G * EPT / 2};
  const int l = threadIdx.x & (G - 1), grp = rn_group<G>();
  RowSlots<G, NV, VW> c(l, a.width);
  const bool has_norm = a.norm != kNone && o.gy != nullptr;
  const bool sum_xn = POST || o.want_gate;
  const bool need_x = sum_xn || (has_norm && !o.h);

  float aw[kSums][VW] = {}, at[kSums][VW] = {};            // dw; dH xn since the gate's row began
  float ab[kBias][VW] = {}, av[kBias][VW] = {};            // db; dH
  float apw[kPost][VW] = {}, apb[kPostBias][VW] = {};      // g times those, of all sections
  float rw[kReg][VW], rp[kReg][VW], rq[kReg][VW];

  // factors of vector j from memory, with the gate's row at `at` (none: 1)
  auto load_factors = [&](const void* gate, int64_t gate_at, int j, bool on, float (&p)[VW], float (&q)[VW]) {
    float g[VW];
    rn_param<T>(c, gate, a.pf32, gate_at, j, 1.f, g, on);
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      p[k] = g[k];
      q[k] = 0.f;
    }
    if constexpr (POST) {
      float w[VW];
      rn_param<T>(c, a.pw, a.pf32, 0, j, 1.f, w, on);
#pragma unroll
      for (int k = 0; k < VW; ++k) p[k] *= w[k];
      if constexpr (LAYER) {
        rn_param<T>(c, a.pb, a.pf32, 0, j, 0.f, q, on);
#pragma unroll
        for (int k = 0; k < VW; ++k) q[k] *= g[k];
      }
    }
  };
  auto keep_factors = [&](int64_t gate_at) {
    if constexpr (!Keep::kLdsSums) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float p[VW], q[VW];
        load_factors(OWN ? nullptr : a.gate, gate_at, j, true, p, q);
        if constexpr (Keep::kLdsFactors) {
          lp.put(l, j, p);
          if constexpr (POST && LAYER) lq.put(l, j, q);
        } else {
#pragma unroll
          for (int k = 0; k < VW; ++k) {
            rp[j][k] = p[k];
            rq[j][k] = q[k];
          }
        }
      }
    }
  };
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if constexpr (Keep::kLdsSums) {
      const float zero[VW] = {};
      lw.put(l, j, zero);
      lp.put(l, j, zero);
    } else {
      float f[VW];
      rn_param<T>(c, a.w, a.pf32, 0, j, 1.f, f);
      if constexpr (Keep::kLdsFactors) {
        lw.put(l, j, f);
      } else {
#pragma unroll
        for (int k = 0; k < VW; ++k) rw[j][k] = f[k];
      }
    }
  }

  // Adds a column sum over the workgroup's groups of rows and hands each
  // thread of the first group its columns' totals.
  auto folded = [&](const float (&s)[VW], int j, auto&& put) {
    if constexpr (ROWS == 1) {
      put(s);
    } else {
      float* mine = fold + (l + j * G) * VW;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < VW; ++k) mine[grp * (G * EPT) + k] = s[k];
      __syncthreads();
      if (grp == 0) {
        float t[VW];
#pragma unroll
        for (int k = 0; k < VW; ++k) t[k] = s[k];
#pragma unroll 1
        for (int g = 1; g < ROWS; ++g) {
#pragma unroll
          for (int k = 0; k < VW; ++k) t[k] += mine[g * (G * EPT) + k];
        }
        put(t);
      }
    }
  };
  float* part = o.part + (int64_t)blockIdx.x * o.sums * a.width;

  // h alone in the place of x and residual: the same sum with factors 1 and 0
  const R* r_rows = static_cast<const R*>(o.h ? o.h : a.res);
  const int64_t r_stride = o.h ? (int64_t)a.width : a.res_stride;
  const float r_scale = o.h ? 1.f : a.scale;
  RnRaw<T, R, NV, VW, OWN> q;
  // What a row does not have, or a group without a row, is zeros.
  auto request = [&](int64_t row, bool active) {
    q.st = active && o.stats ? o.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      q.x[j] = c.template load<true>(static_cast<const T*>(a.x) + row * a.x_stride, j, active && need_x);
      q.r[j] = c.template load<true>(r_rows + row * r_stride, j, active && has_norm);
      q.gy[j] = c.template load<true>(static_cast<const T*>(o.gy) + row * a.width, j, active && has_norm);
      q.gh[j] = c.template load<true>(static_cast<const R*>(o.gh) + row * a.width, j, active && o.gh);
      if constexpr (OWN && Keep::kAhead) {
        if (std::is_same<T, float>::value || a.pf32)
          q.gf[j] = c.template load<true>(static_cast<const float*>(a.gate) + row * a.width, j, active);
        else
          q.gt[j] = c.template load<true>(static_cast<const T*>(a.gate) + row * a.width, j, active);
      }
    }
  };

  int parity = 0;
  const int64_t sec0 = (int64_t)(blockIdx.x / (uint32_t)o.cuts) * o.per;
  const int64_t sec1 = sec0 + o.per < o.sections ? sec0 + o.per : o.sections;
  for (int64_t sec = sec0; sec < sec1; ++sec) {
    const int64_t r0 = sec * o.section + (int64_t)(blockIdx.x % (uint32_t)o.cuts) * o.first;
    const int64_t end = (sec + 1) * o.section < a.rows ? (sec + 1) * o.section : a.rows;
    const int64_t r1 = r0 + o.span < end ? r0 + o.span : end;
    const int64_t gate_at = a.gate ? (int64_t)((uint32_t)r0 / a.period) * a.width : 0;
    keep_factors(gate_at);
    if constexpr (Keep::kAhead) request(r0 + grp, r0 + grp < r1);
    for (int64_t base = r0; base < r1; base += o.step, parity ^= 1) {
      c.renew();
      const int64_t row = base + grp;
      const bool active = ROWS == 1 || row < r1;  // no row: zeros are added and nothing is stored
      if constexpr (!Keep::kAhead) request(row, active);
      const float4 st = q.st;
      // The row as floats: kept while the next row is on its way into q, or
      // (kAhead false, registers for one of the two) formed from q each time.
      constexpr int kRow = Keep::kAhead ? NV : 1;
      float xs[kRow][VW], ns[kRow][VW], das[kRow][VW], dH[NV][VW], s[NS] = {};
      float gs[OWN && Keep::kAhead ? NV : 1][VW];
      auto normalised_x = [&](int j, float (&x)[VW]) {
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          x[k] = row_elem<T, VW>(q.x[j], k);
          if constexpr (POST) x[k] = (LAYER ? x[k] - st.x : x[k]) * st.y;
        }
      };
      auto x_of = [&](int j, float (&x)[VW]) {
        if constexpr (Keep::kAhead) {
#pragma unroll
          for (int k = 0; k < VW; ++k) x[k] = xs[j][k];
        } else {
          normalised_x(j, x);
        }
      };
      auto factors = [&](int j, float (&p)[VW], float (&b)[VW]) {
        if constexpr (Keep::kLdsSums) {
          load_factors(a.gate, OWN ? row * a.width : gate_at, j, active, p, b);
        } else if constexpr (Keep::kLdsFactors) {
          lp.get(l, j, p);
          if constexpr (POST && LAYER) lq.get(l, j, b);
        } else {
#pragma unroll
          for (int k = 0; k < VW; ++k) {
            p[k] = rp[j < kReg ? j : 0][k];
            b[k] = rq[j < kReg ? j : 0][k];
          }
        }
      };
      // the same with the row's own gate in them
      auto gated_factors = [&](int j, float (&p)[VW], float (&b)[VW]) {
        factors(j, p, b);
        if constexpr (OWN && Keep::kAhead) {
#pragma unroll
          for (int k = 0; k < VW; ++k) {
            p[k] *= gs[j][k];
            if constexpr (POST && LAYER) b[k] *= gs[j][k];
          }
        }
      };
      // n = (h - mean) rstd, a = dy w and dy of vector j
      auto normalised_h = [&](int j, float (&n)[VW], float (&da)[VW], float (&dy)[VW]) {
        float x[VW], p[VW], b[VW], w[VW];
        x_of(j, x);
        gated_factors(j, p, b);
        if constexpr (Keep::kLdsFactors) lw.get(l, j, w);
        else if constexpr (Keep::kLdsSums) rn_param<T>(c, a.w, a.pf32, 0, j, 1.f, w);
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          if constexpr (Keep::kRegs) w[k] = rw[j < kReg ? j : 0][k];
          const float u = POST && LAYER ? fmaf(x[k], p[k], b[k]) : x[k] * p[k];
          const float h = fmaf(r_scale, row_elem<R, VW>(q.r[j], k), u);
          dy[k] = row_elem<T, VW>(q.gy[j], k);
          n[k] = (LAYER ? h - st.z : h) * st.w;
          da[k] = dy[k] * w[k];
        }
      };
      // dh plus the norm's part, of one element
      auto through_norm = [&](float n, float da, float dh, float c0, float c1) {
        return fmaf(st.w, fmaf(-n, c1, LAYER ? da - c0 : da), dh);
      };
      // joins the row's sums: the factors of a constant and of the normalised value
      auto joined = [&](bool layer, float* at_lds, float& c0, float& c1) {
        group_sum<G>(s, at_lds);
        c1 = s[0] * a.inv_width;
        c0 = LAYER && layer ? s[NS - 1] * a.inv_width : 0.f;
      };
      if constexpr (Keep::kAhead) {
#pragma unroll
        for (int j = 0; j < NV; ++j) normalised_x(j, xs[j]);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int k = 0; k < VW; ++k) dH[j][k] = row_elem<R, VW>(q.gh[j], k);
        if constexpr (OWN) {
          const bool wide = std::is_same<T, float>::value || a.pf32;
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VW; ++k) gs[j][k] = wide ? row_elem<float, VW>(q.gf[j], k) : row_elem<T, VW>(q.gt[j], k);
        }
      }
      if (has_norm) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float n[VW], da[VW], dy[VW], sum[VW];
          normalised_h(j, n, da, dy);
          if constexpr (Keep::kLdsSums) lw.get(l, j, sum);
#pragma unroll
          for (int k = 0; k < VW; ++k) {
            if constexpr (Keep::kLdsSums) sum[k] = fmaf(dy[k], n[k], sum[k]);
            else aw[j][k] = fmaf(dy[k], n[k], aw[j][k]);
            if constexpr (LAYER) ab[j][k] += dy[k];
            if constexpr (Keep::kAhead) {
              ns[j][k] = n[k];
              das[j][k] = da[k];
            }
          }
          if constexpr (Keep::kLdsSums) lw.put(l, j, sum);
          c.each(j, [&](int k) {
            s[0] = fmaf(da[k], n[k], s[0]);
            if constexpr (LAYER) s[1] += da[k];
          });
        }
        if constexpr (Keep::kAhead) {
          if (base + o.step < r1) request(row + o.step, row + o.step < r1);
        }
        float c0, c1;
        joined(a.norm == kLayer, lds[parity][0], c0, c1);
        if constexpr (!Keep::kAhead) q.hide(), c.renew();
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if constexpr (Keep::kAhead) {
#pragma unroll
            for (int k = 0; k < VW; ++k) dH[j][k] = through_norm(ns[j][k], das[j][k], dH[j][k], c0, c1);
          } else {
            float n[VW], da[VW], dy[VW];
            normalised_h(j, n, da, dy);
#pragma unroll
            for (int k = 0; k < VW; ++k)
              dH[j][k] = through_norm(n[k], da[k], row_elem<R, VW>(q.gh[j], k), c0, c1);
          }
        }
      } else if constexpr (Keep::kAhead) {
        if (base + o.step < r1) request(row + o.step, row + o.step < r1);
      } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int k = 0; k < VW; ++k) dH[j][k] = row_elem<R, VW>(q.gh[j], k);
      }
      if (o.gres) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float t[VW];
#pragma unroll
          for (int k = 0; k < VW; ++k) t[k] = a.scale * dH[j][k];
          c.store(static_cast<R*>(o.gres) + row * a.width, j, t, active);
        }
      }
      if constexpr (OWN) {
        // the gate's gradient is this row's own, and the sums take dH g
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float x[VW], g[VW], u[VW], p[VW], b[VW];
          x_of(j, x);
          if (o.want_gate) {
            if constexpr (Keep::kAhead) factors(j, p, b);
            else load_factors(nullptr, 0, j, active, p, b);
#pragma unroll
            for (int k = 0; k < VW; ++k) u[k] = (POST && LAYER ? fmaf(x[k], p[k], b[k]) : x[k] * p[k]) * dH[j][k];
            rn_param_store<T>(c, o.ggate, a.pf32, row * a.width, j, u, active);
          }
          if constexpr (kTotals) {
#pragma unroll
            for (int k = 0; k < VW; ++k) {
              const float du = dH[j][k] * gs[Keep::kAhead ? j : 0][k];
              apw[j][k] = fmaf(du, x[k], apw[j][k]);
              if constexpr (LAYER) apb[j][k] += du;
            }
          } else if constexpr (POST) {
            float sum[VW];
            rn_param<T>(c, a.gate, a.pf32, row * a.width, j, 1.f, g, active);
            lp.get(l, j, sum);
#pragma unroll
            for (int k = 0; k < VW; ++k) {
              const float du = dH[j][k] * g[k];
              sum[k] = fmaf(du, x[k], sum[k]);
              if constexpr (LAYER) av[j][k] += du;
            }
            lp.put(l, j, sum);
          }
        }
      } else if (sum_xn) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float x[VW], sum[VW];
          x_of(j, x);
          if constexpr (Keep::kLdsSums) lp.get(l, j, sum);
#pragma unroll
          for (int k = 0; k < VW; ++k) {
            if constexpr (Keep::kLdsSums) sum[k] = fmaf(dH[j][k], x[k], sum[k]);
            else at[j][k] = fmaf(dH[j][k], x[k], at[j][k]);
            if constexpr (POST && LAYER) av[j][k] += dH[j][k];
          }
          if constexpr (Keep::kLdsSums) lp.put(l, j, sum);
        }
      }
      if constexpr (POST) {
#pragma unroll
        for (int i = 0; i < NS; ++i) s[i] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float x[VW], p[VW], b[VW];
        gated_factors(j, p, b);
#pragma unroll
        for (int k = 0; k < VW; ++k) dH[j][k] *= p[k];  // the gradient of xn from here on
        if constexpr (POST) {
          x_of(j, x);
          c.each(j, [&](int k) {
            s[0] = fmaf(dH[j][k], x[k], s[0]);
            if constexpr (LAYER) s[1] += dH[j][k];
          });
        }
      }
      if constexpr (POST) {
        float c0, c1;
        joined(a.post == kLayer, lds[parity][1], c0, c1);
        if constexpr (!Keep::kAhead) q.hide(), c.renew();
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float x[VW];
          x_of(j, x);
#pragma unroll
          for (int k = 0; k < VW; ++k) dH[j][k] = st.y * fmaf(-x[k], c1, LAYER ? dH[j][k] - c0 : dH[j][k]);
        }
      }
      if (o.gx) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          c.store(static_cast<T*>(o.gx) + row * a.width, j, dH[j], active);
      }
    }
    if (!OWN && sum_xn) {  // the gate's row ends
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float t[VW], g[VW], one[VW], b[VW];
        if constexpr (Keep::kLdsSums) {
          const float zero[VW] = {};
          lp.get(l, j, t);
          lp.put(l, j, zero);
        } else {
#pragma unroll
          for (int k = 0; k < VW; ++k) {
            t[k] = at[j][k];
            at[j][k] = 0.f;
          }
        }
        if constexpr (POST) rn_param<T>(c, a.gate, a.pf32, gate_at, j, 1.f, g);
        if constexpr (kTotals) {
#pragma unroll
          for (int k = 0; k < VW; ++k) {
            apw[j][k] = fmaf(g[k], t[k], apw[j][k]);
            if constexpr (LAYER) apb[j][k] = fmaf(g[k], av[j][k], apb[j][k]);
          }
        } else if constexpr (POST) {
          float* total = part + (o.want_gate == 1 && o.cuts > 1 ? a.width : 0);
          // to the total that this thread wrote at the last section's end; of the vector
          // that was moved back its own elements alone, as another thread adds the others
          auto add = [&](const auto& s) {
            if (c.whole(j)) {
              RowVec<float, VW> old{};
              if (sec > sec0) old = c.template load<false>(total, j);
              float f[VW];
#pragma unroll
              for (int k = 0; k < VW; ++k) f[k] = fmaf(g[k], s[k], row_elem<float, VW>(old, k));
              c.store(total, j, f);
            } else {
              c.each(j, [&](int k) {
                float* at = total + c.col[j] + k;
                *at = fmaf(g[k], s[k], sec > sec0 ? *at : 0.f);
              });
            }
            total += a.width;
          };
          if (o.want_pw) add(t);
          if constexpr (LAYER) {
            if (o.want_pb) add(av[j]);
          }
        }
        if (o.want_gate) {
          load_factors(nullptr, 0, j, true, one, b);
#pragma unroll
          for (int k = 0; k < VW; ++k) t[k] = POST && LAYER ? fmaf(one[k], t[k], b[k] * av[j][k]) : one[k] * t[k];
          folded(t, j, [&](const float (&f)[VW]) {
            if (o.cuts > 1) c.store(part, j, f);
            else rn_param_store<T>(c, o.ggate, a.pf32, sec * a.width, j, f);
          });
        }
        if constexpr (POST && LAYER) {
#pragma unroll
          for (int k = 0; k < VW; ++k) av[j][k] = 0.f;
        }
      }
    }
  }
  if (o.want_gate == 1 && o.cuts > 1) part += a.width;
  auto put = [&](int want, auto&& sum) {
    if (!want) return;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float t[VW];
      sum(j, t);
      folded(t, j, [&](const float (&f)[VW]) { c.store(part, j, f); });
    }
    part += a.width;
  };
  auto from = [&](const auto& s) {
    return [&](int j, float (&t)[VW]) {
#pragma unroll
      for (int k = 0; k < VW; ++k) t[k] = s[j][k];
    };
  };
  if constexpr (kTotals) {
    put(o.want_pw, from(apw));
    if constexpr (LAYER) put(o.want_pb, from(apb));
  } else if constexpr (POST && OWN) {
    put(o.want_pw, [&](int j, float (&t)[VW]) { lp.get(l, j, t); });
    if constexpr (LAYER) put(o.want_pb, from(av));
  } else if constexpr (POST) {  // written at the sections' ends
    part += (o.want_pw + (LAYER ? o.want_pb : 0)) * (int64_t)a.width;
  }
  if constexpr (Keep::kLdsSums) put(o.want_w, [&](int j, float (&t)[VW]) { lw.get(l, j, t); });
  else put(o.want_w, from(aw));
  if constexpr (LAYER) put(o.want_b, from(ab));
}

// Adds the partials: block (x, y) the columns [64 x, 64 x + 64) of sum y.  The
// gate's sections come first, each over its own `cuts` workgroups.
struct RnSums {
  const float* part;
  void* out[4];       // the sums over all workgroups
  void* gate;
  int32_t gate_sections, cuts, sums, parts, width, pf32;
};
constexpr int kRnSumWaves = 16;
template <typename T>
__global__ void __launch_bounds__(64 * kRnSumWaves) k_residual_norm_sums(RnSums a) {
  __shared__ float lds[kRnSumWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = (int)blockIdx.x * 64 + lane;
  const int y = (int)blockIdx.y;
  const bool gate = y < a.gate_sections;
  const int which = gate ? 0 : y - a.gate_sections + (a.gate_sections > 0 ? 1 : 0);
  const int lo = gate ? y * a.cuts : 0, hi = gate ? lo + a.cuts : a.parts;
  float s = 0.f;
  if (col < a.width) {
    const float* p = a.part + (int64_t)which * a.width + col;
    const int64_t stride = (int64_t)a.sums * a.width;
    s = fold_strided<8>(
        0.f, (int64_t)lo + wave, kRnSumWaves, (int64_t)hi, [&](int64_t i) { return p[i * stride]; },
        [](float u, float v) { return u + v; });
  }
  lds[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && col < a.width) {
#pragma unroll
    for (int w = 1; w < kRnSumWaves; ++w) s += lds[w][lane];
    void* out = gate ? a.gate : a.out[y - a.gate_sections];
    const int64_t at = gate ? (int64_t)y * a.width + col : col;
    if (a.pf32) static_cast<float*>(out)[at] = s;
    else static_cast<T*>(out)[at] = from_arith<T>(s);
  }
}

// The threads a row and the elements a thread, for an x of esize bytes an
// element: the fewest threads that hold the row with 8 elements each; of float32
// twice as many with one vector each where that helped ([6006, 2047] layer norms 41.6
// us with two vectors, 39.3 with one; [8192, 4096] 86, 87; [262144, 72] 70, 76).
template <int esize, typename F> int rn_fwd_shape(int64_t width, F&& go) {
  using std::integral_constant;
  using E4 = integral_constant<int, 4>;
  using E8 = integral_constant<int, 8>;
  if (width <= 128) return go(integral_constant<int, 16>{}, E8{});
  if (width <= 256) return go(integral_constant<int, 32>{}, E8{});
  if (width <= 512) return go(integral_constant<int, 64>{}, E8{});
  if constexpr (esize == 4) {
    if (width <= 1024) return go(integral_constant<int, 256>{}, E4{});
    if (width <= 2048) return go(integral_constant<int, 512>{}, E4{});
  }
  if (width <= 1024) return go(integral_constant<int, 128>{}, E8{});
  if (width <= 2048) return go(integral_constant<int, 256>{}, E8{});
  if (width <= 4096) return go(integral_constant<int, 512>{}, E8{});
  if (width <= 8192) return go(integral_constant<int, 1024>{}, E8{});
  return go(integral_constant<int, 1024>{}, integral_constant<int, 16>{});
}
// The same for the backward, whose threads need more registers: one vector a thread up to 4096 elements ([16384, 1024] float32
// 82 us with two, 73 with one), then 512 threads of 16 elements up to 8192.
template <int esize, typename F> int rn_bwd_shape(int64_t width, F&& go) {
  using std::integral_constant;
  constexpr int E = 16 / esize;
  using V1 = integral_constant<int, E>;
  using E16 = integral_constant<int, 16>;
  if (width <= 16 * E) return go(integral_constant<int, 16>{}, V1{});
  if (width <= 32 * E) return go(integral_constant<int, 32>{}, V1{});
  if (width <= 64 * E) return go(integral_constant<int, 64>{}, V1{});
  if (width <= 128 * E) return go(integral_constant<int, 128>{}, V1{});
  if (width <= 256 * E) return go(integral_constant<int, 256>{}, V1{});
  if (width <= 512 * E) return go(integral_constant<int, 512>{}, V1{});
  if constexpr (esize == 4) {
    if (width <= 1024 * E) return go(integral_constant<int, 1024>{}, V1{});
  }
  if (width <= 8192) return go(integral_constant<int, 512>{}, E16{});
  return go(integral_constant<int, 1024>{}, E16{});
}

inline int rn_check(const supa_amd_residual_norm_desc* d) {
  if (!d || d->rows < 0 || d->width < 1) return SUPA_AMD_EINVAL;
  if (d->width > SUPA_AMD_RESIDUAL_NORM_MAX_WIDTH || d->rows >= (int64_t(1) << 31)) return SUPA_AMD_ELAYOUT;
  if (d->dtype != SUPA_AMD_F32 && d->dtype != SUPA_AMD_BF16 && d->dtype != SUPA_AMD_F16) return SUPA_AMD_EDTYPE;
  if (d->residual_dtype != d->dtype && d->residual_dtype != SUPA_AMD_F32) return SUPA_AMD_EDTYPE;
  if (d->param_dtype != d->dtype && d->param_dtype != SUPA_AMD_F32) return SUPA_AMD_EDTYPE;
  for (int n : {d->post_norm, d->norm})
    if (n < SUPA_AMD_NORM_NONE || n > SUPA_AMD_NORM_LAYER) return SUPA_AMD_EINVAL;
  if (d->gate && d->rows > 0 && (d->gate_period < 1 || d->rows % d->gate_period != 0)) return SUPA_AMD_EINVAL;
  if ((d->post_norm != SUPA_AMD_NORM_LAYER && d->post_bias) || (d->norm != SUPA_AMD_NORM_LAYER && d->bias))
    return SUPA_AMD_EINVAL;
  if ((d->post_norm == SUPA_AMD_NORM_NONE && d->post_weight) || (d->norm == SUPA_AMD_NORM_NONE && d->weight))
    return SUPA_AMD_EINVAL;
  return SUPA_AMD_OK;
}

inline RnArgs rn_args(const supa_amd_residual_norm_desc& d) {
  RnArgs a{};
  a.x = d.x;
  a.res = d.residual;
  a.gate = d.gate;
  a.pw = d.post_weight;
  a.pb = d.post_bias;
  a.w = d.weight;
  a.b = d.bias;
  a.x_stride = d.x_stride;
  a.res_stride = d.residual_stride;
  a.rows = d.rows;
  a.width = (int32_t)d.width;
  a.period = d.gate ? (uint32_t)d.gate_period : 1u;
  a.post = d.post_norm;
  a.norm = d.norm;
  a.pf32 = d.param_dtype == SUPA_AMD_F32;
  a.scale = (float)d.residual_scale;
  a.eps = (float)d.eps;
  a.inv_width = (float)(1.0 / (double)d.width);
  return a;
}

inline bool rn_layer(const supa_amd_residual_norm_desc& d) {
  return d.post_norm == SUPA_AMD_NORM_LAYER || d.norm == SUPA_AMD_NORM_LAYER;
}

// How the backward's rows are shared out; only the sizes decide.
struct RnPlan {
  int64_t section, sections, first, step, span;
  int32_t cuts, per, parts;
  bool elementwise;  // a gate row a row
};
inline RnPlan rn_plan(const supa_amd_residual_norm_desc& d) {
  RnPlan p{};
  int64_t at_once = 1;
  p.elementwise = d.gate && d.gate_period == 1;
  const auto block = [&](auto G, auto E) {
    const bool light = rn_light(dtype_size(d.dtype), E.value, d.post_norm != kNone, rn_layer(d), p.elementwise);
    at_once = rn_bwd_block(G.value, light) / G.value;
    return 0;
  };
  if (d.dtype == SUPA_AMD_F32) rn_bwd_shape<4>(d.width, block);
  else rn_bwd_shape<2>(d.width, block);
  p.section = d.gate && !p.elementwise ? d.gate_period : d.rows;
  p.sections = d.rows / p.section;
  const int64_t steps = (p.section + at_once - 1) / at_once;
  // No more workgroups than CUs: one left over would run alone ([6, 1024, 2048] float32
  // in 258 workgroups 84 us, in 252 67), and 160 CUs come near the memory's rate
  // ([160, 64, 2048] bf16 in 160 workgroups 60 us, in 480 74).
  p.cuts = (int32_t)std::min<int64_t>(steps, std::max<int64_t>(1, kRnParts / p.sections));
  // Rows of one section are dealt out in turn, so that the chip works on
  // neighbouring rows at any time ([8192, 8192] bf16 170 -> 151 us, [8192, 4096] 82 ->
  // 79, [20000, 1500] float32 127 -> 109); of several sections, which lie apart in any case, a
  // workgroup takes consecutive rows ([8, 1024, 4096] bf16 86 us, dealt out 92).
  if (p.sections == 1) {
    p.first = at_once;
    p.step = p.cuts * at_once;
    p.span = p.section;
  } else {
    const int64_t run = (steps + p.cuts - 1) / p.cuts;
    p.cuts = (int32_t)((steps + run - 1) / run);
    p.first = p.span = run * at_once;
    p.step = at_once;
  }
  p.per = p.cuts > 1 ? 1 : (int32_t)((p.sections + kRnParts - 1) / kRnParts);
  p.parts = p.cuts > 1 ? (int32_t)(p.sections * p.cuts) : (int32_t)((p.sections + p.per - 1) / p.per);
  return p;
}

// The launches for one pair of types (residual_norm_*.hip).
template <typename T, typename R>
int rn_forward_t(const supa_amd_residual_norm_desc* d, const RnArgs& a, void* h, void* y, float* stats, hipStream_t st) {
  return rn_fwd_shape<sizeof(T)>(d->width, [&](auto G, auto E) -> int {
    constexpr int BS = G.value > 256 ? G.value : 256, PER = BS / G.value;
    constexpr int64_t kSlab = (int64_t(1) << 31) / BS * PER;  // HIP: fewer than 2^32 threads a launch
    for (int64_t r0 = 0; r0 < d->rows; r0 += kSlab) {
      RnArgs s = a;
      s.row0 = r0;
      s.rows = std::min(d->rows, r0 + kSlab);
      auto go = [&](auto* p, auto layer) {
        using P = std::remove_pointer_t<decltype(p)>;
        k_residual_norm<T, R, P, G.value, E.value, layer.value>
            <<<(unsigned)((s.rows - r0 + PER - 1) / PER), BS, 0, st>>>(s, static_cast<R*>(h), static_cast<T*>(y),
                                                                      reinterpret_cast<float4*>(stats));
      };
      auto typed = [&](auto layer) {
        if (a.pf32) go((float*)nullptr, layer);
        else go((T*)nullptr, layer);
      };
      if (rn_layer(*d)) typed(std::true_type{});
      else typed(std::false_type{});
      const int rl = launch_status();
      if (rl) return rl;
    }
    return SUPA_AMD_OK;
  });
}

template <typename T, typename R>
int rn_backward_t(const supa_amd_residual_norm_desc* d, const RnArgs& a, const RnPlan& p, const RnGrads& o, int gate_sums,
                  void* grad_gate, void* grad_post_weight, void* grad_post_bias, void* grad_weight, void* grad_bias,
                  hipStream_t st) {
  const int rl = rn_bwd_shape<sizeof(T)>(d->width, [&](auto G, auto E) -> int {
    auto go = [&](auto post, auto layer, auto own) -> int {
      constexpr auto kernel = k_residual_norm_backward<T, R, G.value, E.value, post.value, layer.value, own.value>;
      constexpr int lds = RnKeep<G.value, E.value>::bytes(layer.value);
      constexpr int block = rn_bwd_block(G.value, rn_light(sizeof(T), E.value, post.value, layer.value, own.value));
      // with the static part it may take more than a launch has without asking; once a device
      if constexpr (lds > 32768) {
        static std::atomic<uint64_t> asked{0};
        int dev = 0;
        const hipError_t e = hipGetDevice(&dev);
        if (e != hipSuccess) return (int)e;
        if (dev > 63 || !(asked.load() >> dev & 1)) {
          const hipError_t set = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, lds);
          if (set != hipSuccess) return (int)set;
          if (dev <= 63) asked.fetch_or(uint64_t(1) << dev);
        }
      }
      kernel<<<(unsigned)p.parts, block, lds, st>>>(a, o);
      return launch_status();
    };
    using Yes = std::true_type;
    using No = std::false_type;
    auto layered = [&](auto post, auto own) { return rn_layer(*d) ? go(post, Yes{}, own) : go(post, No{}, own); };
    if (d->post_norm != kNone) return p.elementwise ? layered(Yes{}, Yes{}) : layered(Yes{}, No{});
    return p.elementwise ? layered(No{}, Yes{}) : layered(No{}, No{});
  });
  if (rl || o.sums == 0) return rl;
  RnSums f{};
  f.part = o.part;
  int n = 0;
  for (void* out : {grad_post_weight, grad_post_bias, grad_weight, grad_bias})
    if (out) f.out[n++] = out;
  f.gate = grad_gate;
  f.gate_sections = gate_sums ? (int32_t)p.sections : 0;
  f.cuts = p.cuts;
  f.sums = o.sums;
  f.parts = p.parts;
  f.width = a.width;
  f.pf32 = a.pf32;
  k_residual_norm_sums<T><<<dim3((unsigned)((d->width + 63) / 64), (unsigned)(f.gate_sections + n)), 64 * kRnSumWaves, 0,
                            st>>>(f);
  return launch_status();
}

}  // namespace sa

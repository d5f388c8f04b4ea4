// The gated residual with the norms around it: of each row
//   u = N_post(x),  h = s r + g u,  y = N(h)
// (N an RMS or layer norm, or absent), and its gradients.
//
// HBM-bound: the forward reads x and r and writes h and y, once each; the
// backward reads x, r (or h alone where neither gate nor post norm needs x), dh
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
// workgroup takes consecutive rows and keeps its columns' sums in registers,
// writes them as one row of partials, and a second launch adds the partials in
// a fixed order.
#include "row_group.h"

namespace sa {

constexpr int kNone = SUPA_AMD_NORM_NONE, kLayer = SUPA_AMD_NORM_LAYER;
// Threads of a backward workgroup: two wavefronts a SIMD, so that a thread has 256 registers.
constexpr int rn_bwd_block(int g) { return g > 512 ? g : 512; }
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
template <int G, int NV, int VW>
__device__ __forceinline__ float2 rn_stats(const float (&v)[NV][VW], const RowSlots<G, NV, VW>& c, const RnArgs& a,
                                           bool layer, float* lds0, float* lds1) {
  float mean = 0.f;
  if (layer) {
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
      const float d = v[j][k] - mean;
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

template <typename T, typename R, int G, int EPT>
__global__ void __launch_bounds__(G > 256 ? G : 256)
k_residual_norm(RnArgs a, R* __restrict__ h_out, T* __restrict__ y_out, float4* __restrict__ stats) {
  constexpr int BS = G > 256 ? G : 256;
  constexpr int VW = 16 / (int)sizeof(T), NV = EPT / VW;
  __shared__ float lds[4][BS / 64];
  const int l = threadIdx.x & (G - 1);
  const int64_t row = a.row0 + (int64_t)blockIdx.x * (BS / G) + rn_group<G>();
  if (row >= a.rows) return;  // G above 64: a row a workgroup, all of them there
  const RowSlots<G, NV, VW> c(l, a.width);
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const R* res = static_cast<const R*>(a.res) + row * a.res_stride;
  RowVec<T, VW> xq[NV];
  RowVec<R, VW> rq[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) xq[j] = c.template load<true>(x, j);
#pragma unroll
  for (int j = 0; j < NV; ++j) rq[j] = c.template load<true>(res, j);
  float v[NV][VW];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < VW; ++k) v[j][k] = row_elem<T, VW>(xq[j], k);
  float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
  if (a.post != kNone) {
    const float2 m = rn_stats(v, c, a, a.post == kLayer, lds[0], lds[1]);
    st.x = m.x;
    st.y = m.y;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float w[VW], b[VW];
      rn_param<T>(c, a.pw, a.pf32, 0, j, 1.f, w);
      rn_param<T>(c, a.pb, a.pf32, 0, j, 0.f, b);
#pragma unroll
      for (int k = 0; k < VW; ++k) v[j][k] = fmaf((v[j][k] - m.x) * m.y, w[k], b[k]);
    }
  }
  const int64_t gate_at = a.gate ? (int64_t)((uint32_t)row / a.period) * a.width : 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (a.gate) {
      float g[VW];
      rn_param<T>(c, a.gate, a.pf32, gate_at, j, 1.f, g);
#pragma unroll
      for (int k = 0; k < VW; ++k) v[j][k] *= g[k];
    }
#pragma unroll
    for (int k = 0; k < VW; ++k) v[j][k] = fmaf(a.scale, row_elem<R, VW>(rq[j], k), v[j][k]);
    c.store(h_out + row * a.width, j, v[j]);
  }
  if (a.norm != kNone) {
    const float2 m = rn_stats(v, c, a, a.norm == kLayer, lds[2], lds[3]);
    st.z = m.x;
    st.w = m.y;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float w[VW], b[VW];
      rn_param<T>(c, a.w, a.pf32, 0, j, 1.f, w);
      rn_param<T>(c, a.b, a.pf32, 0, j, 0.f, b);
#pragma unroll
      for (int k = 0; k < VW; ++k) v[j][k] = fmaf((v[j][k] - m.x) * m.y, w[k], b[k]);
      c.store(y_out + row * a.width, j, v[j]);
    }
  }
  if (stats && l == 0) stats[row] = st;
}

// The backward's outputs and how its rows are shared out: `sections` of
// `section` rows (the rows of one row of the gate, or all), each cut in `cuts`
// runs of `run` rows, a workgroup each; or (cuts 1) `per` sections a workgroup.
struct RnGrads {
  const void *h, *gh, *gy;
  const float4* stats;
  void *gx, *gres, *ggate;
  float* part;      // [workgroups][sums][width]
  int64_t section, sections, run;
  int32_t cuts, per;
  int32_t sums;     // column sums written: those of the flags below, in their order
  int32_t want_gate, want_pw, want_pb, want_w, want_b;  // want_gate 1: a sum a section, 2: a value an element
};

// A row's operands of the backward as loaded.
template <typename T, typename R, int NV, int VW> struct RnRaw {
  RowVec<T, VW> x[NV], gy[NV];
  RowVec<R, VW> r[NV], gh[NV];
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

// Where the backward keeps what a column needs for all rows.  Up to 8 elements
// a thread parameters and sums fit the registers beside two rows.  With 16, the
// parameters lie in LDS (in global memory their loads, which return in order,
// would wait for the row requested before them); and a workgroup of 1024
// threads, with half the registers each, has the two sums that are always there
// in LDS instead, requests a row when it begins, and reads the parameters again.
template <int G, int EPT> struct RnKeep {
  static constexpr bool kRegParams = EPT == 8;
  static constexpr bool kLdsParams = EPT == 16 && G == 512;
  static constexpr bool kLdsSums = EPT == 16 && G == 1024;
  static constexpr bool kAhead = !kLdsSums;
  // bytes of LDS beside the static ones
  static constexpr int bytes(bool post, bool bias) {
    return kLdsSums ? 2 * G * EPT * 4 : kLdsParams ? (2 + post + (post && bias)) * G * EPT * 4 : 0;
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
// widened, before its sums are joined.
template <typename T, typename R, int G, int EPT, bool POST, bool BIAS>
__global__ void __launch_bounds__(rn_bwd_block(G))
k_residual_norm_backward(RnArgs a, RnGrads o) {
  constexpr int BS = rn_bwd_block(G), ROWS = BS / G;
  constexpr int VW = 16 / (int)sizeof(T), NV = EPT / VW;
  using Keep = RnKeep<G, EPT>;
  using Lds = RnLds<G, NV, VW>;
  constexpr int kReg = Keep::kRegParams ? NV : 1;
  extern __shared__ float4 keep[];
  // parameters (kLdsParams), or the sums of dw and dgate (kLdsSums)
  const Lds lw{keep}, lgate{keep + G * EPT / 4}, lpw{keep + G * EPT / 2}, lpb{keep + 3 * (G * EPT / 4)};
  __shared__ float lds[2][2][2 * BS / 64];
  __shared__ float fold[ROWS > 1 ? BS * EPT : 1];
  const int l = threadIdx.x & (G - 1), grp = rn_group<G>();
  RowSlots<G, NV, VW> c(l, a.width);
  const bool has_norm = a.norm != kNone && o.gy != nullptr;
  const bool need_x = POST || o.want_gate || (has_norm && !o.h);
  constexpr int kSums = Keep::kLdsSums ? 1 : NV;
  float ag[kSums][VW] = {}, aw[kSums][VW] = {};
  float ab[BIAS ? NV : 1][VW] = {}, apw[POST ? NV : 1][VW] = {}, apb[POST && BIAS ? NV : 1][VW] = {};
  float rw[kReg][VW], rgate[kReg][VW], rpw[kReg][VW], rpb[kReg][VW];
  // vector j of the gate's row (where several rows share it)
  auto set_gate = [&](int64_t at) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float f[VW];
      rn_param<T>(c, a.gate, a.pf32, at, j, 1.f, f);
      if constexpr (Keep::kLdsParams) {
        lgate.put(l, j, f);
      } else if constexpr (Keep::kRegParams) {
#pragma unroll
        for (int k = 0; k < VW; ++k) rgate[j][k] = f[k];
      }
    }
  };
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float f[VW];
    rn_param<T>(c, a.w, a.pf32, 0, j, 1.f, f);
    if constexpr (Keep::kRegParams) {
#pragma unroll
      for (int k = 0; k < VW; ++k) rw[j][k] = f[k];
    } else if constexpr (Keep::kLdsParams) {
      lw.put(l, j, f);
    }
    if constexpr (POST) {
      rn_param<T>(c, a.pw, a.pf32, 0, j, 1.f, f);
      if constexpr (Keep::kRegParams) {
#pragma unroll
        for (int k = 0; k < VW; ++k) rpw[j][k] = f[k];
      } else if constexpr (Keep::kLdsParams) {
        lpw.put(l, j, f);
      }
    }
    if constexpr (POST && BIAS) {
      rn_param<T>(c, a.pb, a.pf32, 0, j, 0.f, f);
      if constexpr (Keep::kRegParams) {
#pragma unroll
        for (int k = 0; k < VW; ++k) rpb[j][k] = f[k];
      } else if constexpr (Keep::kLdsParams) {
        lpb.put(l, j, f);
      }
    }
    if constexpr (Keep::kLdsSums) {
      const float zero[VW] = {};
      lw.put(l, j, zero);
      lgate.put(l, j, zero);
    }
  }
  if (!a.gate) set_gate(0);  // ones

  // vector j of a parameter: every thread reads back what it has kept itself
  auto get = [&](const float (&reg)[kReg][VW], const Lds& lds_at, const void* p, int64_t at, int j, float fill,
                 float (&f)[VW]) {
    if constexpr (Keep::kRegParams) {
#pragma unroll
      for (int k = 0; k < VW; ++k) f[k] = reg[j][k];
    } else if constexpr (Keep::kLdsParams) {
      lds_at.get(l, j, f);
    } else {
      rn_param<T>(c, p, a.pf32, at, j, fill, f);
    }
  };

  // Adds a column sum over the workgroup's groups of rows and hands each
  // thread of the first group its columns' totals.
  auto folded = [&](const auto& s, const Lds& at, auto&& put) {
    if constexpr (sizeof(s) < sizeof(float) * NV * VW) {  // kept in LDS, by each thread its own
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float t[VW];
        at.get(l, j, t);
        put(j, t);
      }
    } else if constexpr (ROWS == 1) {
#pragma unroll
      for (int j = 0; j < NV; ++j) put(j, s[j]);
    } else {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VW; ++k) fold[grp * (G * EPT) + (l + j * G) * VW + k] = s[j][k];
      __syncthreads();
      if (grp == 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int first = (l + j * G) * VW;
          float t[VW];
#pragma unroll
          for (int k = 0; k < VW; ++k) t[k] = s[j][k];
#pragma unroll 1
          for (int g = 1; g < ROWS; ++g) {
#pragma unroll
            for (int k = 0; k < VW; ++k) t[k] += fold[g * (G * EPT) + first + k];
          }
          put(j, t);
        }
      }
    }
  };
  float* part = o.part + (int64_t)blockIdx.x * o.sums * a.width;

  // h alone in the place of x and residual: the same sum with factors 1 and 0
  const R* r_rows = static_cast<const R*>(o.h ? o.h : a.res);
  const int64_t r_stride = o.h ? (int64_t)a.width : a.res_stride;
  const float r_scale = o.h ? 1.f : a.scale;
  RnRaw<T, R, NV, VW> q;
  // What a row does not have, or a group without a row, is zeros.
  auto request = [&](int64_t row, bool active) {
    q.st = active && o.stats ? o.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      q.x[j] = c.template load<true>(static_cast<const T*>(a.x) + row * a.x_stride, j, active && need_x);
      q.r[j] = c.template load<true>(r_rows + row * r_stride, j, active && has_norm);
      q.gy[j] = c.template load<true>(static_cast<const T*>(o.gy) + row * a.width, j, active && has_norm);
      q.gh[j] = c.template load<true>(static_cast<const R*>(o.gh) + row * a.width, j, active && o.gh);
    }
  };

  int parity = 0;
  const int64_t sec0 = (int64_t)(blockIdx.x / (uint32_t)o.cuts) * o.per;
  const int64_t sec1 = sec0 + o.per < o.sections ? sec0 + o.per : o.sections;
  for (int64_t sec = sec0; sec < sec1; ++sec) {
    const int64_t r0 = sec * o.section + (int64_t)(blockIdx.x % (uint32_t)o.cuts) * o.run;
    const int64_t end = (sec + 1) * o.section < a.rows ? (sec + 1) * o.section : a.rows;
    const int64_t r1 = r0 + o.run < end ? r0 + o.run : end;
    const int64_t gate_at = a.gate ? (int64_t)((uint32_t)r0 / a.period) * a.width : 0;
    if (a.gate && a.period != 1) set_gate(gate_at);
    if constexpr (Keep::kAhead) request(r0 + grp, r0 + grp < r1);
    for (int64_t base = r0; base < r1; base += ROWS, parity ^= 1) {
      c.renew();
      const int64_t row = base + grp;
      const bool active = ROWS == 1 || row < r1;  // no row: zeros are added and nothing is stored
      if constexpr (!Keep::kAhead) request(row, active);
      const bool own_gate = a.gate && a.period == 1;
      auto gate_of = [&](int j, float (&f)[VW]) {
        if (own_gate) rn_param<T>(c, a.gate, a.pf32, row * a.width, j, 1.f, f, active);
        else get(rgate, lgate, a.gate, gate_at, j, 1.f, f);
      };
      const float4 st = q.st;
      // The row as floats: kept while the next row is on its way into q, or
      // (kAhead false, registers for one of the two) formed from q each time.
      constexpr int kRow = Keep::kAhead ? NV : 1;
      float xs[kRow][VW], ns[kRow][VW], das[kRow][VW], dH[NV][VW], s[2] = {0.f, 0.f};
      auto normalised_x = [&](int j, float (&x)[VW]) {
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          x[k] = row_elem<T, VW>(q.x[j], k);
          if constexpr (POST) x[k] = (x[k] - st.x) * st.y;
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
      // u from the normalised x
      auto post_out = [&](int j, const float (&x)[VW], float (&u)[VW]) {
        float pw[VW], pb[VW];
        if constexpr (POST) get(rpw, lpw, a.pw, 0, j, 1.f, pw);
        if constexpr (POST && BIAS) get(rpb, lpb, a.pb, 0, j, 0.f, pb);
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          u[k] = x[k];
          if constexpr (POST && BIAS) u[k] = fmaf(u[k], pw[k], pb[k]);
          else if constexpr (POST) u[k] *= pw[k];
        }
      };
      // n = (h - mean) rstd and a = dy w of vector j
      auto normalised_h = [&](int j, float (&n)[VW], float (&da)[VW], float (&dy)[VW]) {
        float x[VW], u[VW], w[VW], gate[VW];
        x_of(j, x);
        post_out(j, x, u);
        gate_of(j, gate);
        get(rw, lw, a.w, 0, j, 1.f, w);
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          const float h = fmaf(r_scale, row_elem<R, VW>(q.r[j], k), u[k] * gate[k]);
          dy[k] = row_elem<T, VW>(q.gy[j], k);
          n[k] = (h - st.z) * st.w;
          da[k] = dy[k] * w[k];
        }
      };
      if constexpr (Keep::kAhead) {
#pragma unroll
        for (int j = 0; j < NV; ++j) normalised_x(j, xs[j]);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int k = 0; k < VW; ++k) dH[j][k] = row_elem<R, VW>(q.gh[j], k);
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
            if constexpr (BIAS) ab[j][k] += dy[k];
            if constexpr (Keep::kAhead) {
              ns[j][k] = n[k];
              das[j][k] = da[k];
            }
          }
          if constexpr (Keep::kLdsSums) lw.put(l, j, sum);
          c.each(j, [&](int k) {
            s[0] += da[k];
            s[1] = fmaf(da[k], n[k], s[1]);
          });
        }
        if constexpr (Keep::kAhead) {
          if (base + ROWS < r1) request(row + ROWS, row + ROWS < r1);
        }
        group_sum<G>(s, lds[parity][0]);
        if constexpr (!Keep::kAhead) q.hide(), c.renew();
        const float c0 = a.norm == kLayer ? s[0] * a.inv_width : 0.f, c1 = s[1] * a.inv_width;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if constexpr (Keep::kAhead) {
#pragma unroll
            for (int k = 0; k < VW; ++k) dH[j][k] = fmaf(st.w, fmaf(-ns[j][k], c1, das[j][k] - c0), dH[j][k]);
          } else {
            float n[VW], da[VW], dy[VW];
            normalised_h(j, n, da, dy);
#pragma unroll
            for (int k = 0; k < VW; ++k)
              dH[j][k] = fmaf(st.w, fmaf(-n[k], c1, da[k] - c0), row_elem<R, VW>(q.gh[j], k));
          }
        }
      } else if constexpr (Keep::kAhead) {
        if (base + ROWS < r1) request(row + ROWS, row + ROWS < r1);
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
      if (o.want_gate) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float x[VW], u[VW], sum[VW];
          x_of(j, x);
          post_out(j, x, u);
          if (o.want_gate == 2) {
#pragma unroll
            for (int k = 0; k < VW; ++k) u[k] *= dH[j][k];
            rn_param_store<T>(c, o.ggate, a.pf32, row * a.width, j, u, active);
          } else if constexpr (Keep::kLdsSums) {
            lgate.get(l, j, sum);
#pragma unroll
            for (int k = 0; k < VW; ++k) sum[k] = fmaf(u[k], dH[j][k], sum[k]);
            lgate.put(l, j, sum);
          } else {
#pragma unroll
            for (int k = 0; k < VW; ++k) ag[j][k] = fmaf(u[k], dH[j][k], ag[j][k]);
          }
        }
      }
      s[0] = s[1] = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float x[VW], gate[VW], pw[VW];
        gate_of(j, gate);
        if constexpr (POST) {
          x_of(j, x);
          get(rpw, lpw, a.pw, 0, j, 1.f, pw);
        }
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          dH[j][k] *= gate[k];  // du from here on
          if constexpr (POST) {
            apw[j][k] = fmaf(dH[j][k], x[k], apw[j][k]);
            if constexpr (BIAS) apb[j][k] += dH[j][k];
            dH[j][k] *= pw[k];
          }
        }
        if constexpr (POST)
          c.each(j, [&](int k) {
            s[0] += dH[j][k];
            s[1] = fmaf(dH[j][k], x[k], s[1]);
          });
      }
      if constexpr (POST) {
        group_sum<G>(s, lds[parity][1]);
        if constexpr (!Keep::kAhead) q.hide(), c.renew();
        const float c0 = a.post == kLayer ? s[0] * a.inv_width : 0.f, c1 = s[1] * a.inv_width;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float x[VW];
          x_of(j, x);
#pragma unroll
          for (int k = 0; k < VW; ++k) dH[j][k] = st.y * fmaf(-x[k], c1, dH[j][k] - c0);
        }
      }
      if (o.gx) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          c.store(static_cast<T*>(o.gx) + row * a.width, j, dH[j], active);
      }
    }
    if (o.want_gate == 1) {
      folded(ag, lgate, [&](int j, const float (&t)[VW]) {
        if (o.cuts > 1) c.store(part, j, t);
        else rn_param_store<T>(c, o.ggate, a.pf32, sec * a.width, j, t);
      });
#pragma unroll
      for (int j = 0; j < kSums; ++j)
#pragma unroll
        for (int k = 0; k < VW; ++k) ag[j][k] = 0.f;
      if constexpr (Keep::kLdsSums) {
        const float zero[VW] = {};
#pragma unroll
        for (int j = 0; j < NV; ++j) lgate.put(l, j, zero);
      }
    }
  }
  if (o.want_gate == 1 && o.cuts > 1) part += a.width;
  auto put = [&](int want, const auto& s, const Lds& at) {
    if (!want) return;
    folded(s, at, [&](int j, const float (&t)[VW]) { c.store(part, j, t); });
    part += a.width;
  };
  if constexpr (POST) put(o.want_pw, apw, Lds{nullptr});
  if constexpr (POST && BIAS) put(o.want_pb, apb, Lds{nullptr});
  put(o.want_w, aw, lw);
  if constexpr (BIAS) put(o.want_b, ab, Lds{nullptr});
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

// The threads a row and the elements a thread: the fewest threads that hold the row.
template <typename F> int rn_shape(int64_t width, F&& go) {
  using std::integral_constant;
  using E8 = integral_constant<int, 8>;
  if (width <= 128) return go(integral_constant<int, 16>{}, E8{});
  if (width <= 512) return go(integral_constant<int, 64>{}, E8{});
  if (width <= 2048) return go(integral_constant<int, 256>{}, E8{});
  if (width <= 4096) return go(integral_constant<int, 512>{}, E8{});
  if (width <= 8192) return go(integral_constant<int, 1024>{}, E8{});
  return go(integral_constant<int, 1024>{}, integral_constant<int, 16>{});
}
// The same for the backward, whose threads need more registers: 512 threads up
// to 8192 elements.
template <typename F> int rn_bwd_shape(int64_t width, F&& go) {
  if (width > 4096 && width <= 8192)
    return go(std::integral_constant<int, 512>{}, std::integral_constant<int, 16>{});
  return rn_shape(width, [&](auto G, auto E) -> int {
    if constexpr (G.value == 1024 && E.value == 8) return SUPA_AMD_EINVAL;  // taken above
    else return go(G, E);
  });
}

template <typename F> int rn_types(int dtype, int residual, F&& go) {
  switch (dtype) {
    case SUPA_AMD_F32: return go((float*)nullptr, (float*)nullptr);
    case SUPA_AMD_BF16:
      return residual == SUPA_AMD_F32 ? go((bf16*)nullptr, (float*)nullptr) : go((bf16*)nullptr, (bf16*)nullptr);
    default: return residual == SUPA_AMD_F32 ? go((f16*)nullptr, (float*)nullptr) : go((f16*)nullptr, (f16*)nullptr);
  }
}

int rn_check(const supa_amd_residual_norm_desc* d) {
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

RnArgs rn_args(const supa_amd_residual_norm_desc& d) {
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

// How the backward's rows are shared out; only the sizes decide.
struct RnPlan {
  int64_t section, sections, run;
  int32_t cuts, per, parts;
  bool elementwise;  // a gate row a row
};
RnPlan rn_plan(const supa_amd_residual_norm_desc& d) {
  RnPlan p{};
  int64_t at_once = 1;
  rn_bwd_shape(d.width, [&](auto G, auto) {
    at_once = rn_bwd_block(G.value) / G.value;
    return 0;
  });
  p.elementwise = d.gate && d.gate_period == 1 && d.rows > 1;
  p.section = d.gate && !p.elementwise ? d.gate_period : d.rows;
  p.sections = d.rows / p.section;
  const int64_t steps = (p.section + at_once - 1) / at_once;
  const int64_t cuts = std::min<int64_t>(steps, (kRnParts + p.sections - 1) / p.sections);
  const int64_t run = (steps + cuts - 1) / cuts;
  p.run = run * at_once;
  p.cuts = (int32_t)((steps + run - 1) / run);
  p.per = p.cuts > 1 ? 1 : (int32_t)((p.sections + kRnParts - 1) / kRnParts);
  p.parts = p.cuts > 1 ? (int32_t)(p.sections * p.cuts) : (int32_t)((p.sections + p.per - 1) / p.per);
  return p;
}

}  // namespace sa

using namespace sa;

extern "C" {

int supa_amd_residual_norm_forward(const supa_amd_residual_norm_desc* d, void* h, void* y, float* stats, void* stream) {
  const int rc = rn_check(d);
  if (rc) return rc;
  if (d->rows == 0) return SUPA_AMD_OK;
  if (!d->x || !d->residual || !h || (d->norm != SUPA_AMD_NORM_NONE) != (y != nullptr)) return SUPA_AMD_EINVAL;
  const RnArgs a = rn_args(*d);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return rn_types(d->dtype, d->residual_dtype, [&](auto* t, auto* r) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    using R = std::remove_pointer_t<decltype(r)>;
    return rn_shape(d->width, [&](auto G, auto E) -> int {
      constexpr int BS = G.value > 256 ? G.value : 256, PER = BS / G.value;
      constexpr int64_t kSlab = (int64_t(1) << 31) / BS * PER;  // HIP: fewer than 2^32 threads a launch
      for (int64_t r0 = 0; r0 < d->rows; r0 += kSlab) {
        RnArgs s = a;
        s.row0 = r0;
        s.rows = std::min(d->rows, r0 + kSlab);
        k_residual_norm<T, R, G.value, E.value><<<(unsigned)((s.rows - r0 + PER - 1) / PER), BS, 0, st>>>(
            s, static_cast<R*>(h), static_cast<T*>(y), reinterpret_cast<float4*>(stats));
        const int rl = launch_status();
        if (rl) return rl;
      }
      return SUPA_AMD_OK;
    });
  });
}

int64_t supa_amd_residual_norm_backward_workspace_bytes(const supa_amd_residual_norm_desc* d) {
  const int rc = rn_check(d);
  if (rc) return rc;
  if (d->rows == 0) return 0;
  return (int64_t)rn_plan(*d).parts * 5 * d->width * 4;
}

int supa_amd_residual_norm_backward(const supa_amd_residual_norm_desc* d, const void* h, const void* grad_h,
                                    const void* grad_y, const float* stats, void* grad_x, void* grad_residual,
                                    void* grad_gate, void* grad_post_weight, void* grad_post_bias, void* grad_weight,
                                    void* grad_bias, void* workspace, int64_t ws_bytes, void* stream) {
  const int rc = rn_check(d);
  if (rc) return rc;
  if (d->rows == 0) return SUPA_AMD_EINVAL;  // the caller's zeros
  const bool post = d->post_norm != SUPA_AMD_NORM_NONE, norm = d->norm != SUPA_AMD_NORM_NONE;
  if ((post || d->gate) && h) return SUPA_AMD_EINVAL;
  if ((post || grad_gate || (norm && !h)) && !d->x) return SUPA_AMD_EINVAL;
  if (norm && !h && !d->residual) return SUPA_AMD_EINVAL;
  if ((post || norm) && !stats) return SUPA_AMD_EINVAL;
  if ((!d->gate && grad_gate) || (!post && (grad_post_weight || grad_post_bias)) || (!norm && (grad_weight || grad_bias)))
    return SUPA_AMD_EINVAL;
  const int64_t need = supa_amd_residual_norm_backward_workspace_bytes(d);
  if (!workspace || ws_bytes < need) return SUPA_AMD_EWORKSPACE;
  const RnArgs a = rn_args(*d);
  const RnPlan p = rn_plan(*d);
  RnGrads o{};
  o.h = h;
  o.gh = grad_h;
  o.gy = norm ? grad_y : nullptr;
  o.stats = reinterpret_cast<const float4*>(stats);
  o.gx = grad_x;
  o.gres = grad_residual;
  o.ggate = grad_gate;
  o.part = static_cast<float*>(workspace);
  o.section = p.section;
  o.sections = p.sections;
  o.run = p.run;
  o.cuts = p.cuts;
  o.per = p.per;
  o.want_gate = !grad_gate ? 0 : p.elementwise ? 2 : 1;
  o.want_pw = grad_post_weight != nullptr;
  o.want_pb = grad_post_bias != nullptr;
  o.want_w = grad_weight != nullptr;
  o.want_b = grad_bias != nullptr;
  const int gate_sums = o.want_gate == 1 && p.cuts > 1 ? 1 : 0;
  o.sums = gate_sums + o.want_pw + o.want_pb + o.want_w + o.want_b;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return rn_types(d->dtype, d->residual_dtype, [&](auto* t, auto* r) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    using R = std::remove_pointer_t<decltype(r)>;
    const int rl = rn_bwd_shape(d->width, [&](auto G, auto E) -> int {
      auto go = [&](auto post_c, auto bias_c) -> int {
        constexpr auto kernel = k_residual_norm_backward<T, R, G.value, E.value, post_c.value, bias_c.value>;
        constexpr int lds = RnKeep<G.value, E.value>::bytes(post_c.value, bias_c.value);
        if constexpr (lds > 0) {  // past the 64 KiB that a launch has without asking
          static const hipError_t allowed = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                                hipFuncAttributeMaxDynamicSharedMemorySize, lds);
          if (allowed != hipSuccess) return (int)allowed;
        }
        kernel<<<(unsigned)p.parts, rn_bwd_block(G.value), lds, st>>>(a, o);
        return launch_status();
      };
      using std::bool_constant;
      const bool bias = d->post_bias || d->bias || grad_post_bias || grad_bias;
      if (post) return bias ? go(bool_constant<true>{}, bool_constant<true>{}) : go(bool_constant<true>{}, bool_constant<false>{});
      return bias ? go(bool_constant<false>{}, bool_constant<true>{}) : go(bool_constant<false>{}, bool_constant<false>{});
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
  });
}

}  // extern "C"

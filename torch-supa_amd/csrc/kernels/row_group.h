// Rows held in the registers of a group of threads: G threads (16, a
// wavefront, or several) share a row, thread l holding the vectors l, l + G, ...
// of VW elements, at any element alignment.
#pragma once

#include "softmax_common.h"

namespace sa {

// VW elements of S as loaded.
template <typename S, int VW> struct RowVec {
  uint4 q[VW * sizeof(S) / 16];
};

// Elements [col, col + VW) of a row of `width`; zeros past its end.
template <bool STREAM, int VW, typename S>
__device__ __forceinline__ RowVec<S, VW> row_load(const S* __restrict__ row, int col, int width) {
  RowVec<S, VW> r;
  constexpr int W = (int)(sizeof(r.q) / 16);
  if (col + VW <= width) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const char* p = reinterpret_cast<const char*>(row + col) + 16 * i;
      r.q[i] = STREAM ? ld_any_stream(p) : ld_any(p);
    }
  } else {
    S e[VW];
#pragma unroll
    for (int k = 0; k < VW; ++k) e[k] = col + k < width ? row[col + k] : S{};
    __builtin_memcpy(&r, e, sizeof(r));
  }
  return r;
}
template <typename S, int VW> __device__ __forceinline__ float row_elem(const RowVec<S, VW>& r, int k) {
  constexpr int per = 16 / (int)sizeof(S);
  return elem_f<S>(r.q[k / per], k % per);
}
template <typename S, int VW>
__device__ __forceinline__ void row_store(S* __restrict__ row, int col, int width, const float (&f)[VW]) {
  if (col + VW <= width) {
    store_any<S, VW>(row + col, f);
  } else {
#pragma unroll
    for (int k = 0; k < VW; ++k)
      if (col + k < width) row[col + k] = from_arith<S>(f[k]);
  }
}

// Where a thread's NV vectors lie in a row of `width` elements, the same for
// every row.  The vector that would run past the row's end is moved back
// to it: it computes and stores some elements a second time, with the values
// that the vector before has for them; sums along the row leave them out, and
// what is read, changed and written back has to.  So every access is a whole
// vector, and one instruction; a row narrower than a vector, in groups of 16,
// goes element by element.
template <int G, int NV, int VW> struct RowSlots {
  static constexpr bool kWhole = G > 16;  // callers use them for rows of more than 16 vectors
  uint32_t col[NV];
  int32_t skip[NV];  // elements that another vector holds; VW: no vector here
  int32_t width;

  __device__ __forceinline__ RowSlots(int l, int w) : width(w) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (l + j * G) * VW;
      const int past = c + VW - w;
      col[j] = (uint32_t)c;
      skip[j] = 0;
      if constexpr (kWhole) {
        if (past > 0) {
          skip[j] = past < VW ? past : VW;
          col[j] = past < VW ? (uint32_t)(w - VW) : 0u;
        }
      }
    }
  }
  // At the top of a loop over rows: keeps the compiler from forming every
  // operand's 64-bit addresses ahead of the loop (and spilling them), where a
  // scalar row address and these 32-bit offsets do.
  __device__ __forceinline__ void renew() {
#pragma unroll
    for (int j = 0; j < NV; ++j) asm volatile("" : "+v"(col[j]));
  }
  // Vector j is there and all its elements are its own.
  __device__ __forceinline__ bool whole(int j) const { return kWhole && skip[j] == 0; }
  __device__ __forceinline__ bool live(int j) const { return !kWhole || skip[j] < VW; }
  // f(k) for the elements of vector j that are the row's and no other vector's.
  // The vector that was moved back is one thread's, and takes a branch of its own.
  template <typename F> __device__ __forceinline__ void each(int j, F&& f) const {
    if constexpr (kWhole) {
      if (skip[j] == 0) {
#pragma unroll
        for (int k = 0; k < VW; ++k) f(k);
      } else if (skip[j] < VW) {
#pragma unroll
        for (int k = 0; k < VW; ++k)
          if (k >= skip[j]) f(k);
      }
    } else {
#pragma unroll
      for (int k = 0; k < VW; ++k)
        if ((int)col[j] + k < width) f(k);
    }
  }
  // Vector j of the row at p; zeros where there is none.
  template <bool STREAM, typename S>
  __device__ __forceinline__ RowVec<S, VW> load(const S* __restrict__ p, int j, bool on = true) const {
    if constexpr (kWhole) {
      RowVec<S, VW> r{};
      if (on && live(j)) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(r.q) / 16); ++i) {
          const char* at = reinterpret_cast<const char*>(p) + (col[j] * (uint32_t)sizeof(S) + 16u * i);
          r.q[i] = STREAM ? ld_any_stream(at) : ld_any(at);
        }
      }
      return r;
    } else {
      return row_load<STREAM, VW>(p, (int)col[j], on ? width : 0);
    }
  }
  template <typename S>
  __device__ __forceinline__ void store(S* __restrict__ p, int j, const float (&f)[VW], bool on = true) const {
    if constexpr (kWhole) {
      if (on && live(j))
        store_any<S, VW>(reinterpret_cast<S*>(reinterpret_cast<char*>(p) + col[j] * (uint32_t)sizeof(S)), f);
    } else {
      row_store<S, VW>(p, (int)col[j], on ? width : 0, f);
    }
  }
};

// Sums over 16 lanes by four lane permutations within the row of 16, in every
// lane: neighbours, pairs, then the two mirrors (a mirror pairs lanes that
// hold different halves' sums, as an exchange across 4 and 8 lanes would).
__device__ __forceinline__ float sum16(float v) {
  auto perm = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v += perm(v, std::integral_constant<int, 0xB1>{});   // quad_perm [1, 0, 3, 2]
  v += perm(v, std::integral_constant<int, 0x4E>{});   // quad_perm [2, 3, 0, 1]
  v += perm(v, std::integral_constant<int, 0x141>{});  // row_half_mirror
  v += perm(v, std::integral_constant<int, 0x140>{});  // row_mirror
  return v;
}
__device__ __forceinline__ float sum64(float v) {
  v = sum16(v);
  auto lane = [&](int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); };
  return (lane(0) + lane(16)) + (lane(32) + lane(48));
}

// Sums of N values over the G threads of a row, in every one of them.  lds
// holds N floats for each wavefront of the workgroup; every thread of the
// workgroup makes the call.  One barrier: a caller that comes back to the
// same lds has passed another barrier since.
template <int G, int N> __device__ __forceinline__ void group_sum(float (&v)[N], float* lds) {
  if constexpr (G == 16) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = sum16(v[i]);
  } else if constexpr (G == 32) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = sum16(v[i]);
      v[i] += __shfl_xor(v[i], 16, 64);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = sum64(v[i]);
    if constexpr (G > 64) {
      constexpr int W = G / 64;
      const int wave = threadIdx.x >> 6, first = wave / W * W;
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) lds[wave * N + i] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = lds[first * N + i];
#pragma unroll
      for (int w = 1; w < W; ++w) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += lds[(first + w) * N + i];
      }
    }
  }
}

}  // namespace sa

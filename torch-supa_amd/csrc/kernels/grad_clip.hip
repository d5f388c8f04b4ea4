// The norm of a list of tensors together, and their scaling to a largest norm:
// what clip_grad_norm_ does to a model's gradients before the optimizer step.
//
// HBM-bound: a read of every gradient, then, where the norm exceeds the limit, a
// read and a write (a factor of 1 ends a workgroup before it reads anything).
// The tensors travel in the kernel arguments (mta.h); a workgroup reduces one
// chunk to a partial in float64 -- no square of a float32 overflows or
// underflows there, and a sum over 10^9 terms keeps its digits -- and the
// partials are added in an order of their own, so the norm does not depend on
// timing: by one workgroup in a launch between, or, where they are few, by every
// workgroup of the scaling for itself (24 matrices of 16384 elements: one launch
// of three, 3 us of 13).
//
// Measured on MI355X: 1.2 GB of float32 in 54 tensors 575 us clipped (170 for
// the norm, 7.1 TB/s; 400 for the scaling, 6.1) and 193 within the limit; 600 MB
// of bfloat16 275 and 100.  A tensor at no 16-byte address goes element by element
// (200 MB of bfloat16 within the limit: 86 us, at 16-byte addresses 37).
#include "mta.h"

namespace sa {

constexpr int kClipTensors = 128;  // tensors a launch; the table takes 2.9 KiB of kernel arguments
constexpr int kClipBlock = 256;
// 16-byte vectors a thread.  The norm reads long chunks (600 MB of bfloat16, 4
// vectors a thread 103 us, 16 98: fewer partials); the scaling's are shorter, all
// loads before the first store (1.2 GB, 4 vectors in turn 600 us in all, 8 loaded
// ahead 576), and long enough that a launch with nothing to scale ends soon (4:
// 200 us, 8: 193).
constexpr int kClipNormVecs = 16, kClipScaleVecs = 8;
constexpr int64_t kClipFold = 512;  // most partials that the scaling adds itself

// Tensors of every type share a table: the type, in the low bits of `sized`, is
// one for a workgroup (bfloat16 matrices beside float32 vectors: two launches of five
// less, 50 us -> 43).
struct ClipTable {
  void* p[kClipTensors];
  int64_t sized[kClipTensors];  // elements x 4 + clip_type
  uint32_t chunk_start[kClipTensors + 1];
  int32_t ntensors;
  uint32_t bucket_shift;
  MtaBucket bucket[kMtaBuckets];
};

template <typename T> constexpr int64_t clip_chunk(int vecs) { return (int64_t)kClipBlock * vecs * (16 / (int64_t)sizeof(T)); }

inline int clip_type(int dtype) {
  return dtype == SUPA_AMD_F32 ? 0 : dtype == SUPA_AMD_BF16 ? 1 : dtype == SUPA_AMD_F16 ? 2 : 3;
}

// fn(tensor, lo, hi) for the workgroup's chunk, with the tensor's type.
template <int VECS, typename F> __device__ __forceinline__ void clip_chunk_of(const ClipTable& tab, F&& fn) {
  const int k = find_tensor(tab, blockIdx.x);
  const int64_t c = blockIdx.x - tab.chunk_start[k], n = tab.sized[k] >> 2;
  auto go = [&](auto* x) {
    using T = std::remove_pointer_t<decltype(x)>;
    const int64_t lo = c * clip_chunk<T>(VECS);
    fn(x, lo, lo + clip_chunk<T>(VECS) < n ? lo + clip_chunk<T>(VECS) : n);
  };
  switch (tab.sized[k] & 3) {
    case 0: return go(static_cast<float*>(tab.p[k]));
    case 1: return go(static_cast<bf16*>(tab.p[k]));
    case 2: return go(static_cast<f16*>(tab.p[k]));
    default: return go(static_cast<double*>(tab.p[k]));
  }
}

constexpr int kOrdInf = 0;
template <int ORD> __device__ __forceinline__ double clip_term(double acc, double x) {
  if constexpr (ORD == 2) return fma(x, x, acc);
  else if constexpr (ORD == 1) return acc + fabs(x);
  else return (acc != acc || acc > fabs(x)) ? acc : fabs(x);  // NaN stays
}
template <int ORD> __device__ __forceinline__ double clip_join(double a, double b) {
  if constexpr (ORD == kOrdInf) return (a != a || a > b) ? a : b;
  else return a + b;
}
// Over the workgroup, in thread 0.
template <int ORD, int BS> __device__ __forceinline__ double clip_block(double v) {
  __shared__ double part[BS / 64];
  for (int off = 32; off > 0; off >>= 1) v = clip_join<ORD>(v, __shfl_xor(v, off, 64));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < BS / 64; ++w) v = clip_join<ORD>(v, part[w]);
  }
  return v;
}

template <int ORD>
__global__ void __launch_bounds__(kClipBlock) k_clip_partial(ClipTable tab, double* __restrict__ part) {
  double acc = 0.0;
  clip_chunk_of<kClipNormVecs>(tab, [&](auto* x, int64_t lo, int64_t hi) {
    using T = std::remove_pointer_t<decltype(x)>;
    constexpr int V = 16 / sizeof(T);
    int64_t start = lo;
    if (aligned(x, 16)) {
      const int64_t nv = (hi - lo) / V;
#pragma unroll 4
      for (int64_t v = threadIdx.x; v < nv; v += kClipBlock) {
        const Vec<T, V> w = ld_stream(reinterpret_cast<const Vec<T, V>*>(x + lo + v * V));
#pragma unroll
        for (int i = 0; i < V; ++i) acc = clip_term<ORD>(acc, (double)to_arith(w.v[i]));
      }
      start = lo + nv * V;
    }
    for (int64_t e = start + threadIdx.x; e < hi; e += kClipBlock) acc = clip_term<ORD>(acc, (double)to_arith(x[e]));
  });
  acc = clip_block<ORD, kClipBlock>(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

// The workgroup's sum of all partials, in thread 0, and the norm from it.
template <int ORD, int BS> __device__ __forceinline__ double clip_fold(const double* __restrict__ part, int64_t parts) {
  double acc = fold_strided<8>(
      0.0, (int64_t)threadIdx.x, BS, parts, [&](int64_t i) { return part[i]; },
      [](double a, double b) { return clip_join<ORD>(a, b); });
  acc = clip_block<ORD, BS>(acc);
  return ORD == 2 ? sqrt(acc) : acc;
}
__device__ __forceinline__ void clip_write(double norm, void* out, int out_f64) {
  if (out_f64) *static_cast<double*>(out) = norm;
  else *static_cast<float*>(out) = (float)norm;
}

// The norm of all partials, to ws[0] and to `out`.
constexpr int kClipFinal = 1024;
template <int ORD>
__global__ void __launch_bounds__(kClipFinal)
k_clip_norm(double* __restrict__ ws, int64_t parts, void* __restrict__ out, int out_f64) {
  const double norm = clip_fold<ORD, kClipFinal>(ws + 1, parts);
  if (threadIdx.x == 0) {
    ws[0] = norm;
    clip_write(norm, out, out_f64);
  }
}

// Where the scaling finds the norm: ws[0], or (parts > 0) in the partials, which it then
// adds itself; the workgroup that `out` is given to writes the norm there.
struct ClipNorm {
  const double* ws;
  int64_t parts;
  void* out;
  int out_f64;
};

constexpr int kOrdGiven = 3;  // the norm is in ws[0]
template <int ORD>
__global__ void __launch_bounds__(kClipBlock)
k_clip_scale(ClipTable tab, ClipNorm from, double max_norm) {
  double norm;
  if constexpr (ORD == kOrdGiven) {
    norm = from.ws[0];
  } else {
    __shared__ double shared;
    norm = clip_fold<ORD, kClipBlock>(from.ws + 1, from.parts);
    if (threadIdx.x == 0) {
      shared = norm;
      if (from.out && blockIdx.x == 0) clip_write(norm, from.out, from.out_f64);
    }
    __syncthreads();
    norm = shared;
  }
  const double q = max_norm / (norm + 1e-6);
  if (q >= 1.0) return;  // a NaN goes on
  clip_chunk_of<kClipScaleVecs>(tab, [&](auto* x, int64_t lo, int64_t hi) {
    using T = std::remove_pointer_t<decltype(x)>;
    using A = opmath_t<T>;
    constexpr int V = 16 / sizeof(T), U = kClipScaleVecs;
    const A c = (A)q;
    auto scaled = [&](Vec<T, V> w) {
#pragma unroll
      for (int i = 0; i < V; ++i) w.v[i] = from_arith<T>((A)to_arith(w.v[i]) * c);
      return w;
    };
    int64_t start = lo;
    if (aligned(x, 16)) {
      Vec<T, V>* at = reinterpret_cast<Vec<T, V>*>(x + lo) + threadIdx.x;
      if (hi - lo == clip_chunk<T>(U)) {
        Vec<T, V> w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = ld_stream(at + u * kClipBlock);
#pragma unroll
        for (int u = 0; u < U; ++u) st_stream(at + u * kClipBlock, scaled(w[u]));
        return;
      }
      const int64_t nv = (hi - lo) / V;
      for (int64_t v = threadIdx.x; v < nv; v += kClipBlock, at += kClipBlock) st_stream(at, scaled(ld_stream(at)));
      start = lo + nv * V;
    }
    for (int64_t e = start + threadIdx.x; e < hi; e += kClipBlock) x[e] = from_arith<T>((A)to_arith(x[e]) * c);
  });
}

// Chunks of a tensor, of `vecs` vectors a thread.
inline int64_t clip_chunks(int64_t numel, int dtype, int vecs) {
  const int64_t chunk = (int64_t)kClipBlock * vecs * (16 / dtype_size(dtype));
  return (numel + chunk - 1) / chunk;
}

// Calls fn(tab, chunks) for tables of at most kClipTensors tensors; empty
// tensors are left out.
template <typename F>
int clip_tables(int vecs, int32_t n, void* const* p, const int64_t* numel, const int32_t* dtypes, F&& fn) {
  int i = 0;
  while (i < n) {
    ClipTable tab{};
    int64_t chunks = 0;
    int nt = 0;
    for (; i < n && nt < kClipTensors; ++i) {
      const int64_t c = clip_chunks(numel[i], dtypes[i], vecs);
      if (c == 0) continue;
      if (c >= (int64_t(1) << 24)) return SUPA_AMD_ELAYOUT;
      if (chunks + c >= (int64_t(1) << 24)) break;  // HIP: fewer than 2^32 threads a launch
      tab.p[nt] = p[i];
      tab.sized[nt] = numel[i] * 4 + clip_type(dtypes[i]);
      tab.chunk_start[nt++] = (uint32_t)chunks;
      chunks += c;
    }
    if (nt == 0) continue;
    tab.chunk_start[nt] = (uint32_t)chunks;
    tab.ntensors = nt;
    mta_index(tab, (uint32_t)chunks);
    const int rc = fn(tab, (uint32_t)chunks);
    if (rc) return rc;
  }
  return SUPA_AMD_OK;
}

int clip_check(int32_t n, const void* const* p, const int64_t* numel, const int32_t* dtypes) {
  if (n < 0 || (n > 0 && (!p || !numel || !dtypes))) return SUPA_AMD_EINVAL;
  for (int32_t i = 0; i < n; ++i) {
    if (numel[i] < 0 || (numel[i] > 0 && !p[i])) return SUPA_AMD_EINVAL;
    if (!dtype_is_floating(dtypes[i])) return SUPA_AMD_EDTYPE;
  }
  return SUPA_AMD_OK;
}

// The list and its workspace: the norm, then the partials.
struct ClipList {
  int32_t n;
  void* const* p;
  const int64_t* numel;
  const int32_t* dtypes;
  double* ws;
  hipStream_t st;
};

template <typename F> int clip_ord(double ord, F&& go) {
  if (ord == 2.0) return go(std::integral_constant<int, 2>{});
  if (ord == 1.0) return go(std::integral_constant<int, 1>{});
  return go(std::integral_constant<int, kOrdInf>{});
}

template <int ORD> int clip_partials(const ClipList& l, int64_t& parts) {
  parts = 0;
  return clip_tables(kClipNormVecs, l.n, l.p, l.numel, l.dtypes, [&](const ClipTable& tab, uint32_t chunks) -> int {
    k_clip_partial<ORD><<<chunks, kClipBlock, 0, l.st>>>(tab, l.ws + 1 + parts);
    parts += chunks;
    return launch_status();
  });
}

template <int ORD> int clip_norm(const ClipList& l, int64_t parts, void* out, int32_t out_dtype) {
  k_clip_norm<ORD><<<1, kClipFinal, 0, l.st>>>(l.ws, parts, out, out_dtype == SUPA_AMD_F64);
  return launch_status();
}

template <int ORD> int clip_scale(const ClipList& l, ClipNorm from, double max_norm) {
  return clip_tables(kClipScaleVecs, l.n, l.p, l.numel, l.dtypes, [&](const ClipTable& tab, uint32_t chunks) -> int {
    k_clip_scale<ORD><<<chunks, kClipBlock, 0, l.st>>>(tab, from, max_norm);
    from.out = nullptr;  // the first launch writes it
    return launch_status();
  });
}

// The checks that the norm's entry points share.
int clip_norm_check(int32_t n, const void* const* tensors, const int64_t* numel, const int32_t* dtypes, double ord,
                    const void* norm_out, int32_t norm_dtype, const void* workspace, int64_t ws_bytes) {
  const int rc = clip_check(n, tensors, numel, dtypes);
  if (rc) return rc;
  if (!aligned(workspace, 8)) return SUPA_AMD_EINVAL;
  if (!norm_out || (ord != 1.0 && ord != 2.0 && ord != HUGE_VAL)) return SUPA_AMD_EINVAL;
  if (norm_dtype != SUPA_AMD_F32 && norm_dtype != SUPA_AMD_F64) return SUPA_AMD_EDTYPE;
  const int64_t need = supa_amd_grad_norm_workspace_bytes(n, numel, dtypes);
  if (need < 0) return (int)need;
  return !workspace || ws_bytes < need ? SUPA_AMD_EWORKSPACE : SUPA_AMD_OK;
}

}  // namespace sa

using namespace sa;

extern "C" {

int64_t supa_amd_grad_norm_workspace_bytes(int32_t n, const int64_t* numel, const int32_t* dtypes) {
  if (n < 0 || (n > 0 && (!numel || !dtypes))) return SUPA_AMD_EINVAL;
  int64_t parts = 0;
  for (int32_t i = 0; i < n; ++i) {
    if (numel[i] < 0) return SUPA_AMD_EINVAL;
    if (!dtype_is_floating(dtypes[i])) return SUPA_AMD_EDTYPE;
    const int64_t c = clip_chunks(numel[i], dtypes[i], kClipNormVecs);
    if (c >= (int64_t(1) << 24)) return SUPA_AMD_ELAYOUT;
    parts += c;
  }
  return (1 + parts) * 8;
}

int supa_amd_grad_norm(int32_t n, const void* const* tensors, const int64_t* numel, const int32_t* dtypes, double ord,
                       void* norm_out, int32_t norm_dtype, void* workspace, int64_t ws_bytes, void* stream) {
  const int rc = clip_norm_check(n, tensors, numel, dtypes, ord, norm_out, norm_dtype, workspace, ws_bytes);
  if (rc) return rc;
  const ClipList l{n, const_cast<void* const*>(tensors), numel, dtypes, static_cast<double*>(workspace),
                   static_cast<hipStream_t>(stream)};
  return clip_ord(ord, [&](auto O) -> int {
    int64_t parts;
    const int r = clip_partials<O.value>(l, parts);
    return r ? r : clip_norm<O.value>(l, parts, norm_out, norm_dtype);
  });
}

int supa_amd_grad_scale(int32_t n, void* const* tensors, const int64_t* numel, const int32_t* dtypes, double max_norm,
                        const void* workspace, int64_t ws_bytes, void* stream) {
  const int rc = clip_check(n, tensors, numel, dtypes);
  if (rc) return rc;
  if (!(max_norm >= 0.0) || !aligned(workspace, 8)) return SUPA_AMD_EINVAL;
  if (!workspace || ws_bytes < 8) return SUPA_AMD_EWORKSPACE;
  const ClipList l{n, tensors, numel, dtypes, nullptr, static_cast<hipStream_t>(stream)};
  return clip_scale<kOrdGiven>(l, ClipNorm{static_cast<const double*>(workspace), 0, nullptr, 0}, max_norm);
}

int supa_amd_clip_grad_norm(int32_t n, void* const* tensors, const int64_t* numel, const int32_t* dtypes, double ord,
                            double max_norm, void* norm_out, int32_t norm_dtype, void* workspace, int64_t ws_bytes,
                            void* stream) {
  if (!(max_norm >= 0.0)) return SUPA_AMD_EINVAL;
  const int rc = clip_norm_check(n, tensors, numel, dtypes, ord, norm_out, norm_dtype, workspace, ws_bytes);
  if (rc) return rc;
  const ClipList l{n, tensors, numel, dtypes, static_cast<double*>(workspace), static_cast<hipStream_t>(stream)};
  return clip_ord(ord, [&](auto O) -> int {
    int64_t parts;
    int r = clip_partials<O.value>(l, parts);
    if (r) return r;
    if (parts > 0 && parts <= kClipFold)
      return clip_scale<O.value>(l, ClipNorm{l.ws, parts, norm_out, norm_dtype == SUPA_AMD_F64}, max_norm);
    r = clip_norm<O.value>(l, parts, norm_out, norm_dtype);
    return r ? r : clip_scale<kOrdGiven>(l, ClipNorm{l.ws, 0, nullptr, 0}, max_norm);
  });
}

}  // extern "C"

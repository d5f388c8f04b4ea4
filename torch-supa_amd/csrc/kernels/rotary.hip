// Rotary positions: the pairs of the first `rotary` elements of every head of q
// and k turned by position * frequency (times a scale), the rest copied; with
// the angles negated it is the gradient.
//
// HBM-bound: q and k are read and written once, together in one launch; the
// angles cost 20 bytes a token.  Every head of a token turns by the same
// angles, so a workgroup takes whole tokens: its threads form the sine and
// cosine of each angle once, in LDS, while the first vectors of q and k are on
// their way.  position * frequency is formed in 64 bits and reduced to a
// fraction of a turn there: a float32 angle is off by 0.03 rad at position
// 500 000.  The fraction, its sine and cosine and the rotation are float32.
#include "row_group.h"

namespace sa {

constexpr int kRotBlock = 512;       // most threads of a workgroup
constexpr int kRotMaxPairs = 512;    // most pairs a head
constexpr int kRotTable = 1024;      // angles a workgroup holds

struct RotTensor {
  const void* in;
  void* out;
  int64_t is[3], os[3];  // strides of batch, seq, heads
  int32_t heads;
  int32_t copy;          // the elements past `rotary` are copied
};

struct RotArgs {
  RotTensor t[2];
  const double* freq;
  const void* pos;
  int64_t ps[2], offset;
  int32_t first, tokens;   // the tokens [first, tokens)
  int32_t dim, rotary;
  int32_t per;             // tokens a workgroup
  int32_t slots;           // heads of q and k together
  int32_t turn_units;      // vectors (HALF: pairs of vectors) of a head's rotated part
  int32_t units;           // and with those of its copied part
  int32_t pos64, inverse;
  float scale;
  FastDiv seq, by_token, by_unit;  // token -> (batch, seq); thread's unit -> token, head, unit of the head
};

// One unit of a head: V elements of the rotated part (HALF: V pairs), or of the copied part.
template <typename T, bool HALF> struct RotUnit {
  static constexpr int V = 16 / (int)sizeof(T);
  const T* in;
  T* out;
  int col, part;  // first element; the part's end
  bool turn, live;
  RowVec<T, V> a, b;

  __device__ __forceinline__ void find(const RotArgs& g, uint32_t unit, int32_t token0) {
    uint32_t tk, rest, slot, u;
    g.by_token.divmod(unit, tk, rest);
    g.by_unit.divmod(rest, slot, u);
    const int64_t token = (int64_t)token0 + tk;
    live = (int)tk < g.per && token < g.tokens;
    const bool second = (int)slot >= g.t[0].heads;
    const RotTensor& t = g.t[second ? 1 : 0];
    const int64_t head = (int64_t)slot - (second ? g.t[0].heads : 0);
    turn = (int)u < g.turn_units;
    live = live && (turn || t.copy);
    uint32_t bi, si;
    g.seq.divmod((uint32_t)token, bi, si);
    in = static_cast<const T*>(t.in) + bi * t.is[0] + si * t.is[1] + head * t.is[2];
    out = static_cast<T*>(t.out) + bi * t.os[0] + si * t.os[1] + head * t.os[2];
    if (turn) {
      col = (int)u * V;
      part = HALF ? g.rotary / 2 : g.rotary;
    } else {
      col = g.rotary + ((int)u - g.turn_units) * V;
      part = g.dim;
    }
  }
  __device__ __forceinline__ void load(const RotArgs& g) {
    if (!live) return;
    a = row_load<true, V>(in, col, part);
    if (HALF && turn) b = row_load<true, V>(in + g.rotary / 2, col, part);
  }
  __device__ __forceinline__ void store(const RotArgs& g, const float2* cs) {
    if (!live) return;
    float f[V], h[V];
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = row_elem<T, V>(a, k);
    if (turn) {
      if constexpr (HALF) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float2 w = cs[col + k < part ? col + k : 0];
          const float y = row_elem<T, V>(b, k);
          h[k] = fmaf(y, w.x, f[k] * w.y);
          f[k] = fmaf(f[k], w.x, -(y * w.y));
        }
        row_store<T, V>(out + g.rotary / 2, col, part, h);
      } else {
#pragma unroll
        for (int k = 0; k < V; k += 2) {
          const float2 w = cs[col + k < part ? (col + k) / 2 : 0];
          const float x = f[k], y = f[k + 1];
          f[k] = fmaf(x, w.x, -(y * w.y));
          f[k + 1] = fmaf(y, w.x, x * w.y);
        }
      }
    }
    row_store<T, V>(out, col, part, f);
  }
};

template <typename T, bool HALF>
__global__ void __launch_bounds__(kRotBlock) k_rotary(RotArgs g) {
  __shared__ float2 cs[kRotTable];
  const int32_t token0 = g.first + (int32_t)blockIdx.x * g.per;
  const uint32_t all = (uint32_t)(g.per * g.slots * g.units);
  const int pairs = g.rotary / 2;
  RotUnit<T, HALF> w;
  uint32_t unit = threadIdx.x;
  if (unit < all) {
    w.find(g, unit, token0);
    w.load(g);
  }
  for (int i = threadIdx.x; i < g.per * pairs; i += blockDim.x) {
    const int tk = i / pairs;
    const int32_t token = token0 + tk;
    if (token < g.tokens) {
      uint32_t bi, si;
      g.seq.divmod((uint32_t)token, bi, si);
      int64_t p = si;
      if (g.pos) {
        const int64_t at = bi * g.ps[0] + si * g.ps[1];
        p = g.pos64 ? static_cast<const int64_t*>(g.pos)[at] : (int64_t)static_cast<const int32_t*>(g.pos)[at];
      }
      const double turns = (double)(p + g.offset) * g.freq[i - tk * pairs] * 0.15915494309189533577;
      float s, c;
      sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
      cs[i] = make_float2(g.scale * c, g.scale * (g.inverse ? -s : s));
    }
  }
  __syncthreads();
  for (; unit < all; ) {
    uint32_t tk, rest;
    g.by_token.divmod(unit, tk, rest);
    w.store(g, cs + tk * pairs);
    unit += blockDim.x;
    if (unit < all) {
      w.find(g, unit, token0);
      w.load(g);
    }
  }
}

template <typename T> int rot_launch(const supa_amd_rotary_desc& d, hipStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  RotArgs a{};
  const supa_amd_rotary_tensor* in[2] = {&d.q, &d.k};
  bool copies = false;
  int64_t slots = 0;
  for (int i = 0; i < 2; ++i) {
    RotTensor& t = a.t[i];
    if (!in[i]->in) continue;
    t.in = in[i]->in;
    t.out = in[i]->out;
    for (int k = 0; k < 3; ++k) {
      t.is[k] = in[i]->in_strides[k];
      t.os[k] = in[i]->out_strides[k];
    }
    t.heads = (int32_t)in[i]->heads;
    t.copy = t.in != t.out && d.rotary < d.dim;
    copies = copies || t.copy;
    slots += in[i]->heads;
  }
  if (slots == 0 || d.batch * d.seq == 0) return SUPA_AMD_OK;
  a.freq = d.frequencies;
  a.pos = d.positions;
  a.ps[0] = d.position_strides[0];
  a.ps[1] = d.position_strides[1];
  a.offset = d.offset;
  a.tokens = (int32_t)(d.batch * d.seq);
  a.dim = (int32_t)d.dim;
  a.rotary = (int32_t)d.rotary;
  a.slots = (int32_t)slots;
  const bool half = d.layout == SUPA_AMD_ROTARY_HALF;
  a.turn_units = (int32_t)(((half ? d.rotary / 2 : d.rotary) + V - 1) / V);
  a.units = a.turn_units + (copies ? (int32_t)((d.dim - d.rotary + V - 1) / V) : 0);
  a.pos64 = d.position_dtype == SUPA_AMD_I64;
  a.inverse = d.inverse;
  a.scale = (float)d.scale;
  const int64_t per_token = slots * a.units;
  if (per_token >= (int64_t(1) << 31)) return SUPA_AMD_ELAYOUT;
  // tokens of few heads share a workgroup of 256 threads; a token of many takes
  // up to 512 threads, as many rounds of them as it needs, evenly filled
  const int64_t fit = std::min<int64_t>(256 / per_token, kRotTable / (d.rotary / 2));
  a.per = (int32_t)std::max<int64_t>(1, std::min<int64_t>(fit, a.tokens));
  const int64_t all = a.per * per_token, rounds = (all + kRotBlock - 1) / kRotBlock;
  const int block = (int)((((all + rounds - 1) / rounds) + 63) / 64 * 64);
  a.seq = FastDiv((uint32_t)d.seq);
  a.by_token = FastDiv((uint32_t)per_token);
  a.by_unit = FastDiv((uint32_t)a.units);
  const int64_t slab = (int64_t(1) << 31) / kRotBlock * a.per;  // HIP: fewer than 2^32 threads a launch
  const int64_t tokens = a.tokens;
  for (int64_t first = 0; first < tokens; first += slab) {
    a.first = (int32_t)first;
    a.tokens = (int32_t)std::min(tokens, first + slab);
    const unsigned blocks = (unsigned)((a.tokens - first + a.per - 1) / a.per);
    if (half) k_rotary<T, true><<<blocks, block, 0, st>>>(a);
    else k_rotary<T, false><<<blocks, block, 0, st>>>(a);
    const int rc = launch_status();
    if (rc) return rc;
  }
  return SUPA_AMD_OK;
}

}  // namespace sa

using namespace sa;

extern "C" int supa_amd_rotary(const supa_amd_rotary_desc* d, void* stream) {
  if (!d || d->batch < 0 || d->seq < 0 || d->dim < 1 || d->rotary < 2 || d->rotary % 2 || d->rotary > d->dim)
    return SUPA_AMD_EINVAL;
  if (d->layout != SUPA_AMD_ROTARY_HALF && d->layout != SUPA_AMD_ROTARY_INTERLEAVED) return SUPA_AMD_EINVAL;
  if (d->position_dtype != SUPA_AMD_I64 && d->position_dtype != SUPA_AMD_I32) return SUPA_AMD_EDTYPE;
  if (!d->frequencies) return SUPA_AMD_EINVAL;
  for (const supa_amd_rotary_tensor* t : {&d->q, &d->k})
    if (t->in && (!t->out || t->heads < 0)) return SUPA_AMD_EINVAL;
  if (d->rotary > 2 * kRotMaxPairs || d->dim >= (int64_t(1) << 30) || d->q.heads >= (int64_t(1) << 30) ||
      d->k.heads >= (int64_t(1) << 30) ||
      (d->batch > 0 && d->seq >= (int64_t(1) << 31) / d->batch))
    return SUPA_AMD_ELAYOUT;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_float_storage(d->dtype, [&](auto* tag) -> int {
    return rot_launch<std::remove_pointer_t<decltype(tag)>>(*d, st);
  });
}

// Rotary positions: the pairs of the first `rotary` elements of every head of q
// and k turned by position * frequency (times a scale), the rest copied; with
// the angles negated it is the gradient.
//
// HBM-bound: q and k are read and written once, together in one launch; the
// angles cost 20 bytes a token.  Every head of a token turns by the same
// angles, so a workgroup takes a tile of tokens and heads: its threads form the
// sine and cosine of each angle once, in LDS, while the first vectors of q and k
// are on their way.  Where a token's heads are neighbours in memory the tile is
// all heads of one token (or of a few, if they are small); where a head's tokens
// are, it is a run of tokens of some heads, so that a workgroup reads and writes
// long pieces of memory and shares few lines with others.  position * frequency is formed in 64 bits and reduced there
// to whole quarter turns and the rest: a float32 angle is off by 0.03 rad at position
// 500 000.  The rest, its sine and cosine and the rotation are float32.
//
// Measured on MI355X: [1, 131072, 20, 128] bf16 206 us (6.5 TB/s; its 271
// instructions a wavefront and unit would take some 145 alone), [4, 2048, 40, 128]
// bf16 30 us (5.6 TB/s, launch included), float32 55 us (6.1 TB/s).
#include "row_group.h"

namespace sa {

constexpr int kRotBlock = 512;       // most threads of a workgroup
constexpr int kRotMaxPairs = 512;    // most pairs a head
constexpr int kRotTable = 1024;      // angles a workgroup holds
// Units that a thread has on their way at once: two where their rotation needs
// little else ([4, 2048, 40, 128] bf16 HALF: 31.5 us with one, 29.4 with two; INTERLEAVED
// the same with both).
constexpr int rot_units(bool half) { return half ? 2 : 1; }

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
  int32_t per, heads;      // tokens and heads (of q, then k) of a workgroup's tile
  int32_t slots;           // heads of q and k together
  int32_t head_major;      // a tile's vectors go head by head, not token by token
  int32_t turn_units;      // vectors (HALF: pairs of vectors) of a head's rotated part
  int32_t units;           // and with those of its copied part
  int32_t pos64, inverse;
  float scale;
  FastDiv seq, by_unit, by_inner;  // token -> (batch, seq); a thread's vector -> its place in a head, token and head
};

// One unit of a head: V elements of the rotated part (HALF: V pairs), or of the
// copied part.  A part's last vector is moved back to its end and does some
// elements twice, with the same values; in place, where another thread may have
// written them before, it goes element by element, as does a part shorter than a
// vector.
template <typename T, bool HALF, bool ONE, typename OFF> struct RotUnit {
  static constexpr int V = 16 / (int)sizeof(T);
  const T* in;
  T* out;
  int col, part;  // first element; the part's end
  int tk;         // token of the tile
  bool turn, live;
  RowVec<T, V> a, b;

  __device__ __forceinline__ void find(const RotArgs& g, uint32_t unit, int32_t token0, int32_t slot0) {
    uint32_t v, u;
    g.by_unit.divmod(unit, v, u);
    int32_t slot = slot0 + (int32_t)v;
    tk = 0;
    if constexpr (!ONE) {
      uint32_t outer, inner;
      g.by_inner.divmod(v, outer, inner);
      tk = (int)(g.head_major ? inner : outer);
      slot = slot0 + (int32_t)(g.head_major ? outer : inner);
    }
    const int64_t token = (int64_t)token0 + tk;
    const bool second = slot >= g.t[0].heads;
    // chosen value by value: an indexed pointer would not be known to be global memory
    auto of = [&](auto q, auto k) { return second ? k : q; };
    const RotTensor &q = g.t[0], &k = g.t[1];
    const OFF head = slot - (second ? q.heads : 0);
    auto step = [&](int64_t sq, int64_t sk) { return second ? (OFF)sk : (OFF)sq; };
    turn = (int)u < g.turn_units;
    live = token < g.tokens && slot < g.slots && (turn || of(q.copy, k.copy));
    uint32_t bi, si;
    g.seq.divmod((uint32_t)token, bi, si);
    const OFF ob = (OFF)bi, os = (OFF)si;
    OFF in_at, out_at;
    if constexpr (ONE) {  // the token is the workgroup's: scalar products
      in_at = of((OFF)(ob * (OFF)q.is[0] + os * (OFF)q.is[1]), (OFF)(ob * (OFF)k.is[0] + os * (OFF)k.is[1]));
      out_at = of((OFF)(ob * (OFF)q.os[0] + os * (OFF)q.os[1]), (OFF)(ob * (OFF)k.os[0] + os * (OFF)k.os[1]));
    } else {
      in_at = ob * step(q.is[0], k.is[0]) + os * step(q.is[1], k.is[1]);
      out_at = ob * step(q.os[0], k.os[0]) + os * step(q.os[1], k.os[1]);
    }
    in = static_cast<const T*>(of(q.in, k.in)) + (in_at + head * step(q.is[2], k.is[2]));
    out = static_cast<T*>(of(q.out, k.out)) + (out_at + head * step(q.os[2], k.os[2]));
    int first;
    if (turn) {
      first = 0;
      col = (int)u * V;
      part = HALF ? g.rotary / 2 : g.rotary;
    } else {
      first = g.rotary;
      col = g.rotary + ((int)u - g.turn_units) * V;
      part = g.dim;
    }
    if (col + V > part && part - first >= V && in != out) col = part - V;
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
    auto rotated = [&](auto whole) {
      // the angles of a whole vector are neighbours; past a part's end, any will do
      auto angle = [&](int pair, int e) { return cs[whole.value || e < part ? pair : 0]; };
      if constexpr (HALF) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float2 w = angle(col + k, col + k);
          const float y = row_elem<T, V>(b, k);
          h[k] = fmaf(y, w.x, f[k] * w.y);
          f[k] = fmaf(f[k], w.x, -(y * w.y));
        }
        row_store<T, V>(out + g.rotary / 2, col, part, h);
      } else {
        const int first = col / 2;
#pragma unroll
        for (int k = 0; k < V; k += 2) {
          const float2 w = angle(first + k / 2, col + k);
          const float x = f[k], y = f[k + 1];
          f[k] = fmaf(x, w.x, -(y * w.y));
          f[k + 1] = fmaf(y, w.x, x * w.y);
        }
      }
    };
    if (turn) {
      if (col + V <= part) rotated(std::true_type{});
      else rotated(std::false_type{});
    }
    row_store<T, V>(out, col, part, f);
  }
};

// ONE: a workgroup's tile is one token.  OFF: the type of offsets within a tensor.  A 64-bit product is four 32-bit ones, each
// of a quarter of the rate; with six of them a vector they bounded the kernel
// ([2, 4096, 64, 192] bf16, interleaved: 103 us, 79 with 32-bit offsets, 71 with
// those of a workgroup's one token as scalars).
template <typename T, bool HALF, bool ONE, typename OFF>
__global__ void __launch_bounds__(kRotBlock) k_rotary(RotArgs g) {
  __shared__ float2 cs[kRotTable];
  const int32_t token0 = g.first + (int32_t)blockIdx.x * g.per;
  const int32_t slot0 = (int32_t)blockIdx.y * g.heads;
  const uint32_t all = (uint32_t)(g.per * g.heads * g.units);
  const int pairs = g.rotary / 2;
  constexpr int U = rot_units(HALF);
  RotUnit<T, HALF, ONE, OFF> w[U];
  uint32_t unit = threadIdx.x;
  auto request = [&]() {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      w[i].find(g, unit + i * blockDim.x, token0, slot0);
      if (U > 1) w[i].live = w[i].live && unit + i * blockDim.x < all;
      w[i].load(g);
    }
  };
  if (unit < all) request();
  for (int i = threadIdx.x; i < g.per * pairs; i += blockDim.x) {
    const int tk = i / pairs;
    if (tk < g.tokens - token0) {  // token0 + tk may pass 2^31
      const int32_t token = token0 + tk;
      uint32_t bi, si;
      g.seq.divmod((uint32_t)token, bi, si);
      int64_t p = si;
      if (g.pos) {
        const int64_t at = bi * g.ps[0] + si * g.ps[1];
        p = g.pos64 ? static_cast<const int64_t*>(g.pos)[at] : (int64_t)static_cast<const int32_t*>(g.pos)[at];
      }
      const double turns = (double)(p + g.offset) * g.freq[i - tk * pairs] * 0.15915494309189533577;
      // Whole quarter turns are taken off before the rest, at most an eighth of a turn, is
      // rounded to float32: its sine and cosine keep 24 bits also next to their zeros.
      const double half = 2.0 * (turns - rint(turns)), quarter = rint(2.0 * half);
      const int quarters = (int)quarter & 3;
      float s, c;
      sincospif((float)(half - 0.5 * quarter), &s, &c);
      const float sn = quarters & 1 ? c : s, cn = quarters & 1 ? s : c;
      s = (quarters & 2) != 0 != (g.inverse != 0) ? -sn : sn;
      c = (quarters + 1) & 2 ? -cn : cn;
      cs[i] = make_float2(g.scale * c, g.scale * s);
    }
  }
  __syncthreads();
  while (unit < all) {
#pragma unroll
    for (int i = 0; i < U; ++i) w[i].store(g, cs + w[i].tk * pairs);
    unit += U * blockDim.x;
    if (unit < all) request();
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
  const int64_t table = kRotTable / (d.rotary / 2);  // tokens whose angles fit
  // by the larger tensor's output: its tokens lie closer together than its heads
  const RotTensor& large = a.t[a.t[1].heads > a.t[0].heads ? 1 : 0];
  a.head_major = large.heads > 1 && d.seq > 1 && large.os[1] < large.os[2];
  if (a.head_major) {
    // a run of tokens, and as many heads as fill four steps of 512 threads:
    // [4, 40, 2048, 128] bf16 38 -> 33 us
    a.per = (int32_t)std::min<int64_t>({table, 32, a.tokens});
    a.heads = (int32_t)std::min<int64_t>(slots, std::max<int64_t>(1, 4 * kRotBlock / (a.per * a.units)));
  } else {
    // tokens of few heads share a workgroup of 256 threads
    a.per = (int32_t)std::max<int64_t>(1, std::min<int64_t>({256 / per_token, table, a.tokens}));
    a.heads = (int32_t)slots;
  }
  // up to 512 threads, evenly filled
  const int64_t all = (int64_t)a.per * a.heads * a.units, each = (all + rot_units(half) - 1) / rot_units(half);
  const int64_t steps = (each + kRotBlock - 1) / kRotBlock;
  const int block = (int)((((each + steps - 1) / steps) + 63) / 64 * 64);
  a.seq = FastDiv((uint32_t)d.seq);
  a.by_unit = FastDiv((uint32_t)a.units);
  a.by_inner = FastDiv((uint32_t)(a.head_major ? a.per : a.heads));
  // whether every offset of q and k, and those formed of the tile's places past
  // the last token or head, fits 32 bits
  bool narrow = true;
  for (const RotTensor& t : a.t)
    for (const int64_t* step : {t.is, t.os}) {
      const double most = std::fabs((double)step[0]) * (double)(d.batch + a.per) +
                          std::fabs((double)step[1]) * (double)d.seq +
                          std::fabs((double)step[2]) * (double)(t.heads + a.heads);
      narrow = narrow && most < 2147483648.0;
    }
  const unsigned groups = (unsigned)((slots + a.heads - 1) / a.heads);
  if (groups > 65535) return SUPA_AMD_ELAYOUT;
  const int64_t slab = (int64_t(1) << 31) / kRotBlock / groups * a.per;  // HIP: fewer than 2^32 threads a launch
  const int64_t tokens = a.tokens;
  for (int64_t first = 0; first < tokens; first += slab) {
    a.first = (int32_t)first;
    a.tokens = (int32_t)std::min(tokens, first + slab);
    const unsigned blocks = (unsigned)((a.tokens - first + a.per - 1) / a.per);
    auto go = [&](auto h, auto one, auto* off) {
      k_rotary<T, h.value, one.value, std::remove_pointer_t<decltype(off)>><<<dim3(blocks, groups), block, 0, st>>>(a);
    };
    auto offsets = [&](auto h, auto one) {
      if (narrow) go(h, one, (int32_t*)nullptr);
      else go(h, one, (int64_t*)nullptr);
    };
    auto tile = [&](auto h) {
      if (a.per == 1 && !a.head_major) offsets(h, std::true_type{});
      else offsets(h, std::false_type{});
    };
    if (half) tile(std::true_type{});
    else tile(std::false_type{});
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
  if (d->rotary > 2 * kRotMaxPairs || d->dim >= (int64_t(1) << 24) || d->q.heads >= (int64_t(1) << 30) ||
      d->k.heads >= (int64_t(1) << 30) ||
      (d->batch > 0 && d->seq >= (int64_t(1) << 31) / d->batch))
    return SUPA_AMD_ELAYOUT;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_float_storage(d->dtype, [&](auto* tag) -> int {
    return rot_launch<std::remove_pointer_t<decltype(tag)>>(*d, st);
  });
}

// Rotary positions of new tokens, and their place in the paged cache.
//
// Frequency f turns the pair (x, y) of a query or key head by
// theta = position[axis(f)][t] * omega[f]:
//   x' = x cos(theta) - y sin(theta),  y' = x sin(theta) + y cos(theta)
// with x, y at dims f and F + f (half) or 2f and 2f + 1 (interleaved); dims
// behind the rotated ones pass through.  Text has one axis; images and video
// have several (time, height, width), each turning its share of the
// frequencies.  Positions are the semantic ones, which compaction leaves
// alone; slots are physical.
//
// Every value is read and written once, so memory bounds it.  One workgroup
// takes a token (or a share of its heads where tokens are few): it forms the
// token's F cosines and sines once, in LDS, and all heads use them.  8192 tokens
// of 40 + 8 heads of 128, three axes: 36 us (6.5 TB/s) with the tensors in the
// last-level cache, 48 (4.9, a copy's rate) from HBM.

#include "kvc_common.h"
#include "mfma_common.h"
#include "row_sets.h"

namespace kvc {
namespace {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryMaxFreq = 256;
constexpr int kRotaryMaxAxes = 4;

struct RotaryArgs {
  const uint16_t *q, *k, *v;
  uint16_t *q_out, *k_cache, *v_cache;
  const int64_t* positions;
  const float* omega;
  const int64_t* slots;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head;
  int64_t position_stride, num_slots, page_stride;
  int heads, kv_heads, head_dim, freq, axes, cycled;
  int sections[kRotaryMaxAxes];
};

// Runs of sections[a] frequencies ("blocked"), or the axes in turn while their
// sections last, the rest with the first axis ("cycled").
__device__ __forceinline__ int axis_of(const RotaryArgs& a, int f) {
  if (a.cycled) {
    const int axis = f % a.axes, turn = f / a.axes;
    return turn < a.sections[axis] ? axis : 0;
  }
  int axis = 0, end = a.sections[0];
  while (axis + 1 < a.axes && f >= end) end += a.sections[++axis];
  return axis;
}

template <bool F16>
__device__ __forceinline__ float to_float(uint16_t x) {
  return F16 ? fp16_lo(x) : bf16_lo(x);
}
template <bool F16>
__device__ __forceinline__ uint16_t from_float(float x) {
  return static_cast<uint16_t>(F16 ? pack_f16(x, 0.0f) : pack_bf16(x, 0.0f));
}

template <int VEC>
struct Chunk;
template <>
struct Chunk<8> {
  typedef u32x4 type;
};
template <>
struct Chunk<1> {
  typedef uint16_t type;
};

template <bool F16, int VEC>
__device__ __forceinline__ void unpack(typename Chunk<VEC>::type w, float (&x)[VEC]) {
  if constexpr (VEC == 1) {
    x[0] = to_float<F16>(w);
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      x[2 * i] = MfmaElem<F16>::lo(w[i]);
      x[2 * i + 1] = MfmaElem<F16>::hi(w[i]);
    }
  }
}
template <bool F16, int VEC>
__device__ __forceinline__ typename Chunk<VEC>::type repack(const float (&x)[VEC]) {
  if constexpr (VEC == 1) {
    return from_float<F16>(x[0]);
  } else {
    typename Chunk<VEC>::type w;
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) w[i] = MfmaElem<F16>::pack(x[2 * i], x[2 * i + 1]);
    return w;
  }
}

// One unit: VEC pairs of a head (or, behind the rotated dims, VEC plain
// values).  With interleaved pairs and VEC 8 a unit is one 16-byte chunk of
// four pairs; VEC 1 takes a pair.
template <bool F16, bool IL, int VEC>
__device__ __forceinline__ void turn_unit(const uint16_t* from, uint16_t* to, int unit, int freq, const float2* turns) {
  typedef typename Chunk<VEC>::type word;
  if constexpr (IL && VEC == 8) {
    float x[8];
    const word w = *gptr(reinterpret_cast<const word*>(from + unit * 8));
    if (unit * 4 >= freq) {
      *gptr(reinterpret_cast<word*>(to + unit * 8)) = w;
      return;
    }
    unpack<F16, 8>(w, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 cs = turns[unit * 4 + i];
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = a * cs.x - b * cs.y;
      x[2 * i + 1] = a * cs.y + b * cs.x;
    }
    *gptr(reinterpret_cast<word*>(to + unit * 8)) = repack<F16, 8>(x);
  } else {
    const int f = unit * VEC;
    if (f >= freq) {  // behind the rotated dims
      const int d = freq + f;
      *gptr(reinterpret_cast<word*>(to + d)) = *gptr(reinterpret_cast<const word*>(from + d));
      return;
    }
    const int near = IL ? 2 * f : f, far = IL ? 2 * f + 1 : freq + f;
    float x[VEC], y[VEC];
    unpack<F16, VEC>(*gptr(reinterpret_cast<const word*>(from + near)), x);
    unpack<F16, VEC>(*gptr(reinterpret_cast<const word*>(from + far)), y);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float2 cs = turns[f + i];
      const float a = x[i], b = y[i];
      x[i] = a * cs.x - b * cs.y;
      y[i] = a * cs.y + b * cs.x;
    }
    *gptr(reinterpret_cast<word*>(to + near)) = repack<F16, VEC>(x);
    *gptr(reinterpret_cast<word*>(to + far)) = repack<F16, VEC>(y);
  }
}

template <bool F16, bool IL, int VEC>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a) {
  typedef typename Chunk<VEC>::type word;
  __shared__ float2 turns[kRotaryMaxFreq];
  const int64_t t = blockIdx.x;
  for (int f = threadIdx.x; f < a.freq; f += kRotaryThreads) {
    // The angle in float64, less its whole turns: float32 would lose positions
    // beyond 2^24 / theta turns, and a tenth of a radian at 2^20.
    const double angle = static_cast<double>(a.positions[axis_of(a, f) * a.position_stride + t]) * static_cast<double>(a.omega[f]);
    const double whole = rint(angle * 0.15915494309189535);
    const double part = fma(-whole, 2.4492935982947064e-16, fma(-whole, 6.283185307179586, angle));
    float sn, cs;
    sincosf(static_cast<float>(part), &sn, &cs);
    turns[f] = make_float2(cs, sn);
  }
  const int64_t slot = a.slots[t];
  const bool stored = slot >= 0 && slot < a.num_slots;
  const int64_t place = (slot >> kBlockShift) * a.page_stride + (slot & (kBlockSize - 1)) * static_cast<int64_t>(a.kv_heads) * a.head_dim;
  __syncthreads();
  // Units of a turned head and of a value head.
  const int turned = (IL && VEC == 8) ? a.head_dim / 8 : (a.head_dim - a.freq) / VEC;
  const int plain = a.head_dim / VEC;
  const int q_units = a.heads * turned, k_units = a.kv_heads * turned, v_units = a.kv_heads * plain;
  const int all = stored ? q_units + k_units + v_units : q_units;
  for (int u = blockIdx.y * kRotaryThreads + threadIdx.x; u < all; u += gridDim.y * kRotaryThreads) {
    if (u < q_units) {
      const int h = u / turned, unit = u - h * turned;
      turn_unit<F16, IL, VEC>(a.q + t * a.q_token + h * a.q_head, a.q_out + t * a.out_token + h * a.out_head, unit, a.freq, turns);
    } else if (u < q_units + k_units) {
      const int h = (u - q_units) / turned, unit = u - q_units - h * turned;
      turn_unit<F16, IL, VEC>(a.k + t * a.k_token + h * a.k_head, a.k_cache + place + h * a.head_dim, unit, a.freq, turns);
    } else {
      const int w = u - q_units - k_units, h = w / plain, unit = w - h * plain;
      *gptr(reinterpret_cast<word*>(a.v_cache + place + h * a.head_dim + unit * VEC)) =
          *gptr(reinterpret_cast<const word*>(a.v + t * a.v_token + h * a.v_head + unit * VEC));
    }
  }
}

// Tokens of one dispatch, whose work-items are numbered in 32 bits.
constexpr int64_t kRotaryTokens = 1 << 23;

template <bool F16, bool IL>
int launch(hipStream_t stream, RotaryArgs a, int64_t n, bool wide) {
  // Few tokens: the heads of one are spread over workgroups too.
  const int units = (a.heads + 2 * a.kv_heads) * (a.head_dim / (wide ? 8 : 1));
  const int64_t most = ceil_div(units, kRotaryThreads);
  int64_t shares = n >= 1024 ? 1 : ceil_div(1024, n);
  if (shares > most) shares = most;
  while (n > 0) {
    const int64_t now = n < kRotaryTokens ? n : kRotaryTokens;
    const dim3 grid(static_cast<unsigned>(now), static_cast<unsigned>(shares));
    if (wide)
      rotary_kernel<F16, IL, 8><<<grid, kRotaryThreads, 0, stream>>>(a);
    else
      rotary_kernel<F16, IL, 1><<<grid, kRotaryThreads, 0, stream>>>(a);
    if (int rc = launch_status("kvc_rotate_and_store")) return rc;
    n -= now;
    if (n == 0) break;
    if (a.heads) {
      a.q += now * a.q_token;
      a.q_out += now * a.out_token;
    }
    a.k += now * a.k_token;
    a.v += now * a.v_token;
    a.positions += now;
    a.slots += now;
  }
  return 0;
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" int kvc_rotate_and_store(kvc_stream_t stream, int dtype, int rope_style, int64_t num_tokens, int heads, int kv_heads,
                                    int head_dim, int rotary_dim, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                    const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                    int64_t v_token_stride, int64_t v_head_stride, const int64_t* positions,
                                    int64_t position_stride, int n_axes, const int* sections_host, int cycled, const float* omega,
                                    const int64_t* slot_mapping, void* q_out, int64_t out_token_stride, int64_t out_head_stride,
                                    void* k_cache, void* v_cache, int64_t num_pages, int64_t page_stride) {
  if (dtype != KVC_DTYPE_BF16 && dtype != KVC_DTYPE_FP16)
    return fail(KVC_EINVAL, "kvc_rotate_and_store: dtype must be bf16 or fp16");
  if (rope_style != KVC_ROPE_HALF && rope_style != KVC_ROPE_INTERLEAVED)
    return fail(KVC_EINVAL, "kvc_rotate_and_store: unsupported rope style %d", rope_style);
  if (num_tokens < 0 || num_tokens >= (1ll << 31) || heads < 0 || heads > 4096 || kv_heads <= 0 || kv_heads > 4096)
    return fail(KVC_EINVAL, "kvc_rotate_and_store: bad sizes");
  if (head_dim <= 0 || head_dim > 1024 || rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > head_dim ||
      rotary_dim / 2 > kRotaryMaxFreq)
    return fail(KVC_EINVAL, "kvc_rotate_and_store: rotary_dim %d must be even, at most head_dim %d (at most 1024) and at most %d",
                rotary_dim, head_dim, 2 * kRotaryMaxFreq);
  if (n_axes < 1 || n_axes > kRotaryMaxAxes || !sections_host)
    return fail(KVC_EINVAL, "kvc_rotate_and_store: one to %d axes, each with a section", kRotaryMaxAxes);
  RotaryArgs a = {};
  int sum = 0;
  for (int i = 0; i < n_axes; ++i) {
    if (sections_host[i] < 0 || sections_host[i] > rotary_dim)
      return fail(KVC_EINVAL, "kvc_rotate_and_store: section %d of axis %d is outside [0, rotary_dim]", sections_host[i], i);
    a.sections[i] = sections_host[i];
    sum += sections_host[i];
  }
  if (sum != rotary_dim / 2)
    return fail(KVC_EINVAL, "kvc_rotate_and_store: sections add up to %d, the frequencies are %d", sum, rotary_dim / 2);
  if (num_pages < 0 || page_stride < static_cast<int64_t>(kBlockSize) * kv_heads * head_dim)
    return fail(KVC_EINVAL, "kvc_rotate_and_store: page_stride must be at least one page");
  if (num_tokens == 0) return 0;
  if ((heads > 0 && (!q || !q_out)) || !k || !v || !positions || !omega || !slot_mapping || (num_pages > 0 && (!k_cache || !v_cache)))
    return fail(KVC_EINVAL, "kvc_rotate_and_store: null pointer");
  const RowSet turned = row_set(q_out, out_token_stride, out_head_stride, num_tokens, heads);
  const RowSet queries = row_set(q, q_token_stride, q_head_stride, num_tokens, heads);
  const int64_t row = 2 * head_dim;
  if (rows_share(turned, row)) return fail(KVC_EINVAL, "kvc_rotate_and_store: rows of q_out overlap each other");
  const bool in_place = turned.base == queries.base && turned.token == queries.token && turned.head == queries.head;
  if (!in_place && rows_meet(turned, queries, row))
    return fail(KVC_EINVAL, "kvc_rotate_and_store: q_out overlaps q without being q");
  if (rows_meet(turned, row_set(k, k_token_stride, k_head_stride, num_tokens, kv_heads), row) ||
      rows_meet(turned, row_set(v, v_token_stride, v_head_stride, num_tokens, kv_heads), row))
    return fail(KVC_EINVAL, "kvc_rotate_and_store: q_out overlaps k or v");
  if (num_pages > 0 && k_cache == v_cache)
    return fail(KVC_EINVAL, "kvc_rotate_and_store: k_cache and v_cache are one pool: keys and values would share its rows");
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.k_cache = static_cast<uint16_t*>(k_cache);
  a.v_cache = static_cast<uint16_t*>(v_cache);
  a.positions = positions;
  a.omega = omega;
  a.slots = slot_mapping;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.k_token = k_token_stride;
  a.k_head = k_head_stride;
  a.v_token = v_token_stride;
  a.v_head = v_head_stride;
  a.out_token = out_token_stride;
  a.out_head = out_head_stride;
  a.position_stride = position_stride;
  a.num_slots = num_pages << kBlockShift;
  a.page_stride = page_stride;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.head_dim = head_dim;
  a.freq = rotary_dim / 2;
  a.axes = n_axes;
  a.cycled = cycled != 0;
  // 16-byte words where every row and the pairs' halves start on one.
  const uintptr_t bases = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                          reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache);
  const int64_t steps = q_token_stride | q_head_stride | k_token_stride | k_head_stride | v_token_stride | v_head_stride |
                        out_token_stride | out_head_stride | page_stride | head_dim;
  const bool il = rope_style == KVC_ROPE_INTERLEAVED;
  const bool wide = bases % 16 == 0 && steps % 8 == 0 && a.freq % (il ? 4 : 8) == 0;
  const bool f16 = dtype == KVC_DTYPE_FP16;
  const hipStream_t st = as_stream(stream);
  if (f16) return il ? launch<true, true>(st, a, num_tokens, wide) : launch<true, false>(st, a, num_tokens, wide);
  return il ? launch<false, true>(st, a, num_tokens, wide) : launch<false, false>(st, a, num_tokens, wide);
}

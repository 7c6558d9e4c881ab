// Attention of new tokens over a paged cache: arguments, geometry and helpers
// shared by the two kernels (attend_few.hip, attend_many.hip) and their entry
// (attend.hip).
//
// For a request with `len` cached tokens (its new ones among them) and `fresh`
// new tokens, token i sits at place p = len - fresh + i and sees the keys
//   { j : j <= p  and  (window == 0 or p - j < window or j < sinks) },
// and out = sum_j softmax_j(scale * q.k_j) v_j over them; a row that sees no
// key gives zeros.  The query heads of one KV head are stacked: row
// m = i*qpk + g is query head h*qpk + g of token i, so K and V are read once
// for a whole group of heads.
#pragma once

#include "mfma_common.h"

namespace kvc {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
#define KVC_LDS __attribute__((address_space(3)))

struct AttendArgs {
  const uint16_t* q;
  uint16_t* out;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* start;     // [n_seq + 1] first token of each request
  const int32_t* seq_lens;  // [n_seq]
  const int32_t* table;     // [n_seq][table_stride]
  float* partial;           // joined pieces, see the kernels
  int32_t* header;
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
  int64_t table_stride, num_tokens;
  uint32_t page_bytes;  // from a page to the next
  int num_pages;
  float scale_log2;  // scale * log2(e): weights are powers of two
  int n_seq, kv_heads, qpk, head_dim, max_blocks, window, sinks;
  int few_rows;  // requests of at most this many rows are the few-rows kernel's
};

// An entry of a table that the launch only reads, by a scalar load: a vector one
// would wait for every key and value in flight.
__device__ __forceinline__ int scalar_at(const int32_t* p, int64_t i) {
  return ((__attribute__((address_space(4))) const int32_t*)p)[i];
}

// One request's rows and keys.
struct Request {
  int token0, fresh;  // first token, new tokens
  int len, keys;      // cached tokens; those that the block table covers
};

__device__ __forceinline__ Request request_from(const AttendArgs& a, int start0, int start1, int len) {
  Request s;
  const int64_t total = a.num_tokens;
  int64_t t0 = start0, t1 = start1;
  t0 = t0 < 0 ? 0 : (t0 > total ? total : t0);
  t1 = t1 < t0 ? t0 : (t1 > total ? total : t1);
  s.token0 = static_cast<int>(t0);
  s.fresh = static_cast<int>(t1 - t0);
  s.len = len < 0 ? 0 : len;
  const int64_t most = static_cast<int64_t>(a.max_blocks) << kBlockShift;
  s.keys = s.len < most ? s.len : static_cast<int>(most);
  return s;
}

// Of a request that differs from lane to lane, and of one that does not.
__device__ __forceinline__ Request request_of(const AttendArgs& a, int r) {
  return request_from(a, a.start[r], a.start[r + 1], a.seq_lens[r]);
}
__device__ __forceinline__ Request uniform_request_of(const AttendArgs& a, int r) {
  return request_from(a, scalar_at(a.start, r), scalar_at(a.start, r + 1), scalar_at(a.seq_lens, r));
}

// Key tiles of 2^SHIFT keys that rows at places [first, last] see: the first
// `head` ones (sinks that the window has left behind) and [low, high).
struct TileRange {
  int head, low, high;
  __device__ __forceinline__ int count() const { return head + high - low; }
  __device__ __forceinline__ int tile(int t) const { return t < head ? t : low + t - head; }
};

template <int SHIFT>
__device__ __forceinline__ TileRange tile_range(const AttendArgs& a, const Request& s, int first, int last) {
  TileRange p;
  int end = last + 1 < s.keys ? last + 1 : s.keys;
  if (end < 0) end = 0;
  int begin = a.window ? first - a.window + 1 : 0;
  begin = begin < 0 ? 0 : (begin > end ? end : begin);
  p.low = begin >> SHIFT;
  p.high = (end + (1 << SHIFT) - 1) >> SHIFT;
  const int sink = a.sinks < begin ? a.sinks : begin;
  p.head = (sink + (1 << SHIFT) - 1) >> SHIFT;
  if (p.head > p.low) p.head = p.low;
  return p;
}

// Keys that one row sees: [low, end) and those below `sinks` that are below end.
struct RowSight {
  int end, low;
};

__device__ __forceinline__ RowSight sight_of(const AttendArgs& a, const Request& s, int place) {
  return {place + 1 < s.keys ? place + 1 : s.keys, a.window ? place - a.window + 1 : 0};
}

__device__ __forceinline__ bool sees(const RowSight& s, int sinks, int key) {
  return (key < s.end) & ((key >= s.low) | (key < sinks));  // no branches: 8 to 32 keys a lane ask
}

// The element type of a cache for the 32x32 products.
template <bool F16>
struct AttendElem : MfmaElem<F16> {
  typedef typename MfmaElem<F16>::vec vec;
  // Exponent bits: all set in infinities and NaN.
  static constexpr uint32_t kExponent = F16 ? 0x7c00u : 0x7f80u;
  // A row's largest weight, as a power of two.  fp16 ends at 2^-24: with weights
  // of at most 1 the ones below 2^-25 would be nothing, however many they are
  // (131071 of 2^-25.1 make 2^-8).  bf16 has float32's exponents.
  static constexpr int kRoom = F16 ? 15 : 0;
  __device__ __forceinline__ static f32x16 mfma32(vec a, vec b, f32x16 c) {
    if constexpr (F16)
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // sum + the two values of a word, in float32.
  __device__ __forceinline__ static float add_pair(uint32_t w, float sum) {
    if constexpr (F16)
      return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), __builtin_bit_cast(f16x2, 0x3c003c00u), sum, false);
    else
      return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0x3f803f80u), sum, false);
  }
};

// Four 16-bit values of one column: the 16 lanes of a group give the addresses
// of four rows' 16 columns (lane k: row k/4, columns 4*(k%4)..), and lane k
// gets column k of the four rows (ds_read_b64_tr_b16).
__device__ __forceinline__ s16x4 read_column(const void* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((KVC_LDS s16x4*)p);
}

template <typename V>
__device__ __forceinline__ V join_columns(s16x4 a, s16x4 b) {
  return __builtin_bit_cast(V, s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}

// A value that every lane holds alike, as a scalar.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A request's pages, 64 at a time in the wave's lanes: a page's number then costs
// no wait.  -1 where the table ends.
struct PageIds {
  int first, ids;
  __device__ __forceinline__ void fill(const int32_t* table, int max_blocks, int block) {
    first = block;
    const int mine = block + static_cast<int>(threadIdx.x & 63);
    ids = mine < max_blocks ? *gptr(table + mine) : -1;
    asm volatile("" : "+v"(ids));  // waited for here, not wherever it is used
  }
  __device__ __forceinline__ int at(const int32_t* table, int max_blocks, int block) {
    if (block - first >= 64 || block < first) fill(table, max_blocks, block);
    return __builtin_amdgcn_readlane(ids, block - first);
  }
};

// The same for a walk in order, as places: a lane holds its page's first byte in
// a pool, and whether the page is in it.
struct PagePlaces {
  int first = -(1 << 30);  // nothing yet
  uint32_t low = 0, high = 0, there = 0;
  __device__ __forceinline__ bool covers(int block) const { return static_cast<uint32_t>(block - first) < 64u; }
  __device__ __forceinline__ void refill(const AttendArgs& a, const int32_t* table, int block) {
    first = block;
    const int mine = block + static_cast<int>(threadIdx.x & 63);
    const int page = mine < a.max_blocks ? *gptr(table + mine) : -1;
    const bool in = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.num_pages);
    const uint64_t from = in ? static_cast<uint64_t>(static_cast<uint32_t>(page)) * a.page_bytes : 0;
    low = static_cast<uint32_t>(from);
    high = static_cast<uint32_t>(from >> 32);
    there = in ? 0xffffffffu : 0;
    asm volatile("" : "+v"(low), "+v"(high), "+v"(there));  // waited for here, not wherever they are used
  }
};

// The larger of a lane's value and that of the lane 32 away.
__device__ __forceinline__ float max_across_halves(float x) {
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}

// A buffer of `bytes` bytes, `from` bytes behind a pool's start, for loads with
// lane offsets; past its end they give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t page_rsrc(const uint16_t* pool, uint64_t from, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)(reinterpret_cast<uintptr_t>(pool) + from), 0, bytes, 0x00020000);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr float kNegInf = -__builtin_inff();

// The exponent that a row's weights are taken from, whose largest score is `top`:
// BY below it, so that its weight is 2^BY, in the sum of the weights as in the
// outputs.  Where float32 has no fractions left that difference may become 16, and
// fp16 ends below 2^16: there the largest weight is 1.
template <int BY>
__device__ __forceinline__ float lowered(float top) {
  return BY && fabsf(top) < 8388608.0f ? top - BY : top;
}

// Joins `count` pieces of ROWS rows (first, first + 1, .. below `rows`) of which
// piece i is at piece(i): `floats` unnormalised outputs of DP dims a row, then
// (maximum, sum) pairs.  A workgroup of 256: 256 / ROWS lanes a row find the common
// maximum and sum, then every thread adds four dims at a time of all or of every
// other piece, and such shares meet in LDS.  store(row, dim, f32x4) takes the
// results.
template <int DP, int ROWS, typename Piece, typename Store>
__device__ __forceinline__ void join_pieces(int count, int first, int rows, int head_dim, int floats, Piece piece, Store store) {
  constexpr int kUnits = ROWS * DP / 4, kLanes = 256 / ROWS;
  constexpr int kShares = kUnits <= 128 ? 2 : 1, kEach = (kUnits + 255) / 256;
  __shared__ float top_of[ROWS], inv_of[ROWS];
  __shared__ f32x4 shared_sum[kShares > 1 ? 256 : 1];
  const int tid = threadIdx.x, lane = tid % kLanes, own = first + tid / kLanes;
  if (own < rows) {
    float top = kNegInf;
    for (int i = lane; i < count; i += kLanes) top = fmaxf(top, piece(i)[floats + 2 * own]);
#pragma unroll
    for (int d = kLanes / 2; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float use = top == kNegInf ? 0.0f : top;
    float sum = 0.0f;
    for (int i = lane; i < count; i += kLanes) {
      const f32x2 ml = *reinterpret_cast<const f32x2*>(piece(i) + floats + 2 * own);
      sum += ml[1] * exp2_fast(ml[0] - use);
    }
#pragma unroll
    for (int d = kLanes / 2; d; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) {
      top_of[own - first] = use;
      inv_of[own - first] = sum == 0.0f ? 0.0f : 1.0f / sum;
    }
  }
  __syncthreads();
  f32x4 sums[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int share = kShares > 1 ? tid / kUnits : 0, unit = tid + e * 256 - share * kUnits;
    const int local = unit / (DP / 4), d = (unit - local * (DP / 4)) * 4, row = first + local;
    sums[e] = f32x4{0, 0, 0, 0};
    if (share < kShares && unit < kUnits && row < rows && d < head_dim) {
      const float use = top_of[local];
#pragma unroll 8
      for (int i = share; i < count; i += kShares) {
        const float* p = piece(i);
        sums[e] += *reinterpret_cast<const f32x4*>(p + row * DP + d) * exp2_fast(p[floats + 2 * row] - use);
      }
      sums[e] *= inv_of[local];
    }
  }
  if constexpr (kShares > 1) {
    if (tid >= kUnits && tid < 2 * kUnits) shared_sum[tid - kUnits] = sums[0];
    __syncthreads();
    if (tid < kUnits) sums[0] += shared_sum[tid];
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int unit = tid + e * 256, local = unit / (DP / 4), d = (unit - local * (DP / 4)) * 4, row = first + local;
    if (unit < kUnits && row < rows && d < head_dim) store(row, d, sums[e]);
  }
}

// The many-rows launch: `round` workgroups fit the device at once, `grid` are
// launched, and a (row tile, head)'s keys are split at most `most_splits` times.
struct ManyGrid {
  int round, most_splits;
  uint32_t most_tiles;  // row tiles that the grid and the workspace are for
  int64_t grid;
};

// Entry points of the kernels' files.
int launch_attend_few(hipStream_t stream, bool f16, const AttendArgs& a, int workgroups, int row_tiles);
int launch_attend_many(hipStream_t stream, bool f16, const AttendArgs& a, const ManyGrid& grid);

// Sizes of the workspace's parts.
constexpr int kFewRows = 16;         // rows of one few-rows tile
constexpr int kFewTilesMost = 2;     // tiles of a request that the few-rows kernel takes
constexpr int kFewSequences = 1024;  // requests of one launch (their prefix sums sit in LDS)
// Rows of one many-rows tile, 32 a wave.
constexpr int many_rows(int dim) { return dim <= 192 ? 256 : 128; }
constexpr int many_threads(int dim) { return many_rows(dim) * 2; }

// Few-rows workgroups that a compute unit holds: as many as registers and LDS
// allow, but for head_dim 64 and 96, where one more is slower (16 requests of
// 16384 keys, 8 KV heads, head_dim 64: 117 us with three, 123 with two or four).
constexpr int few_residents(int dim) { return dim <= 64 ? 3 : (dim <= 128 ? 2 : 1); }

// Floats of a piece of `rows` rows: unnormalised outputs, then (max, sum) pairs.
__host__ __device__ inline int64_t piece_floats(int rows, int dim) { return static_cast<int64_t>(rows) * (dim + 2); }

// Head dims are computed in multiples of 32.
inline int padded_dim(int head_dim) {
  const int dims[] = {64, 96, 128, 192, 256};
  for (int d : dims)
    if (head_dim <= d) return d;
  return 0;
}

}  // namespace kvc

// Attention of requests with many rows (chunks of a prompt): the matrix cores
// bound it.  A workgroup takes 128 or 256 rows of one (request, KV head), 32 a
// wave, and walks the key tiles that some row sees; K and V tiles go through
// registers to LDS, where all waves read them.  With few tiles of rows the keys
// are split too, and a second launch joins the splits.
//
// What runs beside the matrix products is what decides.  Up to head_dim 192 two
// waves share a SIMD: two groups of four waves take 128 rows each, the second
// half a tile behind the first, so that one's products run beside the other's
// softmax.  Above that a wave's outputs and queries need more registers than half
// a SIMD's: one group forms a tile's weights between the products of the next
// tile's scores.
//
// 2048 tokens (40 heads on 8, head_dim 128) over 16384 keys: 600 - 615 us, 1.05 -
// 1.07 PFLOP/s, a library product of 16384^3 1.58.  The matrix cores are busy 52% of
// the time, LDS 32%; 1.19 million cycles at 1.93 GHz, where simpler forms took 1.48
// million at 2.19: the clock falls as the matrix cores fill.  16 heads on 2: head_dim
// 64 311 us of 4096 tokens (0.9 PFLOP/s, the softmax's), of 2048 head_dim 192 390 us
// (1.0) and 256 600 us (0.9).
//
// Scores are formed transposed (S^T = K Q^T, 32x32x16): a lane holds one row's
// scores (its other half in lane ^ 32), so the softmax needs one exchange, and
// the packed weights are the right operand of O^T = V^T P^T as they lie, keys
// numbered to match: slot (lane/32, j) of 16 keys is key 8*(j/4) + 4*(lane/32)
// + j%4.  Weights are rounded to the cache's 16-bit type for that product, and the
// rounded ones are what is summed, so that a row's weights add up to one: what is
// left is half a step of how far the values lie from their mean, where the output's
// own rounding is half a step of it: bf16 outputs are 2.2e-3 off float64, 1.7e-3 with
// a second word for each weight, which would take 821 us for 614 (head_dim 192 628
// for 397, 256 754 for 601).  The maxima, sums and outputs are float32.

#include <type_traits>
#include <utility>

#include "attend_internal.h"

namespace kvc {
namespace {

#define KVC_INLINE __attribute__((always_inline))

// f(FROM), f(FROM + 1), .. f(TO - 1) with constant numbers, whatever the compiler
// thinks of unrolling.
template <int FROM, typename F, int... I>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F f) {
  (f(std::integral_constant<int, FROM + I>{}), ...);
}
template <int FROM, int TO, typename F>
__device__ __forceinline__ void each(F f) {
  each_of<FROM>(std::make_integer_sequence<int, TO - FROM>{}, f);
}

constexpr int kJoinThreads = 256, kJoinRows = 16;

// K's and V's place in LDS: rows of 64, 128 or 256 elements whose 16-byte chunks
// are moved, by an exclusive or with a number of the row, so that the 16 rows of
// an operand read (K, one chunk of each) and the four rows of a column read (V,
// four chunks of each) fall on different banks.  A thread holds, of every kStep
// rows, row tid / kSlots and chunk tid % kSlots.
template <int DP>
struct ManyLayout {
  static constexpr int kKeys = DP <= 128 ? 64 : 32;
  static constexpr int kShift = DP <= 128 ? 6 : 5;
  static constexpr int kRow = DP <= 64 ? 64 : (DP <= 128 ? 128 : 256);
  static constexpr int kBytes = kRow * 2;
  static constexpr int kTile = kKeys * kRow;
  static constexpr int kSlots = kRow / 8;
  static constexpr int kGroups = many_rows(DP) / 128;  // of four waves, 32 rows each
  static constexpr int kThreads = many_threads(DP);
  static constexpr int kBuffers = kGroups > 1 ? 3 : 2;  // of K and of V in LDS
  static constexpr int kStep = kThreads / kSlots;
  static constexpr int kLoads = kKeys / kStep;
  __device__ __forceinline__ static constexpr int k_turn(int row) { return (kRow == 64 ? (row >> 1) & 7 : row & 15) << 4; }
  __device__ __forceinline__ static constexpr int v_turn(int row) { return (kRow == 64 ? (row >> 1) & 1 : row & 3) << 6; }
};

// Row tiles of a request that are this kernel's.
template <int ROWS>
__device__ __forceinline__ uint32_t tiles_of(const AttendArgs& a, const Request& s) {
  const int64_t rows = static_cast<int64_t>(s.fresh) * a.qpk;
  return rows > a.few_rows ? static_cast<uint32_t>((rows + ROWS - 1) / ROWS) : 0;
}

// Sums stop at `most` < 2^31, what the launch is for: starts that overlap name
// more tokens than there are.
__device__ __forceinline__ uint32_t add_up_to(uint32_t most, uint32_t x, uint32_t y) { return x + y < most ? x + y : most; }

__device__ __forceinline__ uint32_t sum_up_to_lane(uint32_t most, uint32_t x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t up = __shfl_up(x, d);
    if (lane >= d) x = add_up_to(most, x, up);
  }
  return x;
}

// Row tiles of all requests, counted by one wave: a lane sums its share of them.
template <int ROWS>
struct TileCount {
  int share;           // requests a lane
  uint32_t sum, most;  // tiles up to the end of the lane's
  Request last;        // the lane's last request
  __device__ __forceinline__ TileCount(const AttendArgs& a, const ManyGrid& grid) : most(grid.most_tiles) {
    const int lane = threadIdx.x & 63;
    share = (a.n_seq + 63) / 64;
    last = Request{0, 0, 0, 0};
    uint32_t mine = 0;
    for (int i = 0; i < share; ++i) {
      const int r = lane * share + i;
      if (r >= a.n_seq) break;
      last = request_of(a, r);
      mine = add_up_to(most, mine, tiles_of<ROWS>(a, last));
    }
    sum = sum_up_to_lane(most, mine);
  }
  __device__ __forceinline__ int total() const { return static_cast<int>(__builtin_amdgcn_readlane(sum, 63)); }
  // The request of row tile `tile` < total(), its number, and the tile's in it.
  __device__ __forceinline__ Request find(const AttendArgs& a, int tile, int* request, int* local) const {
    const uint32_t place = static_cast<uint32_t>(tile);
    const int at = __builtin_ctzll(__ballot(sum > place));  // the first lane whose share ends behind it
    uint32_t before = at ? __builtin_amdgcn_readlane(sum, at > 0 ? at - 1 : 0) : 0;
    if (share == 1) {  // a lane holds what would be read again, which would be waited for
      *request = at;
      *local = static_cast<int>(place - before);
      return {__builtin_amdgcn_readlane(last.token0, at), __builtin_amdgcn_readlane(last.fresh, at),
              __builtin_amdgcn_readlane(last.len, at), __builtin_amdgcn_readlane(last.keys, at)};
    }
    for (int base = at * share;; base += 64) {
      const int r = base + static_cast<int>(threadIdx.x & 63);
      const uint32_t up = sum_up_to_lane(most, r < a.n_seq && r < (at + 1) * share ? tiles_of<ROWS>(a, request_of(a, r)) : 0);
      const uint64_t behind = __ballot(before + up > place);
      if (behind || base + 64 >= (at + 1) * share) {
        const int in = behind ? __builtin_ctzll(behind) : 0;
        *request = base + in;
        *local = static_cast<int>(place - before - (in ? __builtin_amdgcn_readlane(up, in > 0 ? in - 1 : 0) : 0));
        return uniform_request_of(a, *request);
      }
      before += __builtin_amdgcn_readlane(up, 63);
    }
  }
};

// How the (row tile, head) items are shared out: whole rounds of the device take
// one item a workgroup; what is left over (or all, where there is no whole
// round) is split along its keys into one more round, however many rounds come
// before it.  40 heads on 8, head_dim 128, split / left whole:
//   1.25 rounds of 16384 keys 601 / 791 us, 3.1 of 32768 2787 / 3335, 6.1 of 40000
//   6290 / 7050, 8.1 of 40000 7935 / 8640;
//   prompts without anything before them, whose first rows are left over and see
//   few keys: 1.2 rounds 78 / 71 us, 3.1 314 / 302, 6.1 1054 / 1043.
// All of them are split alike, by their number: which request is the long one is
// not looked at.  A chunk of 200 over 32768 keys (16 heads on 2) takes 84 us alone
// and 395 beside seven of 200 over 200.
struct ManyShares {
  int total, whole, splits;  // row tiles; those (the last ones) that are not split
  __device__ __forceinline__ ManyShares(const AttendArgs& a, const ManyGrid& grid, int tiles) : total(tiles), whole(tiles), splits(1) {
    const int rounds = tiles * a.kv_heads / grid.round;  // fewer items than workgroups in the grid, below 2^31
    const int left = tiles - rounds * grid.round / a.kv_heads;
    if (left <= 0) return;
    const int fit = grid.round / (left * a.kv_heads);
    splits = fit < grid.most_splits ? fit : grid.most_splits;
    if (splits > 1)
      whole = tiles - left;
    else
      splits = 1;
  }
};

template <bool F16, int DP>
__global__ __launch_bounds__(ManyLayout<DP>::kThreads, ManyLayout<DP>::kGroups) void attend_many_kernel(AttendArgs a, ManyGrid grid) {
  typedef AttendElem<F16> E;
  typedef typename E::vec vec_t;
  typedef ManyLayout<DP> L;
  constexpr int kRows = many_rows(DP);
  constexpr int kSteps = DP / 16;       // 16-dim steps of K Q^T
  constexpr int kBlocks = DP / 32;      // 32-dim blocks of the output
  constexpr int kKeyBlocks = L::kKeys / 32;
  __shared__ __attribute__((aligned(16))) uint16_t k_tile[L::kBuffers][L::kTile];
  __shared__ __attribute__((aligned(16))) uint16_t v_tile[L::kBuffers][L::kTile];

  // The last rows see the most keys: they begin first, and the ones that are
  // split end last.
  const int head = blockIdx.x % a.kv_heads;
  const int order = blockIdx.x / a.kv_heads;
  const TileCount<kRows> counted(a, grid);
  const ManyShares shares(a, grid, counted.total());
  const bool divided = order >= shares.whole;
  const int splits = divided ? shares.splits : 1;
  const int split = divided ? (order - shares.whole) % splits : 0;
  const int item = divided ? (order - shares.whole) / splits : 0;  // of the split ones
  const int tile = shares.total - 1 - (divided ? shares.whole + item : order);
  if (tile < 0) return;
  int request, local;
  const Request s = counted.find(a, tile, &request, &local);
  const int rows = s.fresh * a.qpk, row0 = local * kRows;

  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
  const int wave = uniform(tid >> 6);
  const int place0 = s.len - s.fresh;
  const int wg_last = (row0 + kRows < rows ? row0 + kRows : rows) - 1;
  const TileRange range = tile_range<L::kShift>(a, s, place0 + row0 / a.qpk, place0 + wg_last / a.qpk);
  const int count = range.count();
  const int least = count / splits, more = count - least * splits;  // the first `more` splits take one tile more
  const int t_begin = least * split + (split < more ? split : more);
  const int t_end = t_begin + least + (split < more ? 1 : 0);

  const bool inside = row0 + wave * 32 + col < rows;
  const int token = (inside ? row0 + wave * 32 + col : rows - 1) / a.qpk;
  RowSight sight = sight_of(a, s, place0 + token);
  if (!inside) sight.end = 0;
  // The wave's first and last rows' sights.
  const int m_first = row0 + wave * 32, m_last = m_first + 31 < rows ? m_first + 31 : rows - 1;
  const int token_first = m_first / a.qpk, token_last = (m_first < rows ? m_last : m_first) / a.qpk;
  const RowSight first = sight_of(a, s, place0 + token_first), last = sight_of(a, s, place0 + token_last);

  vec_t qf[kSteps];
  {
    const int g = (inside ? row0 + wave * 32 + col : rows - 1) - token * a.qpk;
    const uint16_t* row = a.q + (s.token0 + token) * a.q_token_stride + (head * a.qpk + g) * a.q_head_stride;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const int d = st * 16 + half * 8;
      u32x4 w = {0, 0, 0, 0};
      if (inside && d < a.head_dim) w = *gptr(reinterpret_cast<const u32x4*>(row + d));
      qf[st] = __builtin_bit_cast(vec_t, w);
    }
  }
  const int row_elems = a.kv_heads * a.head_dim;
  const uint32_t row_bytes = row_elems * 2;
  const int32_t* table = a.table + request * a.table_stride;
  // The thread's chunk of a tile's first rows: where it is (behind everything
  // where the row has none) and where it goes, then where the lane reads.
  const int row_to = tid / L::kSlots, chunk_to = tid & (L::kSlots - 1);
  const uint32_t from = chunk_to * 8 < a.head_dim ? row_to * row_bytes + chunk_to * 16 : 0x7fffffffu;
  const int k_to = row_to * L::kBytes + ((chunk_to << 4) ^ L::k_turn(row_to));
  const int v_to = row_to * L::kBytes + ((chunk_to << 4) ^ L::v_turn(row_to));
  const int k_from = col * L::kBytes + ((half << 4) ^ L::k_turn(col));
  const int v_row = 4 * half + ((lane & 15) >> 2);
  const int v_from = v_row * L::kBytes + L::v_turn(v_row) + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
  u32x4 kst[L::kLoads], vst[L::kLoads];
  // A key tile's place in the pools and its bytes, up to the request's last row:
  // zeros come from behind it, whatever the page holds there, and for tiles behind
  // the last one or of pages outside the pool.  It is worked out in four steps of
  // a few scalar instructions, which the gaps between two products hide.
  PagePlaces pages;
  struct Place {
    uint64_t from;
    uint32_t bytes;
  };
  struct Search {
    int key0, lane;
    uint32_t mask, in_page;
    Place at;
  };
  const uint32_t head_bytes = head * a.head_dim * 2, row_end = a.head_dim * 2;
  auto block_of = [&](int t) { return (range.tile(t < t_end ? t : t_end - 1) << L::kShift) >> kBlockShift; };
  auto ready = [&](int t) KVC_INLINE {  // the page of tile t is in the lanes
    const int block = t_end > 0 ? block_of(t) : 0;
    if (!pages.covers(block)) pages.refill(a, table, block);
  };
  // The queries and the first pages are there before the first tile is asked for:
  // the loop's waits then count its own loads alone.
  pages.refill(a, table, t_end > 0 ? block_of(t_begin) : 0);
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  auto seek = [&](Search& f, int t, int step) KVC_INLINE {
    if (step == 0) {
      f.key0 = range.tile(t < t_end ? t : (t_end > 0 ? t_end - 1 : 0)) << L::kShift;
      f.mask = t < t_end ? 0xffffffffu : 0;
      f.lane = (f.key0 >> kBlockShift) - pages.first;
    } else if (step == 1) {
      f.at.from = static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(pages.high, f.lane))) << 32 |
                  static_cast<uint32_t>(__builtin_amdgcn_readlane(pages.low, f.lane));
      f.mask &= __builtin_amdgcn_readlane(pages.there, f.lane);
    } else if (step == 2) {
      f.in_page = (f.key0 & (kBlockSize - 1)) * row_bytes + head_bytes;
      f.at.from += f.in_page;
    } else {
      const int left = s.keys - f.key0 < L::kKeys ? s.keys - f.key0 : L::kKeys;
      f.at.bytes = ((left - 1) * row_bytes + row_end) & f.mask;
    }
  };
  auto place_of = [&](int t) KVC_INLINE {
    ready(t);
    Search f;
#pragma unroll
    for (int i = 0; i < 4; ++i) seek(f, t, i);
    return f.at;
  };
  auto load = [&](const uint16_t* pool, const Place& p, u32x4 (&to)[L::kLoads]) KVC_INLINE {
    const auto tile = page_rsrc(pool, p.from, p.bytes);
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) to[i] = __builtin_amdgcn_raw_buffer_load_b128(tile, from, i * L::kStep * row_bytes, 0);
  };
  auto store_k = [&](int buffer) KVC_INLINE {
    char* const to = reinterpret_cast<char*>(k_tile[buffer]);
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i)
      *reinterpret_cast<u32x4*>(to + (k_to ^ L::k_turn(i * L::kStep)) + i * L::kStep * L::kBytes) = kst[i];
  };
  auto store_v = [&](int buffer) KVC_INLINE {
    char* const to = reinterpret_cast<char*>(v_tile[buffer]);
#pragma unroll
    for (int i = 0; i < L::kLoads; ++i) *reinterpret_cast<u32x4*>(to + v_to + i * L::kStep * L::kBytes) = vst[i];
  };
  // Of two groups of waves the second is half a tile behind the first, so one's
  // products run beside the other's softmax.  A group loads what the first one
  // needs in the next tile, which is one tile more ahead for the second.
  const int group = L::kGroups > 1 ? wave >> 2 : 0;

  const f32x16 kZero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  f32x16 acc[kBlocks];
  float m_run, l_run;
  // A weight of zero turns an infinity or NaN among V into NaN for rows that do
  // not see it.  That shows in the outputs: a workgroup that finds one there
  // goes over its keys again with care.  Returns whether the thread has one.
  auto go_over = [&](auto care) KVC_INLINE {
    constexpr bool careful = decltype(care)::value;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) acc[b] = kZero;
    m_run = kNegInf;
    // Weights of the tile before, and where its keys begin; none yet.
    vec_t pf[kKeyBlocks][2];
#pragma unroll
    for (int kb = 0; kb < kKeyBlocks; ++kb) pf[kb][0] = pf[kb][1] = __builtin_bit_cast(vec_t, u32x4{0, 0, 0, 0});
    int key0 = 0;
    float tops[4], sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // in four chains: one would wait for itself
    // The products of a tile: S^T = K Q^T (if `scores`) from buffer `now`, then
    // O^T += V^T P^T of the tile before, from buffer `before`.  A left operand is
    // read kAhead products before its use, and the order is the source's (left to
    // itself the compiler reads one into the registers that the product before has
    // just freed, and each waits for LDS).  beside(i) is done between products.
    constexpr int kScores = kKeyBlocks * kSteps, kValues = kKeyBlocks * 2 * kBlocks;
    constexpr int kAhead = 4;  // 6 to 12 are 2 to 7% slower at head_dim 256, one group's
    vec_t ring[kAhead];
    auto k_operand = [&](int buffer, int i) KVC_INLINE {
      const char* at = reinterpret_cast<const char*>(k_tile[buffer]) + (k_from ^ (i / kKeyBlocks << 5)) + (i % kKeyBlocks) * 32 * L::kBytes;
      return __builtin_bit_cast(vec_t, *reinterpret_cast<const u32x4*>(at));
    };
    auto v_operand = [&](int buffer, int i) KVC_INLINE {
      const char* at = reinterpret_cast<const char*>(v_tile[buffer]) + (v_from ^ (i % kBlocks << 6)) + (i / kBlocks) * 16 * L::kBytes;
      return join_columns<vec_t>(read_column(at), read_column(at + 8 * L::kBytes));
    };
    auto products = [&](auto scores, f32x16 (&sc)[kKeyBlocks], int now, int before, auto beside) KVC_INLINE {
      constexpr int kFirst = decltype(scores)::value ? 0 : kScores, kAll = kScores + kValues;
      auto operand = [&](int i) { return i < kScores ? k_operand(now, i) : v_operand(before, i - kScores); };
      each<kFirst, kAll>([&](auto step) KVC_INLINE {
        constexpr int i = decltype(step)::value;
        __builtin_amdgcn_sched_barrier(0);
        vec_t left = ring[(i - kFirst) % kAhead];
        if constexpr (i < kScores) {
          const int kb = i % kKeyBlocks, st = i / kKeyBlocks;
          sc[kb] = E::mfma32(left, qf[st], st ? sc[kb] : kZero);
        } else {
          const int b = (i - kScores) % kBlocks, kh = (i - kScores) / kBlocks, kb = kh >> 1, h = kh & 1;
          if constexpr (careful) {
            // Values that are not finite are added only to the rows that see them,
            // token by token.
            s16x8 raw = __builtin_bit_cast(s16x8, left), odd = {0, 0, 0, 0, 0, 0, 0, 0};
            bool any = false;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if ((static_cast<uint16_t>(raw[j]) & E::kExponent) == E::kExponent) {
                odd[j] = raw[j];
                raw[j] = 0;
                any = true;
              }
            left = __builtin_bit_cast(vec_t, raw);
            if (__any(any)) {
              for (int n = token_first; n <= token_last; ++n) {
                const RowSight one = sight_of(a, s, place0 + n);
                s16x8 seen = odd;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  if (!sees(one, a.sinks, key0 + kb * 32 + h * 16 + 8 * (j >> 2) + 4 * half + (j & 3))) seen[j] = 0;
                const f32x16 more = E::mfma32(__builtin_bit_cast(vec_t, seen), pf[kb][h], kZero);
                if (token == n) acc[b] += more;
              }
            }
          }
          acc[b] = E::mfma32(left, pf[kb][h], acc[b]);
        }
        if (i + kAhead < kAll) ring[(i - kFirst) % kAhead] = operand(i + kAhead);
        beside(i);
      });
      __builtin_amdgcn_sched_barrier(0);
    };
    // The maximum of a lane's scores.
    auto top_of = [&](const f32x16 (&sc)[kKeyBlocks], int e) KVC_INLINE { tops[e & 3] = fmaxf(tops[e & 3], sc[e >> 4][e & 15]); };
    auto all_tops = [&]() KVC_INLINE { return max_across_halves(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]))); };
    constexpr int kLane = kKeyBlocks * 16;  // scores of a lane
    // How far (as a power of two) weights may grow before the maximum moves.  fp16
    // shares its room between that and small weights: of the row's largest, half a
    // step is kept down to 2^-23 and what is below 2^-34 is lost.  With 4, 2^2 less,
    // 2048 tokens over 16384 keys, head_dim 256, take 628 us, with 6 613, with 8 601.
    constexpr int kSlack = F16 ? 6 : 8, kBelow = E::kRoom > kSlack ? E::kRoom - kSlack : 0;
    // The softmax of the scores in `sc`, whose maximum is `top`: masks and the
    // maximum, then the weights two by two, in `pf`.
    float m_use;
    // With one group a SIMD has 512 registers a wave, half of them for the matrix
    // products alone.  The outputs stay in those (left to itself the compiler moves
    // them out for the rare scaling and back at every tile).
    auto hold = [&]() KVC_INLINE {
      if constexpr (L::kGroups == 1) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) asm volatile("" : "+a"(acc[b]));
      }
    };
    auto prepare = [&](f32x16 (&sc)[kKeyBlocks], float top) KVC_INLINE {
      if (!(key0 + L::kKeys <= first.end && (key0 >= last.low || key0 + L::kKeys <= a.sinks))) {
        tops[0] = tops[1] = tops[2] = tops[3] = kNegInf;
#pragma unroll
        for (int e = 0; e < kLane; ++e) {
          const int i = e & 15;
          sc[e >> 4][i] = sees(sight, a.sinks, key0 + (e >> 4) * 32 + 8 * (i >> 2) + 4 * half + (i & 3)) ? sc[e >> 4][i] : kNegInf;
          top_of(sc, e);
        }
        top = all_tops();
      }
      top *= a.scale_log2;
      // The maximum moves only when it grows by more than kSlack: most tiles leave
      // the outputs unscaled.  Their difference is exact where it decides: a sum with
      // the maximum rounds to multiples of 16 where scores reach 2^27.
      const bool moves = top - m_run > kSlack + kBelow;
      if (__any(moves)) {
        const float m_new = moves ? lowered<kBelow>(top) : m_run;
        const float scale = m_new == kNegInf ? 1.0f : exp2_fast(m_run - m_new);
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[i] *= scale;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) acc[b] *= scale;
        m_run = m_new;
        hold();
      }
      m_use = m_run == kNegInf ? 0.0f : m_run;
    };
    auto weigh = [&](const f32x16 (&sc)[kKeyBlocks], int e) KVC_INLINE {
      const int kb = e >> 4, i = e & 15;
      const float p0 = exp2_fast(fmaf(sc[kb][i], a.scale_log2, -m_use)), p1 = exp2_fast(fmaf(sc[kb][i + 1], a.scale_log2, -m_use));
      u32x4 w = __builtin_bit_cast(u32x4, pf[kb][i >> 3]);
      w[i >> 1 & 3] = E::pack(p0, p1);
      sums[i >> 1 & 3] = E::add_pair(w[i >> 1 & 3], sums[i >> 1 & 3]);
      pf[kb][i >> 3] = __builtin_bit_cast(vec_t, w);
    };

    if constexpr (L::kGroups == 1) {
      // One group: a tile's weights are formed beside the scores' products of the
      // next one.
      load(a.k, place_of(t_begin), kst);
      load(a.v, place_of(t_begin), vst);
      uint32_t there = place_of(t_begin).bytes != 0;  // whether the tiles from t on are in the pool, t lowest
      store_k(0);
      store_v(0);
      Place ahead = place_of(t_begin + 1);
      there |= static_cast<uint32_t>(ahead.bytes != 0) << 1;
      load(a.k, ahead, kst);
      load(a.v, ahead, vst);
      store_k(1);
      ahead = place_of(t_begin + 2);  // of tile t + 2
      there |= static_cast<uint32_t>(ahead.bytes != 0) << 2;
      load(a.k, ahead, kst);
      ready(t_begin + 3);
      __syncthreads();
      f32x16 sc[2][kKeyBlocks];
#pragma unroll
      for (int i = 0; i < kScores; ++i) {
        const int kb = i % kKeyBlocks, st = i / kKeyBlocks;
        sc[0][kb] = E::mfma32(k_operand(0, i), qf[st], st ? sc[0][kb] : kZero);
      }
      tops[0] = tops[1] = tops[2] = tops[3] = kNegInf;
#pragma unroll
      for (int e = 0; e < kLane; ++e) top_of(sc[0], e);
      float top = all_tops();
      __syncthreads();
      auto turn = [&](auto parity, int t) KVC_INLINE {
        constexpr int own = decltype(parity)::value, other = 1 - own;  // of tile t and t + 1: buffers, scores
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ring[i] = k_operand(other, i);
        // No key of a page outside the pool is seen: its tile lies behind every row.
        key0 = there & 1 ? range.tile(t) << L::kShift : 1 << 30;
        hold();
        prepare(sc[own], top);
        Search search;
        tops[0] = tops[1] = tops[2] = tops[3] = kNegInf;
        products(std::true_type{}, sc[other], other, own, [&](int i) KVC_INLINE {
#pragma unroll
          for (int e = 0; e < kLane; e += 2)
            if (i == e / 2 * kScores / (kLane / 2)) weigh(sc[own], e);
          if (i == 1) store_k(own);    // tile t + 2; tile t's K was last read a barrier ago
          if (i == 3) store_v(other);  // tile t + 1
          if (i >= 4 && i < 8) seek(search, t + 3, i - 4);
          if (i == 8) load(a.v, ahead, vst);
          if (i == 9) load(a.k, search.at, kst);
          constexpr int kFrom = kScores + 2, kTo = kScores + kValues;  // the scores are there
#pragma unroll
          for (int e = 0; e < kLane; ++e)
            if (i == kFrom + e / 2 * 2 * (kTo - kFrom) / kLane) top_of(sc[other], e);
          if (i == kTo - 1) top = all_tops();
        });
        ahead = search.at;
        there = there >> 1 | static_cast<uint32_t>(search.at.bytes != 0) << 2;
        ready(t + 4);
        __syncthreads();
      };
      for (int t = t_begin; t < t_end; t += 2) {
        turn(std::integral_constant<int, 0>{}, t);
        turn(std::integral_constant<int, 1>{}, t + 1);  // no key of a tile behind the last one is seen
      }
    } else {
      f32x16 sc[kKeyBlocks];
      // The first tile of K, a tile of zeros as V before it, and what the second group
      // stores ahead; the next ones wait in registers.
      int now = 0, next = 1, before = 2;  // buffers of tiles t, t + 1 and t - 1
      Place old = place_of(t_begin);
      uint32_t there = old.bytes != 0;  // whether the last tiles that were asked for are in the pool, the latest lowest
      load(a.k, old, kst);
      store_k(now);
#pragma unroll
      for (int i = 0; i < L::kLoads; ++i) vst[i] = u32x4{0, 0, 0, 0};
      store_v(before);
      Place ahead = place_of(t_begin + 1);
      load(a.k, ahead, kst);
      load(a.v, old, vst);
      there = there << 1 | (ahead.bytes != 0);
      old = ahead;
      if (group) {
        store_k(next);
        store_v(now);
        ahead = place_of(t_begin + 2);
        load(a.k, ahead, kst);
        load(a.v, old, vst);
        there = there << 1 | (ahead.bytes != 0);
        old = ahead;
      }
      ready(t_begin + 2 + group);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kAhead; ++i) ring[i] = k_operand(now, i);
      if (group) __syncthreads();
      for (int t = t_begin; t < t_end; ++t) {
        // Products, beside them the tiles that wait in registers go to LDS, the ones
        // behind those are asked for, and the scores' maximum is taken.
        Search search;
        float top;
        tops[0] = tops[1] = tops[2] = tops[3] = kNegInf;
        __builtin_amdgcn_s_setprio(1);
        products(std::true_type{}, sc, now, before, [&](int i) KVC_INLINE {
          if (i == 1) store_k(group ? before : next);
          if (i == 2) store_v(group ? next : now);
          if (i >= 3 && i < 7) seek(search, t + 2 + group, i - 3);
          if (i == 7) load(a.v, old, vst);
          if (i == 8) load(a.k, search.at, kst);
          constexpr int kFrom = kScores + 2, kTo = kScores + kValues;  // the scores are there
#pragma unroll
          for (int e = 0; e < kLane; ++e)
            if (i == kFrom + e / 2 * 2 * (kTo - kFrom) / kLane) top_of(sc, e);
          if (i == kTo - 1) top = all_tops();
        });
        __builtin_amdgcn_s_setprio(0);
        there = there << 1 | (search.at.bytes != 0);
        old = search.at;
        // No key of a page outside the pool is seen: its tile lies behind every row.
        key0 = there >> (2 + group) & 1 ? range.tile(t) << L::kShift : 1 << 30;
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
        // Softmax.
        prepare(sc, top);
#pragma unroll
        for (int e = 0; e < kLane; e += 2) weigh(sc, e);
        ready(t + 3 + group);
        // The next products' first operands: they have been there for a phase.
        const int free = before;
        before = now;
        now = next;
        next = free;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ring[i] = k_operand(now, i);
        __builtin_amdgcn_sched_barrier(0);
        // Nothing was stored since the last barrier: no wait for LDS before this one.
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) ring[i] = v_operand(before, i);
      products(std::false_type{}, sc, now, before, [](int) {});
      if (!group) __syncthreads();
    }
    l_run = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    bool wild = false;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) wild |= !(fabsf(acc[b][i]) <= 3.4e38f);
    return wild;
  };
  if (__syncthreads_or(go_over(std::false_type{}))) go_over(std::true_type{});

  const float l_all = l_run + __shfl_xor(l_run, 32);
  int thread = tid;
  asm volatile("" : "+v"(thread));  // the row's place is worked out anew, not held through the loop
  const int local_row = (thread >> 6) * 32 + (thread & 31), m = row0 + local_row;
  if (m >= rows) return;
  if (!divided) {
    const float inv = l_all == 0.0f ? 0.0f : 1.0f / l_all;
    const int token = m / a.qpk, g = m - token * a.qpk;
    uint16_t* to = a.out + (s.token0 + token) * a.out_token_stride + (head * a.qpk + g) * a.out_head_stride;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = b * 32 + i * 8 + half * 4;
        if (d < a.head_dim)
          *gptr(reinterpret_cast<u32x2*>(to + d)) =
              u32x2{E::pack(acc[b][4 * i] * inv, acc[b][4 * i + 1] * inv), E::pack(acc[b][4 * i + 2] * inv, acc[b][4 * i + 3] * inv)};
      }
  } else {
    float* const piece = a.partial + ((static_cast<int64_t>(item) * a.kv_heads + head) * splits + split) * piece_floats(kRows, DP);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *gptr(reinterpret_cast<f32x4*>(piece + local_row * DP + b * 32 + i * 8 + half * 4)) =
            f32x4{acc[b][4 * i], acc[b][4 * i + 1], acc[b][4 * i + 2], acc[b][4 * i + 3]};
    if (half == 0) *gptr(reinterpret_cast<f32x2*>(piece + kRows * DP + 2 * local_row)) = f32x2{m_run, l_all};
  }
}

// Joins the splits of a (row tile, KV head), kJoinRows rows a workgroup.
template <bool F16, int DP>
__global__ __launch_bounds__(kJoinThreads) void attend_many_join_kernel(AttendArgs a, ManyGrid grid) {
  typedef AttendElem<F16> E;
  constexpr int kRows = many_rows(DP);
  const int head = blockIdx.x % a.kv_heads, item = blockIdx.x / a.kv_heads;
  const TileCount<kRows> counted(a, grid);
  const ManyShares shares(a, grid, counted.total());
  const int tile = shares.total - 1 - shares.whole - item;
  if (tile < 0) return;
  int request, local_tile;
  const Request s = counted.find(a, tile, &request, &local_tile);
  const int row0 = local_tile * kRows, left = s.fresh * a.qpk - row0;
  const int64_t size = piece_floats(kRows, DP);
  const float* const pieces = a.partial + (static_cast<int64_t>(item) * a.kv_heads + head) * shares.splits * size;
  const int begin = blockIdx.y * kJoinRows;
  join_pieces<DP, kJoinRows>(
      shares.splits, begin, left < begin + kJoinRows ? left : begin + kJoinRows, a.head_dim, kRows * DP,
      [&](int i) { return pieces + i * size; },
      [&](int local, int d, f32x4 x) {
        const int m = row0 + local, token = m / a.qpk, g = m - token * a.qpk;
        uint16_t* to = a.out + (s.token0 + token) * a.out_token_stride + (head * a.qpk + g) * a.out_head_stride;
        *gptr(reinterpret_cast<u32x2*>(to + d)) = u32x2{E::pack(x[0], x[1]), E::pack(x[2], x[3])};
      });
}

template <bool F16, int DP>
int launch(hipStream_t stream, const AttendArgs& a, const ManyGrid& grid) {
  constexpr int kRows = many_rows(DP);
  attend_many_kernel<F16, DP><<<static_cast<unsigned>(grid.grid), ManyLayout<DP>::kThreads, 0, stream>>>(a, grid);
  if (int rc = launch_status("kvc_attend_paged")) return rc;
  // Split items number half a round at most: each has two splits or more.
  const int64_t items = grid.grid - grid.round, split = items < grid.round / 2 ? items : grid.round / 2;
  if (grid.most_splits > 1)
    attend_many_join_kernel<F16, DP><<<dim3(static_cast<unsigned>(split), kRows / kJoinRows), kJoinThreads, 0, stream>>>(a, grid);
  return launch_status("kvc_attend_paged");
}

template <bool F16>
int pick_dim(hipStream_t stream, const AttendArgs& a, const ManyGrid& grid) {
  switch (padded_dim(a.head_dim)) {
    case 64: return launch<F16, 64>(stream, a, grid);
    case 96: return launch<F16, 96>(stream, a, grid);
    case 128: return launch<F16, 128>(stream, a, grid);
    case 192: return launch<F16, 192>(stream, a, grid);
    default: return launch<F16, 256>(stream, a, grid);
  }
}

}  // namespace

int launch_attend_many(hipStream_t stream, bool f16, const AttendArgs& a, const ManyGrid& grid) {
  return f16 ? pick_dim<true>(stream, a, grid) : pick_dim<false>(stream, a, grid);
}

}  // namespace kvc

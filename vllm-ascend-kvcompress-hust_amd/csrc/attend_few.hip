// Attention of requests with few rows (single tokens, a few drafted ones):
// every key is read once for at most 32 query rows, so the cache's bytes bound
// it.  Work is (request, KV head, page) tiles in that order, split evenly over
// the workgroups whatever the requests' lengths, so one long request beside
// short ones takes no longer than its share.  A workgroup's range may begin or
// end inside a (request, head): those pieces go to the workspace and a second
// launch joins them; a (request, head) inside one range is written at once.
//
// A workgroup's four waves take 32 keys each of a page.  Scores are formed
// transposed (S^T = K Q^T, 16x16x32): a lane then holds one query row's scores,
// and the same registers are the right operand of O^T = V^T P^T once keys are
// numbered as they lie in them: slot (lane/16, j) of a product's 32 keys is key
// 16*(j/4) + 4*(lane/16) + j%4.  K goes from memory to registers in operand
// order; V passes through the wave's own LDS, where ds_read_b64_tr_b16 turns
// rows into columns.

#include <type_traits>

#include "attend_internal.h"

namespace kvc {
namespace {

constexpr int kFewThreads = 256;
constexpr int kFewWaves = 4;
constexpr int kSliceKeys = 32;  // keys of a wave's slice of a page
// K and V are read once: non-temporal loads ran a decode batch of 16 x 16384
// tokens in 194 us, plain ones in 202.
constexpr int kNonTemporal = 2;

// V's place in LDS: rows of 64, 128 or 256 elements, whose 32-byte pairs are
// moved (an exclusive or with the row's `turn`) so that eight rows' same columns
// fall on different banks.  Lane l holds, of every kStep rows, row l / kSlots and
// 16-byte chunk l % kSlots.
template <int DP>
struct FewLayout {
  static constexpr int kRow = DP <= 64 ? 64 : (DP <= 128 ? 128 : 256);
  static constexpr int kSlots = kRow / 8;
  static constexpr int kStep = 64 / kSlots;
  static constexpr int kLoads = kSliceKeys / kStep;
  static constexpr int kBytes = kSliceKeys * kRow * 2;
  __device__ __forceinline__ static constexpr int turn(int row) { return kRow == 64 ? (row >> 1) & 3 : row & 7; }
  // Byte place of the lane's chunk of load i: `to` is that of load 0, whose rows
  // are below kStep, so the other rows' turns only set further bits.
  __device__ __forceinline__ static int chunk_at(int to, int i) { return (to ^ (turn(i * kStep) << 5)) + i * kStep * kRow * 2; }
};

// Workgroups of a compute unit (waves of a SIMD): as many as leave registers for
// the outputs, the queries, and a slice's K and V ahead of their use; each wave
// then has 64 x DP bytes in flight.
template <bool F16, int DP, int NQ>
__global__ __launch_bounds__(kFewThreads, few_residents(DP)) void attend_few_kernel(AttendArgs a) {
  typedef AttendElem<F16> E;
  typedef typename E::vec vec_t;
  constexpr int kSteps = DP / 32;   // 32-dim steps of K Q^T
  constexpr int kBlocks = DP / 16;  // 16-dim blocks of the output
  constexpr int kRows = 16 * NQ;
  typedef FewLayout<DP> Layout;
  __shared__ __attribute__((aligned(16))) uint16_t v_stage[kFewWaves][kSliceKeys * Layout::kRow];
  // Two row tiles' queries are read from LDS where they are used, in operand
  // order: held in registers they pushed others out to memory (16 requests of 3
  // tokens x 8 heads on 8 KV heads, head_dim 128, 16384 keys: 240 us, now 209).
  constexpr bool kQueriesHeld = NQ == 1;
  __shared__ u32x4 q_stage[kQueriesHeld ? 1 : NQ * kSteps * 64];
  __shared__ int before[kFewSequences + 1];
  __shared__ float wave_m[kFewWaves][kRows], wave_l[kFewWaves][kRows];
  __shared__ int wave_sum[kFewWaves];

  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, group = lane >> 4;
  const int wave = uniform(tid >> 6);

  // Tiles before each request.
  if (tid == 0) before[0] = 0;
  int carried = 0;
  for (int base = 0; base < a.n_seq; base += kFewThreads) {
    const int r = base + tid;
    int tiles = 0;
    if (r < a.n_seq) {
      const Request s = request_of(a, r);
      if (s.fresh > 0 && static_cast<int64_t>(s.fresh) * a.qpk <= a.few_rows) {
        tiles = tile_range<kBlockShift>(a, s, s.len - s.fresh, s.len - 1).count();
        tiles = (tiles < 1 ? 1 : tiles) * a.kv_heads;  // a request without keys is written by one empty tile a head
      }
    }
    int sum = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    int add = carried, all = 0;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
      if (w < wave) add += wave_sum[w];
      all += wave_sum[w];
    }
    if (r < a.n_seq) before[r + 1] = sum + add;
    carried += all;
    __syncthreads();
  }
  const int total = uniform(before[a.n_seq]);
  const int per = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  const int wg = blockIdx.x;
  if (tid == 0) a.header[4 * wg + 2] = 0;  // no pieces to join until one begins here
  int at = wg * per;
  const int range_begin = at;
  const int range_end = at + per < total ? at + per : total;
  if (at >= range_end) return;

  // The request that holds tile `at`.
  int r = 0;
  for (int span = kFewSequences / 2; span; span >>= 1)
    if (r + span < a.n_seq && before[r + span] <= at) r += span;

  const int row_elems = a.kv_heads * a.head_dim;
  // The lane's places in a slice, in bytes: its K chunk of row `col`, its V chunk
  // of the first rows (behind everything where the row has none), where that
  // chunk goes, and the column it reads first.
  const uint32_t row_bytes = row_elems * 2, k_lane = col * row_bytes + group * 16;
  const int v_row = lane / Layout::kSlots, v_chunk = lane & (Layout::kSlots - 1), read_row = 4 * group + (col >> 2);
  const uint32_t v_lane = v_chunk * 8 < a.head_dim ? v_row * row_bytes + v_chunk * 16 : 0x7fffffffu;
  char* const stage = reinterpret_cast<char*>(&v_stage[wave][0]);
  const int v_to = v_row * Layout::kRow * 2 + ((v_chunk * 16) ^ (Layout::turn(v_row) << 5));
  const int v_from = read_row * Layout::kRow * 2 + (Layout::turn(read_row) << 5) + (col & 3) * 8;
  while (at < range_end) {
    while (before[r + 1] <= at) ++r;
    r = uniform(r);
    const Request s = uniform_request_of(a, r);
    const TileRange pages = tile_range<kBlockShift>(a, s, s.len - s.fresh, s.len - 1);
    const int request_begin = uniform(before[r]);
    const int tiles = (uniform(before[r + 1]) - request_begin) / a.kv_heads;
    const int head = (at - request_begin) / tiles;
    const int whole_begin = request_begin + head * tiles;
    const int piece_first = at - whole_begin;
    const int piece_end = whole_begin + tiles < range_end ? whole_begin + tiles : range_end;
    const int piece_last = piece_end - whole_begin;
    const int32_t* const table = a.table + r * a.table_stride;
    const int rows = s.fresh * a.qpk;
    const int place0 = s.len - s.fresh;

    vec_t qf[kQueriesHeld ? kSteps : 1];
    RowSight sight[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int m = n * 16 + col;
      const int token = m / a.qpk, g = m - token * a.qpk;
      const bool inside = m < rows;
      const int place = place0 + token;
      sight[n] = sight_of(a, s, place);
      if (!inside) sight[n].end = 0;
      const uint16_t* row = a.q + (s.token0 + (inside ? token : 0)) * a.q_token_stride +
                            (head * a.qpk + (inside ? g : 0)) * a.q_head_stride;
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        const int d = st * 32 + group * 8;
        u32x4 w = {0, 0, 0, 0};
        if (!kQueriesHeld && (n * kSteps + st) % kFewWaves != wave) continue;
        if (inside && d < a.head_dim) w = *gptr(reinterpret_cast<const u32x4*>(row + d));
        if constexpr (kQueriesHeld)
          qf[st] = __builtin_bit_cast(vec_t, w);
        else
          q_stage[(n * kSteps + st) * 64 + lane] = w;
      }
    }
    if constexpr (!kQueriesHeld) __syncthreads();
    auto query = [&](int n, int st) {
      if constexpr (kQueriesHeld)
        return qf[st];
      else
        return __builtin_bit_cast(vec_t, q_stage[(n * kSteps + st) * 64 + lane]);
    };
    // The first pages' numbers beside the queries, both there before the loop: its
    // waits count its own loads alone.
    PageIds ids;
    ids.fill(table, a.max_blocks, pages.count() ? pages.tile(piece_first) : 0);
    __builtin_amdgcn_s_waitcnt(0x0f70);
    // Keys that some row sees, and those that every row sees.
    const int last_end = place0 + s.fresh < s.keys ? place0 + s.fresh : s.keys;
    const int first_end = place0 + 1 < s.keys ? place0 + 1 : s.keys;
    const int first_low = a.window ? place0 - a.window + 1 : 0;
    const int last_low = a.window ? s.len - a.window : 0;

    // The next slice of this wave, from tile t on, that some row sees and whose
    // page is in the pool.
    struct Slice {
      int tile, key0;
      uint64_t base;  // bytes
    };
    auto find = [&](int t) {
      Slice f = {t, 0, 0};
      if (pages.count() == 0) f.tile = piece_last;
      for (; f.tile < piece_last; ++f.tile) {
        const int block = pages.tile(f.tile);
        f.key0 = (block << kBlockShift) + wave * kSliceKeys;
        if (f.key0 >= last_end || (f.key0 + kSliceKeys <= first_low && f.key0 >= a.sinks)) continue;
        const int page = ids.at(table, a.max_blocks, block);
        if (page < 0 || page >= a.num_pages) continue;
        f.base = static_cast<uint64_t>(static_cast<uint32_t>(page)) * a.page_bytes + wave * kSliceKeys * row_bytes + head * a.head_dim * 2;
        break;
      }
      return f;
    };
    // Buffer loads: a scalar base, 32-bit lane offsets, and zeros from behind the
    // page (K) or the request's last row (V: whatever the page holds there).
    u32x4 kw[2][kSteps], vw[Layout::kLoads];
    auto load_k = [&](const Slice& f) {
      const auto from = page_rsrc(a.k, f.base, kSliceKeys * row_bytes - head * a.head_dim * 2);
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int st = 0; st < kSteps; ++st)
          kw[b][st] = __builtin_amdgcn_raw_buffer_load_b128(from, k_lane + st * 64, b * 16 * row_bytes, kNonTemporal);
    };
    auto load_v = [&](const Slice& f) {
      const int left = s.keys - f.key0 < kSliceKeys ? s.keys - f.key0 : kSliceKeys;
      const auto from = page_rsrc(a.v, f.base, (left - 1) * row_bytes + a.head_dim * 2);
#pragma unroll
      for (int i = 0; i < Layout::kLoads; ++i)
        vw[i] = __builtin_amdgcn_raw_buffer_load_b128(from, v_lane, i * Layout::kStep * row_bytes, kNonTemporal);
    };

    f32x4 acc[NQ][kBlocks];
    float m_run[NQ], l_run[NQ];
    // Weights of zero, and second words of any sign, turn an infinity or NaN
    // among V into NaN for rows that do not see it.  That shows in the outputs:
    // a wave that finds one there goes over its keys again with care.  Returns
    // whether there is one.
    auto go_over = [&](auto care) {
      constexpr bool careful = decltype(care)::value;
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        m_run[n] = kNegInf;
        l_run[n] = 0.0f;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) acc[n][b] = f32x4{0, 0, 0, 0};
      }

      Slice now = find(piece_first);
      if (now.tile < piece_last) {
        load_k(now);
        load_v(now);
      }
      while (now.tile < piece_last) {
        const int key0 = now.key0;
        // Worked out anew: places held through the loop are registers that loads ahead need.
        int to = v_to, column = v_from;
        asm volatile("" : "+v"(to), "+v"(column));
        const bool whole = key0 + kSliceKeys <= first_end && (key0 >= last_low || key0 + kSliceKeys <= a.sinks);
        const Slice next = find(now.tile + 1);
        if (a.head_dim != DP) {
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int st = 0; st < kSteps; ++st)
              if (st * 32 + group * 8 >= a.head_dim) kw[b][st] = u32x4{0, 0, 0, 0};
        }

        f32x4 sc[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            sc[n][b] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int st = 0; st < kSteps; ++st) sc[n][b] = E::mfma(__builtin_bit_cast(vec_t, kw[b][st]), query(n, st), sc[n][b]);
          }
        if (!careful && next.tile < piece_last) load_k(next);

        vec_t hi[NQ], lo[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          float x[8], top = kNegInf;
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = sc[n][j >> 2][j & 3] * a.scale_log2;
          if (!whole) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              x[j] = sees(sight[n], a.sinks, key0 + 16 * (j >> 2) + 4 * group + (j & 3)) ? x[j] : kNegInf;
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) top = fmaxf(top, x[j]);
          top = fmaxf(top, __shfl_xor(top, 16));
          top = max_across_halves(top);
          const float m_new = fmaxf(m_run[n], lowered<E::kRoom>(top));
          const float m_use = m_new == kNegInf ? 0.0f : m_new;
          const float scale = exp2_fast(m_run[n] - m_use);
          m_run[n] = m_new;
          float sum = 0.0f;
          u32x4 hw, lw;
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const float p0 = exp2_fast(x[j] - m_use), p1 = exp2_fast(x[j + 1] - m_use);
            sum += p0 + p1;
            // Weights in two 16-bit words (2^-16 of them left; in fp16 2^-22, or
            // 2^-40 of the row's largest): the second product costs nothing beside
            // the cache's bytes.
            hw[j >> 1] = E::pack(p0, p1);
            lw[j >> 1] = E::pack(p0 - E::lo(hw[j >> 1]), p1 - E::hi(hw[j >> 1]));
          }
          hi[n] = __builtin_bit_cast(vec_t, hw);
          lo[n] = __builtin_bit_cast(vec_t, lw);
          l_run[n] = l_run[n] * scale + sum;
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) acc[n][b] *= scale;
        }

#pragma unroll
        for (int i = 0; i < Layout::kLoads; ++i) *reinterpret_cast<u32x4*>(stage + Layout::chunk_at(to, i)) = vw[i];
        if (!careful && next.tile < piece_last) load_v(next);
        // The wave reads what it wrote itself: its LDS operations keep their order.
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          const char* from = stage + (column ^ ((b & 7) << 5)) + (b >> 3) * 256;
          const s16x4 v0 = read_column(from);
          const s16x4 v1 = read_column(from + 16 * Layout::kRow * 2);
          vec_t vf = join_columns<vec_t>(v0, v1);
          if constexpr (careful) {
            // Values that are not finite are added only to the rows that see them,
            // token by token, by the first word of their weights.
            s16x8 raw = __builtin_bit_cast(s16x8, vf), odd = {0, 0, 0, 0, 0, 0, 0, 0};
            bool any = false;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if ((static_cast<uint16_t>(raw[j]) & E::kExponent) == E::kExponent) {
                odd[j] = raw[j];
                raw[j] = 0;
                any = true;
              }
            vf = __builtin_bit_cast(vec_t, raw);
            if (__any(any)) {
              for (int i = 0; i < s.fresh; ++i) {
                const RowSight one = sight_of(a, s, place0 + i);
                s16x8 seen = odd;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  if (!sees(one, a.sinks, key0 + 16 * (j >> 2) + 4 * group + (j & 3))) seen[j] = 0;
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                  const f32x4 more = E::mfma(__builtin_bit_cast(vec_t, seen), hi[n], f32x4{0, 0, 0, 0});
                  if ((n * 16 + col) / a.qpk == i) acc[n][b] += more;
                }
              }
            }
          }
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            acc[n][b] = E::mfma(vf, hi[n], acc[n][b]);
            acc[n][b] = E::mfma(vf, lo[n], acc[n][b]);
          }
        }
        __builtin_amdgcn_wave_barrier();
        if (careful && next.tile < piece_last) {  // not ahead: registers that the fast pass has no use for
          load_k(next);
          load_v(next);
        }
        now = next;
      }
      bool wild = false;
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) wild |= !(fabsf(acc[n][b][i]) <= 3.4e38f);
      return wild;
    };
    if (__any(go_over(std::false_type{}))) go_over(std::true_type{});

    // Join the four waves: a common maximum, then sums.
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float l = l_run[n];
      l += __shfl_xor(l, 16);
      l += __shfl_xor(l, 32);
      l_run[n] = l;
      if (group == 0) {
        wave_m[wave][n * 16 + col] = m_run[n];
        wave_l[wave][n * 16 + col] = l;
      }
    }
    __syncthreads();
    float m_all[NQ], l_all[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int m = n * 16 + col;
      float top = kNegInf;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) top = fmaxf(top, wave_m[w][m]);
      const float use = top == kNegInf ? 0.0f : top;
      float l = 0.0f;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) l += wave_l[w][m] * exp2_fast(wave_m[w][m] - use);
      const float scale = exp2_fast(m_run[n] - use);
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) acc[n][b] *= scale;
      m_all[n] = top;
      l_all[n] = l;
    }
    // 16 rows x DP floats a tile and wave, waves 2, 3 then 1 into 0, 1 then 0.
    float* const pool = reinterpret_cast<float*>(&v_stage[0][0]);
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int half = 2; half >= 1; half >>= 1) {
        __syncthreads();
        if (wave >= half && wave < 2 * half) {
          float* to = pool + (wave - half) * (DP * 16);
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) *reinterpret_cast<f32x4*>(to + (b * 64 + lane) * 4) = acc[n][b];
        }
        __syncthreads();
        if (wave < half) {
          const float* from = pool + wave * (DP * 16);
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) acc[n][b] += *reinterpret_cast<const f32x4*>(from + (b * 64 + lane) * 4);
        }
      }

    const bool complete = piece_first == 0 && piece_last == tiles;
    if (wave == 0) {
      const int kind = at == range_begin ? 0 : 1;
      float* const piece = a.partial + (2 * static_cast<int64_t>(wg) + kind) * piece_floats(kRows, DP);
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int m = n * 16 + col;
        if (m >= rows) continue;
        if (complete) {
          const float inv = l_all[n] == 0.0f ? 0.0f : 1.0f / l_all[n];
          const int token = m / a.qpk, g = m - token * a.qpk;
          uint16_t* to = a.out + (s.token0 + token) * a.out_token_stride + (head * a.qpk + g) * a.out_head_stride;
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            const int d = b * 16 + group * 4;
            if (d < a.head_dim)
              *gptr(reinterpret_cast<u32x2*>(to + d)) =
                  u32x2{E::pack(acc[n][b][0] * inv, acc[n][b][1] * inv), E::pack(acc[n][b][2] * inv, acc[n][b][3] * inv)};
          }
        } else {
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) *gptr(reinterpret_cast<f32x4*>(piece + m * DP + b * 16 + group * 4)) = acc[n][b];
          if (group == 0) *gptr(reinterpret_cast<f32x2*>(piece + kRows * DP + 2 * m)) = f32x2{m_all[n], l_all[n]};
        }
      }
      if (!complete && piece_first == 0 && lane == 0) {
        // The (request, head) goes on in the next workgroups: `count` pieces in all.
        a.header[4 * wg] = s.token0;
        a.header[4 * wg + 1] = rows;
        a.header[4 * wg + 2] = (whole_begin + tiles - 1) / per - wg + 1;
        a.header[4 * wg + 3] = head << 1 | kind;
      }
    }
    at = piece_end;
    __syncthreads();
  }
}

// Joins the pieces of the (request, head) that begins in workgroup blockIdx.x
// and ends in a later one, four rows a workgroup:
// out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.
template <bool F16, int DP, int NQ>
__global__ __launch_bounds__(kFewThreads) void attend_few_join_kernel(AttendArgs a) {
  typedef AttendElem<F16> E;
  constexpr int kRows = 16 * NQ;
  const int wg = blockIdx.x, row0 = blockIdx.y * 4;
  const int count = scalar_at(a.header, 4 * wg + 2);
  if (count < 2) return;
  const int token0 = scalar_at(a.header, 4 * wg), rows = scalar_at(a.header, 4 * wg + 1);
  const int head = scalar_at(a.header, 4 * wg + 3) >> 1, kind = scalar_at(a.header, 4 * wg + 3) & 1;
  if (row0 >= rows) return;
  const int64_t size = piece_floats(kRows, DP);
  const float* const first = a.partial + (2 * static_cast<int64_t>(wg) + kind) * size;
  const float* const rest = a.partial + 2 * static_cast<int64_t>(wg) * size;  // piece i > 0 at 2*i*size
  join_pieces<DP, 4>(
      count, row0, rows, a.head_dim, kRows * DP, [&](int i) { return i ? rest + 2 * i * size : first; },
      [&](int m, int d, f32x4 x) {
        const int token = m / a.qpk, g = m - token * a.qpk;
        uint16_t* to = a.out + (token0 + token) * a.out_token_stride + (head * a.qpk + g) * a.out_head_stride;
        *gptr(reinterpret_cast<u32x2*>(to + d)) = u32x2{E::pack(x[0], x[1]), E::pack(x[2], x[3])};
      });
}

template <bool F16, int DP, int NQ>
int launch(hipStream_t stream, const AttendArgs& a, int workgroups) {
  attend_few_kernel<F16, DP, NQ><<<workgroups, kFewThreads, 0, stream>>>(a);
  if (int rc = launch_status("kvc_attend_paged")) return rc;
  if (workgroups > 1) attend_few_join_kernel<F16, DP, NQ><<<dim3(workgroups, 4 * NQ), kFewThreads, 0, stream>>>(a);
  return launch_status("kvc_attend_paged");
}

template <bool F16, int DP>
int pick_rows(hipStream_t stream, const AttendArgs& a, int workgroups, int row_tiles) {
  return row_tiles == 1 ? launch<F16, DP, 1>(stream, a, workgroups) : launch<F16, DP, 2>(stream, a, workgroups);
}

template <bool F16>
int pick_dim(hipStream_t stream, const AttendArgs& a, int workgroups, int row_tiles) {
  switch (padded_dim(a.head_dim)) {
    case 64: return pick_rows<F16, 64>(stream, a, workgroups, row_tiles);
    case 96: return pick_rows<F16, 96>(stream, a, workgroups, row_tiles);
    case 128: return pick_rows<F16, 128>(stream, a, workgroups, row_tiles);
    case 192: return pick_rows<F16, 192>(stream, a, workgroups, row_tiles);
    default: return pick_rows<F16, 256>(stream, a, workgroups, row_tiles);
  }
}

}  // namespace

int launch_attend_few(hipStream_t stream, bool f16, const AttendArgs& a, int workgroups, int row_tiles) {
  return f16 ? pick_dim<true>(stream, a, workgroups, row_tiles) : pick_dim<false>(stream, a, workgroups, row_tiles);
}

}  // namespace kvc

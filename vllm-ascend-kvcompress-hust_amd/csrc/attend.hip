// Entry of the attention over a paged cache: checks, launch sizes, workspace.

#include <math.h>

#include "attend_internal.h"
#include "row_sets.h"

namespace kvc {
namespace {

constexpr int kCompute = 256;  // compute units of the device
// Rows (tokens x query heads a KV head) of a call: the kernels number them, and the
// places of a last tile behind them, in 32 bits.
constexpr int64_t kMostRows = (1ll << 31) - 256;

// How a call is launched; the workspace query and the call agree by sharing it.
struct AttendPlan {
  int row_tiles;    // 16-row tiles a request of the few-rows kernel has at most; 0: kernel not needed
  int workgroups;   // of the few-rows kernel
  ManyGrid many;    // of the many-rows kernel; no grid: kernel not needed
  size_t bytes;     // workspace
};

AttendPlan make_plan(int kv_heads, int qpk, int head_dim, int n_seq, int64_t num_tokens, int max_query_len, int max_seq_len) {
  AttendPlan p = {};
  const int dim = padded_dim(head_dim);
  const int64_t most_rows = static_cast<int64_t>(max_query_len) * qpk;
  const int64_t pages = ceil_div(max_seq_len > 0 ? max_seq_len : 1, kBlockSize);
  size_t few = 0, many = 0;
  // A small batch that needs the many-rows kernel leaves it the few rows too: its
  // padding costs less than a launch of each kind.  Requests of one to four tokens
  // (8 heads each) beside a chunk of 256, head_dim 64 / 128 / 256:
  //   7 of 4096 keys, 2 KV heads   40 / 48 / 67 us, apart 60 / 75 / 100
  //   31 of 2048, 8 KV heads       70 / 97 / 158,   apart 89 / 114 / 176
  //   63 of 4096, 8 KV heads       195 / 298 / 480, apart 185 / 263 / 482
  // The lengths of one batch are alike there.  The rule sees the longest one's bound
  // only: a token at 32768 keys beside six at 700 and the chunk (2 KV heads, head_dim
  // 128) takes 110 us, apart 65; and it counts keys that a window hides: 15 tokens at
  // 32768 keys with a window of 1024 (8 KV heads) take 68 apart, together 50.
  const bool together = most_rows > kFewRows * kFewTilesMost &&
                        static_cast<int64_t>(n_seq) * kv_heads * max_seq_len <= (1 << 19);
  if (qpk <= kFewRows * kFewTilesMost) {
    const int row_tiles = most_rows <= kFewRows ? 1 : kFewTilesMost;
    const int64_t sequences = n_seq < kFewSequences ? n_seq : kFewSequences;
    const int64_t bound = sequences * kv_heads * pages;
    const int64_t resident = kCompute * few_residents(dim);
    const int workgroups = static_cast<int>(bound < resident ? bound : resident);
    // Asked for also where the many-rows kernel takes all: a workspace for the
    // largest step then serves the smaller ones too.
    few = static_cast<size_t>(workgroups) * (16 + 8 * piece_floats(kFewRows * row_tiles, dim));
    if (!together) {
      p.row_tiles = row_tiles;
      p.workgroups = workgroups;
    }
  }
  if (most_rows > kFewRows * p.row_tiles) {
    // Row tiles are at most as many as all rows fill, and a partly filled one more
    // for each request that has more rows than the few-rows kernel takes; one
    // round more of workgroups is there for the items that are split, into one
    // piece for every 512 keys of the longest request at most (a shorter one's
    // pieces hold fewer keys, or none).
    const int64_t rows = num_tokens * qpk, most = rows / (kFewRows * p.row_tiles + 1);
    const int64_t tiles = rows / many_rows(dim) + (most < n_seq ? most : n_seq);
    p.many.round = kCompute;  // one workgroup a compute unit
    p.many.grid = tiles * kv_heads + p.many.round;
    p.many.most_tiles = static_cast<uint32_t>(tiles);
    const int64_t by_keys = pages * kBlockSize / 512;
    p.many.most_splits = static_cast<int>(by_keys < 1 ? 1 : (by_keys > p.many.round ? p.many.round : by_keys));
    if (p.many.most_splits > 1) many = static_cast<size_t>(p.many.round) * piece_floats(many_rows(dim), dim) * 4;
  }
  p.bytes = few > many ? few : many;
  if (p.bytes == 0) p.bytes = 16;
  return p;
}

bool good_shape(int kv_heads, int qpk, int head_dim, int n_seq, int64_t num_tokens, int max_query_len, int max_seq_len) {
  return kv_heads > 0 && qpk > 0 && kv_heads <= 1024 && qpk <= 1024 && head_dim > 0 && head_dim % 8 == 0 && padded_dim(head_dim) &&
         n_seq >= 0 && num_tokens >= 0 && num_tokens < (1 << 24) && n_seq < (1 << 24) && max_query_len >= 0 && max_seq_len >= 0 &&
         num_tokens * qpk < kMostRows;
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" size_t kvc_attend_workspace_bytes(int kv_heads, int qpk, int head_dim, int n_seq, int64_t num_tokens,
                                             int max_query_len, int max_seq_len) {
  if (!good_shape(kv_heads, qpk, head_dim, n_seq, num_tokens, max_query_len, max_seq_len)) return 0;
  return make_plan(kv_heads, qpk, head_dim, n_seq, num_tokens, max_query_len, max_seq_len).bytes;
}

extern "C" int kvc_attend_paged(kvc_stream_t stream, int dtype, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                const void* k_cache, const void* v_cache, int64_t num_pages, int64_t page_stride, int kv_heads,
                                int qpk, int head_dim, int n_seq, int64_t num_tokens, const int32_t* query_start_loc,
                                const int32_t* seq_lens, const int32_t* block_table, int64_t block_table_stride, int max_blocks,
                                int max_query_len, int max_seq_len, float scale, int window, int sinks, void* out,
                                int64_t out_token_stride, int64_t out_head_stride, void* workspace, size_t workspace_bytes) {
  if (dtype != KVC_DTYPE_BF16 && dtype != KVC_DTYPE_FP16) return fail(KVC_EINVAL, "kvc_attend_paged: dtype must be bf16 or fp16");
  if (!good_shape(kv_heads, qpk, head_dim, n_seq, num_tokens, max_query_len, max_seq_len))
    return fail(KVC_EINVAL,
                "kvc_attend_paged: bad sizes (head_dim %d must be a multiple of 8 up to 256; kv_heads %d, qpk %d at most 1024; "
                "n_seq %d, num_tokens %lld below 2^24, num_tokens * qpk below 2^31 - 256)",
                head_dim, kv_heads, qpk, n_seq, static_cast<long long>(num_tokens));
  if (num_pages < 0 || page_stride < static_cast<int64_t>(kBlockSize) * kv_heads * head_dim || page_stride % 8 ||
      page_stride >= (1ll << 31))
    return fail(KVC_EINVAL, "kvc_attend_paged: page_stride must be a multiple of 8 elements, at least one page and below 2^31");
  if (max_blocks < 0 || max_blocks >= (1 << 23) || block_table_stride < max_blocks)
    return fail(KVC_EINVAL, "kvc_attend_paged: max_blocks must be below 2^23 and at most block_table_stride");
  if (!(scale > 0.0f) || !isfinite(scale)) return fail(KVC_EINVAL, "kvc_attend_paged: scale must be positive and finite");
  if (window < 0 || sinks < 0) return fail(KVC_EINVAL, "kvc_attend_paged: window and sinks must be non-negative");
  if (n_seq == 0 || num_tokens == 0 || max_query_len == 0) return 0;
  if (!q || !out || !query_start_loc || !seq_lens || (max_blocks > 0 && !block_table) || (num_pages > 0 && (!k_cache || !v_cache)))
    return fail(KVC_EINVAL, "kvc_attend_paged: null pointer");
  const uintptr_t bases = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(k_cache) |
                          reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(workspace);
  if (bases % 16 || (q_token_stride | q_head_stride | out_token_stride | out_head_stride) % 8)
    return fail(KVC_EINVAL, "kvc_attend_paged: pointers must be 16-byte aligned and strides multiples of 8 elements");
  const AttendPlan plan = make_plan(kv_heads, qpk, head_dim, n_seq, num_tokens, max_query_len, max_seq_len);
  if (!workspace || workspace_bytes < plan.bytes)
    return fail(KVC_EINVAL, "kvc_attend_paged: workspace too small (%zu of %zu bytes)", workspace_bytes, plan.bytes);
  if (plan.many.grid * many_threads(padded_dim(head_dim)) > kMaxDispatchItems)
    return fail(KVC_EINVAL, "kvc_attend_paged: too many rows for one launch (num_tokens * query heads / %d x %d threads, below 2^32)",
                many_rows(padded_dim(head_dim)), many_threads(padded_dim(head_dim)));
  // Tile numbers are 32-bit: requests x heads x pages of a few-rows launch stay below 2^30.
  const int64_t each = static_cast<int64_t>(kv_heads) * (max_blocks > 0 ? max_blocks : 1);
  if (plan.row_tiles && each > (1 << 30)) return fail(KVC_EINVAL, "kvc_attend_paged: kv_heads x max_blocks must be at most 2^30");
  const RowSet read = row_set(q, q_token_stride, q_head_stride, num_tokens, kv_heads * qpk);
  const RowSet written = row_set(out, out_token_stride, out_head_stride, num_tokens, kv_heads * qpk);
  if (rows_share(written, 2 * head_dim)) return fail(KVC_EINVAL, "kvc_attend_paged: rows of out overlap each other");
  if (rows_meet(written, read, 2 * head_dim)) return fail(KVC_EINVAL, "kvc_attend_paged: out overlaps q");

  AttendArgs a = {};
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.k = static_cast<const uint16_t*>(k_cache);
  a.v = static_cast<const uint16_t*>(v_cache);
  a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.out_token_stride = out_token_stride;
  a.out_head_stride = out_head_stride;
  a.num_pages = num_pages < 0x7fffffff ? static_cast<int>(num_pages) : 0x7fffffff;
  a.page_bytes = static_cast<uint32_t>(page_stride * 2);
  a.table_stride = block_table_stride;
  a.num_tokens = num_tokens;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.kv_heads = kv_heads;
  a.qpk = qpk;
  a.head_dim = head_dim;
  a.max_blocks = max_blocks;
  a.window = window < (1 << 30) ? window : 0;  // the table covers fewer keys than that
  a.sinks = sinks;
  a.few_rows = kFewRows * plan.row_tiles;
  const hipStream_t st = as_stream(stream);
  const bool f16 = dtype == KVC_DTYPE_FP16;
  if (plan.row_tiles) {
    a.header = static_cast<int32_t*>(workspace);
    a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + 16 * static_cast<size_t>(plan.workgroups));
    int64_t chunk = (1 << 30) / each;
    if (chunk > kFewSequences) chunk = kFewSequences;
    for (int64_t base = 0; base < n_seq; base += chunk) {
      a.n_seq = static_cast<int>(n_seq - base < chunk ? n_seq - base : chunk);
      a.start = query_start_loc + base;
      a.seq_lens = seq_lens + base;
      a.table = block_table + base * block_table_stride;
      if (int rc = launch_attend_few(st, f16, a, plan.workgroups, plan.row_tiles)) return rc;
    }
  }
  if (plan.many.grid) {
    a.n_seq = n_seq;
    a.start = query_start_loc;
    a.seq_lens = seq_lens;
    a.table = block_table;
    a.partial = static_cast<float*>(workspace);
    ManyGrid grid = plan.many;
    if (a.window) {  // a row tile's keys are fewer than the request's
      const int64_t most = (static_cast<int64_t>(a.window) + sinks + many_rows(padded_dim(head_dim))) / 512;
      if (most < grid.most_splits) grid.most_splits = most < 1 ? 1 : static_cast<int>(most);
    }
    if (int rc = launch_attend_many(st, f16, a, grid)) return rc;
  }
  return 0;
}

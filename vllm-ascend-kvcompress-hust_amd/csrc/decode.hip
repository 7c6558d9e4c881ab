// Decode-side consumers of a compacted cache: physical positions, slot
// mapping and attention lengths.
//
// Compaction keeps semantic RoPE positions monotonic; only where a token's K/V
// row lives moves.  A request compacted from semantic length S to physical
// length P carries offset S - P (pkg/provider.py:52-54), and every later token
// of that request is written at physical position semantic - offset
// (shift_positions, tri/kernels.py:35-47, used by the slot-mapping hook
// pkg/provider.py:687-705 ahead of the host's compute_slot_mapping).  The
// attention lengths shrink by the same offset (pkg/provider.py:707-728).
//
// All three are integer gathers over a few thousand entries per step: one
// thread per entry, no LDS.  The step tables form all of them, and the block
// table itself, from the requests' lengths in one launch.

#include "kvc_common.h"
#include "row_sets.h"

namespace kvc {
namespace {

constexpr int kDecodeThreads = 256;

__device__ __forceinline__ int64_t load_index(const void* p, int bytes, int64_t i) {
  return bytes == 4 ? static_cast<int64_t>(static_cast<const int32_t*>(p)[i]) : static_cast<const int64_t*>(p)[i];
}

__global__ __launch_bounds__(kDecodeThreads) void shift_positions_kernel(const int64_t* __restrict__ positions,
                                                                         const void* __restrict__ request_indices,
                                                                         int index_bytes,
                                                                         const int64_t* __restrict__ offsets, int64_t n,
                                                                         int64_t* __restrict__ out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kDecodeThreads + threadIdx.x;
  if (i >= n) return;
  out[i] = positions[i] - offsets[load_index(request_indices, index_bytes, i)];
}

// One workgroup per request (grid-stride over requests); the request's tokens
// are [query_start_loc[r], query_start_loc[r+1]).  Tokens past the last
// request (graph padding) get -1, as do positions outside the block table.
__global__ __launch_bounds__(kDecodeThreads) void slot_mapping_kernel(
    int num_reqs, const int32_t* __restrict__ query_start_loc, const int64_t* __restrict__ positions,
    const int64_t* __restrict__ offsets, const int32_t* __restrict__ block_table, int64_t table_stride,
    int max_blocks, int block_size, int64_t num_tokens, int64_t* __restrict__ slot_mapping,
    int64_t* __restrict__ physical_out) {
  for (int r = blockIdx.x; r <= num_reqs; r += gridDim.x) {
    if (r == num_reqs) {
      // Padding tokens after the last request.
      for (int64_t i = query_start_loc[num_reqs] + threadIdx.x; i < num_tokens; i += kDecodeThreads) {
        slot_mapping[i] = -1;
        if (physical_out) physical_out[i] = positions[i];
      }
      continue;
    }
    const int64_t begin = query_start_loc[r];
    const int64_t end = query_start_loc[r + 1];
    const int64_t off = offsets ? offsets[r] : 0;
    const int32_t* row = block_table + static_cast<int64_t>(r) * table_stride;
    for (int64_t i = begin + threadIdx.x; i < end && i < num_tokens; i += kDecodeThreads) {
      const int64_t p = positions[i] - off;
      const int64_t blk = p >= 0 ? p / block_size : -1;
      int64_t slot = -1;
      if (blk >= 0 && blk < max_blocks) {
        const int64_t page = row[blk];
        if (page >= 0) slot = page * block_size + (p - blk * block_size);
      }
      slot_mapping[i] = slot;
      if (physical_out) physical_out[i] = p;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kDecodeThreads) void shift_lengths_kernel(T* __restrict__ seq_lens,
                                                                       const int64_t* __restrict__ offsets,
                                                                       int num_reqs) {
  const int r = blockIdx.x * kDecodeThreads + threadIdx.x;
  if (r >= num_reqs) return;
  seq_lens[r] = static_cast<T>(static_cast<int64_t>(seq_lens[r]) - offsets[r]);
}

struct StepTables {
  const int32_t *computed, *fresh;
  const int64_t *offsets, *ids, *id_offsets;
  int32_t *start, *seq_lens, *table;
  int64_t *positions, *slots;
  int64_t table_stride, num_tokens;
  int n_seq, expand, max_blocks, shares;
};

// Page j (of 128 tokens) of a request whose scheduler pages are ids[0 .. count),
// each `expand` pages long; -1 where there is none.
__device__ __forceinline__ int32_t step_page(const int64_t* ids, int64_t count, int expand, int j) {
  const int at = j / expand;
  if (at >= count) return -1;
  const int64_t id = ids[at];
  if (id < 0 || id > (0x7fffffffll - expand) / expand) return -1;
  return static_cast<int32_t>(id) * expand + (j - at * expand);
}

// Workgroup (r, share) writes request r's row of every table, the row's entries
// and tokens spread over the shares; the workgroups behind the last request
// write the padding tokens.  Each adds up the new tokens of all requests before its
// own itself (n^2 / 2 reads of 4 bytes a share, from L2): no launch or wait between
// the sum and its readers.  64 requests 3.6 us, 512 with 24 chunks among them 5.3:
// the dependent loads, the tables' bytes take less than 1.
__global__ __launch_bounds__(kDecodeThreads) void step_tables_kernel(StepTables a) {
  __shared__ int64_t part[kDecodeThreads / 64];
  const int r = blockIdx.x / a.shares, share = blockIdx.x - r * a.shares;
  int64_t sum = 0;
  for (int i = threadIdx.x; i < r; i += kDecodeThreads) {
    const int n = a.fresh[i];
    sum += n > 0 ? n : 0;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int w = 0; w < kDecodeThreads / 64; ++w) sum += part[w];
  // Tokens that the buffers have no room for are dropped, here and for every request behind.
  const int64_t start = sum < a.num_tokens ? sum : a.num_tokens;
  const int thread = share * kDecodeThreads + threadIdx.x, threads = a.shares * kDecodeThreads;
  if (r == a.n_seq) {
    if (thread == 0) a.start[r] = static_cast<int32_t>(start);
    for (int64_t i = start + thread; i < a.num_tokens; i += threads) {
      a.slots[i] = -1;
      a.positions[i] = 0;
    }
    return;
  }
  const int64_t wanted = a.fresh[r] > 0 ? a.fresh[r] : 0;
  const int64_t fresh = wanted < a.num_tokens - start ? wanted : a.num_tokens - start;
  const int64_t computed = a.computed[r], offset = a.offsets ? a.offsets[r] : 0;
  int64_t len = computed + fresh - offset;
  len = len < 0 ? 0 : (len > 0x7fffffff ? 0x7fffffff : len);
  if (thread == 0) {
    a.start[r] = static_cast<int32_t>(start);
    a.seq_lens[r] = static_cast<int32_t>(len);
  }
  const int64_t first = a.id_offsets[r], count = a.id_offsets[r + 1] - first;
  const int64_t* ids = a.ids + first;
  for (int j = thread; j < a.max_blocks; j += threads)
    a.table[r * a.table_stride + j] =
        static_cast<int64_t>(j) << kBlockShift < len ? step_page(ids, count, a.expand, j) : -1;
  for (int64_t i = thread; i < fresh; i += threads) {
    const int64_t p = computed + i - offset, j = p >> kBlockShift;
    int64_t slot = -1;
    if (p >= 0 && j < a.max_blocks) {
      const int64_t page = step_page(ids, count, a.expand, static_cast<int>(j));
      if (page >= 0) slot = (page << kBlockShift) + (p & (kBlockSize - 1));
    }
    a.slots[start + i] = slot;
    a.positions[start + i] = computed + i;
  }
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" int kvc_shift_positions(kvc_stream_t stream, const int64_t* positions, const void* request_indices,
                                   int index_bytes, const int64_t* request_offsets, int64_t n,
                                   int64_t* output) {
  if (n < 0) return fail(KVC_EINVAL, "kvc_shift_positions: n must be non-negative");
  if (index_bytes != 4 && index_bytes != 8)
    return fail(KVC_EINVAL, "kvc_shift_positions: index_bytes must be 4 or 8");
  if (n == 0) return 0;
  if (!positions || !request_indices || !request_offsets || !output)
    return fail(KVC_EINVAL, "kvc_shift_positions: null pointer");
  shift_positions_kernel<<<static_cast<unsigned>(ceil_div(n, kDecodeThreads)), kDecodeThreads, 0,
                           as_stream(stream)>>>(positions, request_indices, index_bytes, request_offsets, n,
                                                output);
  return launch_status("kvc_shift_positions");
}

extern "C" int kvc_physical_slot_mapping(kvc_stream_t stream, int num_reqs, const int32_t* query_start_loc,
                                         const int64_t* positions, const int64_t* request_offsets,
                                         const int32_t* block_table, int64_t block_table_stride, int max_blocks,
                                         int block_size, int64_t num_tokens, int64_t* slot_mapping,
                                         int64_t* physical_positions) {
  if (num_reqs < 0 || num_tokens < 0 || max_blocks < 0 || block_size <= 0)
    return fail(KVC_EINVAL, "kvc_physical_slot_mapping: bad sizes");
  if (block_table_stride < max_blocks)
    return fail(KVC_EINVAL, "kvc_physical_slot_mapping: block_table_stride < max_blocks");
  if (num_tokens == 0) return 0;
  if (!query_start_loc || !positions || !slot_mapping || (num_reqs > 0 && !block_table))
    return fail(KVC_EINVAL, "kvc_physical_slot_mapping: null pointer");
  const unsigned blocks = static_cast<unsigned>(num_reqs + 1 < 4096 ? num_reqs + 1 : 4096);
  slot_mapping_kernel<<<blocks, kDecodeThreads, 0, as_stream(stream)>>>(
      num_reqs, query_start_loc, positions, request_offsets, block_table, block_table_stride, max_blocks,
      block_size, num_tokens, slot_mapping, physical_positions);
  return launch_status("kvc_physical_slot_mapping");
}

extern "C" int kvc_shift_lengths(kvc_stream_t stream, void* seq_lens, int elem_bytes, const int64_t* request_offsets,
                                 int num_reqs) {
  if (num_reqs < 0) return fail(KVC_EINVAL, "kvc_shift_lengths: num_reqs must be non-negative");
  if (elem_bytes != 4 && elem_bytes != 8) return fail(KVC_EINVAL, "kvc_shift_lengths: elem_bytes must be 4 or 8");
  if (num_reqs == 0) return 0;
  if (!seq_lens || !request_offsets) return fail(KVC_EINVAL, "kvc_shift_lengths: null pointer");
  const unsigned blocks = static_cast<unsigned>(ceil_div(num_reqs, kDecodeThreads));
  if (elem_bytes == 4)
    shift_lengths_kernel<int32_t><<<blocks, kDecodeThreads, 0, as_stream(stream)>>>(static_cast<int32_t*>(seq_lens),
                                                                                     request_offsets, num_reqs);
  else
    shift_lengths_kernel<int64_t><<<blocks, kDecodeThreads, 0, as_stream(stream)>>>(static_cast<int64_t*>(seq_lens),
                                                                                     request_offsets, num_reqs);
  return launch_status("kvc_shift_lengths");
}

extern "C" int kvc_step_tables(kvc_stream_t stream, int n_seq, const int32_t* computed_tokens, const int32_t* new_tokens,
                               const int64_t* request_offsets, const int64_t* block_ids, const int64_t* block_offsets,
                               int page_tokens, int max_query_len, int64_t num_tokens, int max_blocks, int64_t block_table_stride,
                               int32_t* query_start_loc, int32_t* seq_lens, int64_t* positions, int64_t* slot_mapping,
                               int32_t* block_table) {
  // A workgroup a request and one for the padding, in one dispatch of less than 2^32 work-items.
  if (n_seq < 0 || n_seq >= (1 << 24) - 1 || num_tokens < 0 || num_tokens >= (1ll << 31) || max_query_len < 0)
    return fail(KVC_EINVAL, "kvc_step_tables: bad sizes");
  if (page_tokens <= 0 || page_tokens % kBlockSize)
    return fail(KVC_EINVAL, "kvc_step_tables: page_tokens must be a positive multiple of %d", kBlockSize);
  if (max_blocks < 0 || max_blocks >= (1 << 24) || block_table_stride < max_blocks)
    return fail(KVC_EINVAL, "kvc_step_tables: max_blocks must be below 2^24 and at most block_table_stride");
  if (!query_start_loc || (num_tokens > 0 && (!positions || !slot_mapping)) ||
      (n_seq > 0 && (!computed_tokens || !new_tokens || !block_offsets || !seq_lens || (max_blocks > 0 && !block_table))))
    return fail(KVC_EINVAL, "kvc_step_tables: null pointer");
  // Workgroups read other requests' lengths while the tables are written.
  const int64_t n = n_seq;
  const Rows read[] = {vector_rows(computed_tokens, 4 * n), vector_rows(new_tokens, 4 * n), vector_rows(request_offsets, 8 * n),
                       vector_rows(block_offsets, n ? 8 * (n + 1) : 0)};
  const Rows written[] = {vector_rows(query_start_loc, 4 * (n + 1)), vector_rows(seq_lens, 4 * n), vector_rows(positions, 8 * num_tokens),
                          vector_rows(slot_mapping, 8 * num_tokens)};
  const Rows table = {static_cast<int64_t>(reinterpret_cast<uintptr_t>(block_table)), 4 * block_table_stride, max_blocks ? n : 0,
                      4ll * max_blocks};
  for (const Rows& x : read) {
    bool meets = vector_meets(x, table);
    for (const Rows& y : written) meets |= vector_meets(x, y);
    if (meets) return fail(KVC_EINVAL, "kvc_step_tables: inputs and outputs overlap");
  }
  for (int i = 0; i < 4; ++i) {
    bool meets = vector_meets(written[i], table);
    for (int j = 0; j < i; ++j) meets |= vector_meets(written[i], written[j]);
    if (meets) return fail(KVC_EINVAL, "kvc_step_tables: outputs overlap each other");
  }
  // About four entries or tokens a thread, as far as the device has room for workgroups.
  const int64_t most = max_query_len > max_blocks ? max_query_len : max_blocks;
  int64_t shares = ceil_div(most, 4 * kDecodeThreads);
  const int64_t room = ceil_div(4096, n_seq + 1);
  if (shares > room) shares = room;
  if (shares < 1) shares = 1;
  StepTables a = {computed_tokens, new_tokens, request_offsets, block_ids, block_offsets, query_start_loc, seq_lens, block_table,
                  positions, slot_mapping, block_table_stride, num_tokens, n_seq, page_tokens / kBlockSize, max_blocks,
                  static_cast<int>(shares)};
  step_tables_kernel<<<static_cast<unsigned>((n_seq + 1) * shares), kDecodeThreads, 0, as_stream(stream)>>>(a);
  return launch_status("kvc_step_tables");
}

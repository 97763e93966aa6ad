// amf_slot_maps.hip - block tables grown from a free list and the slots of a
// step's new tokens, from the sequences' lengths on the device.
//
// Sequence i holds c_i tokens and gets n_i more: it needs
// ceil((c_i + n_i) / block) - ceil(c_i / block) pages, taken from the free list
// in sequence order, and its token c_i + j is row start_i + j of the step, with
// start the exclusive sum of n.  (The host form is AMFReqMeta.make,
// korith_vllm_ext/amf_kv_connector.py:90-115 of the reference, per request.)
//
// Every workgroup owns kTokens rows of the step and walks the sequences in
// tiles of one per thread, summing n and the pages grown as it goes, until its
// rows are covered; the owner of a row finds its sequence by bisection in the
// tile, and the row that starts a page writes the block table's entry.  Nothing
// read is written (lengths and the free count come out in buffers of their
// own), so workgroups need no order, and a step is one launch.
#include <algorithm>

#include "amf_paged.h"

namespace {

using namespace amf;

// 1000 prompts of 131 tokens 8.4 us (256 threads 11.8, 1024 8.1), one token of 32
// sequences 4.8 (4.3, 6.6): latencies of a few barriers, far from the bytes.
constexpr int kThreads = 512;
constexpr int kTokens = 1024;  // rows of a workgroup

struct SlotArgs {
  const int32_t* context_lens;
  const int32_t* new_tokens;
  int32_t* block_tables;
  int64_t bt_stride;
  int32_t table_pages;
  int32_t block_size;
  int64_t pool_pages;
  const int32_t* free_pages;
  int64_t n_free;
  const int32_t* free_used;
  int32_t num_seqs;
  int64_t num_tokens;
  int64_t* slot_mapping;
  int64_t* positions;
  int32_t* query_start;
  int32_t* context_out;
  int32_t* free_used_out;
  int32_t* err_flag;
};

__global__ __launch_bounds__(kThreads) void slot_maps_kernel(SlotArgs a) {
  __shared__ int64_t tmp[kThreads / 64];
  __shared__ int64_t first_row[kThreads];   // row of the sequence's first new token
  __shared__ int64_t first_free[kThreads];  // its first page's place in the free list; -1: no pages
  __shared__ int32_t context[kThreads];
  const int tid = threadIdx.x;
  const bool lead = blockIdx.x == 0;  // writes the sequences' outputs
  const int64_t row0 = (int64_t)blockIdx.x * kTokens;
  const int64_t row1 = min(row0 + kTokens, a.num_tokens);
  const int64_t used = a.free_used ? max(*a.free_used, 0) : 0;
  const int64_t avail = max(a.n_free - used, (int64_t)0);
  int64_t rows = 0, grown = 0, granted = 0;
  int flags = 0;
  for (int s0 = 0; s0 < a.num_seqs; s0 += kThreads) {
    const int s = s0 + tid;
    int64_t c = 0, n = 0, grow = 0;
    bool fits = true;
    if (s < a.num_seqs) {
      c = max(a.context_lens[s], 0);
      n = max(a.new_tokens[s], 0);
    }
    int64_t rows_all, grown_all;
    const int64_t row = rows + block_exclusive<kThreads>(n, tmp, &rows_all);
    if (s < a.num_seqs) {
      const int64_t need = (c + n + a.block_size - 1) / a.block_size;
      fits = need <= a.table_pages && c + n <= 0x7FFFFFFF && (n == 0 || row + n <= a.num_tokens);
      if (fits) grow = need - (c + a.block_size - 1) / a.block_size;
    }
    const int64_t place = grown + block_exclusive<kThreads>(grow, tmp, &grown_all);
    if (!fits) flags |= AMF_ERRFLAG_CONTEXT;
    if (fits && grow > 0 && place + grow > avail) {
      fits = false;
      flags |= AMF_ERRFLAG_FREE_LIST;
    }
    first_row[tid] = row;
    first_free[tid] = fits ? used + place : -1;
    context[tid] = (int32_t)c;
    if (lead && s < a.num_seqs) {
      a.query_start[s] = (int32_t)min(row, (int64_t)0x7FFFFFFF);
      a.context_out[s] = (int32_t)(fits ? c + n : c);
      if (fits && grow > 0) granted = max(granted, place + grow);
    }
    __syncthreads();
    const int seqs = min(kThreads, a.num_seqs - s0);
    for (int64_t r = max(row0, rows) + tid; r < min(row1, rows + rows_all); r += kThreads) {
      int lo = 0, hi = seqs;  // the last sequence that starts at or before row r
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first_row[mid] <= r) lo = mid; else hi = mid;
      }
      const int64_t cl = context[lo], pos = cl + (r - first_row[lo]);
      const int64_t have = (cl + a.block_size - 1) / a.block_size;
      const int64_t page = pos / a.block_size, at = pos - page * a.block_size;
      int64_t id = -1;
      if (first_free[lo] >= 0) {
        int32_t* entry = a.block_tables + (int64_t)(s0 + lo) * a.bt_stride + page;
        id = page < have ? *entry : a.free_pages[first_free[lo] + page - have];
        if (id < 0 || id >= a.pool_pages) {
          id = -1;
          flags |= AMF_ERRFLAG_BLOCK_RANGE;
        }
        // -1 for an id outside the pool: the next step must not take what the row held
        // before for this sequence's page
        if (page >= have && at == 0) *entry = (int32_t)id;
      }
      a.slot_mapping[r] = id < 0 ? -1 : id * a.block_size + at;
      a.positions[r] = pos;
    }
    rows += rows_all;
    grown += grown_all;
    if (!lead && rows >= row1) break;
    __syncthreads();
  }
  for (int64_t r = max(row0, rows) + tid; r < row1; r += kThreads) {
    a.slot_mapping[r] = -1;
    a.positions[r] = 0;
  }
  if (lead) {
    // the largest end of a granted run, over the workgroup
    __shared__ int64_t ends[kThreads];
    ends[tid] = granted;
    __syncthreads();
    for (int o = kThreads / 2; o > 0; o >>= 1) {
      if (tid < o) ends[tid] = max(ends[tid], ends[tid + o]);
      __syncthreads();
    }
    if (tid == 0) {
      a.query_start[a.num_seqs] = (int32_t)min(rows, (int64_t)0x7FFFFFFF);
      if (a.free_used_out) *a.free_used_out = (int32_t)(used + ends[0]);
    }
  }
  if (flags && a.err_flag) atomicOr(a.err_flag, flags);
}

}  // namespace

extern "C" int amf_build_slot_maps(const int32_t* context_lens, const int32_t* new_tokens,
                                   int32_t num_seqs, int32_t* block_tables, int64_t bt_stride,
                                   int32_t table_pages, int32_t block_size, int64_t pool_pages,
                                   const int32_t* free_pages, int64_t n_free,
                                   const int32_t* free_used, int64_t num_tokens,
                                   int64_t* slot_mapping, int64_t* positions,
                                   int32_t* query_start, int32_t* context_out,
                                   int32_t* free_used_out, int32_t* err_flag, void* stream) {
  const char* who = "amf_build_slot_maps";
  if (num_seqs < 0 || num_tokens < 0 || num_tokens > 0x7FFFFFFF || n_free < 0 ||
      n_free > 0x7FFFFFFF)
    return fail(AMF_ERR_INVALID_ARG, "%s: bad num_seqs=%d num_tokens=%lld n_free=%lld", who,
                num_seqs, (long long)num_tokens, (long long)n_free);
  if (block_size <= 0 || table_pages < 0 || bt_stride < table_pages || pool_pages <= 0)
    return fail(AMF_ERR_INVALID_ARG,
                "%s: bad block_size=%d table_pages=%d bt_stride=%lld pool_pages=%lld", who,
                block_size, table_pages, (long long)bt_stride, (long long)pool_pages);
  if (!query_start || (num_tokens > 0 && (!slot_mapping || !positions)) ||
      (num_seqs > 0 && (!context_lens || !new_tokens || !context_out ||
                        (table_pages > 0 && !block_tables))) ||
      (n_free > 0 && !free_pages))
    return fail(AMF_ERR_INVALID_ARG, "%s: null pointer", who);
  const SlotArgs a{context_lens, new_tokens, block_tables, bt_stride, table_pages, block_size,
                   pool_pages, free_pages, n_free, free_used, num_seqs, num_tokens, slot_mapping,
                   positions, query_start, context_out, free_used_out, err_flag};
  const int64_t groups = std::max<int64_t>(1, (num_tokens + kTokens - 1) / kTokens);
  slot_maps_kernel<<<dim3((unsigned)groups), kThreads, 0, as_stream(stream)>>>(a);
  return check_launch(who);
}

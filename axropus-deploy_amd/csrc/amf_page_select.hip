// amf_page_select.hip - which pages of a long context a query attends to.
//
// page_key_bounds keeps the smallest and largest key of every page, per KV head
// and channel: lo[d] = min_t k[t, d], hi[d] = max_t k[t, d].  No key of the page
// scores more against q than
//   u = sum_d max(q_d lo_d, q_d hi_d) = sum_d q_d (q_d >= 0 ? hi_d : lo_d),
// and a page's rank for a KV head is the largest u of the query heads that share
// it.  select_pages takes the num_pages best pages of each (sequence, KV head).
//
// u is summed in 64 bits: thousands of pages lie close together around the last
// one taken, where the order of an fp32 sum would decide between two of them.
#include <algorithm>
#include <type_traits>

#include "amf_paged.h"

namespace {

using namespace amf;

constexpr int kThreads = 256;

// ---- bounds --------------------------------------------------------------------

struct BoundsArgs {
  const uint8_t* k;
  int64_t page_stride, token_stride, head_stride;  // bytes
  int64_t pool_pages;
  const int32_t* block_tables;
  int64_t bt_stride;
  int32_t table_pages;
  const int32_t* context_lens;
  const int32_t* first_tokens;
  uint16_t* bounds;
  int32_t num_kv_heads, head_dim, block_size;
  int32_t chunks;        // of 8 channels, of all heads
  int32_t* err_flag;
};

template <int DT>
__device__ __forceinline__ void load_keys8(const uint8_t* p, float* x) {
  if constexpr (DT == AMF_DTYPE_E4M3) {
    const u32x2 w = ld_stream(reinterpret_cast<const u32x2*>(p));
    e4m3x4_to_f32(w[0], x);
    e4m3x4_to_f32(w[1], x + 4);
  } else {
    load8_stream<DT>(p, x);
  }
}

// One thread takes 8 channels of one page: block_size loads of 16 (fp8: 8)
// bytes, neighbouring threads on neighbouring channels.  BF16: of the bounds.
template <int DT, bool BF16>
__global__ __launch_bounds__(kThreads) void page_key_bounds_kernel(BoundsArgs a) {
  const int s = blockIdx.y;
  const int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t c = a.context_lens[s];
  int64_t page = item / a.chunks;
  const int chunk = (int)(item - page * a.chunks);
  if (a.first_tokens) page += max(a.first_tokens[s], 0) / a.block_size;
  if (page * a.block_size >= c) return;
  if (page >= a.table_pages) {
    if (a.err_flag) atomicOr(a.err_flag, AMF_ERRFLAG_CONTEXT);
    return;
  }
  const int64_t id = a.block_tables[s * a.bt_stride + page];
  if (id < 0 || id >= a.pool_pages) {
    if (a.err_flag) atomicOr(a.err_flag, AMF_ERRFLAG_BLOCK_RANGE);
    return;
  }
  const int n = (int)min((int64_t)a.block_size, c - page * a.block_size);
  const int per_head = a.head_dim / 8;
  const int h = chunk / per_head, d = 8 * (chunk - h * per_head);
  constexpr int ES = DT == AMF_DTYPE_E4M3 ? 1 : 2;
  const uint8_t* p = a.k + id * a.page_stride + h * a.head_stride + d * ES;
  float lo[8], hi[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo[e] = INFINITY;
    hi[e] = -INFINITY;
  }
#pragma unroll 8
  for (int t = 0; t < n; ++t, p += a.token_stride) {
    float x[8];
    load_keys8<DT>(p, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // a NaN stays: the page is then always taken
      lo[e] = __builtin_elementwise_minimum(lo[e], x[e]);
      hi[e] = __builtin_elementwise_maximum(hi[e], x[e]);
    }
  }
  uint16_t* o = a.bounds + ((id * a.num_kv_heads + h) * 2) * a.head_dim + d;
  *reinterpret_cast<u32x4*>(o) = pack8<BF16>(lo);
  *reinterpret_cast<u32x4*>(o + a.head_dim) = pack8<BF16>(hi);
}

// ---- scores --------------------------------------------------------------------

struct SelectArgs {
  const uint16_t* q;
  int64_t q_seq, q_head;  // strides, elements
  const uint16_t* bounds;
  int64_t pool_pages;
  const int32_t* block_tables;
  int64_t bt_stride;
  int32_t table_pages;
  const int32_t* context_lens;
  int32_t num_seqs, group, num_kv_heads, head_dim, block_size;
  int32_t num_pages, first_pages, last_pages;
  int64_t max_pages;  // of a sequence: the table's, or what max_context_len allows
  uint64_t* keys;     // [seq][KV head][max_pages]
  int32_t* pages;
  int32_t* counts;
  int32_t* err_flag;
};

// Pages of sequence s, at most what its table holds.
__device__ __forceinline__ int64_t seq_pages(const SelectArgs& a, int s) {
  const int64_t c = max(a.context_lens[s], 0);
  return min((c + a.block_size - 1) / a.block_size, a.max_pages);
}

// Unsigned words in the order of the doubles they stand for.
__device__ __forceinline__ uint64_t order_key(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);  // -0 as 0
  return (u >> 63) ? ~u : u | (1ull << 63);
}
constexpr uint64_t kForced = ~0ull;  // first and last pages
constexpr uint64_t kInfinite = 0xFFF0000000000000ull;  // order_key(inf)

template <bool BF16>
__device__ __forceinline__ float elem16(uint16_t w) {
  return BF16 ? bf16_to_f32(w) : (float)__builtin_bit_cast(_Float16, w);
}

// LP lanes share a page, 8 channels each.
constexpr int kScorePages = 64;  // pages of a workgroup

template <bool BF16, int LP>
__global__ __launch_bounds__(kThreads) void page_score_kernel(SelectArgs a) {
  const int s = blockIdx.z, h = blockIdx.y;
  const int64_t n = seq_pages(a, s);
  const int64_t p0 = (int64_t)blockIdx.x * kScorePages;
  if (p0 >= n || n <= a.num_pages) return;
  const int sub = threadIdx.x % LP, d = 8 * sub;
  const bool live = d < a.head_dim;
  const uint16_t* q0 = a.q + s * a.q_seq + (int64_t)h * a.group * a.q_head + d;
  uint64_t* keys = a.keys + ((int64_t)s * a.num_kv_heads + h) * a.max_pages;
  for (int64_t p = p0 + threadIdx.x / LP; p < min(p0 + kScorePages, n); p += kThreads / LP) {
    const int64_t id = a.block_tables[s * a.bt_stride + p];
    const bool ok = id >= 0 && id < a.pool_pages;
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) lo[e] = hi[e] = 0.0f;
    if (ok && live) {
      const uint16_t* b = a.bounds + ((id * a.num_kv_heads + h) * 2) * a.head_dim + d;
      unpack8<BF16>(ld_stream(reinterpret_cast<const u32x4*>(b)), lo);
      unpack8<BF16>(ld_stream(reinterpret_cast<const u32x4*>(b + a.head_dim)), hi);
    }
    bool finite = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) finite = finite && fabsf(lo[e]) < INFINITY && fabsf(hi[e]) < INFINITY;
    double best = -INFINITY;
    for (int g = 0; g < a.group; ++g) {
      double u = 0.0;
      if (live) {
        float x[8];
        unpack8<BF16>(*reinterpret_cast<const u32x4*>(q0 + g * a.q_head), x);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          u = __builtin_fma((double)x[e], (double)(x[e] >= 0.0f ? hi[e] : lo[e]), u);
      }
#pragma unroll
      for (int o = LP / 2; o > 0; o >>= 1) u += __shfl_xor(u, o, LP);
      finite = finite && u - u == 0.0;
      best = max(best, u);
    }
    // a NaN or an infinity anywhere: above every finite score
#pragma unroll
    for (int o = LP / 2; o > 0; o >>= 1) finite = __shfl_xor((int)finite, o, LP) && finite;
    if (sub == 0) {
      uint64_t key = finite ? order_key(best) : kInfinite;
      if (!ok) {
        key = 0;  // never scored: behind every page that can be read
        if (a.err_flag) atomicOr(a.err_flag, AMF_ERRFLAG_BLOCK_RANGE);
      }
      if (p < a.first_pages || p >= n - a.last_pages) key = kForced;
      keys[p] = key;
    }
  }
}

// ---- choice --------------------------------------------------------------------

constexpr int kPickThreads = 1024;

// The num_pages largest keys of one (sequence, KV head), the lower page first
// among equals, in page order.  The key of the last one taken is found digit by
// digit (8 bits, a histogram in LDS), then the pages above it and the first of
// its equals are written at their ranks.
__global__ __launch_bounds__(kPickThreads) void page_pick_kernel(SelectArgs a) {
  __shared__ uint32_t hist[256];
  __shared__ int64_t tmp[kPickThreads / 64];
  __shared__ uint64_t s_prefix;
  __shared__ int32_t s_left;
  __shared__ int s_done;
  const int s = blockIdx.y, h = blockIdx.x, tid = threadIdx.x;
  const int64_t n = seq_pages(a, s);
  const int64_t row = (int64_t)s * a.num_kv_heads + h;
  int32_t* out = a.pages + row * a.num_pages;
  const int32_t K = a.num_pages;
  const int32_t count = (int32_t)min(n, (int64_t)K);
  if (tid == 0) {
    a.counts[row] = count;
    if (h == 0 && a.err_flag && (int64_t)a.context_lens[s] > a.max_pages * a.block_size)
      atomicOr(a.err_flag, AMF_ERRFLAG_CONTEXT);
  }
  for (int i = count + tid; i < K; i += kPickThreads) out[i] = -1;
  if (n <= K) {
    for (int i = tid; i < count; i += kPickThreads) out[i] = i;
    return;
  }
  const uint64_t* keys = a.keys + row * a.max_pages;
  uint64_t prefix = 0;  // the digits found, in place
  int32_t left = K;     // of the keys with these digits, how many are taken
  int shift = 56;
  for (;; shift -= 8) {
    for (int i = tid; i < 256; i += kPickThreads) hist[i] = 0;
    __syncthreads();
    for (int64_t i = tid; i < n; i += kPickThreads) {
      const uint64_t k = keys[i];
      if (shift == 56 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&hist[(k >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid < 64) {  // the digit below which `left` keys do not fit; lane l: digits 4l ..
      uint32_t c[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += c[i] = hist[4 * tid + i];
      int64_t all;
      int64_t above = wave_exclusive(sum, &all);
      above = all - above - sum;  // keys with larger digits than this lane's
#pragma unroll
      for (int i = 3; i >= 0; --i) {
        if (above < left && above + c[i] >= left) {
          s_prefix = prefix | (uint64_t)(4 * tid + i) << shift;
          s_left = left - (int32_t)above;
          s_done = above + c[i] == left;  // all of them are taken
        }
        above += c[i];
      }
    }
    __syncthreads();
    prefix = s_prefix;
    left = s_left;
    if (s_done || shift == 0) break;
    __syncthreads();
  }
  // taken: keys whose digits are above the prefix, and `left` of its equals
  const uint64_t cut = prefix >> shift;
  int64_t gt0 = 0, eq0 = 0;
  for (int64_t i0 = 0; i0 < n; i0 += kPickThreads) {
    const int64_t i = i0 + tid;
    const uint64_t k = i < n ? keys[i] >> shift : 0;
    const bool gt = i < n && k > cut, eq = i < n && k == cut;
    int64_t all;
    const int64_t both = block_exclusive<kPickThreads>((int64_t)gt << 32 | (int64_t)eq, tmp, &all);
    const int64_t eq_before = eq0 + (both & 0xFFFFFFFF), gt_before = gt0 + (both >> 32);
    if (gt || (eq && eq_before < left)) out[gt_before + min(eq_before, (int64_t)left)] = (int32_t)i;
    gt0 += all >> 32;
    eq0 += all & 0xFFFFFFFF;
  }
}

template <bool BF16>
void launch_score(const SelectArgs& a, dim3 grid, hipStream_t st) {
  const int lanes = a.head_dim / 8;
  if (lanes <= 8)
    page_score_kernel<BF16, 8><<<grid, kThreads, 0, st>>>(a);
  else if (lanes <= 16)
    page_score_kernel<BF16, 16><<<grid, kThreads, 0, st>>>(a);
  else
    page_score_kernel<BF16, 32><<<grid, kThreads, 0, st>>>(a);
}

int64_t select_max_pages(int32_t table_pages, int32_t block_size, int32_t max_context_len) {
  return std::min<int64_t>(table_pages, ((int64_t)max_context_len + block_size - 1) / block_size);
}

}  // namespace

extern "C" int amf_page_key_bounds(const void* k, int32_t kv_dtype, int64_t page_stride,
                                   int64_t token_stride, int64_t head_stride, int64_t pool_pages,
                                   const int32_t* block_tables, int64_t bt_stride,
                                   int32_t table_pages, const int32_t* context_lens,
                                   const int32_t* first_tokens, int32_t max_new_tokens,
                                   int32_t num_seqs, int32_t num_kv_heads, int32_t head_dim,
                                   int32_t block_size, void* bounds, int32_t bounds_dtype,
                                   int32_t* err_flag, void* stream) {
  const char* who = "amf_page_key_bounds";
  const int es = kv_elem_bytes(kv_dtype);
  if (num_seqs < 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || table_pages < 0 ||
      bt_stride < table_pages || pool_pages <= 0 || max_new_tokens < 0)
    return fail(AMF_ERR_INVALID_ARG,
                "%s: bad num_seqs=%d num_kv_heads=%d head_dim=%d block_size=%d table_pages=%d "
                "bt_stride=%lld pool_pages=%lld max_new_tokens=%d",
                who, num_seqs, num_kv_heads, head_dim, block_size, table_pages,
                (long long)bt_stride, (long long)pool_pages, max_new_tokens);
  if (es == 0 || es == 4 || head_dim % 8 != 0 || head_dim > 256 || num_seqs > 65535)
    return fail(AMF_ERR_UNSUPPORTED,
                "%s: dtype %d, head_dim %d (a multiple of 8 up to 256), %d sequences (at most "
                "65535); fp32 caches have no bounds",
                who, kv_dtype, head_dim, num_seqs);
  if ((bounds_dtype != AMF_DTYPE_BF16 && bounds_dtype != AMF_DTYPE_F16) ||
      (es == 2 && bounds_dtype != kv_dtype))
    return fail(AMF_ERR_INVALID_ARG, "%s: bounds of type %d for a cache of type %d", who,
                bounds_dtype, kv_dtype);
  if (num_seqs == 0 || table_pages == 0) return ok();
  if (!k || !block_tables || !context_lens || !bounds)
    return fail(AMF_ERR_INVALID_ARG, "%s: null pointer", who);
  const int align = 8 * es;  // bytes of a thread's load
  if ((page_stride * es) % align || (token_stride * es) % align || (head_stride * es) % align ||
      (uintptr_t)k % align || (uintptr_t)bounds % 16)
    return fail(AMF_ERR_INVALID_ARG, "%s: keys and strides need %d-byte alignment, bounds 16", who,
                align);
  // pages that a sequence's new tokens can lie in
  int64_t pages = table_pages;
  if (first_tokens && max_new_tokens > 0)
    pages = std::min<int64_t>(pages, ((int64_t)max_new_tokens + block_size - 2) / block_size + 1);
  const int64_t chunks = (int64_t)num_kv_heads * head_dim / 8;
  const int64_t groups = (pages * chunks + kThreads - 1) / kThreads;
  if (chunks > 0x7FFFFFFF || groups > 0x7FFFFFFF)
    return fail(AMF_ERR_UNSUPPORTED, "%s: %lld pages of %lld channels", who, (long long)pages,
                (long long)chunks * 8);
  const BoundsArgs a{static_cast<const uint8_t*>(k), page_stride * es, token_stride * es,
                     head_stride * es, pool_pages, block_tables, bt_stride, table_pages,
                     context_lens, first_tokens, static_cast<uint16_t*>(bounds), num_kv_heads,
                     head_dim, block_size, (int32_t)chunks, err_flag};
  const dim3 grid((unsigned)groups, (unsigned)num_seqs);
  hipStream_t st = as_stream(stream);
  if (kv_dtype == AMF_DTYPE_BF16)
    page_key_bounds_kernel<AMF_DTYPE_BF16, true><<<grid, kThreads, 0, st>>>(a);
  else if (kv_dtype == AMF_DTYPE_F16)
    page_key_bounds_kernel<AMF_DTYPE_F16, false><<<grid, kThreads, 0, st>>>(a);
  else if (bounds_dtype == AMF_DTYPE_BF16)
    page_key_bounds_kernel<AMF_DTYPE_E4M3, true><<<grid, kThreads, 0, st>>>(a);
  else
    page_key_bounds_kernel<AMF_DTYPE_E4M3, false><<<grid, kThreads, 0, st>>>(a);
  return check_launch(who);
}

extern "C" int64_t amf_select_pages_workspace_bytes(int32_t num_seqs, int32_t num_kv_heads,
                                                    int32_t table_pages, int32_t block_size,
                                                    int32_t max_context_len) {
  if (num_seqs <= 0 || num_kv_heads <= 0 || table_pages <= 0 || block_size <= 0 ||
      max_context_len <= 0)
    return 0;
  return 8 * (int64_t)num_seqs * num_kv_heads *
         select_max_pages(table_pages, block_size, max_context_len);
}

extern "C" int amf_select_pages(const void* q, int32_t dtype, int64_t q_seq_stride,
                                int64_t q_head_stride, const void* bounds, int64_t pool_pages,
                                const int32_t* block_tables, int64_t bt_stride,
                                int32_t table_pages, const int32_t* context_lens,
                                int32_t max_context_len, int32_t num_seqs, int32_t num_q_heads,
                                int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                int32_t num_pages, int32_t first_pages, int32_t last_pages,
                                int32_t* pages, int32_t* page_counts, void* workspace,
                                int64_t workspace_bytes, int32_t* err_flag, void* stream) {
  const char* who = "amf_select_pages";
  if (num_seqs < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 ||
      head_dim <= 0 || block_size <= 0 || table_pages < 0 || bt_stride < table_pages ||
      pool_pages <= 0 || max_context_len < 0)
    return fail(AMF_ERR_INVALID_ARG,
                "%s: bad num_seqs=%d heads=%d/%d (a multiple) head_dim=%d block_size=%d "
                "table_pages=%d bt_stride=%lld pool_pages=%lld max_context_len=%d",
                who, num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, table_pages,
                (long long)bt_stride, (long long)pool_pages, max_context_len);
  if (num_pages <= 0 || first_pages < 0 || last_pages < 0 ||
      (int64_t)first_pages + last_pages > num_pages)
    return fail(AMF_ERR_INVALID_ARG, "%s: num_pages=%d has to hold first_pages=%d and last_pages=%d",
                who, num_pages, first_pages, last_pages);
  if ((dtype != AMF_DTYPE_BF16 && dtype != AMF_DTYPE_F16) || head_dim % 8 != 0 || head_dim > 256 ||
      num_seqs > 65535 || num_kv_heads > 65535)
    return fail(AMF_ERR_UNSUPPORTED,
                "%s: dtype %d (bf16, fp16), head_dim %d (a multiple of 8 up to 256), %d sequences "
                "and %d KV heads (at most 65535)",
                who, dtype, head_dim, num_seqs, num_kv_heads);
  if (num_seqs == 0) return ok();
  if (!q || !bounds || !context_lens || !pages || !page_counts || (table_pages > 0 && !block_tables))
    return fail(AMF_ERR_INVALID_ARG, "%s: null pointer", who);
  if ((uintptr_t)q % 16 || (uintptr_t)bounds % 16 || q_seq_stride % 8 || q_head_stride % 8)
    return fail(AMF_ERR_INVALID_ARG, "%s: q, its strides and bounds need 16-byte alignment", who);
  const int64_t max_pages = select_max_pages(table_pages, block_size, max_context_len);
  const int64_t need = amf_select_pages_workspace_bytes(num_seqs, num_kv_heads, table_pages,
                                                        block_size, max_context_len);
  const bool scored = max_pages > num_pages;  // else every page is taken
  if (scored && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 8))
    return fail(AMF_ERR_WORKSPACE, "%s: workspace of %lld bytes needed, got %lld", who,
                (long long)need, (long long)workspace_bytes);
  const SelectArgs a{static_cast<const uint16_t*>(q), q_seq_stride, q_head_stride,
                     static_cast<const uint16_t*>(bounds), pool_pages, block_tables, bt_stride,
                     table_pages, context_lens, num_seqs, num_q_heads / num_kv_heads,
                     num_kv_heads, head_dim, block_size, num_pages, first_pages, last_pages,
                     max_pages, static_cast<uint64_t*>(workspace), pages, page_counts, err_flag};
  hipStream_t st = as_stream(stream);
  if (scored) {
    const dim3 grid((unsigned)((max_pages + kScorePages - 1) / kScorePages),
                    (unsigned)num_kv_heads, (unsigned)num_seqs);
    if (dtype == AMF_DTYPE_BF16)
      launch_score<true>(a, grid, st);
    else
      launch_score<false>(a, grid, st);
    if (int rc = check_launch(who)) return rc;
  }
  page_pick_kernel<<<dim3((unsigned)num_kv_heads, (unsigned)num_seqs), kPickThreads, 0, st>>>(a);
  return check_launch(who);
}

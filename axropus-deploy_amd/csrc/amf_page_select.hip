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
// Bound by HBM: 30000 tokens of 8 heads of 128, 65 MB, 11.9 us, 5.5 TB/s; the pages of
// one step of 64 sequences 4.1 us, latency.
template <int DT, bool BF16>
__global__ __launch_bounds__(kThreads) void page_key_bounds_kernel(BoundsArgs a) {
  const int s = blockIdx.y;
  const int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t c = a.context_lens[s];
  // here, not where a page is missed: the grid may end with the table's pages
  if (item == 0 && a.err_flag && c > (int64_t)a.table_pages * a.block_size)
    atomicOr(a.err_flag, AMF_ERRFLAG_CONTEXT);
  int64_t page = item / a.chunks;
  const int chunk = (int)(item - page * a.chunks);
  if (a.first_tokens) page += max(a.first_tokens[s], 0) / a.block_size;
  if (page * a.block_size >= c || page >= a.table_pages) return;
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

// A wave scores 16 pages against SETS times 4 query heads with 4x4x4 products in
// 64 bits, four blocks side by side: lane (lo, hi) = (lane % 16, lane / 16) holds
// page lo's bounds in dims 32 c + 8 hi + e as the A operand of step (c, e), and as B
// head lo % 4's q in that dim, split as max(q, 0) against hi and min(q, 0) against
// lo; D gives it page 4 (lo / 4) + hi of head lo % 4.  q waits in LDS as doubles.
//
// 8 sequences x 65000 tokens, 64 / 8 heads of 128, 133 MB of bounds: 39 us, of which
// the products and conversions (16 cycles each) take about 22 and the reads 30, partly
// at the same time.  On the vector units it was 95 us: a conversion, a choice and a
// product per element and head, and a reduction over lanes.  fp32 products with an
// error bound each, and 64 bits only for the pages that it leaves in doubt, were as
// slow (53 us) and made the choice 23 us longer.
constexpr int kScorePages = kThreads / 64 * 16;  // pages that a workgroup takes at once
constexpr int kHeadSet = 4;

__device__ __forceinline__ double max64(double x, double y) { return x > y ? x : y; }

// NC chunks of 32 dims; SETS of heads share a bound's conversion to a double.  The
// heads' workgroups of a page run side by side: their bounds lie together.  A wave
// takes one tile of 16 pages; walking several with the next one's bounds in flight
// needs twice the registers and was slower (2 tiles 82 -> 87 us a selection with its
// attention, 4 93).
template <bool BF16, int NC, int SETS>
__global__ __launch_bounds__(kThreads) void page_score_kernel(SelectArgs a) {
  // [dim in step order][set][hi][head] -> (max(q, 0), min(q, 0))
  __shared__ __attribute__((aligned(16))) double q_lds[NC * 8][SETS][4][kHeadSet][2];
  constexpr int kItems = NC * 4 * SETS * kHeadSet;  // 8 dims of a head to a thread
  static_assert(kItems <= kThreads, "a thread takes at most one");
  const int s = blockIdx.z, h = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int q_g = tid % (SETS * kHeadSet), q_d = tid / (SETS * kHeadSet);
  auto load_q = [&](int g0) {
    u32x4 x{0, 0, 0, 0};
    if (tid < kItems && 8 * q_d < a.head_dim && g0 + q_g < a.group)
      x = *reinterpret_cast<const u32x4*>(
          a.q + s * a.q_seq + ((int64_t)h * a.group + g0 + q_g) * a.q_head + 8 * q_d);
    return x;
  };
  u32x4 q_raw = load_q(0);  // on its way before the lengths are known
  const int64_t n = seq_pages(a, s);
  const int64_t p0 = (int64_t)blockIdx.y * kScorePages;
  if (p0 >= n || n <= a.num_pages) return;
  const int lo = lane & 15, hi = lane >> 4;
  const int64_t base = p0 + wave * 16;
  const int64_t id = base + lo < n ? a.block_tables[s * a.bt_stride + base + lo] : -1;
  const bool ok = id >= 0 && id < a.pool_pages;
  u32x4 b[2][NC];
  {
    const uint16_t* src = a.bounds + ((ok ? id : 0) * a.num_kv_heads + h) * 2 * a.head_dim + 8 * hi;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      b[0][c] = b[1][c] = u32x4{0, 0, 0, 0};
      if (ok && 32 * c + 8 * hi < a.head_dim) {
        b[0][c] = ld_stream(reinterpret_cast<const u32x4*>(src + 32 * c));
        b[1][c] = ld_stream(reinterpret_cast<const u32x4*>(src + a.head_dim + 32 * c));
      }
    }
  }
  double best = -INFINITY;
  int fin = 1;
  for (int g0 = 0; g0 < a.group; g0 += SETS * kHeadSet) {
    if (g0 > 0) {
      q_raw = load_q(g0);
      __syncthreads();
    }
    if (tid < kItems) {
      float x[8];
      unpack8<BF16>(q_raw, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        double* o = q_lds[8 * (q_d / 4) + e][q_g / kHeadSet][q_d % 4][q_g % kHeadSet];
        o[0] = x[e] < 0.0f ? 0.0f : x[e];  // a NaN stays one
        o[1] = x[e] < 0.0f ? x[e] : 0.0f;
      }
    }
    __syncthreads();
    double u[SETS];
#pragma unroll
    for (int k = 0; k < SETS; ++k) u[k] = 0.0;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t wl = b[0][c][e / 2], wh = b[1][c][e / 2];
        asm volatile("" : "+v"(wl), "+v"(wh));  // converted here, not before the loop
        const double l = e % 2 ? half_hi<BF16>(wl) : half_lo<BF16>(wl);
        const double m = e % 2 ? half_hi<BF16>(wh) : half_lo<BF16>(wh);
#pragma unroll
        for (int k = 0; k < SETS; ++k) {
          const double* q = q_lds[8 * c + e][k][hi][lo % 4];
          u[k] = __builtin_amdgcn_mfma_f64_4x4x4f64(m, q[0], u[k], 0, 0, 0);
          u[k] = __builtin_amdgcn_mfma_f64_4x4x4f64(l, q[1], u[k], 0, 0, 0);
        }
      }
#pragma unroll
    for (int k = 0; k < SETS; ++k) {
      fin &= u[k] - u[k] == 0.0;
      if (g0 + k * kHeadSet + lo % 4 < a.group) best = max64(best, u[k]);
    }
  }
  // the best of the heads, in the four lanes of a page
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    best = max64(best, __shfl_xor(best, o));
    fin &= __shfl_xor(fin, o);
  }
  const int place = 4 * (lo / 4) + hi;
  const int good = __shfl((int)ok, place);
  const int64_t p = base + place;
  if (lo % 4 == 0 && p < n) {
    uint64_t key = fin ? order_key(best) : kInfinite;
    if (!good) {
      key = 0;  // never scored: behind every page that can be read
      if (a.err_flag) atomicOr(a.err_flag, AMF_ERRFLAG_BLOCK_RANGE);
    }
    if (p < a.first_pages || p >= n - a.last_pages) key = kForced;
    a.keys[((int64_t)s * a.num_kv_heads + h) * a.max_pages + p] = key;
  }
}

// ---- choice --------------------------------------------------------------------

constexpr int kDigit = 11;    // bits
constexpr int kBins = 1 << kDigit;

// Sum over the threads before this one, and over all in *total; tmp holds a
// word per wave and is not used again before the next barrier but one.  One
// barrier.
template <int NT>
__device__ __forceinline__ uint32_t pick_exclusive(uint32_t v, uint32_t* tmp, uint32_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  if (lane == 63) tmp[wave] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    const uint32_t y = tmp[w];
    if (w < wave) before += y;
    all += y;
  }
  *total = all;
  return before + x - v;
}

// The num_pages largest keys of one (sequence, KV head), the lower page first
// among equals, in page order.  The key of the last one taken is found digit by
// digit (a histogram in LDS each), from the first bit in which the keys differ,
// so that one or two digits separate scores that share sign and exponent; then
// the pages above it and the first of its equals are written at their ranks.
// Forced pages are left out of the search.  A thread takes KEYS consecutive keys;
// up to NT * KEYS of a row stay in registers (MANY: they are read again for each
// pass).
//
// Bound by its barriers, three a digit, and by the 64-bit shifts of a thread's keys:
// 4063 pages, 8 / 16 / 32 keys a thread on 1024 / 512 / 256 threads, 9.7 / 12.0 /
// 16.7 us.
template <int NT, int KEYS, bool MANY>
__global__ __launch_bounds__(NT) void page_pick_kernel(SelectArgs a) {
  constexpr int kTile = NT * KEYS;
  constexpr int kMine = kBins / NT;  // bins of a thread
  __shared__ uint32_t hist[2][kBins];
  __shared__ uint32_t tmp[2][NT / 64];
  __shared__ uint64_t s_lo[NT / 64], s_hi[NT / 64];
  __shared__ uint32_t s_digit, s_left, s_all;
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
  for (int i = count + tid; i < K; i += NT) out[i] = -1;
  if (n <= K) {
    for (int i = tid; i < count; i += NT) out[i] = i;
    return;
  }
  const uint64_t* keys = a.keys + row * a.max_pages;
  uint64_t kept[KEYS];
  auto load = [&](int64_t t0) {  // this thread's keys of a tile; 0 behind the last
#pragma unroll
    for (int e = 0; e < KEYS; ++e) {
      const int64_t i = t0 + (int64_t)tid * KEYS + e;
      kept[e] = i < n ? keys[i] : 0;
    }
  };
  auto each_tile = [&](auto&& body) {
    if constexpr (MANY) {
      for (int64_t t0 = 0; t0 < n; t0 += kTile) {
        load(t0);
        body(t0);
      }
    } else {
      body((int64_t)0);
    }
  };
  if constexpr (!MANY) load(0);
  auto searched = [&](int64_t t0, int e) {
    return t0 + (int64_t)tid * KEYS + e < n && kept[e] != kForced;
  };
#pragma unroll
  for (int k = 0; k < kMine; ++k) hist[0][tid + k * NT] = 0;
  // range of the keys searched
  uint64_t lo = ~0ull, hi = 0;
  each_tile([&](int64_t t0) {
#pragma unroll
    for (int e = 0; e < KEYS; ++e)
      if (searched(t0, e)) {
        lo = min(lo, kept[e]);
        hi = max(hi, kept[e]);
      }
  });
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    lo = min(lo, (uint64_t)__shfl_xor((unsigned long long)lo, o));
    hi = max(hi, (uint64_t)__shfl_xor((unsigned long long)hi, o));
  }
  if ((tid & 63) == 0) {
    s_lo[tid >> 6] = lo;
    s_hi[tid >> 6] = hi;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    lo = min(lo, s_lo[w]);
    hi = max(hi, s_hi[w]);
  }
  // n > K, so first_pages + last_pages pages are forced
  uint32_t left = (uint32_t)(K - a.first_pages - a.last_pages);
  uint64_t cut = lo;  // keys of these digits: `left` of them are taken
  int shift = lo < hi ? 64 - __builtin_clzll(lo ^ hi) : 0;  // bits not decided yet
  if (left == 0) {  // nothing but the forced pages
    cut = kForced;
    shift = 0;
  }
  int now = 0;
  while (shift > 0) {  // uniform
    const int next = max(shift - kDigit, 0), bins = 1 << (shift - next);
    const uint64_t above = shift == 64 ? 0 : cut >> shift;
    each_tile([&](int64_t t0) {
#pragma unroll
      for (int e = 0; e < KEYS; ++e)
        if (searched(t0, e) && (shift == 64 || kept[e] >> shift == above))
          atomicAdd(&hist[now][(kept[e] >> next) & (bins - 1)], 1u);
    });
    __syncthreads();
    // bins from the top, kMine a thread: the one in which `left` keys are reached
    uint32_t c[kMine], sum = 0, all;
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int bin = bins - 1 - (tid * kMine + k);
      sum += c[k] = bin >= 0 ? hist[now][bin] : 0;
      hist[now ^ 1][tid + k * NT] = 0;
    }
    uint32_t before = pick_exclusive<NT>(sum, tmp[now], &all);
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      if (before < left && before + c[k] >= left) {
        s_digit = bins - 1 - (tid * kMine + k);
        s_left = left - before;
        s_all = before + c[k] == left;
      }
      before += c[k];
    }
    __syncthreads();
    cut = (cut >> next >> (shift - next) << (shift - next) | s_digit) << next;
    left = s_left;
    shift = next;
    now ^= 1;
    if (s_all) break;  // s_*: written again after the next histogram's barrier
  }
  // taken: keys whose digits are above the cut's, and `left` of its equals
  cut >>= shift;
  uint32_t gt0 = 0, eq0 = 0;
  each_tile([&](int64_t t0) {
    uint32_t gt = 0, eq = 0;
#pragma unroll
    for (int e = 0; e < KEYS; ++e) {
      const bool in = t0 + (int64_t)tid * KEYS + e < n;
      gt += in && (kept[e] == kForced || kept[e] >> shift > cut);
      eq += in && kept[e] != kForced && kept[e] >> shift == cut;
    }
    uint32_t all;  // both below 2^14 in a tile
    const uint32_t both = pick_exclusive<NT>(gt << 16 | eq, tmp[now], &all);
    now ^= 1;
    uint32_t g = gt0 + (both >> 16), q = eq0 + (both & 0xFFFFu);
#pragma unroll
    for (int e = 0; e < KEYS; ++e) {
      const int64_t i = t0 + (int64_t)tid * KEYS + e;
      if (i >= n) continue;
      const bool above = kept[e] == kForced || kept[e] >> shift > cut;
      const bool equal = kept[e] != kForced && kept[e] >> shift == cut;
      if (above || (equal && q < left)) out[g + min(q, left)] = (int32_t)i;
      g += above;
      q += equal;
    }
    gt0 += all >> 16;
    eq0 += all & 0xFFFFu;
  });
}

template <bool BF16, int NC>
void launch_score_sets(const SelectArgs& a, dim3 grid, hipStream_t st) {
  if (a.group <= kHeadSet)
    page_score_kernel<BF16, NC, 1><<<grid, kThreads, 0, st>>>(a);
  else
    page_score_kernel<BF16, NC, 2><<<grid, kThreads, 0, st>>>(a);
}

template <bool BF16>
void launch_score(const SelectArgs& a, dim3 grid, hipStream_t st) {
  if (a.head_dim <= 64)
    launch_score_sets<BF16, 2>(a, grid, st);
  else if (a.head_dim <= 128)
    launch_score_sets<BF16, 4>(a, grid, st);
  else
    launch_score_sets<BF16, 8>(a, grid, st);
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
  if (num_seqs == 0 || (table_pages == 0 && !err_flag)) return ok();
  if (!k || (table_pages > 0 && !block_tables) || !context_lens || !bounds)
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
  // one at least, for the flag
  const int64_t groups = std::max<int64_t>(1, (pages * chunks + kThreads - 1) / kThreads);
  if (chunks > 0x7FFFFFFF || groups > 0xFFFFFF)
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
    const int64_t chunks = (max_pages + kScorePages - 1) / kScorePages;
    if (chunks > 65535)
      return fail(AMF_ERR_UNSUPPORTED, "%s: %lld pages of a sequence", who, (long long)max_pages);
    const dim3 grid((unsigned)num_kv_heads, (unsigned)chunks, (unsigned)num_seqs);
    if (dtype == AMF_DTYPE_BF16)
      launch_score<true>(a, grid, st);
    else
      launch_score<false>(a, grid, st);
    if (int rc = check_launch(who)) return rc;
  }
  const dim3 rows((unsigned)num_kv_heads, (unsigned)num_seqs);
  if (max_pages <= 1024)
    page_pick_kernel<256, 4, false><<<rows, 256, 0, st>>>(a);
  else if (max_pages <= 4096)
    page_pick_kernel<1024, 4, false><<<rows, 1024, 0, st>>>(a);
  else if (max_pages <= 8192)
    page_pick_kernel<1024, 8, false><<<rows, 1024, 0, st>>>(a);
  else
    page_pick_kernel<1024, 8, true><<<rows, 1024, 0, st>>>(a);
  return check_launch(who);
}

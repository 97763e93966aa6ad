// amf_paged_attn.hip - attention of one new token per sequence over a paged
// K/V cache as vLLM keeps it (bf16, fp16, fp32 or FP8 e4m3 elements in pages
// [token][head][dim], read in place through the block table), split over the
// context and joined.
//
//   out[s, h] = v_scale * sum_t softmax_t(k_scale * scale * q[s, h] . k[t]) v[t]
//
// over the context_lens[s] tokens of the sequence, or those of the pages listed
// for its KV head.  Each K and V element is read once, for all query heads that
// share it, and meets the running maximum m and sum l of each head's softmax.
//
// Work.  Steps of NW waves x 32 tokens; the steps of all (sequence, KV head,
// head tile) pairs, sequence-major, are cut into equal shares, one per
// workgroup of a grid that is resident as a whole, so every workgroup reads
// about the same number of tokens whatever the mix of context lengths.  A
// workgroup finds its share by summing the lengths itself (they are on the
// device), its waves take 32 tokens of a step each and are joined in LDS.  A
// pair inside one share is finished there; one that several
// share leaves a partial (acc, m, l) per workgroup, and a second launch joins
// those.
#include <algorithm>

#include "amf_attn.h"
#include "amf_paged.h"

// Held to a tolerance, as the other attention kernels: multiplies and adds may
// fuse.
#pragma clang fp contract(fast)

namespace {

using namespace amf;

constexpr int kChunk = 32;  // tokens of a wave's step
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kStep = kWaves * kChunk;
constexpr int kMaxDim = 256;

struct PagedArgs {
  const void* q;
  int64_t q_seq, q_head;  // strides, elements
  void* out;
  const uint8_t* k;
  const uint8_t* v;
  int64_t page_stride, token_stride, head_stride;  // bytes
  int64_t pool_pages;
  const int32_t* block_tables;
  int64_t bt_stride;
  int32_t table_pages;
  const int32_t* context_lens;
  const int32_t* pages;        // [seq][KV head][max_pages], or null: every page
  const int32_t* page_counts;  // [seq][KV head]
  int32_t max_pages;
  int32_t num_seqs, num_q_heads, num_kv_heads, head_dim, block_size;
  int32_t block_shift;  // log2(block_size), or -1
  int32_t group;        // query heads of a KV head
  int32_t tiles;        // head tiles of a group
  int32_t out_dtype;
  float score_scale;    // softmax scale * k_scale * log2(e)
  float v_scale;
  float* part;          // [workgroup][2][heads of a tile][head_dim + kPartPad]
  int64_t part_stride;  // floats of one partial
  int32_t* err_flag;
};

// ---- shares --------------------------------------------------------------------

// Tokens that sequence s reads for a KV head: its context, or, with page lists,
// the pages of its longest list.
__device__ __forceinline__ int64_t seq_tokens(const PagedArgs& a, int s) {
  const int64_t c = a.context_lens[s];
  if (c <= 0) return 0;
  if (a.pages) {
    int n = 0;
    for (int h = 0; h < a.num_kv_heads; ++h)
      n = max(n, a.page_counts[(int64_t)s * a.num_kv_heads + h]);
    return (int64_t)min(n, a.max_pages) * a.block_size;
  }
  return min(c, (int64_t)a.table_pages * a.block_size);
}

__device__ __forceinline__ int64_t seq_steps(const PagedArgs& a, int s) {
  return (seq_tokens(a, s) + kStep - 1) / kStep;
}

// Where a unit (a step of a pair) lies.
struct Unit {
  int64_t total;  // units of the launch
  int64_t share;  // units of a workgroup
  int seq;
  int64_t start;  // first unit of that sequence
  int64_t steps;  // of each of its pairs
};

// The place of unit at(share), the same in every thread; seq is -1 behind the
// last unit.
template <typename At>
__device__ __forceinline__ Unit find_unit(const PagedArgs& a, int64_t groups, const At& at) {
  __shared__ int64_t tmp[kWaves];
  __shared__ Unit found;
  const int64_t pairs = (int64_t)a.num_kv_heads * a.tiles;
  const int tid = threadIdx.x;
  Unit r{};
  int64_t steps = 0, before = 0;
  if (a.num_seqs <= kThreads) {  // one scan gives the total and the places
    if (tid < a.num_seqs) steps = seq_steps(a, tid);
    before = block_exclusive<kThreads>(steps * pairs, tmp, &r.total);
  } else {
    int64_t mine = 0;
    for (int s = tid; s < a.num_seqs; s += kThreads) mine += seq_steps(a, s) * pairs;
    block_exclusive<kThreads>(mine, tmp, &r.total);
  }
  r.share = (r.total + groups - 1) / groups;
  const int64_t u = at(r.share);
  if (u >= r.total) {
    r.seq = -1;
    return r;
  }
  if (a.num_seqs <= kThreads) {
    if (before <= u && u < before + steps * pairs) found = Unit{r.total, r.share, tid, before, steps};
    __syncthreads();
    return found;
  }
  int64_t base = 0;
  for (int s0 = 0;; s0 += kThreads) {
    const int s = s0 + tid;
    int64_t all;
    steps = s < a.num_seqs ? seq_steps(a, s) : 0;
    before = base + block_exclusive<kThreads>(steps * pairs, tmp, &all);
    if (u < base + all) {  // uniform; u < total, so this comes
      if (before <= u && u < before + steps * pairs) found = Unit{r.total, r.share, s, before, steps};
      __syncthreads();
      return found;
    }
    base += all;
  }
}

// ---- tokens --------------------------------------------------------------------

// Byte offset of token i of the list of (s, hkv) from the cache's start, -1 for
// one that is not there.
__device__ __forceinline__ int64_t token_offset(const PagedArgs& a, int s, int hkv, int64_t i,
                                                int64_t ctx) {
  int64_t j = a.block_shift >= 0 ? i >> a.block_shift : i / a.block_size;
  const int at = (int)(i - j * a.block_size);
  if (a.pages) {
    const int64_t row = (int64_t)s * a.num_kv_heads + hkv;
    if (j >= min(a.page_counts[row], a.max_pages)) return -1;
    j = a.pages[row * a.max_pages + j];
    if (j < 0) return -1;
  }
  if (j * a.block_size + at >= ctx) return -1;
  const int64_t id = j < a.table_pages ? a.block_tables[s * a.bt_stride + j] : -1;
  if (id < 0 || id >= a.pool_pages) {
    if (a.err_flag) atomicOr(a.err_flag, AMF_ERRFLAG_BLOCK_RANGE);
    return -1;
  }
  return id * a.page_stride + at * a.token_stride + hkv * a.head_stride;
}

// ---- joining -------------------------------------------------------------------

// 2^(m - top), 1 where they are equal (-inf: nothing seen yet, or only scores
// of -inf, whose sum is NaN already).
__device__ __forceinline__ float weight_to(float m, float top) {
  return m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
}

// The larger, NaN if either is.
__device__ __forceinline__ float max_nan(float x, float y) {
  return __builtin_elementwise_maximum(x, y);
}

__device__ __forceinline__ void store_out(const PagedArgs& a, int64_t i, float x) {
  if (a.out_dtype == AMF_DTYPE_F32) {
    static_cast<float*>(a.out)[i] = x;
  } else {
    static_cast<uint16_t*>(a.out)[i] =
        (uint16_t)(a.out_dtype == AMF_DTYPE_BF16 ? pack2<true>(x, 0.0f) : pack2<false>(x, 0.0f));
  }
}

// Zeros for the sequences without tokens, and the flag of contexts that their
// block tables do not hold; the workgroups take turns.
__device__ __forceinline__ void empty_seqs(const PagedArgs& a) {
  const int64_t row = (int64_t)a.num_q_heads * a.head_dim;
  for (int64_t s = blockIdx.x; s < a.num_seqs; s += gridDim.x) {
    if (seq_tokens(a, (int)s) == 0)
      for (int64_t i = threadIdx.x; i < row; i += kThreads) store_out(a, s * row + i, 0.0f);
    if (threadIdx.x == 0 && a.err_flag &&
        (int64_t)a.context_lens[s] > (int64_t)a.table_pages * a.block_size)
      atomicOr(a.err_flag, AMF_ERRFLAG_CONTEXT);
  }
}

// ---- general kernel ------------------------------------------------------------
//
// Any element type, head_dim up to 256, strides and alignment: element loads.
// A lane scores one token of the chunk (two lanes share its dims) and, for PV,
// owns dims lane, lane + 64, ...
constexpr int kGenHeads = 4;  // query heads of a tile

template <int QDT, int KDT>
__global__ __launch_bounds__(kThreads) void paged_attn_general_kernel(PagedArgs a) {
  constexpr int ES = KDT == AMF_DTYPE_F32 ? 4 : KDT == AMF_DTYPE_E4M3 ? 1 : 2;
  constexpr int QS = QDT == AMF_DTYPE_F32 ? 4 : 2;
  constexpr int DI = kMaxDim / 64;
  __shared__ float q_lds[kGenHeads][kMaxDim];
  __shared__ float p_lds[kWaves][kGenHeads][kChunk];
  __shared__ float acc_lds[kWaves][kGenHeads][kMaxDim];
  __shared__ float m_lds[kWaves][kGenHeads], l_lds[kWaves][kGenHeads];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int D = a.head_dim, half = lane >> 5;
  const int d0 = half ? (D + 1) / 2 : 0, d1 = half ? D : (D + 1) / 2;
  empty_seqs(a);
  Unit un = find_unit(a, gridDim.x, [](int64_t share) { return (int64_t)blockIdx.x * share; });
  if (un.seq < 0) return;
  const int64_t pairs = (int64_t)a.num_kv_heads * a.tiles;
  const int64_t u0 = blockIdx.x * un.share, u1 = min(u0 + un.share, un.total);
  for (int64_t u = u0; u < u1;) {
    const int64_t pair = (u - un.start) / un.steps;
    const int64_t st0 = (u - un.start) % un.steps, st1 = min(un.steps, st0 + (u1 - u));
    const int s = un.seq, hkv = (int)(pair / a.tiles), tile = (int)(pair % a.tiles);
    const int heads = min(kGenHeads, a.group - tile * kGenHeads);
    const int head0 = hkv * a.group + tile * kGenHeads;
    const int64_t ctx = a.context_lens[s], len = seq_tokens(a, s);
    __syncthreads();
    for (int i = tid; i < kGenHeads * D; i += kThreads) {
      const int g = i / D, d = i - g * D;
      q_lds[g][d] = g < heads ? kv_elem<QDT>(static_cast<const uint8_t*>(a.q) +
                                             (s * a.q_seq + (head0 + g) * a.q_head + d) * QS)
                              : 0.0f;
    }
    __syncthreads();
    float m[kGenHeads], l[kGenHeads], acc[kGenHeads][DI];
#pragma unroll
    for (int g = 0; g < kGenHeads; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.0f;
#pragma unroll
      for (int i = 0; i < DI; ++i) acc[g][i] = 0.0f;
    }
    for (int64_t st = st0; st < st1; ++st) {
      const int64_t t = st * kStep + wave * kChunk + (lane & 31);
      const int64_t off = t < len ? token_offset(a, s, hkv, t, ctx) : -1;
      const bool ok = off >= 0;
      if (!__any(ok)) continue;
      float x[kGenHeads];
#pragma unroll
      for (int g = 0; g < kGenHeads; ++g) x[g] = 0.0f;
      if (ok) {
        for (int d = d0; d < d1; ++d) {
          const float kd = kv_elem<KDT>(a.k + off + d * ES);
#pragma unroll
          for (int g = 0; g < kGenHeads; ++g) x[g] = __builtin_fmaf(q_lds[g][d], kd, x[g]);
        }
      }
#pragma unroll
      for (int g = 0; g < kGenHeads; ++g) {
        x[g] += __shfl_xor(x[g], 32);
        float top = ok ? x[g] * a.score_scale : -INFINITY;
        for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor(top, o));
        const float mn = max_nan(m[g], top);
        const float p = ok ? __builtin_amdgcn_exp2f(__builtin_fmaf(x[g], a.score_scale, -mn)) : 0.0f;
        const float w = weight_to(m[g], mn);
        m[g] = mn;
        l[g] = l[g] * w + (half ? 0.0f : p);
#pragma unroll
        for (int i = 0; i < DI; ++i) acc[g][i] *= w;
        if (!half) p_lds[wave][g][lane] = p;
      }
      __builtin_amdgcn_wave_barrier();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      for (int j = 0; j < kChunk; ++j) {
        const int64_t row = __shfl(off, j);
        if (row < 0) continue;
        float w[kGenHeads];
#pragma unroll
        for (int g = 0; g < kGenHeads; ++g) w[g] = p_lds[wave][g][j];
#pragma unroll
        for (int i = 0; i < DI; ++i) {
          const int d = lane + 64 * i;
          if (d >= D) continue;
          const float vd = kv_elem<KDT>(a.v + row + d * ES);
#pragma unroll
          for (int g = 0; g < kGenHeads; ++g) acc[g][i] = __builtin_fmaf(w[g], vd, acc[g][i]);
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int g = 0; g < kGenHeads; ++g) {
      float sum = l[g];
      for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
      if (lane == 0) {
        m_lds[wave][g] = m[g];
        l_lds[wave][g] = sum;
      }
#pragma unroll
      for (int i = 0; i < DI; ++i) acc_lds[wave][g][lane + 64 * i] = acc[g][i];
    }
    __syncthreads();
    const bool whole = st0 == 0 && st1 == un.steps;
    float* part = whole ? nullptr : a.part + (2 * (int64_t)blockIdx.x + (u != u0)) * a.part_stride;
    for (int i = tid; i < heads * D; i += kThreads) {
      const int g = i / D, d = i - g * D;
      float top = m_lds[0][g], sum = 0.0f, x = 0.0f;
      for (int w = 1; w < kWaves; ++w) top = max_nan(top, m_lds[w][g]);
      for (int w = 0; w < kWaves; ++w) {
        const float f = weight_to(m_lds[w][g], top);
        sum = __builtin_fmaf(l_lds[w][g], f, sum);
        x = __builtin_fmaf(acc_lds[w][g][d], f, x);
      }
      if (whole) {
        store_out(a, ((int64_t)s * a.num_q_heads + head0 + g) * D + d,
                  sum == 0.0f ? 0.0f : x * (a.v_scale / sum));
      } else {
        part[g * (D + kPartPad) + d] = x;
        if (d == 0) {
          part[g * (D + kPartPad) + D] = top;
          part[g * (D + kPartPad) + D + 1] = sum;
        }
      }
    }
    // the next pair, perhaps of the next sequence with tokens
    u += st1 - st0;
    if (u < u1 && u == un.start + pairs * un.steps) {
      un.start = u;
      do {
        ++un.seq;
        un.steps = seq_steps(a, un.seq);
      } while (un.steps == 0);
    }
  }
}

// ---- merge ---------------------------------------------------------------------
//
// Workgroup b looks at the boundary between shares b and b + 1.  When it cuts a
// pair, and is the first that does, the workgroup joins the pair's partials:
// slot 1 of the workgroup the pair begins in (slot 0 if it begins the share),
// slot 0 of the others.
template <int TILE>
__global__ __launch_bounds__(kThreads) void paged_attn_merge_kernel(PagedArgs a, int64_t groups) {
  const int64_t b = blockIdx.x;
  const Unit un = find_unit(a, groups, [b](int64_t share) { return (b + 1) * share; });
  if (un.seq < 0) return;
  const int64_t ub = (b + 1) * un.share;
  const int64_t pair = (ub - un.start) / un.steps;
  const int64_t begin = un.start + pair * un.steps, end = begin + un.steps;
  if (begin == ub || begin < ub - un.share) return;
  const int64_t last = (end - 1) / un.share;
  const int hkv = (int)(pair / a.tiles), tile = (int)(pair % a.tiles);
  const int heads = min(TILE, a.group - tile * TILE);
  const int D = a.head_dim, row = D + kPartPad;
  const int64_t head0 = (int64_t)un.seq * a.num_q_heads + hkv * a.group + tile * TILE;
  for (int i = threadIdx.x; i < heads * D; i += kThreads) {
    const int g = i / D, d = i - g * D;
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    for (int64_t w = b; w <= last; ++w) {
      const int slot = w == b && begin != b * un.share;
      const float* p = a.part + (2 * w + slot) * a.part_stride + g * row;
      const float pm = p[D], top = max_nan(m, pm);
      const float f = weight_to(m, top), pf = weight_to(pm, top);
      l = l * f + p[D + 1] * pf;
      acc = acc * f + p[d] * pf;
      m = top;
    }
    store_out(a, (head0 + g) * D + d, l == 0.0f ? 0.0f : acc * (a.v_scale / l));
  }
}

// ---- launch --------------------------------------------------------------------

constexpr int64_t kGroups = 1024;  // workgroups of a launch

int tile_heads(int32_t group) { return std::min<int32_t>(group, kGenHeads); }

int64_t part_floats(int32_t group, int32_t head_dim) {
  return (int64_t)tile_heads(group) * (head_dim + kPartPad);
}

template <int QDT, int KDT>
void launch_general(const PagedArgs& a, hipStream_t st) {
  paged_attn_general_kernel<QDT, KDT><<<dim3((unsigned)kGroups), kThreads, 0, st>>>(a);
}

}  // namespace

extern "C" int64_t amf_paged_decode_workspace_bytes(int32_t num_q_heads, int32_t num_kv_heads,
                                                    int32_t head_dim) {
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 || head_dim <= 0 ||
      head_dim > kMaxDim)
    return 0;
  return 2 * kGroups * part_floats(num_q_heads / num_kv_heads, head_dim) * (int64_t)sizeof(float);
}

extern "C" int amf_paged_decode_attn(
    const void* q, int32_t q_dtype, int64_t q_seq_stride, int64_t q_head_stride, void* out,
    int32_t out_dtype, const void* k, const void* v, int32_t kv_dtype, int64_t page_stride,
    int64_t token_stride, int64_t head_stride, int64_t pool_pages, const int32_t* block_tables,
    int64_t bt_stride, int32_t table_pages, const int32_t* context_lens, const int32_t* pages,
    const int32_t* page_counts, int32_t max_pages, int32_t num_seqs, int32_t num_q_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int32_t max_context_len,
    float softmax_scale, float k_scale, float v_scale, void* workspace, int64_t workspace_bytes,
    int32_t* err_flag, void* stream) {
  const char* who = "amf_paged_decode_attn";
  if (num_seqs < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 ||
      head_dim <= 0 || block_size <= 0 || table_pages < 0 || bt_stride < table_pages ||
      pool_pages <= 0 || max_pages < 0 || max_context_len < 0)
    return fail(AMF_ERR_INVALID_ARG,
                "%s: bad num_seqs=%d heads=%d/%d (a multiple) head_dim=%d block_size=%d "
                "table_pages=%d bt_stride=%lld pool_pages=%lld max_pages=%d max_context_len=%d",
                who, num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, table_pages,
                (long long)bt_stride, (long long)pool_pages, max_pages, max_context_len);
  const int es = kv_elem_bytes(kv_dtype);
  if (es == 0 || head_dim > kMaxDim)
    return fail(AMF_ERR_UNSUPPORTED, "%s: cache dtype %d, head_dim %d (at most %d)", who, kv_dtype,
                head_dim, kMaxDim);
  if (cache_elem_bytes(q_dtype) == 0 || cache_elem_bytes(out_dtype) == 0 ||
      (es == 1 ? q_dtype == AMF_DTYPE_F32 : q_dtype != kv_dtype))
    return fail(AMF_ERR_INVALID_ARG,
                "%s: q of type %d and out of type %d with a cache of type %d (q has the cache's "
                "type, with FP8 bf16 or fp16)",
                who, q_dtype, out_dtype, kv_dtype);
  if (num_seqs == 0) return ok();
  if (!q || !out || !k || !v || !context_lens || (table_pages > 0 && !block_tables) ||
      (pages && !page_counts))
    return fail(AMF_ERR_INVALID_ARG, "%s: null pointer", who);
  const int qs = cache_elem_bytes(q_dtype);
  if ((uintptr_t)q % qs || (uintptr_t)k % es || (uintptr_t)v % es ||
      (uintptr_t)out % cache_elem_bytes(out_dtype))
    return fail(AMF_ERR_INVALID_ARG, "%s: a tensor is not aligned to its elements", who);
  const int64_t need = amf_paged_decode_workspace_bytes(num_q_heads, num_kv_heads, head_dim);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
    return fail(AMF_ERR_WORKSPACE, "%s: workspace of %lld bytes (16-byte aligned) needed, got %lld",
                who, (long long)need, (long long)workspace_bytes);
  PagedArgs a{};
  a.q = q;
  a.q_seq = q_seq_stride;
  a.q_head = q_head_stride;
  a.out = out;
  a.k = static_cast<const uint8_t*>(k);
  a.v = static_cast<const uint8_t*>(v);
  a.page_stride = page_stride * es;
  a.token_stride = token_stride * es;
  a.head_stride = head_stride * es;
  a.pool_pages = pool_pages;
  a.block_tables = block_tables;
  a.bt_stride = bt_stride;
  a.table_pages = table_pages;
  a.context_lens = context_lens;
  a.pages = pages;
  a.page_counts = page_counts;
  a.max_pages = max_pages;
  a.num_seqs = num_seqs;
  a.num_q_heads = num_q_heads;
  a.num_kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.block_size = block_size;
  a.block_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
  a.group = num_q_heads / num_kv_heads;
  a.tiles = (a.group + kGenHeads - 1) / kGenHeads;
  a.out_dtype = out_dtype;
  a.score_scale = (softmax_scale > 0.0f ? softmax_scale : 1.0f / sqrtf((float)head_dim)) *
                  k_scale * kLog2e;
  a.v_scale = v_scale;
  a.part = static_cast<float*>(workspace);
  a.part_stride = part_floats(a.group, head_dim);
  a.err_flag = err_flag;
  hipStream_t st = as_stream(stream);
  if (kv_dtype == AMF_DTYPE_BF16)
    launch_general<AMF_DTYPE_BF16, AMF_DTYPE_BF16>(a, st);
  else if (kv_dtype == AMF_DTYPE_F16)
    launch_general<AMF_DTYPE_F16, AMF_DTYPE_F16>(a, st);
  else if (kv_dtype == AMF_DTYPE_F32)
    launch_general<AMF_DTYPE_F32, AMF_DTYPE_F32>(a, st);
  else if (q_dtype == AMF_DTYPE_BF16)
    launch_general<AMF_DTYPE_BF16, AMF_DTYPE_E4M3>(a, st);
  else
    launch_general<AMF_DTYPE_F16, AMF_DTYPE_E4M3>(a, st);
  if (int rc = check_launch(who)) return rc;
  paged_attn_merge_kernel<kGenHeads><<<dim3((unsigned)(kGroups - 1)), kThreads, 0, st>>>(a, kGroups);
  return check_launch(who);
}

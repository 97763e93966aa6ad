// amf_paged_attn.hip - attention of one new token per sequence over a paged
// K/V cache as vLLM keeps it (bf16, fp16, fp32 or FP8 e4m3 elements in pages
// [token][head][dim], read in place through the block table), split over the
// context and joined.
//
//   out[s, h] = v_scale * sum_t softmax_t(k_scale * scale * q[s, h] . k[t]) v[t]
//
// over the context_lens[s] tokens of the sequence, or those of the pages listed
// for its KV head.  Each K and V element is read once for a tile of the query heads
// that share it (up to 16 in the matrix kernel, 4 in the general one; larger groups
// read it again for each tile), and meets the running maximum m and sum l of each
// head's softmax.
//
// Work.  The contexts of all sequences, one after the other, are steps, cut into
// equal shares; a share is taken by a few workgroups side by side, each for one, two
// or four (KV head, head tile) pairs.  They read the same pages at the same time,
// and the grid is resident as a whole, so every workgroup reads about the same
// number of tokens whatever the mix of context lengths.  A workgroup finds its share
// by summing the lengths itself (they are on the device); waves of the same pair
// split a step's tokens and are joined in LDS.  What of a sequence lies inside one
// share is finished there; where several share it, each leaves a partial (acc, m,
// l), and a second launch joins those.  Short contexts take a workgroup per
// sequence and pair and no second launch.
//
// Measured (MI355X, bytes of K and V over the call's time): 32 sequences of 1K-32K
// tokens, bf16, 32 / 8 heads of 128, 340 us, 6.5 TB/s; 8 x 126K tokens, FP8, 64 / 8
// heads, 336 us, 6.1 TB/s; 200 chats of 1-1200 tokens, fp16, 105 us, 4.7 TB/s (a share
// is two sequences there, and the beginning of each is latency); two short contexts
// 11 us, nothing but latency.  The large ones are bound by HBM.
#include <algorithm>

#include "amf_attn.h"
#include "amf_paged.h"

// Held to a tolerance, as the other attention kernels: multiplies and adds may
// fuse.
#pragma clang fp contract(fast)

namespace {

using namespace amf;

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
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
  int32_t step_shift;   // log2 of the tokens of a step (of all waves)
  int32_t group;        // query heads of a KV head
  int32_t tiles;        // head tiles of a group
  int32_t side;         // (KV head, head tile) pairs of a workgroup: 1, 2 or 4
  int32_t out_dtype;
  float score_scale;    // softmax scale * k_scale * log2(e)
  float v_scale;
  bool whole;           // a share is a whole sequence
  bool by_seq;          // cuts are kept by sequence (fewer than shares), else by share
  struct Cut* cuts;     // [sequence or share][pair]
  float* part;          // [share][pair][2][heads of a tile][head_dim + kPartPad]
  int64_t part_stride;  // floats of one partial
  int32_t* err_flag;
};

// A pair that does not end in the share where it begins: its partials are slot
// `slot` of that share's place and slot 0 of the `more` next shares' for the pair.
struct Cut {
  int32_t heads;  // 0: no such pair
  int32_t head0;  // of the step's rows
  int32_t more;
  int32_t place;  // 2 * place + slot
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
  return (seq_tokens(a, s) + (1 << a.step_shift) - 1) >> a.step_shift;
}

// The step at which a workgroup's share begins, counted over the sequences.
struct Unit {
  int64_t total;  // steps of the launch
  int64_t share;  // steps of a workgroup
  int64_t first;  // of this workgroup
  int seq;        // the sequence it lies in, -1: there is none
  int64_t start;  // first step of that sequence
  int64_t steps;  // its steps
};

__device__ __forceinline__ int pairs_of(const PagedArgs& a) { return a.num_kv_heads * a.tiles; }
// Workgroups of a share.
__device__ __forceinline__ int teams_of(const PagedArgs& a) { return pairs_of(a) / a.side; }

// The same in every thread.
__device__ __forceinline__ Unit find_unit(const PagedArgs& a) {
  __shared__ int64_t tmp[kWaves];
  __shared__ int found_seq;
  __shared__ int64_t found_start, found_steps;
  const int teams = teams_of(a);
  const int64_t shares = gridDim.x / teams, mine = blockIdx.x / teams;
  const int tid = threadIdx.x;
  Unit r{};
  if (a.whole) {
    r.seq = (int)mine;
    r.total = r.share = r.steps = seq_steps(a, r.seq);
    if (r.steps == 0) r.seq = -1;
    return r;
  }
  int64_t steps = 0, before = 0;
  if (a.num_seqs <= kThreads) {  // one scan gives the total and the places
    if (tid < a.num_seqs) steps = seq_steps(a, tid);
    before = block_exclusive<kThreads>(steps, tmp, &r.total);
  } else {
    int64_t sum = 0;
    for (int s = tid; s < a.num_seqs; s += kThreads) sum += seq_steps(a, s);
    block_exclusive<kThreads>(sum, tmp, &r.total);
  }
  r.share = (r.total + shares - 1) / shares;
  r.first = mine * r.share;
  if (r.first >= r.total) {
    r.seq = -1;
    return r;
  }
  int64_t base = 0;
  for (int s0 = 0;; s0 += kThreads) {
    if (a.num_seqs > kThreads) {
      int64_t all;
      steps = s0 + tid < a.num_seqs ? seq_steps(a, s0 + tid) : 0;
      before = base + block_exclusive<kThreads>(steps, tmp, &all);
      base += all;
      if (r.first >= base) continue;  // uniform; first < total, so this ends
    }
    if (before <= r.first && r.first < before + steps) {
      found_seq = s0 + tid;
      found_start = before;
      found_steps = steps;
    }
    __syncthreads();
    r.seq = found_seq;
    r.start = found_start;
    r.steps = found_steps;
    return r;
  }
}

// ---- segments ------------------------------------------------------------------

// The steps of one pair that lie in a share.
struct Segment {
  int seq, hkv, heads;
  int64_t head0;     // first query head, of the step's rows
  int64_t st0, st1;  // steps
  int64_t ctx;
  bool whole;        // all steps of the pair
  float* part;       // where the partial goes otherwise
};

// The segment from step u of sequence un.seq on, for pair n of the workgroup; the
// share ends at u1.
template <int TILE>
__device__ __forceinline__ Segment segment_at(const PagedArgs& a, const Unit& un, int64_t u,
                                              int64_t u1, int n) {
  Segment g;
  const int teams = teams_of(a), pair = (blockIdx.x % teams) * a.side + n;
  const int64_t share = blockIdx.x / teams, place = share * pairs_of(a) + pair;
  g.st0 = u - un.start;
  g.st1 = min(un.steps, g.st0 + (u1 - u));
  g.seq = un.seq;
  g.hkv = pair / a.tiles;
  const int tile = pair - g.hkv * a.tiles;
  g.heads = min(TILE, a.group - tile * TILE);
  g.head0 = (int64_t)un.seq * a.num_q_heads + g.hkv * a.group + tile * TILE;
  g.ctx = a.context_lens[un.seq];
  g.whole = g.st0 == 0 && g.st1 == un.steps;
  g.part = a.part + (2 * place + (u != un.first)) * a.part_stride;
  return g;
}

// Notes whether the pair of a segment that begins it is cut.
__device__ __forceinline__ void note_cut(const PagedArgs& a, const Unit& un, const Segment& g,
                                         int64_t u, int n) {
  if (a.whole || g.st0 != 0 || (g.whole && !a.by_seq)) return;
  const int teams = teams_of(a), pairs = pairs_of(a), pair = (blockIdx.x % teams) * a.side + n;
  const int64_t share = blockIdx.x / teams;
  a.cuts[(a.by_seq ? g.seq : share) * pairs + pair] =
      Cut{g.whole ? 0 : g.heads, (int32_t)g.head0,
          (int32_t)((u + un.steps - 1) / un.share - share),
          (int32_t)(2 * (share * pairs + pair) + (u != un.first))};
}

// Moves on to step u, perhaps of the next sequence with tokens; u lies in the
// launch.
__device__ __forceinline__ void advance(const PagedArgs& a, Unit& un, int64_t u) {
  if (u < un.start + un.steps) return;
  un.start = u;
  do {
    ++un.seq;
    un.steps = seq_steps(a, un.seq);
  } while (un.steps == 0);
}

// The pages of a run of steps, looked up by the workgroup and kept in LDS: the
// loads of K and V then depend on no load but their own.
constexpr int kPageSlots = 1024;
struct PageRun {
  int32_t id[kPageSlots];
  int32_t tokens[kPageSlots];  // of the page that count; 0 where there is none
};

// Steps that a run holds: kPageSlots pages, one of them begun before the run.
__device__ __forceinline__ int64_t run_steps(const PagedArgs& a) {
  return max((int64_t)1, (int64_t)(kPageSlots - 1) * a.block_size >> a.step_shift);
}

__device__ __forceinline__ int64_t page_of(const PagedArgs& a, int64_t t) {
  return a.block_shift >= 0 ? t >> a.block_shift : t / a.block_size;
}

__device__ __forceinline__ void load_pages(const PagedArgs& a, const Segment& g, int64_t st0,
                                           int64_t st1, PageRun& run) {
  __syncthreads();  // the last run has been read
  const int64_t j0 = page_of(a, st0 << a.step_shift);
  const int64_t j1 = page_of(a, (st1 << a.step_shift) - 1);
  const int64_t row = (int64_t)g.seq * a.num_kv_heads + g.hkv;
  const int64_t count = a.pages ? min(a.page_counts[row], a.max_pages) : a.table_pages;
  for (int64_t j = j0 + threadIdx.x; j <= j1; j += kThreads) {
    int64_t p = -1, left = 0;
    int32_t id = 0;
    if (j < count) p = a.pages ? a.pages[row * a.max_pages + j] : j;
    if (p >= 0) left = min(g.ctx - p * a.block_size, (int64_t)a.block_size);
    if (left > 0) {
      id = p < a.table_pages ? a.block_tables[g.seq * a.bt_stride + p] : -1;
      if (id < 0 || id >= a.pool_pages) {
        if (a.err_flag) atomicOr(a.err_flag, AMF_ERRFLAG_BLOCK_RANGE);
        id = 0;
        left = 0;
      }
    }
    run.id[j - j0] = id;
    run.tokens[j - j0] = (int32_t)max(left, (int64_t)0);
  }
  __syncthreads();
}

// Byte offset of token t's row from the cache's start, -1 for a token that does
// not count; the run begins with page j0.
__device__ __forceinline__ int64_t token_offset(const PagedArgs& a, const Segment& g,
                                                const PageRun& run, int64_t j0, int64_t t) {
  const int64_t j = page_of(a, t);
  const int at = (int)(t - j * a.block_size);
  if (at >= run.tokens[j - j0]) return -1;
  return run.id[j - j0] * a.page_stride + at * a.token_stride + g.hkv * a.head_stride;
}

// ---- joining -------------------------------------------------------------------

// A part with m = -inf has seen no token (l = 0) or only scores of -inf (l > 0, which
// no longer sums weights).  Next to a finite score both weigh nothing.

// 2^(m - top), 1 where they are equal.
__device__ __forceinline__ float weight_to(float m, float top) {
  return m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
}

// What is taken from a score before 2^x: the maximum, or 0 where that is -inf (the
// difference would be NaN, and stay, where another part has finite scores).
__device__ __forceinline__ float exp_base(float m) { return m == -INFINITY ? 0.0f : m; }

// The factor of a head's weighted rows, for l > 0: NaN where all scores are -inf.
__device__ __forceinline__ float row_factor(float v_scale, float m, float l) {
  return m == -INFINITY ? __builtin_nanf("") : v_scale / l;
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
// block tables do not hold (the workgroups take turns); no cut, until one is noted.
__device__ __forceinline__ void empty_seqs(const PagedArgs& a) {
  const int64_t row = (int64_t)a.num_q_heads * a.head_dim;
  if (!a.whole && !a.by_seq && threadIdx.x < a.side)  // until a cut is found
    a.cuts[(int64_t)blockIdx.x * a.side + threadIdx.x].heads = 0;
  for (int64_t s = blockIdx.x; s < a.num_seqs; s += gridDim.x) {
    if (seq_tokens(a, (int)s) == 0) {
      for (int64_t i = threadIdx.x; i < row; i += kThreads) store_out(a, s * row + i, 0.0f);
      if (!a.whole && a.by_seq)
        for (int i = threadIdx.x; i < pairs_of(a); i += kThreads)
          a.cuts[s * pairs_of(a) + i].heads = 0;
    }
    if (threadIdx.x == 0 && a.err_flag &&
        (int64_t)a.context_lens[s] > (int64_t)a.table_pages * a.block_size)
      atomicOr(a.err_flag, AMF_ERRFLAG_CONTEXT);
  }
}

// ---- general kernel ------------------------------------------------------------
//
// Any element type, head_dim up to 256, strides and alignment.  LPR lanes share a
// token's row, 8 dims each (one or two 16-byte loads, or element by element where
// rows are not aligned or end inside one), so a wave reads 64 / LPR rows at once,
// kGenAhead of them after each other in flight; every such group of lanes keeps its
// own m, l and output for 4 query heads, and all groups of the workgroup are joined in
// LDS.
// fp32, 12 / 4 heads of 96, 2 x 9500 tokens, 58 MB: 33 us, 1.75 TB/s; 32 / 8 of 128, 4 x
// 9500, 311 MB: 78 us, 4.0 TB/s, where the beginning and the merge are some 20 us; 64 / 8
// of 128, whose K and V are read twice, 111 us; 36 dims of fp16, element by element, 37
// MB in 58 us.  Tried, against 34 and 79 us of the first two: a branch around the loads,
// in place of page 0's rows, 37 and 79; the next step's rows asked for before this one's
// are used, 34 and 79; a lane per token for the scores and a lane per dim for the
// output, with element loads, 88 for the first.
constexpr int kGenHeads = 4;  // query heads of a tile
constexpr int kGenAhead = 4;  // rows of a group of lanes in a step

// Eight consecutive elements, `n` of which are there.  ROWS: all or none are, and the
// first 8 at p can be read all the same: no branch, whose end would wait for the load.
template <int DT, bool ROWS>
__device__ __forceinline__ void load_row8(const uint8_t* p, int n, float* x) {
  constexpr int ES = DT == AMF_DTYPE_F32 ? 4 : DT == AMF_DTYPE_E4M3 ? 1 : 2;
  if constexpr (ROWS) {
    if constexpr (DT == AMF_DTYPE_E4M3) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(p);
      e4m3x4_to_f32(w[0], x);
      e4m3x4_to_f32(w[1], x + 4);
    } else {
      load8<DT>(p, x);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = n > 0 ? x[e] : 0.0f;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = e < n ? kv_elem<DT>(p + e * ES) : 0.0f;
  }
}

template <int QDT, int KDT, int LPR, bool ROWS>
__global__ __launch_bounds__(kThreads) void paged_attn_general_kernel(PagedArgs a) {
  constexpr int ES = KDT == AMF_DTYPE_F32 ? 4 : KDT == AMF_DTYPE_E4M3 ? 1 : 2;
  constexpr int QS = QDT == AMF_DTYPE_F32 ? 4 : 2;
  constexpr int RG = 64 / LPR;          // groups of a wave
  constexpr int PARTS = kWaves * RG;    // of the workgroup
  __shared__ PageRun run;
  __shared__ __attribute__((aligned(16))) float acc_lds[PARTS][kGenHeads][8 * LPR];
  __shared__ float m_lds[PARTS][kGenHeads], l_lds[PARTS][kGenHeads];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int D = a.head_dim, c = lane % LPR, grp = lane / LPR, part_id = wave * RG + grp;
  const int dims = min(8, D - 8 * c);  // of this lane; none below 1
  empty_seqs(a);
  Unit un = find_unit(a);
  if (un.seq < 0) return;
  const int64_t u1 = min(un.first + un.share, un.total);
  for (int64_t u = un.first; u < u1;) {
    advance(a, un, u);
    const Segment sg = segment_at<kGenHeads>(a, un, u, u1, 0);
    if (tid == 0) note_cut(a, un, sg, u, 0);
    u += sg.st1 - sg.st0;
    // where there is no row, page 0's is read, and its first dims where there are none
    const int64_t head_off = sg.hkv * a.head_stride, at = ROWS && dims <= 0 ? 0 : 8 * c * ES;
    float q[kGenHeads][8];
#pragma unroll
    for (int g = 0; g < kGenHeads; ++g) {
      const int64_t head = sg.head0 - (int64_t)sg.seq * a.num_q_heads + g;
      const uint8_t* p = static_cast<const uint8_t*>(a.q) +
                         (sg.seq * a.q_seq + head * a.q_head + 8 * c) * QS;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        q[g][e] = g < sg.heads && e < dims ? kv_elem<QDT>(p + e * QS) : 0.0f;
    }
    float m[kGenHeads], l[kGenHeads], acc[kGenHeads][8];
#pragma unroll
    for (int g = 0; g < kGenHeads; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[g][e] = 0.0f;
    }
    const int64_t hold = run_steps(a);
    for (int64_t r0 = sg.st0; r0 < sg.st1; r0 += hold) {
      const int64_t r1 = min(r0 + hold, sg.st1), j0 = page_of(a, r0 << a.step_shift);
      load_pages(a, sg, r0, r1, run);
      for (int64_t st = r0; st < r1; ++st) {
        float k[kGenAhead][8], v[kGenAhead][8];
        bool ok[kGenAhead], any = false;
#pragma unroll
        for (int i = 0; i < kGenAhead; ++i) {
          const int64_t t = (st << a.step_shift) + (wave * kGenAhead + i) * RG + grp;
          const int64_t off = token_offset(a, sg, run, j0, t);
          ok[i] = off >= 0;
          any |= ok[i];
          const int n = ok[i] ? dims : 0;
          const int64_t o = (ROWS && off < 0 ? head_off : off) + at;
          load_row8<KDT, ROWS>(a.k + o, n, k[i]);
          load_row8<KDT, ROWS>(a.v + o, n, v[i]);
        }
#pragma unroll
        for (int g = 0; g < kGenHeads; ++g) {
          float x[kGenAhead], top = -INFINITY;
#pragma unroll
          for (int i = 0; i < kGenAhead; ++i) {
            x[i] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i] = __builtin_fmaf(q[g][e], k[i][e], x[i]);
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) x[i] += __shfl_xor(x[i], o, LPR);
            top = max_nan(top, ok[i] ? x[i] * a.score_scale : -INFINITY);
          }
          const float mn = max_nan(m[g], top), w = weight_to(m[g], mn), base = exp_base(mn);
          m[g] = mn;
          l[g] *= w;
          if (mn == -INFINITY && any) l[g] = 1.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[g][e] *= w;
#pragma unroll
          for (int i = 0; i < kGenAhead; ++i) {
            const float p =
                ok[i] ? __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], a.score_scale, -base)) : 0.0f;
            l[g] += p;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[g][e] = __builtin_fmaf(p, v[i][e], acc[g][e]);
          }
        }
      }
    }
    __syncthreads();  // the last pair's parts have been read
#pragma unroll
    for (int g = 0; g < kGenHeads; ++g) {
      if (c == 0) {
        m_lds[part_id][g] = m[g];
        l_lds[part_id][g] = l[g];
      }
#pragma unroll
      for (int e = 0; e < 8; e += 4)
        *reinterpret_cast<f32x4*>(&acc_lds[part_id][g][8 * c + e]) =
            f32x4{acc[g][e], acc[g][e + 1], acc[g][e + 2], acc[g][e + 3]};
    }
    __syncthreads();
    for (int i = tid; i < sg.heads * D; i += kThreads) {
      const int g = i / D, d = i - g * D;
      float top = m_lds[0][g], sum = 0.0f, x = 0.0f;
      for (int w = 1; w < PARTS; ++w) top = max_nan(top, m_lds[w][g]);
      for (int w = 0; w < PARTS; ++w) {
        const float f = weight_to(m_lds[w][g], top);
        sum = __builtin_fmaf(l_lds[w][g], f, sum);
        x = __builtin_fmaf(acc_lds[w][g][d], f, x);
      }
      if (sg.whole) {
        store_out(a, (sg.head0 + g) * D + d,
                  sum == 0.0f ? 0.0f : x * row_factor(a.v_scale, top, sum));
      } else {
        float* part = sg.part + g * (D + kPartPad);
        part[d] = x;
        if (d == 0) {
          part[D] = top;
          part[D + 1] = sum;
        }
      }
    }
  }
}

// ---- matrix kernel -------------------------------------------------------------
//
// bf16 and fp16 queries, head_dim a multiple of 16, rows of whole 16-byte vectors.
// A wave takes blocks of 32 tokens and up to 16 query heads on 16x16x32 tiles; lane
// (lo, hi) = (lane % 16, lane / 16).
//
//   scores   S^T = K Q^T: K rows as the A operand straight from memory (16 bytes
//            of row lo), the heads' q as B, kept in registers.  Lane (lo, hi)
//            gets head lo's scores of tokens 4 hi + r and 16 + 4 hi + r, r < 4.
//   weights  so a head's m and l are per-lane scalars (joined over hi), and its
//            8 weights are the B operand of the second product as they are, its
//            k slots taking those tokens.
//   output   O^T = V^T P^T: the A operand holds, of tokens 4 hi + r and 16 + 4 hi
//            + r, dims DP lo .. DP lo + DP - 1 (DP = head_dim / 16): 8 row pieces
//            that lie side by side in memory for the lanes of a row, transposed
//            in registers by byte permutes, and no K or V goes through LDS.
//
// Precision: products of 16-bit K and q are exact and summed in fp32.  Weights
// are fp32 and enter as three bf16 terms whose sum is the weight; fp16 V enters
// as two bf16 terms (11 bits), of which the lower meets the weight's first two
// terms (the third's product is below 2^-24 of the whole).  FP8 elements are
// exact in either 16-bit type.
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

template <int DT>
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (DT == AMF_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// Two of the four e4m3 codes of w (the low or the high two) as a pair of DT.
template <int DT, bool HIGH>
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {
  if constexpr (DT == AMF_DTYPE_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HIGH));
}

constexpr int kTileHeads = 16;
// Waves per SIMD, at least.  256 dims of 16 bits spill at two (164 sequences of 4700
// fp16 tokens 272 -> 434 us); of FP8 they are faster with 12 to 15 words spilled (the same
// 170 -> 163, 200 chats 53 -> 48).
constexpr int matrix_waves(int D, int es) { return D == 256 && es == 2 ? 1 : 2; }
// Tokens of a wave's step.  64 of 64 dims (two sequences of 700 tokens 12.3 -> 11.6
// us; fewer, larger steps); 64 of 128 FP8 dims are as many bytes but slower than 32
// (8 x 128K 342 / 335 us).
constexpr int matrix_chunk(int D) { return D <= 64 ? 64 : 32; }

// D: the head_dim, or (FULL false) the next of 64, 128 and 256 above a multiple of
// 16, with zeros in the dims that are not there.
template <int QDT, int KDT, int D, bool FULL>
__global__ __launch_bounds__(kThreads, matrix_waves(D, KDT == AMF_DTYPE_E4M3 ? 1 : 2)) void
paged_attn_matrix_kernel(PagedArgs a) {
  constexpr bool FP8 = KDT == AMF_DTYPE_E4M3;
  constexpr bool V16 = KDT == AMF_DTYPE_F16;  // V in two terms
  constexpr int ES = FP8 ? 1 : 2;
  constexpr int CH = matrix_chunk(D), NB = CH / 32;
  constexpr int KS = D / 32;          // k steps of a score tile
  constexpr int KL = KS * ES / 2;     // 16-byte loads of a K row per lane
  constexpr int DP = D / 16;          // dims of a V row per lane
  constexpr int VW = DP * ES / 4;     // their words
  constexpr int ROW = D + 4;          // LDS row of a head's output, 4 banks on
  __shared__ PageRun run;
  __shared__ __attribute__((aligned(16))) float acc_lds[kWaves][kTileHeads][ROW];
  __shared__ float m_lds[kWaves][kTileHeads], l_lds[kWaves][kTileHeads];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lo = lane & 15, hi = lane >> 4;
  const int dim = FULL ? D : a.head_dim;
  empty_seqs(a);
  Unit un = find_unit(a);
  if (un.seq < 0) return;
  const int64_t u1 = min(un.first + un.share, un.total);
  for (int64_t u = un.first; u < u1;) {
    advance(a, un, u);
    const Segment sg = segment_at<kTileHeads>(a, un, u, u1, wave % a.side);
    if (lane == 0 && wave < a.side) note_cut(a, un, sg, u, wave);
    const int64_t u_here = u;
    u += sg.st1 - sg.st0;
    // q of head lo, dims 32 ks + 8 hi .. (FP8: the dims of the K bytes that the
    // lane loads, 64 j + 16 hi .., two k steps)
    u32x4 qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = FP8 ? 64 * (ks / 2) + 16 * hi + 8 * (ks % 2) : 32 * ks + 8 * hi;
      qf[ks] = u32x4{0, 0, 0, 0};
      if (lo < sg.heads && (FULL || d < dim)) {
        const int64_t head = sg.head0 - (int64_t)sg.seq * a.num_q_heads + lo;
        qf[ks] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) +
                                                 sg.seq * a.q_seq + head * a.q_head + d);
      }
    }
    float m = -INFINITY, l = 0.0f;
    f32x4 acc[DP];
#pragma unroll
    for (int j = 0; j < DP; ++j) acc[j] = f32x4{0, 0, 0, 0};
    u32x4 kr[2 * NB][KL];
    uint32_t vr[8 * NB][VW];
    const int64_t head_off = sg.hkv * a.head_stride;
    // rows of K: tokens 16 i + lo; tokens that do not count read page 0
    auto load_k = [&](int64_t off) {
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) {
        const int64_t o = __shfl(off, 16 * i + lo);
        const uint8_t* p = a.k + (o < 0 ? head_off : o) + 16 * hi;
#pragma unroll
        for (int n = 0; n < KL; ++n) {
          if (!FULL) kr[i][n] = u32x4{0, 0, 0, 0};
          if (FULL || 16 * hi + 64 * n < dim * ES)
            kr[i][n] = *reinterpret_cast<const u32x4*>(p + 64 * n);
        }
      }
    };
    auto load_v = [&](int64_t off) {
#pragma unroll
      for (int r = 0; r < 8 * NB; ++r) {
        const int64_t o = __shfl(off, 16 * (r / 4) + 4 * hi + r % 4);
        const uint8_t* p = a.v + (o < 0 ? head_off : o) + DP * ES * lo;
        if (!FULL) {
#pragma unroll
          for (int w = 0; w < VW; ++w) vr[r][w] = 0;
          if (DP * lo >= dim) continue;
        }
        if constexpr (VW >= 4) {
#pragma unroll
          for (int n = 0; n < VW / 4; ++n) {
            const u32x4 x = ld_stream(reinterpret_cast<const u32x4*>(p) + n);
#pragma unroll
            for (int w = 0; w < 4; ++w) vr[r][4 * n + w] = x[w];
          }
        } else if constexpr (VW == 2) {
          const u32x2 x = ld_stream(reinterpret_cast<const u32x2*>(p));
          vr[r][0] = x[0];
          vr[r][1] = x[1];
        } else {
          vr[r][0] = ld_stream(reinterpret_cast<const uint32_t*>(p));
        }
      }
    };
    const int64_t hold = run_steps(a);
    for (int64_t r0 = sg.st0; r0 < sg.st1; r0 += hold) {
      const int64_t r1 = min(r0 + hold, sg.st1), j0 = page_of(a, r0 << a.step_shift);
      load_pages(a, sg, r0, r1, run);
      const int64_t t = (wave / a.side) * CH + (lane & (CH - 1));
      int64_t off = token_offset(a, sg, run, j0, (r0 << a.step_shift) + t);
      uint64_t seen = __ballot(off >= 0);
      if (seen) {
        load_k(off);
        load_v(off);
      }
      for (int64_t st = r0; st < r1; ++st) {
        // the next step's rows
        int64_t next = -1;
        if (st + 1 < r1) next = token_offset(a, sg, run, j0, ((st + 1) << a.step_shift) + t);
        const uint64_t seen_next = __ballot(next >= 0);
        f32x4 s[2 * NB];
        if (seen) {
#pragma unroll
          for (int i = 0; i < 2 * NB; ++i) {
            s[i] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              u32x4 kf;
              if constexpr (FP8) {
                const uint32_t w0 = kr[i][ks / 2][2 * (ks % 2)], w1 = kr[i][ks / 2][2 * (ks % 2) + 1];
                kf = u32x4{e4m3_pair<QDT, false>(w0), e4m3_pair<QDT, true>(w0),
                           e4m3_pair<QDT, false>(w1), e4m3_pair<QDT, true>(w1)};
              } else {
                kf = kr[i][ks];
              }
              s[i] = mfma16<QDT>(kf, qf[ks], s[i]);
            }
          }
        }
        if (seen_next) load_k(next);
        if (seen) {
          const bool full = seen == ~0ull;
          // whether this lane's token r of block b counts
          auto counts = [&](int b, int r) {
            return full || ((uint32_t)(seen >> (32 * b)) >> (4 * hi) >> (16 * (r / 4) + r % 4) & 1);
          };
          float x[NB][8], p[NB][8], top = -INFINITY;
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              x[b][r] = s[2 * b + r / 4][r % 4];
              top = max_nan(top, counts(b, r) ? x[b][r] * a.score_scale : -INFINITY);
            }
          top = max_nan(top, __shfl_xor(top, 16));
          top = max_nan(top, __shfl_xor(top, 32));
          const float mn = max_nan(m, top);
          const float w = weight_to(m, mn), base = exp_base(mn);
          m = mn;
          float sum = 0.0f;
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              p[b][r] = counts(b, r) ? __builtin_amdgcn_exp2f(
                                           __builtin_fmaf(x[b][r], a.score_scale, -base))
                                     : 0.0f;
              sum += p[b][r];
            }
          l = mn == -INFINITY ? 1.0f : l * w + sum;
          if (__any(w != 1.0f)) {
#pragma unroll
            for (int j = 0; j < DP; ++j) acc[j] *= w;
          }
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            u32x4 pb[kTerms];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              uint32_t t3[kTerms];
              weight_split(p[b][2 * n], p[b][2 * n + 1], t3);
#pragma unroll
              for (int k = 0; k < kTerms; ++k) pb[k][n] = t3[k];
            }
            if (!full) {  // V rows that do not count: zeros, not what page 0 holds
#pragma unroll
              for (int r = 0; r < 8; ++r)
                if (!counts(b, r)) {
#pragma unroll
                  for (int n = 0; n < VW; ++n) vr[8 * b + r][n] = 0;
                }
            }
#pragma unroll
            for (int j = 0; j < DP; j += 2) {  // dims j and j + 1 of each lane's piece
              uint32_t v2[8];
#pragma unroll
              for (int r = 0; r < 8; ++r) {
                if constexpr (FP8)
                  v2[r] = j % 4 ? e4m3_pair<AMF_DTYPE_BF16, true>(vr[8 * b + r][j / 4])
                                : e4m3_pair<AMF_DTYPE_BF16, false>(vr[8 * b + r][j / 4]);
                else
                  v2[r] = vr[8 * b + r][j / 2];
              }
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                u32x4 va, vl;
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                  va[n] = __builtin_amdgcn_perm(v2[2 * n + 1], v2[2 * n],
                                                e ? 0x07060302u : 0x05040100u);
                  if constexpr (V16) {
                    uint32_t h2, l2;
                    v_split(va[n], h2, l2);
                    va[n] = h2;
                    vl[n] = l2;
                  }
                }
#pragma unroll
                for (int k = 0; k < kTerms; ++k) {
                  acc[j + e] = mfma16<AMF_DTYPE_BF16>(va, pb[k], acc[j + e]);
                  if constexpr (V16) {
                    if (k < 2) acc[j + e] = mfma16<AMF_DTYPE_BF16>(vl, pb[k], acc[j + e]);
                  }
                }
              }
            }
          }
        }
        if (seen_next) load_v(next);
        seen = seen_next;
      }
    }
    // the four waves' parts
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    __syncthreads();  // the last pair's parts have been read
    if (lo < sg.heads) {
      if (hi == 0) {
        m_lds[wave][lo] = m;
        l_lds[wave][lo] = l;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float* o = &acc_lds[wave][lo][DP * (4 * hi + r)];
#pragma unroll
        for (int j = 0; j < DP; j += 4)
          *reinterpret_cast<f32x4*>(o + j) =
              f32x4{acc[j][r], acc[j + 1][r], acc[j + 2][r], acc[j + 3][r]};
      }
    }
    __syncthreads();
    for (int n = 0; n < a.side; ++n) {
      const Segment sn = segment_at<kTileHeads>(a, un, u_here, u1, n);
      for (int i = tid; i < sn.heads * (dim / 4); i += kThreads) {
        const int g = i / (dim / 4), d = 4 * (i - g * (dim / 4));
        float top = m_lds[n][g], sum = 0.0f;
        f32x4 x{0, 0, 0, 0};
        for (int w = n + a.side; w < kWaves; w += a.side) top = max_nan(top, m_lds[w][g]);
        for (int w = n; w < kWaves; w += a.side) {
          const float f = weight_to(m_lds[w][g], top);
          sum += l_lds[w][g] * f;
          x += *reinterpret_cast<const f32x4*>(&acc_lds[w][g][d]) * f;
        }
        if (sn.whole) {
          if (sum == 0.0f)
            x = f32x4{0, 0, 0, 0};
          else
            x *= row_factor(a.v_scale, top, sum);
          store4(a.out, a.out_dtype, (sn.head0 + g) * dim + d, x);
        } else {
          float* part = sn.part + g * (dim + kPartPad);
          *reinterpret_cast<f32x4*>(part + d) = x;
          if (d == 0) {
            part[dim] = top;
            part[dim + 1] = sum;
          }
        }
      }
    }
  }
}

// ---- merge ---------------------------------------------------------------------
//
// A workgroup per pair that may be cut and `heads` of its heads: threads take W
// dims of every n-th partial, several partials loaded ahead of their use, and are
// joined in LDS.
template <int W, int NT>
__global__ __launch_bounds__(NT) void paged_attn_merge_kernel(PagedArgs a, int heads) {
  constexpr int kAhead = 8;
  __shared__ float x_lds[NT][W], m_lds[NT], l_lds[NT];
  const Cut cut = a.cuts[blockIdx.x];
  const int tid = threadIdx.x, D = a.head_dim;
  if ((int)blockIdx.y * heads >= cut.heads) return;
  const int cols = (D + W - 1) / W, rows = NT / (cols * heads);
  const int r = tid / (cols * heads), g = (int)blockIdx.y * heads + tid % (cols * heads) / cols;
  const int col = tid % cols, row = g * (D + kPartPad);
  float m = -INFINITY, l = 0.0f, x[W];
#pragma unroll
  for (int e = 0; e < W; ++e) x[e] = 0.0f;
  if (r < rows && g < cut.heads) {
    const int n = cut.more + 1, pairs = pairs_of(a);
    for (int i0 = r; i0 < n; i0 += kAhead * rows) {
      float pm[kAhead], pl[kAhead], px[kAhead][W];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = i0 + k * rows;
        pm[k] = -INFINITY;
        pl[k] = 0.0f;
#pragma unroll
        for (int e = 0; e < W; ++e) px[k][e] = 0.0f;
        if (i < n) {
          const int64_t place = i == 0 ? cut.place : (cut.place & ~1) + 2 * (int64_t)i * pairs;
          const float* p = a.part + place * a.part_stride + row;
          pm[k] = p[D];
          pl[k] = p[D + 1];
          if constexpr (W == 4) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(p + 4 * col);
#pragma unroll
            for (int e = 0; e < 4; ++e) px[k][e] = v[e];
          } else {
            px[k][0] = p[col];
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const float top = max_nan(m, pm[k]);
        const float f = weight_to(m, top), pf = weight_to(pm[k], top);
        l = l * f + pl[k] * pf;
#pragma unroll
        for (int e = 0; e < W; ++e) x[e] = x[e] * f + px[k][e] * pf;
        m = top;
      }
    }
  }
  m_lds[tid] = m;
  l_lds[tid] = l;
#pragma unroll
  for (int e = 0; e < W; ++e) x_lds[tid][e] = x[e];
  __syncthreads();
  if (r > 0 || g >= cut.heads) return;
  for (int k = 1; k < rows; ++k) {
    const int o = tid + k * cols * heads;
    const float pm = m_lds[o], top = max_nan(m, pm);
    const float f = weight_to(m, top), pf = weight_to(pm, top);
    l = l * f + l_lds[o] * pf;
#pragma unroll
    for (int e = 0; e < W; ++e) x[e] = x[e] * f + x_lds[o][e] * pf;
    m = top;
  }
  const float scale = l == 0.0f ? 0.0f : row_factor(a.v_scale, m, l);
  const int64_t at = (int64_t)(cut.head0 + g) * D + W * col;
  if constexpr (W == 4)
    store4(a.out, a.out_dtype, at,
           l == 0.0f ? f32x4{0, 0, 0, 0}
                     : f32x4{x[0] * scale, x[1] * scale, x[2] * scale, x[3] * scale});
  else
    store_out(a, at, l == 0.0f ? 0.0f : x[0] * scale);
}

// ---- launch --------------------------------------------------------------------

// Workgroups that share a launch's steps: two a CU, all resident (32 sequences of
// 1K-32K tokens 337 us; 256: 343, 1024: 348; 8 x 126K FP8 tokens 339, 483, 360; a
// selection and 4096 listed tokens each of 8 sequences 80, 80, 86).
constexpr int64_t kGroups = 512;
// Short contexts take a workgroup a (sequence, pair) and no merge: at most so many
// steps and pairs.  8 KV heads of 128, bf16, split / whole, us: 1 x 128 tokens 12.5 / 7.0,
// 1 x 500 12.9 / 11.4, 64 x 500 33 / 26, 160 x 500 68 / 66; but 1 x 1000 13.4 / 17.2, 256
// x 128 30 / 37.  (Equal lengths; of mixed ones the longest would decide.)  FP8 and 64
// dims are alike (1 x 500 12.7 / 11.1, 12.3 / 9.2; 160 x 500 47 / 43, 20 / 15), fp32 by
// rows too (12 / 4 heads of 96, 1 x 128 12.8 / 11.8).  256 dims of 16 bits, whose step is
// twice the bytes at one workgroup a CU, are slower whole but for one short sequence (2
// KV heads, 1 x 128 15.7 / 11.7; 1 x 500 16 / 25, 160 x 128 23 / 25, 160 x 500 48 / 54):
// the rule does not look at that yet.
constexpr int64_t kWholeSteps = 4;
constexpr int64_t kWholePairs = 3 * kGroups;

// Floats of a partial, for either kernel.
int64_t part_floats(int32_t group, int32_t head_dim) {
  return (int64_t)std::min<int32_t>(group, kTileHeads) * (head_dim + kPartPad);
}

// Places for partials: every pair of a launch's shares, of which there is one at
// least.
int64_t part_places(int32_t num_kv_heads, int32_t group) {
  return std::max<int64_t>(kGroups * kWaves,
                           (int64_t)num_kv_heads * ((group + kGenHeads - 1) / kGenHeads));
}

// The tile of head_dim in the matrix kernel.
int matrix_dim(int32_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

// Lanes that share a row in the general kernel.
int general_lanes(int32_t head_dim) {
  return head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : 32;
}

template <int QDT, int KDT, int D>
void launch_matrix(const PagedArgs& a, dim3 grid, hipStream_t st) {
  if (a.head_dim == D)
    paged_attn_matrix_kernel<QDT, KDT, D, true><<<grid, kThreads, 0, st>>>(a);
  else
    paged_attn_matrix_kernel<QDT, KDT, D, false><<<grid, kThreads, 0, st>>>(a);
}

template <int QDT, int KDT, int LPR>
void launch_general(const PagedArgs& a, dim3 grid, bool rows, hipStream_t st) {
  if (rows)
    paged_attn_general_kernel<QDT, KDT, LPR, true><<<grid, kThreads, 0, st>>>(a);
  else
    paged_attn_general_kernel<QDT, KDT, LPR, false><<<grid, kThreads, 0, st>>>(a);
}

template <int QDT, int KDT>
void launch(const PagedArgs& a, int64_t groups, bool matrix, bool rows, hipStream_t st) {
  const dim3 grid((unsigned)groups);
  if constexpr (QDT != AMF_DTYPE_F32) {
    if (matrix) {
      switch (matrix_dim(a.head_dim)) {
        case 64: return launch_matrix<QDT, KDT, 64>(a, grid, st);
        case 128: return launch_matrix<QDT, KDT, 128>(a, grid, st);
        default: return launch_matrix<QDT, KDT, 256>(a, grid, st);
      }
    }
  }
  switch (general_lanes(a.head_dim)) {
    case 8: return launch_general<QDT, KDT, 8>(a, grid, rows, st);
    case 16: return launch_general<QDT, KDT, 16>(a, grid, rows, st);
    default: return launch_general<QDT, KDT, 32>(a, grid, rows, st);
  }
}

}  // namespace

extern "C" int64_t amf_paged_decode_workspace_bytes(int32_t num_q_heads, int32_t num_kv_heads,
                                                    int32_t head_dim) {
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 || head_dim <= 0 ||
      head_dim > kMaxDim)
    return 0;
  const int32_t group = num_q_heads / num_kv_heads;
  return part_places(num_kv_heads, group) *
         ((int64_t)sizeof(Cut) + 2 * part_floats(group, head_dim) * (int64_t)sizeof(float));
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
  // rows that 16-byte loads and stores reach; 8 elements at a time in the general
  // kernel
  const int64_t bits = (int64_t)((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) |
                       a.page_stride | a.token_stride | a.head_stride |
                       (q_seq_stride * qs) | (q_head_stride * qs);
  const bool matrix = qs == 2 && head_dim % 16 == 0 && aligned16(bits);
  const bool rows = head_dim % 8 == 0 && ((((uintptr_t)k | (uintptr_t)v) | a.page_stride |
                                           a.token_stride | a.head_stride) &
                                          (8 * es > 16 ? 15 : 8 * es - 1)) == 0;
  const int tile = matrix ? kTileHeads : kGenHeads;
  a.tiles = (a.group + tile - 1) / tile;
  a.out_dtype = out_dtype;
  a.score_scale = (float)((softmax_scale > 0.0f ? (double)softmax_scale : 1.0 / sqrt((double)head_dim)) *
                          (double)k_scale * 1.4426950408889634);
  a.v_scale = v_scale;
  // the most steps that a pair can have, as far as the host knows
  const int64_t tokens = pages ? (int64_t)max_pages * block_size
                               : std::min<int64_t>(max_context_len, (int64_t)table_pages * block_size);
  const int chunk = matrix ? matrix_chunk(matrix_dim(head_dim))
                           : 64 / general_lanes(head_dim) * kGenAhead;
  a.step_shift = __builtin_ctz(chunk * kWaves);
  const int64_t steps = std::max<int64_t>(1, (tokens + chunk * kWaves - 1) / (chunk * kWaves));
  const int64_t pairs = (int64_t)num_seqs * num_kv_heads * a.tiles;
  if (pairs > 0xFFFFFF || (int64_t)num_seqs * num_q_heads > 0x7FFFFFFF)
    return fail(AMF_ERR_UNSUPPORTED, "%s: %d sequences of %d heads", who, num_seqs, num_q_heads);
  a.whole = steps <= kWholeSteps && pairs <= kWholePairs;
  // pairs side by side on the waves of a workgroup: their rows lie side by side in
  // memory and are asked for at the same time.  32 sequences of 1K-32K tokens 365 us
  // with one pair a workgroup, 337 with four (8 x 126K FP8 389, 339); page lists differ
  // from head to head, and a whole sequence has too few workgroups.
  const int64_t heads = (int64_t)num_kv_heads * a.tiles;
  a.side = 1;
  if (matrix && !a.whole && !pages) a.side = heads % 4 == 0 ? 4 : heads % 2 == 0 ? 2 : 1;
  if (a.side > 1) a.step_shift -= a.side / 2;
  const int64_t teams = heads / a.side;
  const int64_t most_steps = num_seqs * ((tokens + (1 << a.step_shift) - 1) >> a.step_shift);
  // one workgroup a CU where two do not fit: 512 shares of 256 dims are taken in two
  // rounds (164 sequences of 4700 fp16 tokens 289 us, 272 with 256)
  const bool half = matrix && matrix_waves(matrix_dim(head_dim), es) == 1;
  const int64_t resident = half ? kGroups / 2 : kGroups;
  const int64_t shares =
      std::max<int64_t>(1, std::min(std::max<int64_t>(resident / teams, 1), most_steps));
  const int64_t groups = (a.whole ? num_seqs : shares) * teams;
  a.by_seq = num_seqs < shares;
  a.cuts = static_cast<Cut*>(workspace);
  a.part = reinterpret_cast<float*>(a.cuts + part_places(num_kv_heads, a.group));
  a.part_stride = part_floats(a.group, head_dim);
  a.err_flag = err_flag;
  hipStream_t st = as_stream(stream);
  if (kv_dtype == AMF_DTYPE_BF16)
    launch<AMF_DTYPE_BF16, AMF_DTYPE_BF16>(a, groups, matrix, rows, st);
  else if (kv_dtype == AMF_DTYPE_F16)
    launch<AMF_DTYPE_F16, AMF_DTYPE_F16>(a, groups, matrix, rows, st);
  else if (kv_dtype == AMF_DTYPE_F32)
    launch<AMF_DTYPE_F32, AMF_DTYPE_F32>(a, groups, matrix, rows, st);
  else if (q_dtype == AMF_DTYPE_BF16)
    launch<AMF_DTYPE_BF16, AMF_DTYPE_E4M3>(a, groups, matrix, rows, st);
  else
    launch<AMF_DTYPE_F16, AMF_DTYPE_E4M3>(a, groups, matrix, rows, st);
  if (int rc = check_launch(who)) return rc;
  if (a.whole) return ok();
  // partials of a pair, about: many take a workgroup a head, hundreds (one long
  // context) a larger one (131072 tokens of one KV head 44 -> 27 us a call)
  const int64_t parts = shares / num_seqs;
  const int32_t tile_heads = std::min<int32_t>(a.group, tile);
  const int cols = matrix ? head_dim / 4 : head_dim;
  const int per = std::min<int>(tile_heads, std::max(1, kThreads / cols / (parts >= 4 ? 8 : 2)));
  const dim3 grid((unsigned)(std::min<int64_t>(num_seqs, shares) * heads),
                  (unsigned)((tile_heads + per - 1) / per));
  if (!matrix)
    paged_attn_merge_kernel<1, kThreads><<<grid, kThreads, 0, st>>>(a, per);
  else if (parts >= 64)
    paged_attn_merge_kernel<4, 1024><<<grid, 1024, 0, st>>>(a, per);
  else
    paged_attn_merge_kernel<4, kThreads><<<grid, kThreads, 0, st>>>(a, per);
  return check_launch(who);
}

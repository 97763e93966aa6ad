// amf_paged_rows.hip - causal attention of several new rows per sequence (prompt
// chunks, drafted tokens, single rows among them) over a paged K/V cache (bf16,
// fp16, fp32, FP8 e4m3) or an INT4_ASYM_G32 pool, read in place.
//
//   out[r, h] = v_scale * sum_{t <= p} softmax_t(k_scale * scale * q[r, h] . k[t]) v[t]
//
// for row j of sequence s with n rows at position p = context - n + j.  FP8 codes
// enter as their values, INT4 ones as u * s + z rounded to q's type.
//
// Tiles.  The query heads of a KV head and kRows / group tokens are the up to
// kRows columns of a workgroup's 32x32x16 matrix products, 32 columns a wave.  K and
// V come through LDS, BT tokens at a time, so each element is loaded and
// dequantised once for all columns.  The scores are formed transposed, S^T = K Q^T: a
// lane holds one column (lane % 32) and 16 of 32 tokens, so the softmax statistics are
// per lane (one exchange with lane ^ 32 for the maximum) and the weights are in the
// B layout of O^T = V^T P^T as they are.  V^T comes out of LDS by the transposing read.
//
// Shares.  Tile j of a sequence reads its first e_j tokens; the tiles of all
// (KV head, sequence, tile) one after the other, each as long as it reads plus a
// constant, are cut into equal shares, one a workgroup, so a mix of long chunks and
// single rows fills the chip.  e_j grows linearly in j, so a workgroup finds its
// place from sums over the sequences alone.  A tile inside one share is finished
// there; one that several share leaves partials (acc, m, l), joined by a second
// launch.
//
// Precision.  Products of Q and K are exact and summed in fp32; maximum, sum and
// accumulators are fp32.  The weights enter the second product in one term: bf16 (8
// bits) beside a bf16 V, which adds to the result what its own rounding to bf16 does
// (their sum is within 2^-7 of the weighted |v|), fp16 (11 bits) beside an fp16 or an
// FP8 one, whose values fp16 holds exactly; three bf16 terms would cost twice the
// matrix time of the whole for bits that the result's type drops.
#include <algorithm>

#include "amf_attn.h"
#include "amf_int4_asym.h"
#include "amf_paged.h"

// Held to a tolerance, as the other attention kernels: multiplies and adds may
// fuse.
#pragma clang fp contract(fast)

namespace {

using namespace amf;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef s16x4 __attribute__((address_space(3))) lds_s16x4;

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows = 32 * kWaves;  // columns of a workgroup
constexpr int kMaxDim = 256;
constexpr int kMaxShares = 512;     // two workgroups a CU
constexpr int kMinShare = 256;      // tokens
constexpr int kTileCost = 64;       // tokens' worth of a tile's beginning and end, >= BT
constexpr int kMaxContext = 1 << 30;
constexpr int kInt4 = 16;           // beside the AMF_DTYPE_* of a cache

// A tile that does not end in the share where it begins.
struct Cut {
  int32_t more;   // shares after it that hold pieces, 0: there is none
  int32_t share;
  int32_t row0;   // the tile's first row
  int32_t cols;   // its columns
  int32_t head;   // KV head
  int32_t pad[3];
};

struct RowsArgs {
  const uint8_t* q;
  int64_t q_row, q_head;  // bytes
  uint16_t* out;
  int64_t n_rows;
  const int32_t* query_start;
  const uint8_t* k;  // or codes
  const uint8_t* v;
  const uint32_t* kp;  // INT4 params
  const uint32_t* vp;
  int64_t page_stride, token_stride, head_stride;  // bytes
  int64_t pool_pages;
  const int32_t* block_tables;
  int64_t bt_stride;
  int32_t table_pages;
  const int32_t* context_lens;
  int32_t num_seqs, num_q_heads, num_kv_heads, head_dim, block_size;
  int32_t block_shift;  // log2(block_size), or -1
  int32_t group;        // query heads of a KV head
  int32_t tile_rows;    // query rows of a tile
  bool by16;            // 16 tokens at a multiple of 16 lie in one page
  int32_t shares;       // of the grid
  float score_scale;    // softmax scale * k_scale * log2(e)
  float v_scale;
  Cut* cuts;            // [workgroup]
  float* part;          // [share][2][kRows][head_dim + kPartPad]
  int32_t* err_flag;
};

// ---- sequences and shares ------------------------------------------------------

struct Seq {
  int row0, rows;  // its rows of the step
  int pos0;        // position of the first
  int lim;         // tokens that the block table holds of its context
  int base;        // pos0, or more where the table is too short, at least 0
  int tiles;
};

__device__ __forceinline__ Seq get_seq(const RowsArgs& a, int s, int* flags) {
  const int lo = a.query_start[s], hi = a.query_start[s + 1];
  const int ctx = max(a.context_lens[s], 0);
  const int cap = a.table_pages * a.block_size;  // at most kMaxContext
  Seq r;
  const bool ok = lo >= 0 && lo <= hi && hi <= a.n_rows;
  r.row0 = ok ? lo : 0;
  r.rows = ok ? hi - lo : 0;
  r.pos0 = ctx - r.rows;
  r.lim = min(ctx, cap);
  r.base = ctx > cap ? cap : max(r.pos0, 0);
  r.tiles = (r.rows + a.tile_rows - 1) / a.tile_rows;
  if (!ok || (ctx > cap && r.rows > 0)) *flags |= AMF_ERRFLAG_CONTEXT;
  return r;
}

// Tile j is base + min((j + 1) tile_rows, rows) + kTileCost long.
__device__ __forceinline__ int64_t tiles_before(const RowsArgs& a, const Seq& s, int64_t j) {
  return j * ((int64_t)s.base + kTileCost) + a.tile_rows * (j * (j + 1) / 2);
}
__device__ __forceinline__ int64_t seq_length(const RowsArgs& a, const Seq& s) {
  return s.tiles ? tiles_before(a, s, s.tiles - 1) + s.base + kTileCost + s.rows : 0;
}

struct Share {
  int64_t index, length;  // of every share
  int64_t first, end;     // of this one
  int64_t seq_start;      // where the sequence starts that `first` lies in
  int32_t head, seq;      // seq -1: nothing to do
};

// The same in every thread; workgroup 0 flags.
__device__ __forceinline__ Share find_share(const RowsArgs& a) {
  __shared__ int64_t tmp[kWaves];
  __shared__ int64_t found_start;
  __shared__ int found_seq;
  const int tid = threadIdx.x;
  int64_t total = 0, len = 0, before = 0;
  int flags = 0;
  for (int s0 = 0; s0 < a.num_seqs; s0 += kThreads) {
    const int s = s0 + tid;
    len = s < a.num_seqs ? seq_length(a, get_seq(a, s, &flags)) : 0;
    int64_t sum;
    before = total + block_exclusive<kThreads>(len, tmp, &sum);
    total += sum;
  }
  if (flags && blockIdx.x == 0 && a.err_flag) atomicOr(a.err_flag, flags);
  Share r{};
  r.seq = -1;
  const int64_t all = total * a.num_kv_heads;
  if (all == 0) return r;
  r.length = max((all + a.shares - 1) / a.shares, (int64_t)kMinShare);
  const int64_t n = (all + r.length - 1) / r.length;
  // consecutive shares on one XCD: they read the same tokens
  const int64_t per = (n + kXcds - 1) / kXcds, slot = blockIdx.x / kXcds;
  r.index = (blockIdx.x % kXcds) * per + slot;
  if (slot >= per || r.index >= n) return r;
  r.first = r.index * r.length;
  r.end = min(all, r.first + r.length);
  r.head = (int32_t)(r.first / total);
  const int64_t at = r.first - r.head * total;
  if (a.num_seqs <= kThreads) {
    if (before <= at && at < before + len) {
      found_seq = tid;
      found_start = before;
    }
  } else {
    int64_t sum = 0;
    for (int s0 = 0; s0 < a.num_seqs && sum <= at; s0 += kThreads) {
      const int s = s0 + tid;
      len = s < a.num_seqs ? seq_length(a, get_seq(a, s, &flags)) : 0;
      int64_t part;
      before = sum + block_exclusive<kThreads>(len, tmp, &part);
      sum += part;
      if (before <= at && at < before + len) {
        found_seq = s;
        found_start = before;
      }
    }
  }
  __syncthreads();
  r.seq = found_seq;
  r.seq_start = r.head * total + found_start;
  return r;
}

// ---- K and V of a tile into LDS --------------------------------------------------

constexpr int tile_tokens(int D) { return D == 256 ? 32 : 64; }
// LDS row strides in bytes.  K rows are read as 16-byte vectors of 32 consecutive
// rows: 16 more than the row moves each by 4 banks.  V rows are read by the
// transposing read, 4 rows of 64 bytes per half wave: 64 more than the row puts them
// 16 banks apart.
constexpr int k_stride(int D) { return 2 * D + 16; }
constexpr int v_stride(int D) { return 2 * D + 64; }

// Two fp32 values as a pair of type T in one conversion, round to nearest even.
template <int T>
__device__ __forceinline__ uint32_t pair16(float a, float b) {
  if constexpr (T == AMF_DTYPE_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2_t));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2_t));
}

// Read by the scalar unit: nothing that a launch writes.
typedef const __attribute__((address_space(4))) int32_t scalar_i32;
__device__ __forceinline__ int32_t scalar_load(const int32_t* p, int i) {
  return ((scalar_i32*)(uintptr_t)p)[i];
}

// Whether a pair of 16-bit values holds one that is not finite.
template <int T>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  constexpr uint32_t m = T == AMF_DTYPE_BF16 ? 0x7F80u : 0x7C00u;
  return (w & m) == m || (w >> 16 & m) == m;
}

// What a thread moves of a tile of BT tokens of one (page table, KV head): raw values
// in registers between fetch() and stage().
template <int QT, int KV, int D>
struct Mover {
  static constexpr int BT = tile_tokens(D), KS = k_stride(D), VS = v_stride(D);
  // types of K and V in LDS; FP8 values are exact in both
  static constexpr int VT = KV == AMF_DTYPE_E4M3 ? AMF_DTYPE_F16 : QT;
  static constexpr int EB = KV == AMF_DTYPE_E4M3 ? 1 : 2;    // bytes of a cache element
  static constexpr int CPR = D * EB / 16;                    // 16-byte chunks of a row
  static constexpr int CH = BT * CPR / kThreads;             // chunks of a thread
  static constexpr int STEP = kThreads / CPR;                // rows between them
  static_assert(CH >= 1 && kThreads % CPR == 0, "a tile is whole chunks per thread");

  const RowsArgs& a;
  const int32_t* table;
  int head;
  int end;  // tokens behind it are not read
  int32_t ids[CH];
  u32x4 kr[CH], vr[CH];

  __device__ __forceinline__ Mover(const RowsArgs& args) : a(args) {}
  __device__ __forceinline__ int row(int i) const { return threadIdx.x / CPR + i * STEP; }
  // the wave's first row: its rows lie in one aligned group of 16
  static_assert(64 / CPR <= 16, "a wave's rows lie in a page of 16 tokens or more");
  __device__ __forceinline__ int wave_row(int i) const {
    return __builtin_amdgcn_readfirstlane(row(i));
  }
  __device__ __forceinline__ bool good(int32_t id) const { return id >= 0 && id < a.pool_pages; }
  __device__ __forceinline__ int page_of(int t) const {
    return a.block_shift >= 0 ? t >> a.block_shift : (int)((uint32_t)t / (uint32_t)a.block_size);
  }
  __device__ __forceinline__ void start(int seq, int h, int e) {
    table = a.block_tables + seq * a.bt_stride;
    head = h;
    end = e;
  }
  // Page ids of a tile: of the wave's rows, or of each lane's.
  __device__ __forceinline__ void pages(int t0) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      ids[i] = -1;
      if (a.by16) {
        const int t = t0 + wave_row(i);
        if (t < end) ids[i] = scalar_load(table, page_of(t));
      } else if (t0 + row(i) < end) {
        ids[i] = table[page_of(t0 + row(i))];
      }
    }
  }
  __device__ __forceinline__ void fetch(int t0) {
    if (a.by16) {
      bool all = t0 + BT <= end;
#pragma unroll
      for (int i = 0; i < CH; ++i) all = all && good(__builtin_amdgcn_readfirstlane(ids[i]));
      if (all) {
        // a uniform base and one offset a lane
        const uint32_t lane = (threadIdx.x % 64) / CPR * (uint32_t)a.token_stride +
                              threadIdx.x % CPR * 16;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int t = t0 + wave_row(i);
          const int64_t off = __builtin_amdgcn_readfirstlane(ids[i]) * a.page_stride +
                              (t - page_of(t) * a.block_size) * a.token_stride +
                              head * a.head_stride;
          kr[i] = *reinterpret_cast<const u32x4*>(a.k + off + lane);
          vr[i] = *reinterpret_cast<const u32x4*>(a.v + off + lane);
        }
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int t = t0 + row(i);
      kr[i] = vr[i] = u32x4{0, 0, 0, 0};
      if (t < end && good(ids[i])) {
        const int64_t off = ids[i] * a.page_stride +
                            (t - page_of(t) * a.block_size) * a.token_stride +
                            head * a.head_stride + threadIdx.x % CPR * 16;
        kr[i] = *reinterpret_cast<const u32x4*>(a.k + off);
        vr[i] = *reinterpret_cast<const u32x4*>(a.v + off);
      }
    }
  }
  // bad: bits of the tile's tokens whose page is none
  __device__ __forceinline__ void note_pages(int t0, uint32_t* bad) const {
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (!good(ids[i]) && t0 + row(i) < end) atomicOr(bad + row(i) / 32, 1u << (row(i) % 32));
  }
  // wild: bits of the tokens with a V element that is not finite, which is stored as 0
  template <bool CHECK>
  __device__ __forceinline__ void stage(uint8_t* k_lds, uint8_t* v_lds, uint32_t* wild) const {
    const int c = threadIdx.x % CPR;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      u32x4 k[2 / EB], v[2 / EB];
      if constexpr (EB == 2) {
        k[0] = kr[i];
        v[0] = vr[i];
      } else {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          k[w / 2][2 * (w % 2)] = fp8_pair<QT, false>(kr[i][w]);
          k[w / 2][2 * (w % 2) + 1] = fp8_pair<QT, true>(kr[i][w]);
          v[w / 2][2 * (w % 2)] = fp8_pair<VT, false>(vr[i][w]);
          v[w / 2][2 * (w % 2) + 1] = fp8_pair<VT, true>(vr[i][w]);
        }
      }
      if constexpr (CHECK) clean(v, 2 / EB, row(i), wild);
#pragma unroll
      for (int n = 0; n < 2 / EB; ++n) {
        *reinterpret_cast<u32x4*>(k_lds + row(i) * KS + (2 / EB) * 16 * c + 16 * n) = k[n];
        *reinterpret_cast<u32x4*>(v_lds + row(i) * VS + (2 / EB) * 16 * c + 16 * n) = v[n];
      }
    }
  }
  template <int T, bool HIGH>
  static __device__ __forceinline__ uint32_t fp8_pair(uint32_t w) {
    if constexpr (T == AMF_DTYPE_BF16)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HIGH));
  }
  static __device__ __forceinline__ void clean(u32x4* v, int n, int r, uint32_t* wild) {
    bool found = false;
    for (int m = 0; m < n; ++m)
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (not_finite<VT>(v[m][w])) {
          found = true;
          if (not_finite<VT>(v[m][w] & 0xFFFFu)) v[m][w] &= 0xFFFF0000u;
          if (not_finite<VT>(v[m][w] & 0xFFFF0000u)) v[m][w] &= 0xFFFFu;
        }
    if (found) atomicOr(wild + r / 32, 1u << (r % 32));
  }
  // Element d of token t's V row, from memory (pages are good where this is asked).
  __device__ __forceinline__ float v_elem(int t, int d) const {
    const int64_t off = table[t / a.block_size] * a.page_stride +
                        t % a.block_size * a.token_stride + head * a.head_stride;
    return kv_elem<KV>(a.v + off + d * EB);
  }
};

// INT4 pages: K rows of 32 dims (16 bytes, one param) a thread, V in chunks of 4 dims
// by 8 tokens (16 bytes, 8 params).  At head_dim 64 half the threads move K, half V.
template <int QT, int D>
struct Mover<QT, kInt4, D> {
  static constexpr int BT = tile_tokens(D), KS = k_stride(D), VS = v_stride(D);
  static constexpr int VT = QT, G = D / 32, N = BT * G;  // items of K, and of V
  static constexpr bool HALF = N * 2 == kThreads;
  static_assert(HALF || N == kThreads, "an item per thread");

  const RowsArgs& a;
  const int32_t* table;
  int end;
  int32_t head;
  int32_t k_id, v_id;
  u32x4 kr, vr, vs[2];
  uint32_t ks;

  __device__ __forceinline__ Mover(const RowsArgs& args) : a(args) {}
  __device__ __forceinline__ bool has_k() const { return !HALF || threadIdx.x < N; }
  __device__ __forceinline__ bool has_v() const { return !HALF || threadIdx.x >= N; }
  __device__ __forceinline__ int item() const { return threadIdx.x % N; }
  __device__ __forceinline__ int k_row() const { return item() / G; }
  __device__ __forceinline__ int v_page() const { return item() / (D / 2); }
  __device__ __forceinline__ void start(int seq, int h, int e) {
    table = a.block_tables + seq * a.bt_stride;
    head = h;
    end = e;
  }
  __device__ __forceinline__ void pages(int64_t t0) {
    k_id = v_id = -1;
    if (t0 + k_row() < end) k_id = table[(t0 + k_row()) / 16];
    if (t0 + 16 * v_page() < end) v_id = table[t0 / 16 + v_page()];
  }
  __device__ __forceinline__ bool good(int32_t id) const { return id >= 0 && id < a.pool_pages; }
  __device__ __forceinline__ void fetch(int t0) {
    kr = vr = vs[0] = vs[1] = u32x4{0, 0, 0, 0};
    ks = 0;
    const int i = item();
    if (has_k() && good(k_id)) {
      // K items of a (page, head) block follow each other
      const int64_t block = (int64_t)k_id * a.num_kv_heads + head;
      const uint32_t at = i % (16 * G);
      kr = *reinterpret_cast<const u32x4*>(a.k + block * 8 * D + 16 * at);
      ks = a.kp[block * 16 * G + at];
    }
    if (has_v() && good(v_id)) {
      const int64_t block = (int64_t)v_id * a.num_kv_heads + head;
      const uint32_t x = i % (D / 2);
      vr = *reinterpret_cast<const u32x4*>(a.v + block * 8 * D + 16 * x);
      const u32x4* p = reinterpret_cast<const u32x4*>(a.vp + block * 16 * G);
      const uint32_t q = x / 16 * 4 + x / 2 % 2 * 2;
      vs[0] = p[q];
      vs[1] = p[q + 1];
    }
  }
  __device__ __forceinline__ void note_pages(int t0, uint32_t* bad) const {
    if (!good(k_id) && has_k() && t0 + k_row() < end)
      atomicOr(bad + k_row() / 32, 1u << (k_row() % 32));
  }
  // The 8 nibbles of w as bytes' fp32 values, in order.
  static __device__ __forceinline__ void nibbles(uint32_t w, float* x) {
    uint32_t ev = w & 0x0F0F0F0Fu, od = (w >> 4) & 0x0F0F0F0Fu;
    asm("" : "+v"(ev));
    asm("" : "+v"(od));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = (float)((ev >> (8 * i)) & 0xFFu);
      x[2 * i + 1] = (float)((od >> (8 * i)) & 0xFFu);
    }
  }
  template <bool CHECK>
  __device__ __forceinline__ void stage(uint8_t* k_lds, uint8_t* v_lds, uint32_t* wild) const {
    const int i = item();
    // u * s is exact (4 bits by 11), so the fma rounds as the codec's multiply and add
    if (has_k()) {
      const float s = param_scale(ks), z = param_zero(ks);
      uint8_t* o = k_lds + k_row() * KS + 64 * (i % G);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float x[8];
        nibbles(kr[w], x);
        u32x4 y;
#pragma unroll
        for (int n = 0; n < 4; ++n)
          y[n] = pair16<QT>(__builtin_fmaf(x[2 * n], s, z), __builtin_fmaf(x[2 * n + 1], s, z));
        *reinterpret_cast<u32x4*>(o + 16 * w) = y;
      }
    }
    if (has_v()) {
      const int x0 = i % (D / 2);
      const int r0 = 16 * v_page() + x0 / 2 % 2 * 8;
      uint8_t* o = v_lds + r0 * VS + (x0 / 4 * 8 + x0 % 2 * 4) * 2;
      float x[4][8];
#pragma unroll
      for (int d = 0; d < 4; ++d) nibbles(vr[d], x[d]);
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const uint32_t p = vs[t / 4][t % 4];
        const float s = param_scale(p), z = param_zero(p);
        u32x2 y = {pair16<QT>(__builtin_fmaf(x[0][t], s, z), __builtin_fmaf(x[1][t], s, z)),
                   pair16<QT>(__builtin_fmaf(x[2][t], s, z), __builtin_fmaf(x[3][t], s, z))};
        if constexpr (CHECK) {
          if (not_finite<VT>(y[0]) || not_finite<VT>(y[1])) {
            atomicOr(wild + (r0 + t) / 32, 1u << ((r0 + t) % 32));
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              if (not_finite<VT>(y[n] & 0xFFFFu)) y[n] &= 0xFFFF0000u;
              if (not_finite<VT>(y[n] & 0xFFFF0000u)) y[n] &= 0xFFFFu;
            }
          }
        }
        *reinterpret_cast<u32x2*>(o + t * VS) = y;
      }
    }
  }
  __device__ __forceinline__ float v_elem(int t, int d) const {
    const int64_t block = (int64_t)table[t / 16] * a.num_kv_heads + head;
    const int at = t % 16;
    const uint8_t c = a.v[block * 8 * D + 64 * (d / 8) + 32 * (at / 8) + 4 * (d % 8) + at % 8 / 2];
    const uint32_t p = a.vp[(block * G + d / 32) * 16 + at];
    return round_to<QT>(
        __builtin_fmaf((float)(at % 2 ? c >> 4 : c & 15), param_scale(p), param_zero(p)));
  }
};

// ---- the matrix kernel -------------------------------------------------------------

template <int T>
__device__ __forceinline__ f32x16 mfma32(const u32x4& x, const u32x4& y, const f32x16& c) {
  if constexpr (T == AMF_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, x),
                                                   __builtin_bit_cast(bf16x8_t, y), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, x),
                                                  __builtin_bit_cast(f16x8_t, y), c, 0, 0, 0);
}

// The running maximum is raised, and sum and accumulators scaled, only when a score
// exceeds it by 2^kSlack; weights run to 2^kSlack then, which fp32 sums hold as well.
// Weights in fp16 run to 2^(7 + kSlack) instead, so that those down to 2^-21 of the
// largest keep their 11 bits.
constexpr float kSlack = 8.0f;
template <int T>
constexpr float weight_shift() {
  return T == AMF_DTYPE_F16 ? 7.0f : 0.0f;
}

template <int QT, int KV, int D>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void rows_kernel(RowsArgs a) {
  using Move = Mover<QT, KV, D>;
  constexpr int BT = Move::BT, KS = Move::KS, VS = Move::VS, VT = Move::VT;
  __shared__ __attribute__((aligned(16))) uint8_t k_lds[BT * KS];
  __shared__ __attribute__((aligned(16))) uint8_t v_lds[BT * VS];
  __shared__ uint32_t marks[2][4];  // of even and odd tiles: bad pages (2 words), wild V (2)
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lc = lane & 31, h = lane >> 5;

  Cut cut{};
  const Share sh = find_share(a);
  if (sh.seq < 0) {
    if (tid == 0) a.cuts[blockIdx.x] = cut;
    return;
  }
  if (tid < 8) marks[tid >> 2][tid & 3] = 0;
  int flags = 0;
  Move mv(a);
  int head = sh.head, seq = sh.seq;
  Seq sq = get_seq(a, seq, &flags);
  int j = 0;  // the tile that the share begins in
  {
    const int64_t at = sh.first - sh.seq_start;
    int hi = sq.tiles;
    while (hi - j > 1) {
      const int mid = (j + hi) >> 1;
      if (tiles_before(a, sq, mid) <= at) j = mid; else hi = mid;
    }
  }
  int64_t start = sh.seq_start + tiles_before(a, sq, j);
  const int G = a.group;
  const float c2 = a.score_scale;
  bool bad_seen = false;
  int par = 0;  // of the tiles, over all pieces

  // addresses of this lane's LDS reads
  const uint8_t* k_rd = k_lds + lc * KS + 16 * h;
  const int l16 = lane & 15;
  const uint8_t* v_rd = v_lds + (4 * h + (l16 >> 2)) * VS + 32 * ((lane >> 4) & 1) + 8 * (l16 & 3);
  // A operand of V^T: dims 32 d .. + 31, 16 tokens in the order of the scores
  auto read_v = [](const uint8_t* vp) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vp));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vp + 8 * VS));
    const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
    return u32x4{l2[0], l2[1], h2[0], h2[1]};
  };

  while (start < sh.end) {
    const int row_lo = j * a.tile_rows;
    const int rows = min(a.tile_rows, sq.rows - row_lo);
    const int pos0 = sq.pos0 + row_lo;  // position of the tile's first row
    const int length = sq.base + row_lo + rows + kTileCost;
    const int e = max(min(sq.lim, pos0 + rows), 0);
    // the share's part of [0, length)
    const bool begins = sh.first <= start;
    const int lo = begins ? 0 : (int)(sh.first - start);
    const int hi = (int)min(sh.end - start, (int64_t)length);
    const int t_lo = min(e, lo / BT * BT);
    const int t_hi = hi == length ? e : min(e, hi / BT * BT);
    if (begins || t_lo < e) {
      const int cols = rows * G;
      const int col = wave * 32 + lc;
      const int qi = min(col, cols - 1) / G;
      const int qh = head * G + min(col, cols - 1) - qi * G;
      const int qrow = sq.row0 + row_lo + qi;
      const bool wave_on = wave * 32 < cols;
      const int wave_first = wave * 32 / G;                         // rows of the wave
      const int wave_last = (min(wave * 32 + 32, cols) - 1) / G;
      u32x4 qb[D / 16];  // B operand: dims 16 ks + 8 h .. + 7
      {
        const uint8_t* qp = a.q + qrow * a.q_row + qh * a.q_head + 16 * h;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          qb[ks] = *reinterpret_cast<const u32x4*>(qp + 32 * ks);
      }
      // the row's last token
      const int last = min(pos0 + qi, t_hi - 1);
      float m_run = -INFINITY, l_run = 0.0f;  // l_run: this lane's tokens
      bool seen = false;                      // a token that the row attends to
      f32x16 acc[D / 32];
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;

      mv.start(seq, head, t_hi);
      mv.pages(t_lo);
      mv.fetch(t_lo);
      for (int t0 = t_lo; t0 < t_hi; t0 += BT, par ^= 1) {
        __syncthreads();  // the previous tile has been read
        mv.note_pages(t0, &marks[par][0]);
        // tokens that some rows see and others do not: V has to be finite there, as 0 * inf
        // is not 0
        const bool diagonal = t0 + BT > pos0 + 1;
        if (diagonal)
          mv.template stage<true>(k_lds, v_lds, &marks[par][2]);
        else
          mv.template stage<false>(k_lds, v_lds, nullptr);
        if (t0 + BT < t_hi) {
          mv.pages(t0 + BT);
          mv.fetch(t0 + BT);
        }
        __syncthreads();
        auto mark = [&](int i) {
          return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(marks[par][i]);
        };
        const uint64_t bad = mark(1) << 32 | mark(0), wild = mark(3) << 32 | mark(2);
        if (tid < 4) marks[par ^ 1][tid] = 0;
        bad_seen |= bad != 0;
        if (!wave_on || t0 > pos0 + wave_last) continue;  // nothing for this wave

        f32x16 s[BT / 32];
#pragma unroll
        for (int tb = 0; tb < BT / 32; ++tb) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[tb][i] = 0.0f;
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
            s[tb] = mfma32<QT>(*reinterpret_cast<const u32x4*>(k_rd + 32 * tb * KS + 32 * ks),
                               qb[ks], s[tb]);
        }
        // token of score element i of block tb: t0 + 32 tb + 8 (i / 4) + 4 h + i % 4
        if (t0 + BT > t_hi || t0 + BT - 1 > pos0 + wave_first || bad) {
          const int left = last - t0 - 4 * h;
#pragma unroll
          for (int tb = 0; tb < BT / 32; ++tb) {
            uint32_t gone = (uint32_t)(bad >> (32 * tb)) >> (4 * h);
            asm volatile("" : "+v"(gone));  // no masks kept over the loop
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int t = 32 * tb + 8 * (i >> 2) + (i & 3);
              const bool hide = t > left || (gone >> (t % 32) & 1);
              if (hide) s[tb][i] = -INFINITY;
              seen |= !hide;
            }
          }
        } else {
          seen = true;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int tb = 0; tb < BT / 32; ++tb)
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[tb][i]);
        mx = fmaxf(mx, __shfl_xor(mx, 32)) * c2 - weight_shift<VT>();
        // a row with every score so far -inf keeps l = 0 and acc = 0
        if (__any(mx > m_run + kSlack)) {
          const float m_new = fmaxf(m_run, mx);
          const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.0f : m_new));
          l_run *= alpha;
#pragma unroll
          for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[d][i] *= alpha;
          m_run = m_new;
        }
        const float m_use = m_run == -INFINITY ? 0.0f : m_run;
        if (wild) {
          // elements that are not finite, for the rows that see their token
          for (uint64_t w = wild; w; w &= w - 1) {
            const int t = __ffsll((unsigned long long)w) - 1;
            const int e0 = t / 32 * 16 + t % 32 / 8 * 4 + t % 4;  // its element, in half t / 4 % 2
            float x = 0.0f;
#pragma unroll
            for (int i = 0; i < BT / 2; ++i) x = i == e0 ? s[i / 16][i % 16] : x;
            const float p = __builtin_amdgcn_exp2f(__shfl(x, lc + t / 4 % 2 * 32) * c2 - m_use);
            if (t0 + t > last) continue;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
              for (int n = 0; n < 16; ++n) {
                const float v = mv.v_elem(t0 + t, 32 * d + 8 * (n >> 2) + 4 * h + (n & 3));
                if (!(fabsf(v) < INFINITY)) acc[d][n] += p * v;
              }
          }
        }
#pragma unroll
        for (int st = 0; st < BT / 16; ++st) {
          u32x4 pb;  // weights of 16 tokens, 8 per lane
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float p0 =
                __builtin_amdgcn_exp2f(s[st >> 1][8 * (st & 1) + 2 * n] * c2 - m_use);
            const float p1 =
                __builtin_amdgcn_exp2f(s[st >> 1][8 * (st & 1) + 2 * n + 1] * c2 - m_use);
            l_run += p0;
            l_run += p1;
            pb[n] = pair16<VT>(p0, p1);
          }
#pragma unroll
          for (int d = 0; d < D / 32; ++d)
            acc[d] = mfma32<VT>(read_v(v_rd + 16 * st * VS + 64 * d), pb, acc[d]);
        }
      }

      float l = l_run + __shfl_xor(l_run, 32);
      seen |= __shfl_xor((int)seen, 32) != 0;
      const bool whole = begins && t_hi == e;
      if (!whole && begins) {
        const int64_t reach = start + (e + BT - 1) / BT * BT - 1;
        cut.more = (int32_t)(reach / sh.length - sh.index);
        cut.share = (int32_t)sh.index;
        cut.row0 = sq.row0 + row_lo;
        cut.cols = cols;
        cut.head = head;
      }
      if (col < cols) {
        if (whole) {
          // no token: zeros; every score -inf: 0 / 0 = NaN, as softmax gives
          const float f = seen ? a.v_scale / l : 0.0f;
          const int64_t o = ((int64_t)qrow * a.num_q_heads + qh) * D;
#pragma unroll
          for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              f32x4 x = {acc[d][4 * n], acc[d][4 * n + 1], acc[d][4 * n + 2], acc[d][4 * n + 3]};
              store4(a.out, QT, o + 32 * d + 8 * n + 4 * h, x * f);
            }
        } else {
          float* p = a.part + ((sh.index * 2 + begins) * kRows + col) * (D + kPartPad);
#pragma unroll
          for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int n = 0; n < 4; ++n)
              *reinterpret_cast<f32x4*>(p + 32 * d + 8 * n + 4 * h) =
                  f32x4{acc[d][4 * n], acc[d][4 * n + 1], acc[d][4 * n + 2], acc[d][4 * n + 3]};
          if (h == 0) {
            p[D] = m_run;
            p[D + 1] = seen && l == 0.0f ? -1.0f : l;  // -1: tokens, all of them -inf
          }
        }
      }
    }
    start += length;
    if (++j == sq.tiles) {
      j = 0;
      do {
        if (++seq == a.num_seqs) {
          seq = 0;
          ++head;
        }
        if (head == a.num_kv_heads) break;
        sq = get_seq(a, seq, &flags);
      } while (sq.tiles == 0);
      if (head == a.num_kv_heads) break;
    }
  }
  if (tid == 0) a.cuts[blockIdx.x] = cut;
  if (bad_seen && tid == 0 && a.err_flag) atomicOr(a.err_flag, AMF_ERRFLAG_BLOCK_RANGE);
}

// out = v_scale sum_k f_k acc_k / sum_k f_k l_k, f_k = 2^(m_k - M), over the pieces of a
// cut tile; D / 4 lanes a column, kMergeParts workgroups a tile.
constexpr int kMergeParts = 4;

template <int QT, int D>
__global__ __launch_bounds__(kThreads) void rows_merge_kernel(RowsArgs a) {
  constexpr int Q = D / 4, RP = kThreads / Q;
  __shared__ float f_lds[RP][kMaxShares + 1];
  const Cut cut = a.cuts[blockIdx.x];
  if (cut.more == 0) return;
  const int quad = threadIdx.x % Q, r = threadIdx.x / Q, n = cut.more + 1;
  constexpr int64_t PS = D + kPartPad;
  for (int c0 = blockIdx.y * RP; c0 < cut.cols; c0 += kMergeParts * RP) {
    const int col = min(c0 + r, cut.cols - 1);
    auto piece = [&](int k) {
      const int64_t slot = k == 0 ? (int64_t)cut.share * 2 + 1 : ((int64_t)cut.share + k) * 2;
      return a.part + (slot * kRows + col) * PS;
    };
    float M = -INFINITY;
    for (int k = quad; k < n; k += Q) M = fmaxf(M, piece(k)[D]);
#pragma unroll
    for (int o = 1; o < Q; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
    float den = 0.0f;
    bool seen = false;
    for (int k = quad; k < n; k += Q) {
      const float* p = piece(k);
      const float m = p[D], l = p[D + 1];
      seen |= l != 0.0f;
      // a piece of no tokens, or of -inf scores, weighs nothing; one of NaN scores stays
      const float f = m != -INFINITY ? __builtin_amdgcn_exp2f(m - M) : l != l ? 1.0f : 0.0f;
      f_lds[r][k] = f;
      if (f != 0.0f || l != l) den = fmaf(l, f, den);
    }
#pragma unroll
    for (int o = 1; o < Q; o <<= 1) {
      den += __shfl_xor(den, o);
      seen |= __shfl_xor((int)seen, o) != 0;
    }
    __syncthreads();
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int k = 0; k < n; ++k) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(piece(k) + 4 * quad);
      const float f = f_lds[r][k];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(f, f != 0.0f ? x[e] : 0.0f, acc[e]);
    }
    if (c0 + r < cut.cols) {
      const int qi = col / a.group, qh = cut.head * a.group + col - qi * a.group;
      const float f = seen ? a.v_scale / den : 0.0f;
      store4(a.out, QT, (((int64_t)cut.row0 + qi) * a.num_q_heads + qh) * D + 4 * quad, acc * f);
    }
    __syncthreads();
  }
}

// ---- the general kernel --------------------------------------------------------------

// A wave per (row, query head): 64 tokens at a time, one a lane for the scores, then
// the dims on the lanes for the values.  For fp32, head dims other than 64, 128 and
// 256, rows that are not 16-byte aligned and groups of more than kRows heads; every
// K and V element is read again for each row and head.
template <int KV, int QT>
__global__ __launch_bounds__(kThreads) void rows_general_kernel(RowsArgs a) {
  __shared__ float q_lds[kWaves][kMaxDim];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, D = a.head_dim;
  const int64_t id = (int64_t)blockIdx.x * kWaves + wave;
  const int64_t row = id / a.num_q_heads;
  const int qh = (int)(id - row * a.num_q_heads), head = qh / a.group;
  int seq = -1;
  int64_t ctx = 0, pos = -1;
  int flags = 0;
  if (row < a.n_rows && a.num_seqs > 0) {  // the last sequence that starts at or before it
    int lo = 0, hi = a.num_seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.query_start[mid] <= row) lo = mid; else hi = mid;
    }
    const int64_t first = a.query_start[lo], end = a.query_start[lo + 1];
    if (first >= 0 && first <= row && row < end && end <= a.n_rows) {
      seq = lo;
      ctx = max(a.context_lens[lo], 0);
      pos = ctx - (end - row);
    }
  }
  if (seq >= 0) {
    const uint8_t* q = a.q + row * a.q_row + qh * a.q_head;
    for (int d = lane; d < D; d += 64) q_lds[wave][d] = kv_elem<QT>(q + d * elem_bytes<QT>());
  }
  __syncthreads();
  if (seq < 0) return;
  const int64_t cap = (int64_t)a.table_pages * a.block_size;
  if (ctx > cap) flags |= AMF_ERRFLAG_CONTEXT;
  const int64_t n = min(min(pos + 1, ctx), cap);
  const int32_t* table = a.block_tables + seq * a.bt_stride;
  constexpr int EB = KV == kInt4 ? 0 : KV == AMF_DTYPE_E4M3 ? 1 : elem_bytes<KV == kInt4 ? 0 : KV>();
  const int G = D / 32;
  float m = -INFINITY, l = 0.0f, acc[kMaxDim / 64] = {0.0f, 0.0f, 0.0f, 0.0f};
  bool seen = false;
  for (int64_t t0 = 0; t0 < n; t0 += 64) {
    const int64_t t = t0 + lane;
    int64_t place = -1;  // byte offset of the token's row; INT4: (page, head) block * 16 + token
    if (t < n) {
      const int64_t page = table[t / a.block_size];
      if (page < 0 || page >= a.pool_pages)
        flags |= AMF_ERRFLAG_BLOCK_RANGE;
      else if constexpr (KV == kInt4)
        place = (page * a.num_kv_heads + head) * 16 + t % 16;
      else
        place = page * a.page_stride + t % a.block_size * a.token_stride + head * a.head_stride;
    }
    float s = -INFINITY;
    if (place >= 0) {
      float x = 0.0f;
      for (int d = 0; d < D; ++d) {
        float k;
        if constexpr (KV == kInt4) {
          const uint8_t c = a.k[place * (D / 2) + d / 2];
          const uint32_t p = a.kp[place * G + d / 32];
          k = round_to<QT>(
              __builtin_fmaf((float)(d % 2 ? c >> 4 : c & 15), param_scale(p), param_zero(p)));
        } else {
          k = kv_elem<KV>(a.k + place + d * EB);
        }
        x = fmaf(q_lds[wave][d], k, x);
      }
      s = x * a.score_scale;
    }
    float mx = s;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
    const float m_new = fmaxf(m, mx), m_use = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - m_use);
    m = m_new;
    const float p = place >= 0 ? __builtin_amdgcn_exp2f(s - m_use) : 0.0f;
    l = l * alpha + p;
#pragma unroll
    for (int i = 0; i < kMaxDim / 64; ++i) acc[i] *= alpha;
    uint64_t on = __ballot(place >= 0);
    seen |= on != 0;
    for (; on; on &= on - 1) {
      const int b = __ffsll((unsigned long long)on) - 1;
      const float w = __shfl(p, b);
      const int64_t at = __shfl(place, b);
#pragma unroll
      for (int i = 0; i < kMaxDim / 64; ++i) {
        const int d = lane + 64 * i;
        if (d >= D) continue;
        float v;
        if constexpr (KV == kInt4) {
          const int tk = (int)(at % 16);
          const int64_t block = at / 16;
          const uint8_t c =
              a.v[block * 8 * D + 64 * (d / 8) + 32 * (tk / 8) + 4 * (d % 8) + tk % 8 / 2];
          const uint32_t pr = a.vp[(block * G + d / 32) * 16 + tk];
          v = round_to<QT>(
              __builtin_fmaf((float)(tk % 2 ? c >> 4 : c & 15), param_scale(pr), param_zero(pr)));
        } else {
          v = kv_elem<KV>(a.v + at + d * EB);
        }
        acc[i] = fmaf(w, v, acc[i]);
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o);
  const float f = seen ? a.v_scale / l : 0.0f;
  uint8_t* out = reinterpret_cast<uint8_t*>(a.out) +
                 (row * a.num_q_heads + qh) * D * elem_bytes<QT>();
#pragma unroll
  for (int i = 0; i < kMaxDim / 64; ++i) {
    const int d = lane + 64 * i;
    if (d >= D) continue;
    const float x = seen ? acc[i] * f : 0.0f;
    if constexpr (QT == AMF_DTYPE_F32)
      reinterpret_cast<float*>(out)[d] = x;
    else
      reinterpret_cast<uint16_t*>(out)[d] = (uint16_t)pair16<QT>(x, 0.0f);
  }
  if (flags && a.err_flag) atomicOr(a.err_flag, flags);
}

// ------------------------------------------------------------------ host ----

bool matrix_dim(int D) { return D == 64 || D == 128 || D == 256; }

int64_t part_floats(int D) { return (int64_t)2 * kRows * (D + kPartPad); }

template <int QT, int KV>
void launch_matrix(const RowsArgs& a, hipStream_t st) {
  const dim3 grid(a.shares), merge(a.shares, kMergeParts);
#define AMF_ROWS(DD)                                       \
  rows_kernel<QT, KV, DD><<<grid, kThreads, 0, st>>>(a);   \
  rows_merge_kernel<QT, DD><<<merge, kThreads, 0, st>>>(a)
  if (a.head_dim == 64) {
    AMF_ROWS(64);
  } else if (a.head_dim == 128) {
    AMF_ROWS(128);
  } else {
    AMF_ROWS(256);
  }
#undef AMF_ROWS
}

template <int QT, int KV>
void launch_general(const RowsArgs& a, hipStream_t st) {
  const int64_t waves = a.n_rows * a.num_q_heads;
  rows_general_kernel<KV, QT>
      <<<dim3((unsigned)((waves + kWaves - 1) / kWaves)), kThreads, 0, st>>>(a);
}

int check(const char* who, const RowsArgs& a, int32_t q_dtype, const void* workspace,
          int64_t workspace_bytes, int64_t need) {
  if (a.num_seqs < 0 || a.n_rows < 0 || a.num_q_heads <= 0 || a.num_kv_heads <= 0 ||
      a.num_q_heads % a.num_kv_heads || a.head_dim <= 0 || a.block_size <= 0 ||
      a.table_pages < 0 || a.bt_stride < a.table_pages || a.pool_pages <= 0)
    return fail(AMF_ERR_INVALID_ARG,
                "%s: bad num_seqs=%d n_rows=%lld heads=%d/%d (a multiple) head_dim=%d "
                "block_size=%d table_pages=%d bt_stride=%lld pool_pages=%lld",
                who, a.num_seqs, (long long)a.n_rows, a.num_q_heads, a.num_kv_heads, a.head_dim,
                a.block_size, a.table_pages, (long long)a.bt_stride, (long long)a.pool_pages);
  if (a.head_dim > kMaxDim || a.n_rows * a.num_q_heads > (int64_t)1 << 26)
    return fail(AMF_ERR_UNSUPPORTED, "%s: head_dim=%d (at most %d) or %lld rows of %d heads", who,
                a.head_dim, kMaxDim, (long long)a.n_rows, a.num_q_heads);
  if (!cache_elem_bytes(q_dtype))
    return fail(AMF_ERR_UNSUPPORTED, "%s: q dtype %d", who, q_dtype);
  if ((int64_t)a.table_pages * a.block_size > kMaxContext)
    return fail(AMF_ERR_UNSUPPORTED, "%s: block tables of %d pages of %d tokens", who,
                a.table_pages, a.block_size);
  if (a.n_rows == 0 || a.num_seqs == 0) return AMF_OK;
  if (!a.q || !a.out || !a.k || !a.v || !a.query_start || !a.context_lens ||
      (a.table_pages > 0 && !a.block_tables))
    return fail(AMF_ERR_INVALID_ARG, "%s: null pointer", who);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
    return fail(AMF_ERR_WORKSPACE, "%s: workspace of %lld bytes (16-byte aligned) needed, got %lld",
                who, (long long)need, (long long)workspace_bytes);
  return AMF_OK;
}

void finish_args(RowsArgs* a, void* workspace, float softmax_scale, float k_scale) {
  a->group = a->num_q_heads / a->num_kv_heads;
  a->tile_rows = std::max(1, kRows / a->group);
  const int b = a->block_size;
  a->block_shift = (b & (b - 1)) == 0 ? __builtin_ctz((unsigned)b) : -1;
  a->by16 = b % 16 == 0 && a->token_stride >= 0 && a->token_stride < (1 << 27);
  const float scale =
      softmax_scale > 0.0f ? softmax_scale : 1.0f / __builtin_sqrtf((float)a->head_dim);
  a->score_scale = scale * k_scale * kLog2e;
  // shares of kMinShare that the longest contexts of the tables could fill
  const int64_t tiles = a->n_rows / a->tile_rows + std::min<int64_t>(a->num_seqs, a->n_rows);
  const int64_t cap = (int64_t)a->table_pages * a->block_size + a->tile_rows + kTileCost;
  const int64_t most = (tiles * a->num_kv_heads * cap + kMinShare - 1) / kMinShare;
  // whole rounds of the XCDs
  a->shares = (int)std::min<int64_t>(kMaxShares, (most + kXcds - 1) / kXcds * kXcds);
  a->cuts = static_cast<Cut*>(workspace);
  a->part = reinterpret_cast<float*>(a->cuts + kMaxShares);
}

}  // namespace

extern "C" int64_t amf_paged_attn_rows_workspace_bytes(int32_t num_q_heads, int32_t num_kv_heads,
                                                       int32_t head_dim) {
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || head_dim <= 0 ||
      head_dim > kMaxDim)
    return 0;
  if (!matrix_dim(head_dim)) return 16;
  return kMaxShares * ((int64_t)sizeof(Cut) + part_floats(head_dim) * (int64_t)sizeof(float));
}

extern "C" int amf_paged_attn_rows(
    const void* q, int32_t q_dtype, int64_t q_row_stride, int64_t q_head_stride, void* out,
    int64_t n_rows, const int32_t* query_start, const void* k, const void* v, int32_t kv_dtype,
    int64_t page_stride, int64_t token_stride, int64_t head_stride, int64_t pool_pages,
    const int32_t* block_tables, int64_t bt_stride, int32_t table_pages,
    const int32_t* context_lens, int32_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads,
    int32_t head_dim, int32_t block_size, float softmax_scale, float k_scale, float v_scale,
    void* workspace, int64_t workspace_bytes, int32_t* err_flag, void* stream) {
  const char* who = "amf_paged_attn_rows";
  const int es = kv_elem_bytes(kv_dtype), qs = cache_elem_bytes(q_dtype);
  RowsArgs a{};
  a.q = static_cast<const uint8_t*>(q);
  a.q_row = q_row_stride * qs;
  a.q_head = q_head_stride * qs;
  a.out = static_cast<uint16_t*>(out);
  a.n_rows = n_rows;
  a.query_start = query_start;
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
  a.num_seqs = num_seqs;
  a.num_q_heads = num_q_heads;
  a.num_kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.block_size = block_size;
  a.v_scale = v_scale;
  a.err_flag = err_flag;
  const int rc = check(who, a, q_dtype, workspace, workspace_bytes,
                       amf_paged_attn_rows_workspace_bytes(num_q_heads, num_kv_heads, head_dim));
  if (rc) return rc;
  const bool fp8 = kv_dtype == AMF_DTYPE_E4M3;
  if (!(fp8 ? q_dtype != AMF_DTYPE_F32 : kv_dtype == q_dtype))
    return fail(AMF_ERR_UNSUPPORTED, "%s: q of type %d over a cache of type %d", who, q_dtype,
                kv_dtype);
  if (!(k_scale > 0.0f) || !(v_scale > 0.0f))
    return fail(AMF_ERR_INVALID_ARG, "%s: scales must be positive", who);
  if (n_rows == 0 || num_seqs == 0) return ok();
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)a.page_stride | (uintptr_t)a.token_stride |
       (uintptr_t)a.head_stride) % es ||
      ((uintptr_t)q | (uintptr_t)out) % qs)
    return fail(AMF_ERR_INVALID_ARG, "%s: elements must be aligned", who);
  finish_args(&a, workspace, softmax_scale, k_scale);
  const bool vec = ((uintptr_t)q | (uintptr_t)a.q_row | (uintptr_t)a.q_head | (uintptr_t)out |
                    (uintptr_t)k | (uintptr_t)v | (uintptr_t)a.page_stride |
                    (uintptr_t)a.token_stride | (uintptr_t)a.head_stride) %
                       16 == 0;
  const bool matrix = q_dtype != AMF_DTYPE_F32 && matrix_dim(head_dim) && vec && a.group <= kRows;
  hipStream_t st = as_stream(stream);
#define AMF_PICK(QT, KV) (matrix ? launch_matrix<QT, KV>(a, st) : launch_general<QT, KV>(a, st))
  if (q_dtype == AMF_DTYPE_F32)
    launch_general<AMF_DTYPE_F32, AMF_DTYPE_F32>(a, st);
  else if (q_dtype == AMF_DTYPE_BF16)
    fp8 ? AMF_PICK(AMF_DTYPE_BF16, AMF_DTYPE_E4M3) : AMF_PICK(AMF_DTYPE_BF16, AMF_DTYPE_BF16);
  else
    fp8 ? AMF_PICK(AMF_DTYPE_F16, AMF_DTYPE_E4M3) : AMF_PICK(AMF_DTYPE_F16, AMF_DTYPE_F16);
#undef AMF_PICK
  return check_launch(who);
}

extern "C" int amf_int4_paged_attn_rows(
    const void* q, int32_t q_dtype, int64_t q_row_stride, int64_t q_head_stride, void* out,
    int64_t n_rows, const int32_t* query_start, const void* k_codes, const void* k_params,
    const void* v_codes, const void* v_params, int64_t pool_pages, const int32_t* block_tables,
    int64_t bt_stride, int32_t table_pages, const int32_t* context_lens, int32_t num_seqs,
    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, float softmax_scale,
    void* workspace, int64_t workspace_bytes, int32_t* err_flag, void* stream) {
  const char* who = "amf_int4_paged_attn_rows";
  const int qs = cache_elem_bytes(q_dtype);
  RowsArgs a{};
  a.q = static_cast<const uint8_t*>(q);
  a.q_row = q_row_stride * qs;
  a.q_head = q_head_stride * qs;
  a.out = static_cast<uint16_t*>(out);
  a.n_rows = n_rows;
  a.query_start = query_start;
  a.k = static_cast<const uint8_t*>(k_codes);
  a.v = static_cast<const uint8_t*>(v_codes);
  a.kp = static_cast<const uint32_t*>(k_params);
  a.vp = static_cast<const uint32_t*>(v_params);
  a.pool_pages = pool_pages;
  a.block_tables = block_tables;
  a.bt_stride = bt_stride;
  a.table_pages = table_pages;
  a.context_lens = context_lens;
  a.num_seqs = num_seqs;
  a.num_q_heads = num_q_heads;
  a.num_kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.block_size = 16;
  a.v_scale = 1.0f;
  a.err_flag = err_flag;
  const int rc = check(who, a, q_dtype, workspace, workspace_bytes,
                       amf_paged_attn_rows_workspace_bytes(num_q_heads, num_kv_heads, head_dim));
  if (rc) return rc;
  if (head_dim % 32 || q_dtype == AMF_DTYPE_F32)
    return fail(AMF_ERR_UNSUPPORTED, "%s: head_dim %d (a multiple of 32), q dtype %d", who,
                head_dim, q_dtype);
  if (n_rows == 0 || num_seqs == 0) return ok();
  if (!k_params || !v_params) return fail(AMF_ERR_INVALID_ARG, "%s: null pointer", who);
  if (((uintptr_t)k_codes | (uintptr_t)k_params | (uintptr_t)v_codes | (uintptr_t)v_params) % 16 ||
      ((uintptr_t)q | (uintptr_t)out) % qs)
    return fail(AMF_ERR_INVALID_ARG, "%s: elements and the pool's planes must be aligned", who);
  finish_args(&a, workspace, softmax_scale, 1.0f);
  const bool vec =
      ((uintptr_t)q | (uintptr_t)a.q_row | (uintptr_t)a.q_head | (uintptr_t)out) % 16 == 0;
  const bool matrix = matrix_dim(head_dim) && vec && a.group <= kRows;
  hipStream_t st = as_stream(stream);
  if (q_dtype == AMF_DTYPE_BF16)
    matrix ? launch_matrix<AMF_DTYPE_BF16, kInt4>(a, st)
           : launch_general<AMF_DTYPE_BF16, kInt4>(a, st);
  else
    matrix ? launch_matrix<AMF_DTYPE_F16, kInt4>(a, st)
           : launch_general<AMF_DTYPE_F16, kInt4>(a, st);
  return check_launch(who);
}

// amf_paged_rows.h - what a workgroup of the attention of several rows reads of K and
// V: its arguments, and tiles of a paged cache or an INT4 pool brought into LDS.
#pragma once

#include "amf_attn.h"
#include "amf_int4_asym.h"
#include "amf_paged.h"

namespace amf {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef s16x4 __attribute__((address_space(3))) lds_s16x4;
typedef uint8_t __attribute__((address_space(3))) lds_u8;
typedef u32x4 __attribute__((address_space(3))) lds_u32x4;

__device__ __forceinline__ uint32_t lds_address(const uint8_t* p) {
  return (uint32_t)(uintptr_t)(lds_u8*)p;
}

constexpr int kRowsWaves = 4;
constexpr int kRowsThreads = 64 * kRowsWaves;
constexpr int kInt4 = 16;  // beside the AMF_DTYPE_* of a cache

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
  uint32_t pages;  // pool_pages, or 2^31: every id from 0 on
  const int32_t* block_tables;
  int64_t bt_stride;
  int32_t table_pages;
  const int32_t* context_lens;
  int32_t num_seqs, num_q_heads, num_kv_heads, head_dim, block_size;
  int32_t block_shift;  // by16: log2(block_size)
  int32_t group;        // query heads of a KV head
  int32_t tile_rows;    // query rows of a tile
  bool by16;            // block_size is 16, 32, 64, .., and page and token strides are
  uint32_t page_units, token_units;  // these many times 16 bytes, a plane below 2^32 of them
  int32_t shares;       // of the grid
  float score_scale;    // softmax scale * k_scale * log2(e)
  float v_scale;
  Cut* cuts;            // [workgroup]
  float* part;          // [share][2][kRows][head_dim + kPartPad]
  int32_t* err_flag;
};

// Tokens of a tile in LDS.
constexpr int tile_tokens(int D) { return D == 256 ? 32 : 64; }

// A row of D 16-bit values in LDS, its 16-byte chunks permuted so that reads meet each
// bank once: chunk c of row r lies at place c ^ swizzle(r).  K is read as the same chunk
// of 16 consecutive rows, V (by the transposing read) as 64 bytes of 4 consecutive rows.
template <int D>
__device__ __forceinline__ int k_swizzle(int r) {
  return D == 64 ? r >> 1 & 7 : r & 15;
}
template <int D>
__device__ __forceinline__ int v_swizzle(int r) {
  return D == 64 ? (r >> 1 & 1) << 2 : (r & 3) << 2;
}
template <int D>
__device__ __forceinline__ int k_place(int r, int c) {
  return r * 2 * D + ((c ^ k_swizzle<D>(r)) << 4);
}
template <int D>
__device__ __forceinline__ int v_place(int r, int c) {
  return r * 2 * D + ((c ^ v_swizzle<D>(r)) << 4);
}

// Two fp32 values as a pair of type T in one conversion, round to nearest even.
template <int T>
__device__ __forceinline__ uint32_t pair16(float a, float b) {
  if constexpr (T == AMF_DTYPE_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2_t));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2_t));
}

// Two fp32 numbers a, b >= 0 as pairs hi + lo of type T.  lo is above 0, so that an infinite
// factor stays one (a zero or negative lo would make it NaN): bf16, the number cut to 8 bits and
// what is left with 2^-23 of the number; fp16, a step less than the number cut to 11 bits and
// what is left.  That is at most 2^-7 (2^-9) of the number's leading bit and rounded to 8 (11)
// bits: hi + lo is within 2^-16 + 2^-23 (2^-21) of the number, or in fp16 2^-25 of it.  (fp16
// numbers below 2^-23 have hi = 0.)
struct TwoTerms {
  uint32_t hi, lo;
};
template <int T>
__device__ __forceinline__ TwoTerms two_terms(float a, float b) {
  if constexpr (T == AMF_DTYPE_BF16) {
    constexpr float up = 1.0f + 0x1p-23f;
    const uint32_t x = f2u(a), y = f2u(b);
    return {__builtin_amdgcn_perm(y, x, 0x07060302u),
            pair16<T>(__builtin_fmaf(a, up, -u2f(x & 0xFFFF0000u)),
                      __builtin_fmaf(b, up, -u2f(y & 0xFFFF0000u)))};
  } else {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    const u16x2 cut = __builtin_bit_cast(u16x2, __builtin_amdgcn_cvt_pkrtz(a, b));
    const u16x2 x = __builtin_elementwise_sub_sat(cut, (u16x2){1, 1});
    const f16x2_t h = __builtin_bit_cast(f16x2_t, x);
    return {__builtin_bit_cast(uint32_t, x), pair16<T>(a - (float)h[0], b - (float)h[1])};
  }
}

// Sets values that are not finite to 0; whether there were any.
template <int T, int N>
__device__ __forceinline__ bool clean(uint32_t (&v)[N]) {
  constexpr uint32_t m = T == AMF_DTYPE_BF16 ? 0x7F80u : 0x7C00u;
  bool found = false;
#pragma unroll
  for (int w = 0; w < N; ++w) {
    const bool lo = (v[w] & m) == m, hi = (v[w] >> 16 & m) == m;
    v[w] &= (lo ? 0xFFFF0000u : ~0u) & (hi ? 0xFFFFu : ~0u);
    found |= lo | hi;
  }
  return found;
}

// x, of which the compiler knows nothing: what seldom branches derive from it is not
// computed ahead and kept in registers over the loop.
__device__ __forceinline__ int opaque(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// The thread's index, for addresses that the turns of a piece keep in registers (KEEP; `id`
// is the piece's own, so that they are not kept over all pieces) or compute again each.
template <bool KEEP>
__device__ __forceinline__ int thread(int id) {
  return KEEP ? id : opaque(threadIdx.x);
}

// Marks row r where `is`.
__device__ __forceinline__ void mark_row(uint32_t* marks, int r, bool is) {
  atomicOr(marks + r / 32, is ? 1u << (r % 32) : 0u);
}

// A mover brings tiles of one (block table, KV head) into LDS, K one tile ahead of V:
// next(t) finds the pages, and of quantised caches loads, K of the tile at t and V of the
// one before; store_k and store_v put what the last next() found into LDS, complete
// after settle() and a barrier.  kInRegisters: what it found can be copied, and stored after
// the following next().  `end`: tokens that are read; behind them K rows hold anything
// (they are hidden), V rows zeros.  Rows whose page is none are marked by store_k, and
// are zeros in V.  check: V values that are not finite become 0, *wild != 0 then.
//
// KEEP: there are registers for addresses.  Branches in next() and the stores are the same
// for all lanes of a wave, or select.

// What movers of caches (EB bytes an element) share.  Wave w of the workgroup takes rows
// RPW w .. of a tile, which lie in one aligned group of 16: with pages of 16, 32, 64 ..
// tokens (BY16) it looks up one page a tile (with every wave's rows spread over the tile's
// pages each looked up them all, in 420 scalar instructions: more than the products
// take).  A lane takes 16 bytes of a row, CH rows RPI apart.
template <int EB, int D, bool BY16>
struct CacheMover {
  static constexpr int BT = tile_tokens(D);
  static constexpr int CPR = D * EB / 16;          // 16-byte chunks of a row
  static constexpr int RPI = 64 / CPR;             // rows of a load instruction
  static constexpr int RPW = BT / kRowsWaves;      // rows of a wave
  static constexpr int CH = RPW / RPI;
  static_assert(CH >= 1 && RPW <= 16 && 64 % CPR == 0, "a wave's rows are whole loads");

  const RowsArgs& a;
  const int32_t* table;
  int end;
  int id;                  // of the thread
  const uint8_t *kb, *vb;  // the KV head's
  int32_t k_id, v_id;      // BY16: pages of the wave's rows; -1 behind `end`
  uint32_t k_off, v_off;   // and their place, in units of 16 bytes
  int32_t ahead;           // BY16: the table's entry for the tile after K's

  __device__ __forceinline__ CacheMover(const RowsArgs& args) : a(args) {}
  static __device__ __forceinline__ int wave_row() {
    return __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * RPW;
  }
  static __device__ __forceinline__ int lane_row(int i, int tid = threadIdx.x) {
    return tid % 64 / CPR + i * RPI;
  }
  static __device__ __forceinline__ int row(int i, int tid = threadIdx.x) {
    return tid / 64 * RPW + lane_row(i, tid);
  }
  __device__ __forceinline__ bool good(int32_t id) const { return (uint32_t)id < a.pages; }
  // Byte offset of token t's row in page id, of any block size.
  __device__ __forceinline__ int page_of(int t) const {
    return (int)((uint32_t)t / (uint32_t)a.block_size);
  }
  __device__ __forceinline__ int64_t place(int32_t id, int t) const {
    return id * a.page_stride + (t - page_of(t) * a.block_size) * a.token_stride;
  }
  __device__ __forceinline__ void start(int seq, int head, int t0, int e) {
    table = a.block_tables + seq * a.bt_stride;
    end = e;
    id = opaque(threadIdx.x);
    kb = a.k + head * a.head_stride;
    vb = a.v + head * a.head_stride;
    k_id = -1;
    k_off = 0;
    if (BY16 && e > 0) look_up(t0);
  }
  // BY16: goes on to the K tile at t0.  The table's entry was asked for a turn before, as
  // the tile's loads depend on it, by a vector load: reads of LDS behind a scalar one
  // wait for it.
  __device__ __forceinline__ void advance(int t0) {
    v_id = k_id;
    v_off = k_off;
    const int t = t0 + wave_row();
    const int32_t page = __builtin_amdgcn_readfirstlane(ahead);
    k_id = t < end ? page : -1;
    k_off = (uint32_t)page * a.page_units + (uint32_t)(t & (a.block_size - 1)) * a.token_units;
    look_up(t0 + BT);
  }
  __device__ __forceinline__ void look_up(int t0) {
    ahead = table[opaque(min(t0 + wave_row(), end - 1) >> a.block_shift)];
  }
  // The wave's rows behind `off`, and a lane's bytes of row i behind that.
  static __device__ __forceinline__ const uint8_t* base(const uint8_t* plane, uint32_t off) {
    return plane + ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(off) << 4);
  }
  __device__ __forceinline__ uint32_t lane_off(int i, int chunk, int lane) const {
    return (lane_row(i, lane) * a.token_units + chunk) << 4;
  }
  // 16 bytes of token t's row from byte c on, zeros where it is not there; *bad: its page
  // is none.
  __device__ __forceinline__ u32x4 lane_row_of(const uint8_t* plane, int t, int c,
                                               bool* bad) const {
    const int32_t id = table[page_of(min(t, end - 1))];
    const bool ok = t < end && good(id);
    *bad = t < end && !good(id);
    u32x4 x = *reinterpret_cast<const u32x4*>(plane + place(ok ? id : 0, ok ? t : 0) + c);
#pragma unroll
    for (int w = 0; w < 4; ++w) x[w] = ok ? x[w] : 0u;
    return x;
  }
  __device__ __forceinline__ bool there(int t) const { return good(table[page_of(t)]); }
  // Element d of token t's row of K or V, from memory.
  template <int KV>
  __device__ __forceinline__ float elem(const uint8_t* plane, int t, int d) const {
    return kv_elem<KV>(plane + place(table[page_of(t)], t) + d * EB);
  }
};

// 16-bit rows go to LDS directly (no registers; a lane's 16 bytes land at its place, so
// it loads the chunk that belongs there), in kParts loads that the caller spreads over its
// products: all at once they hold up the wave, as the CU takes 16 cycles for each.  They
// are issued for tiles and pages that are not there as well, from page 0, and what they
// bring is hidden or made zeros.  Pages of other sizes pass through registers.
template <int QT, int KV, int D, bool BY16>
struct Mover : CacheMover<2, D, BY16> {
  using Base = CacheMover<2, D, BY16>;
  using Base::a, Base::id, Base::row, Base::end, Base::kb, Base::vb, Base::k_id, Base::v_id;
  static constexpr int VT = QT, BT = Base::BT, CH = Base::CH, RB = 2 * D;
  static constexpr bool kInRegisters = false;
  static constexpr int kParts = 2 * CH;

  uint32_t row_off, k_chunk, v_chunk;  // of the lane's bytes of row(0)
  const uint8_t *k_src, *v_src;        // the wave's rows
  uint32_t k_dst, v_dst;
  // V rows of this wave that are to be looked at when they are there.
  bool look;
  int look_t;

  __device__ __forceinline__ Mover(const RowsArgs& args) : Base(args), look(false) {}
  __device__ __forceinline__ void start(int seq, int head, int t0, int e) {
    Base::start(seq, head, t0, e);
    const int r = row(0, id), c = id % Base::CPR;
    row_off = (Base::lane_row(0, id) * a.token_units) << 4;
    k_chunk = (c ^ k_swizzle<D>(r)) << 4;
    v_chunk = (c ^ v_swizzle<D>(r)) << 4;
  }
  // 16 bytes of each lane, at base + off, to 16 lane bytes behind `lds` + further.  In
  // assembly, as
  // the compiler waits for all loads in flight before LDS reads that it cannot tell from
  // what they write; settle() does that.
  static __device__ __forceinline__ void load_lds(const uint8_t* base, uint32_t off,
                                                  uint32_t lds, int further) {
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 : : "v"(off), "s"(base), "s"(lds), "i"(further) : "memory", "m0", "scc");
  }
  template <bool KEEP>
  __device__ __forceinline__ void next(int t0) {
    if (BY16) this->advance(t0);
  }
  // Part p: the wave's K rows, then its V rows, from row(p) on.
  __device__ __forceinline__ void part(int p) const {
    if (!BY16) return;
    const int i = p % CH;  // rows RPI i further on: bits of the swizzles of their own
    const uint8_t* src = (p < CH ? k_src : v_src) + (uint32_t)(i * Base::RPI * 16) * a.token_units;
    const uint32_t chunk = p < CH ? k_chunk ^ k_swizzle<D>(i * Base::RPI) << 4
                                  : v_chunk ^ v_swizzle<D>(i * Base::RPI) << 4;
    load_lds(src, chunk + row_off, p < CH ? k_dst : v_dst, i * Base::RPI * RB);
  }
  template <bool KEEP>
  __device__ __forceinline__ void store_k(int t0, uint8_t* lds, bool wanted, uint32_t* bad) {
    if (BY16) {
      const int32_t page = __builtin_amdgcn_readfirstlane(k_id);
      const int wr = Base::wave_row();
      const bool ok = this->good(page);
      k_src = Base::base(kb, ok ? this->k_off : 0u);
      k_dst = __builtin_amdgcn_readfirstlane(lds_address(lds) + wr * RB);
      if (wanted && !ok && t0 + wr < end)
        for (int i = 0; i < CH; ++i) mark_row(bad, row(i, opaque(threadIdx.x)), true);
      return;
    }
    if (!wanted) return;
    const int tid = thread<KEEP>(id), c = tid % Base::CPR;
#pragma unroll 1
    for (int i = 0; i < CH; ++i) {
      const int r = row(i, tid);
      bool none;
      const u32x4 k = this->lane_row_of(kb, t0 + r, 16 * c, &none);
      mark_row(bad, r, none);
      *reinterpret_cast<u32x4*>(lds + k_place<D>(r, c)) = k;
    }
  }
  template <bool KEEP>
  __device__ __forceinline__ void store_v(int t0, uint8_t* lds, bool wanted, bool check,
                                          uint32_t* wild) {
    if (BY16) {
      const bool ok = this->good(__builtin_amdgcn_readfirstlane(v_id));
      // (in other tiles `end` is a page's, so a wave's rows lie all before it or all behind)
      look = wanted && (check || !ok);
      look_t = ok ? t0 : end;
      v_src = Base::base(vb, ok ? this->v_off : 0u);
      v_dst = __builtin_amdgcn_readfirstlane(lds_address(lds) + Base::wave_row() * RB);
      return;
    }
    if (!wanted) return;
    const int tid = thread<KEEP>(id), c = tid % Base::CPR;
#pragma unroll 1
    for (int i = 0; i < CH; ++i) {
      const int r = row(i, tid);
      bool none;
      const u32x4 x = this->lane_row_of(vb, t0 + r, 16 * c, &none);
      uint32_t w[4] = {x[0], x[1], x[2], x[3]};
      if (check) {
        const bool found = clean<VT>(w);
        mark_row(wild, 0, found);
      }
      *reinterpret_cast<u32x4*>(lds + v_place<D>(r, c)) = u32x4{w[0], w[1], w[2], w[3]};
    }
  }
  __device__ __forceinline__ void settle(uint32_t* wild) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (!look) return;
    look = false;
    const int tid = opaque(threadIdx.x);
    lds_u32x4* p = (lds_u32x4*)(v_dst + tid % 64 * 16);
    bool found = false;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const bool in = look_t + row(i, tid) < end;
      const u32x4 x = p[64 * i];
      uint32_t w[4] = {in ? x[0] : 0u, in ? x[1] : 0u, in ? x[2] : 0u, in ? x[3] : 0u};
      found |= clean<VT>(w);
      p[64 * i] = u32x4{w[0], w[1], w[2], w[3]};
    }
    mark_row(wild, 0, found);
  }
  __device__ __forceinline__ float k_elem(int t, int d) const {
    return this->template elem<KV>(kb, t, d);
  }
  __device__ __forceinline__ float v_elem(int t, int d) const {
    return this->template elem<KV>(vb, t, d);
  }
};

// FP8 rows: 16 values a chunk, converted on their way from registers to LDS.  V becomes
// fp16, which holds its values exactly as bf16 does.
template <int QT, int D, bool BY16>
struct Mover<QT, AMF_DTYPE_E4M3, D, BY16> : CacheMover<1, D, BY16> {
  using Base = CacheMover<1, D, BY16>;
  using Base::a, Base::id, Base::row, Base::end, Base::kb, Base::vb, Base::k_id, Base::v_id;
  static constexpr int VT = AMF_DTYPE_F16, BT = Base::BT;
  static constexpr bool kInRegisters = true;
  u32x4 kr[Base::CH], vr[Base::CH];
  int bad;    // bits of the lane's K rows whose pages are none
  bool none;  // BY16: no page for the wave's V rows

  __device__ __forceinline__ Mover(const RowsArgs& args) : Base(args) {}
  static __device__ __forceinline__ void settle(uint32_t*) {}
  // As many loads on every way, so that a wait for the tile before is not one for this.
  // Where no page is, any is read.
  template <bool KEEP>
  __device__ __forceinline__ void next(int t0) {
    bad = 0;
    if (BY16) {
      this->advance(t0);
      const int32_t ki = __builtin_amdgcn_readfirstlane(k_id);
      const int32_t vi = __builtin_amdgcn_readfirstlane(v_id);
      const int tid = thread<KEEP>(id), c = tid % Base::CPR;
      const uint8_t* kp = Base::base(kb, this->good(ki) ? this->k_off : 0u);
      const uint8_t* vp = Base::base(vb, this->good(vi) ? this->v_off : 0u);
#pragma unroll
      for (int i = 0; i < Base::CH; ++i) {
        kr[i] = *reinterpret_cast<const u32x4*>(kp + this->lane_off(i, c, tid));
        vr[i] = *reinterpret_cast<const u32x4*>(vp + this->lane_off(i, c, tid));
        bad |= (!this->good(ki) && t0 + row(i, tid) < end) << i;
      }
      none = !this->good(vi);
      return;
    }
    none = false;
    const int tid = thread<KEEP>(id), c = tid % Base::CPR * 16;
#pragma unroll
    for (int i = 0; i < Base::CH; ++i) {
      const int t = t0 + row(i, tid);
      bool gone;
      kr[i] = this->lane_row_of(kb, t, c, &gone);
      bad |= gone ? 1 << i : 0;
      vr[i] = this->lane_row_of(vb, max(t - BT, 0), c, &gone);
    }
  }
  template <int T, bool HIGH>
  static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    if constexpr (T == AMF_DTYPE_BF16)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HIGH));
  }
  template <bool KEEP>
  __device__ __forceinline__ void store_k(int, uint8_t* lds, uint32_t* marks) const {
    const int tid = thread<KEEP>(id), c = tid % Base::CPR * 2;
    if (__any(bad)) {
#pragma unroll
      for (int i = 0; i < Base::CH; ++i) mark_row(marks, row(i, tid), bad >> i & 1);
    }
#pragma unroll
    for (int i = 0; i < Base::CH; ++i)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint32_t x = kr[i][2 * n], y = kr[i][2 * n + 1];
        *reinterpret_cast<u32x4*>(lds + k_place<D>(row(i, tid), c + n)) =
            u32x4{pair<QT, false>(x), pair<QT, true>(x), pair<QT, false>(y), pair<QT, true>(y)};
      }
  }
  template <bool KEEP>
  __device__ __forceinline__ void store_v(int t0, uint8_t* lds, bool check,
                                          uint32_t* wild) const {
    const int tid = thread<KEEP>(id), c = tid % Base::CPR * 2;
#pragma unroll
    for (int i = 0; i < Base::CH; ++i) {
      uint32_t w[8];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        w[2 * n] = pair<VT, false>(vr[i][n]);
        w[2 * n + 1] = pair<VT, true>(vr[i][n]);
      }
      if (check || none) {
        const bool in = !none && t0 + row(i, tid) < end;
#pragma unroll
        for (int n = 0; n < 8; ++n) w[n] = in ? w[n] : 0u;
        const bool found = clean<VT>(w);
        mark_row(wild, 0, found);
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
        *reinterpret_cast<u32x4*>(lds + v_place<D>(row(i, tid), c + n)) =
            u32x4{w[4 * n], w[4 * n + 1], w[4 * n + 2], w[4 * n + 3]};
    }
  }
  __device__ __forceinline__ float k_elem(int t, int d) const {
    return this->template elem<AMF_DTYPE_E4M3>(kb, t, d);
  }
  __device__ __forceinline__ float v_elem(int t, int d) const {
    return this->template elem<AMF_DTYPE_E4M3>(vb, t, d);
  }
};

// INT4 pages: K rows of 32 dims (16 bytes, one param) a thread, V in chunks of 4 dims
// by 8 tokens (16 bytes, 8 params), dequantised on their way from registers to LDS.  At
// head_dim 64 half the threads move K, half V.
template <int QT, int D>
struct Mover<QT, kInt4, D, true> {
  static constexpr int BT = tile_tokens(D);
  static constexpr int VT = QT, G = D / 32, N = BT * G;  // items of K, and of V
  static constexpr bool HALF = N * 2 == kRowsThreads;
  static_assert(HALF || N == kRowsThreads, "an item per thread");
  static constexpr bool kInRegisters = true;

  const RowsArgs& a;
  const int32_t* table;
  int head;
  int end;
  const uint8_t *kc, *vc, *kp, *vp;  // the head's codes and parameters in page 0
  int id;  // of the thread
  u32x4 kr, vr, vs[2];
  uint32_t ks;
  bool k_none, v_none; // no page for the items of K (or not in the context), of V
  int32_t k_id, ahead; // the items' page, of K, and in the tile after

  __device__ __forceinline__ Mover(const RowsArgs& args) : a(args) {}
  static __device__ __forceinline__ void settle(uint32_t*) {}
  // the same in a wave
  static __device__ __forceinline__ bool has_k() {
    return !HALF || __builtin_amdgcn_readfirstlane(threadIdx.x) < N;
  }
  static __device__ __forceinline__ bool has_v() {
    return !HALF || __builtin_amdgcn_readfirstlane(threadIdx.x) >= N;
  }
  static __device__ __forceinline__ int item(int tid = threadIdx.x) { return tid % N; }
  static __device__ __forceinline__ int k_row(int tid = threadIdx.x) { return item(tid) / G; }
  // First token of the page that the lane's items lie in, of K and of V: one page a wave,
  // or (HALF) one for each half of it.
  static __device__ __forceinline__ int page_row(int tid = threadIdx.x) {
    const int x = item(tid) / (D / 2) * 16;
    return HALF ? x : __builtin_amdgcn_readfirstlane(x);
  }
  __device__ __forceinline__ bool good(int32_t id) const { return (uint32_t)id < a.pages; }
  __device__ __forceinline__ void start(int seq, int h, int t0, int e) {
    table = a.block_tables + seq * a.bt_stride;
    head = h;
    end = e;
    kc = a.k + h * 8 * D;
    vc = a.v + h * 8 * D;
    kp = reinterpret_cast<const uint8_t*>(a.kp) + h * 2 * D;
    vp = reinterpret_cast<const uint8_t*>(a.vp) + h * 2 * D;
    id = opaque(threadIdx.x);
    k_id = -1;
    if (e > 0) look_up(t0);
  }
  // As for a cache.
  __device__ __forceinline__ void look_up(int t0) {
    ahead = table[opaque(min(t0 + page_row(), end - 1) / 16)];
  }
  // Bytes of parameters before page id's, a quarter of those of codes.
  __device__ __forceinline__ uint64_t page_off(int32_t id) const {
    uint32_t x = good(id) ? id : 0;
    if constexpr (!HALF) x = __builtin_amdgcn_readfirstlane(x);
    return (uint64_t)x * (uint32_t)(a.num_kv_heads * 2 * D);
  }
  template <bool KEEP>
  __device__ __forceinline__ void next(int t0) {
    const int tid = thread<KEEP>(id);
    const uint32_t i = item(tid);
    const int32_t v_id = k_id;
    k_id = t0 + page_row(tid) < end ? ahead : -1;
    look_up(t0 + BT);
    k_none = !good(k_id);
    v_none = !good(v_id);
    if (has_k()) {  // items of a (page, head) block follow each other
      const uint64_t off = page_off(k_id);
      const uint32_t at = i % (16 * G);
      kr = *reinterpret_cast<const u32x4*>(kc + 4 * off + 16 * at);
      ks = *reinterpret_cast<const uint32_t*>(kp + off + 4 * at);
    }
    if (has_v()) {
      const uint64_t off = page_off(v_id);
      const uint32_t x = i % (D / 2), q = x / 16 * 4 + x / 2 % 2 * 2;
      vr = *reinterpret_cast<const u32x4*>(vc + 4 * off + 16 * x);
      vs[0] = *reinterpret_cast<const u32x4*>(vp + off + 16 * q);
      vs[1] = *reinterpret_cast<const u32x4*>(vp + off + 16 * q + 16);
    }
  }
  // Codes as fp16 numbers, two an instruction: a code u in the low bits of an fp16 is
  // u 2^-24, four bits further u 2^-20, and its scale comes 2^24 or 2^20 times as large.
  // c[i]: codes i and 4 + i of w, at i odd four bits further.
  static __device__ __forceinline__ void codes(uint32_t w, uint32_t (&c)[4]) {
    const uint32_t x = w >> 8;
    c[0] = w & 0x000F000Fu;
    c[1] = w & 0x00F000F0u;
    c[2] = x & 0x000F000Fu;
    c[3] = x & 0x00F000F0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("" : "+v"(c[i]));
  }
  static constexpr float unit(int i) { return i % 2 ? 0x1p20f : 0x1p24f; }
  // Code i of c.  The product with its scale is exact (4 bits by 11), so the fma rounds as the
  // codec's multiply and add.
  static __device__ __forceinline__ float value(const uint32_t (&c)[4], int i, float s,
                                                float z) {
    const f16x2_t u = __builtin_bit_cast(f16x2_t, c[i % 4]);
    return __builtin_fmaf((float)u[i / 4], s, z);
  }
  template <bool KEEP>
  __device__ __forceinline__ void store_k(int t0, uint8_t* lds, uint32_t* marks) const {
    if (!has_k()) return;
    const int tid = thread<KEEP>(id);
    if (__any(k_none)) mark_row(marks, k_row(tid), k_none && t0 + k_row(tid) < end);
    const float z = param_zero(ks), s[2] = {param_scale(ks) * unit(0), param_scale(ks) * unit(1)};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t c[4];
      codes(kr[w], c);
      u32x4 y;
#pragma unroll
      for (int n = 0; n < 4; ++n)
        y[n] = pair16<QT>(value(c, 2 * n, s[0], z), value(c, 2 * n + 1, s[1], z));
      *reinterpret_cast<u32x4*>(lds + k_place<D>(k_row(tid), 4 * (item(tid) % G) + w)) = y;
    }
  }
  template <bool KEEP>
  __device__ __forceinline__ void store_v(int t0, uint8_t* lds, bool check,
                                          uint32_t* wild) const {
    if (!has_v()) return;
    const int tid = thread<KEEP>(id), c = item(tid) % (D / 2);
    const int r0 = item(tid) / (D / 2) * 16 + c / 2 % 2 * 8;
    uint32_t x[4][4], y[16];
#pragma unroll
    for (int d = 0; d < 4; ++d) codes(vr[d], x[d]);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const uint32_t p = vs[t / 4][t % 4];
      const float s = param_scale(p) * unit(t), z = param_zero(p);
      y[2 * t] = pair16<QT>(value(x[0], t, s, z), value(x[1], t, s, z));
      y[2 * t + 1] = pair16<QT>(value(x[2], t, s, z), value(x[3], t, s, z));
    }
    if (check || __any(v_none)) {
#pragma unroll
      for (int t = 0; t < 16; ++t) y[t] = !v_none && t0 + r0 + t / 2 < end ? y[t] : 0u;
      if (!HALF || check) {  // (HALF: half of the wave's items may have a page)
        const bool found = clean<VT>(y);
        mark_row(wild, 0, found);
      }
    }
#pragma unroll
    for (int t = 0; t < 8; ++t)
      *reinterpret_cast<u32x2*>(lds + v_place<D>(r0 + t, c / 4) + c % 2 * 8) =
          u32x2{y[2 * t], y[2 * t + 1]};
  }
  __device__ __forceinline__ bool there(int t) const { return good(table[t / 16]); }
  __device__ __forceinline__ float k_elem(int t, int d) const {
    const int64_t line = ((int64_t)table[t / 16] * a.num_kv_heads + head) * 16 + t % 16;
    const uint8_t c = a.k[line * (D / 2) + d / 2];
    const uint32_t p = a.kp[line * G + d / 32];
    return round_to<QT>(
        __builtin_fmaf((float)(d % 2 ? c >> 4 : c & 15), param_scale(p), param_zero(p)));
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

}  // namespace amf

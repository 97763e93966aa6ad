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
// Tiles of 64 columns and fewer (decoded and drafted rows, short ends) are shared: two or
// four waves take parts of the tokens and of V's dims (with one wave at work 32 x 5 drafted
// rows over INT4 took 240 us, so 204, before the steps below).
//
// What bounds it.  With two workgroups of four waves a CU, a SIMD has two waves, and each
// issues an instruction every five cycles or so: a turn's time goes with its number of
// instructions of all kinds, and with its products (1536 of a SIMD's 2800 cycles a turn).
// So the turn is written out: weights, loads and maxima stand between the products, the
// accumulators are changed by products alone, one wave looks up one page, and what can be
// known before the turns is.  32 / 8 heads of 128: prompt of 12000 rows 1525 us, 0.77
// PFLOP/s in what the formula counts, 1.16 in what is multiplied (a library product reaches 1.2
// to 1.3); 64 x 32 rows of 8192 tokens 457 us, 4.7 TB/s; one row each 392 us, 5.5 TB/s, bound by
// the reads (FP8 246, 4.4); 48 decoded rows beside a chunk of 2048 rows of 8192 tokens 449 us,
// 0.54 PFLOP/s and 2.0 TB/s; 32 x 5 drafted rows over INT4 160 us, 2.2 TB/s, where taking out
// the codes is a third of a turn's instructions; prompt of 4096 rows over FP8 256, INT4 274.
//
// Shares.  Tile j of a sequence reads its first e_j tokens; the tiles of all
// (KV head, sequence, tile) one after the other, each as long as it reads plus a
// constant, are cut into equal shares, one a workgroup, so a mix of long chunks and
// single rows fills the chip.  e_j grows linearly in j, so a workgroup finds its
// place from sums over the sequences alone.  A tile inside one share is finished
// there; one that several share leaves partials (acc, m, l), joined by a second
// launch.  The constant is what a tile's beginning and end take, 448 tokens' time (8 prompts of
// 2048: with 256 tokens 478 us, 352 464, 448 455, 576 467).
// The older of a CU's two workgroups goes first wherever both could and ends at 4/5 of the
// other's time, which then is alone; the younger has a higher priority in every second turn
// (prompt of 12000 rows 1684 us without, 1543 with, and no loss where the reads bind; longer
// shares for the older gave the same here and lost 10 % there).
//
// Precision.  Products of Q and K are exact and summed in fp32; maximum, sum and
// accumulators are fp32.  A weight enters the second product as two terms of the type
// beside it: bf16 beside a bf16 V (16 bits of the weight), fp16 beside an fp16 or an FP8
// one (21 bits; fp16 holds FP8 values exactly).  The result is then off by 2^-16 of the
// weighted |v|, where rounding it to bf16 takes 2^-8 of itself (2^-21 and 2^-11 for fp16).
// With one term it was off by as much again as that rounding, and by more in values that cancel:
// those rounded weights are what a result near 0 consists of (prompt of 12000 rows
// 1209 us with one, 1525 with two; 64 single rows of 8192 tokens 392, so 402); a third bf16 term
// would cost another 16 products to the turn's 48, for bits that the result's type drops.
#include <algorithm>
#include <type_traits>

#include "amf_paged_rows.h"

// Held to a tolerance, as the other attention kernels: multiplies and adds may
// fuse.
#pragma clang fp contract(fast)

namespace {

using namespace amf;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr int kWaves = kRowsWaves;
constexpr int kThreads = kRowsThreads;
constexpr int kRows = 32 * kWaves;  // columns of a workgroup
constexpr int kMaxDim = 256;
constexpr int kMaxShares = 512;     // two workgroups a CU
// Lengths of tiles and shares.  A token of a tile of more than 64 columns counts kWide, of a
// narrower one kNarrow (48 decoded rows beside a chunk: 4/6 471 us, 5/6 452, 6/6 477).  Shares
// are of 256 tokens at least (a prompt of 512 rows: 128 tokens 50 us, 256 47, 2048 68).
constexpr int kWide = 6, kNarrow = 5;
constexpr int kMinShare = 256 * kWide;
constexpr int kTileCost = 448 * kWide;  // a tile's beginning and end; at least BT tokens
constexpr int kCusXcd = 32;
constexpr int kMaxContext = 1 << 30;

// ---- sequences and shares ------------------------------------------------------

struct Seq {
  int row0, rows;  // its rows of the step
  int pos0;        // position of the first
  int lim;         // tokens that the block table holds of its context
  int base;        // pos0, or more where the table is too short, at least 0
  int tiles;
  int weight;      // of a token of its tiles
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
  r.weight = min(r.rows, a.tile_rows) * a.group > 64 ? kWide : kNarrow;
  if (!ok || (ctx > cap && r.rows > 0)) *flags |= AMF_ERRFLAG_CONTEXT;
  return r;
}

// Tile j is weight (base + min((j + 1) tile_rows, rows)) + kTileCost long.
__device__ __forceinline__ int64_t tiles_before(const RowsArgs& a, const Seq& s, int64_t j) {
  return j * ((int64_t)s.weight * s.base + kTileCost) +
         (int64_t)s.weight * a.tile_rows * (j * (j + 1) / 2);
}
__device__ __forceinline__ int64_t seq_length(const RowsArgs& a, const Seq& s) {
  return s.tiles ? tiles_before(a, s, s.tiles - 1) + s.weight * ((int64_t)s.base + s.rows) +
                       kTileCost
                 : 0;
}

struct Share {
  int64_t index;
  int64_t length;         // of every share
  int64_t first, end;     // of this one
  int64_t seq_start;      // where the sequence starts that `first` lies in
  int32_t head, seq;      // seq -1: nothing to do
  bool young;             // not the first of its CU's workgroups
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
  r.young = slot >= kCusXcd;
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
// exceeds it by 2^kSlack.  Weights in bf16 are held 2^-kSlack times as large as the maximum
// makes them, so at most 1: finite values whose average is finite leave finite sums, as with
// the exact maximum, and weights down to 2^-118 of the largest keep their bits.  Weights in
// fp16 are held 2^7 times as large, at most 2^15 (values of at most 2^16 cannot exceed fp32):
// those down to 2^-21 of the largest keep the 11 bits of their first term.  (2^30 for bf16, in
// the maximum's own size, was no faster: prompt of 12000 rows 1542 us, with 2^8 1503.)
constexpr float kSlack = 8.0f;
template <int T>
constexpr float weight_shift() {
  return T == AMF_DTYPE_F16 ? 7.0f : -kSlack;
}

// The larger of x here and in lane ^ 32.
__device__ __forceinline__ float max_of_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return fmaxf(u2f(r[0]), u2f(r[1]));
}

template <int QT, int KV, int D, bool BY16>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void rows_kernel(RowsArgs a) {
  using Move = Mover<QT, KV, D, BY16>;
  constexpr int BT = Move::BT, VT = Move::VT, RB = 2 * D;
  // Two buffers each: while the values of a tile and the keys of the next are multiplied,
  // the next values and the keys after are on their way, with one barrier a tile.
  constexpr int TB = BT * RB;
  __shared__ __attribute__((aligned(2 * D))) uint8_t k_lds[2 * TB];
  __shared__ __attribute__((aligned(2 * D))) uint8_t v_lds[2 * TB];
  __shared__ uint32_t marks[4][2];  // of K tiles, by turns; [3]: the piece's wild V
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lc = lane & 31, h = lane >> 5;

  Cut cut{};
  const Share sh = find_share(a);
  if (sh.seq < 0) {
    if (tid == 0) a.cuts[blockIdx.x] = cut;
    return;
  }
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

  // This lane's LDS reads.  K: chunk 2 ks + h of row lc, whose swizzle the rows 32
  // further share.  V: 8 bytes of row 4 h + l16 / 4, whose swizzle depends on l16 alone,
  // for dims 32 d of each d.  Rows are aligned to their length, so ks and d flip bits
  // of one address.
  const int l16 = lane & 15, v_row = 4 * h + (l16 >> 2);
  const uint32_t k_at = lds_address(k_lds) + k_place<D>(lc, h);
  const uint32_t v_at = lds_address(v_lds) + 8 * (l16 & 1) +
                        v_place<D>(v_row, (lane >> 4 & 1) * 2 + (l16 >> 1 & 1));
  // A operand of V^T: dims 32 d .. + 31, 16 tokens in the order of the scores
  auto read_v = [](uint32_t at) __attribute__((always_inline)) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 8 * RB));
    const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
    return u32x4{l2[0], l2[1], h2[0], h2[1]};
  };

  while (start < sh.end) {
    const int row_lo = j * a.tile_rows;
    const int rows = min(a.tile_rows, sq.rows - row_lo);
    const int pos0 = sq.pos0 + row_lo;  // position of the tile's first row
    const int64_t length = (int64_t)sq.weight * (sq.base + row_lo + rows) + kTileCost;
    const int e = max(min(sq.lim, pos0 + rows), 0);
    // the share's part of [0, length)
    const bool begins = sh.first <= start;
    const int64_t lo = begins ? 0 : sh.first - start, hi = min(sh.end - start, length);
    const int unit = sq.weight * BT;
    const int t_lo = (int)min((int64_t)e, lo / unit * BT);
    const int t_hi = hi == length ? e : (int)min((int64_t)e, hi / unit * BT);
    const int cols = rows * G;
    // CG groups of 32 columns.  With fewer groups than waves, several waves work on one:
    // TS of them on 32 tokens of a tile each, DS on parts of V's dims.
    auto piece = [&](auto groups) __attribute__((always_inline)) {
      constexpr int CG = decltype(groups)::value, NW = kWaves / CG;
      constexpr bool KEEP = CG < kWaves;
      constexpr int TS = NW < BT / 32 ? NW : BT / 32, DS = NW / TS;
      constexpr int NB = BT / 32 / TS, DN = D / 32 / DS;  // a wave's blocks of 32: tokens, dims
      // its products of K and q of 32 tokens, and of all; of V
      constexpr int KS = D / 16, QN = NB * KS, PN = 2 * NB * DN;
      const int cg = wave % CG, tok = wave / CG % TS * 32, dim = wave / CG / TS * DN * 32;
      const uint32_t k_wave = k_at + tok * RB, v_wave = (v_at ^ (2 * dim)) + tok * RB;
      const int col = cg * 32 + lc;
      const int qi = min(col, cols - 1) / G;
      const int qh = head * G + min(col, cols - 1) - qi * G;
      const int qrow = sq.row0 + row_lo + qi;
      const bool wave_on = cg * 32 < cols;
      const int wave_first = cg * 32 / G;  // the wave's first row
      u32x4 qb[KS];  // B operand: dims 16 ks + 8 h .. + 7
      {
        const uint8_t* qp = a.q + qrow * a.q_row + qh * a.q_head + 16 * h;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          qb[ks] = *reinterpret_cast<const u32x4*>(qp + 32 * ks);
      }
      // the row's last token
      const int last = min(pos0 + qi, t_hi - 1);
      float m_run = -INFINITY, l_run = 0.0f;  // l_run: this lane's tokens
      bool seen = false;                      // a token that the row attends to
      f32x16 acc[DN], s[NB];
#pragma unroll
      for (int d = 0; d < DN; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;

      const int n = (t_hi - t_lo + BT - 1) / BT;  // tiles
      mv.start(seq, head, t_lo, t_hi);
      __syncthreads();  // the last piece's marks have been read
      marks[tid & 3][tid >> 2 & 1] = 0;
      __syncthreads();
      // Turn i stores K of tile i + 2 and V of tile i + 1, and multiplies V of tile i and K
      // of tile i + 1.
      int m0 = 0, m1 = 1, m2 = 2;  // marks of K tiles i + 2, i + 3, i + 1
      auto move = [&](int i) __attribute__((always_inline)) {
        const int t2 = t_lo + (i + 2) * BT, t1 = t2 - BT;
        if (sh.young) {
          if (i & 1)
            __builtin_amdgcn_s_setprio(1);
          else
            __builtin_amdgcn_s_setprio(0);
        }
        marks[m1][tid & 1] = 0;
        // tokens that some rows see and others do not: V has to be finite there, as
        // 0 * inf is not 0
        const bool check = t1 + BT > pos0 + 1;
        uint8_t *k_to = k_lds + (i & 1) * TB, *v_to = v_lds + (i + 1 & 1) * TB;
        const bool more_k = i + 2 < n, more_v = i >= -1 && i + 1 < n;
        if constexpr (Move::kInRegisters) {
          const Move now = mv;
          mv.template next<KEEP>(t2 + BT);
          if (more_k) now.template store_k<KEEP>(t2, k_to, marks[m0]);
          if (more_v) now.template store_v<KEEP>(t1, v_to, check, marks[3]);
        } else {
          mv.template next<KEEP>(t2);
          mv.template store_k<KEEP>(t2, k_to, more_k, marks[m0]);
          mv.template store_v<KEEP>(t1, v_to, more_v, check, marks[3]);
        }
        const int m = m2;
        m2 = m0;
        m0 = m1;
        m1 = m;
      };
      // What of move() is spread: every second of 2 kParts calls issues a load.
      auto load = [&](int p) __attribute__((always_inline)) {
        if constexpr (!Move::kInRegisters)
          if (p % 2 == 0 && p / 2 < Move::kParts) mv.part(p / 2);
      };
      // K fragment q of a tile: dims 16 (q % KS) .. of tokens 32 (q / KS) ..
      auto read_k = [&](uint32_t at, int q) __attribute__((always_inline)) {
        return *(const lds_u32x4*)((at ^ (32 * (q % KS))) + 32 * (q / KS) * RB);
      };
      // Whether tile i holds tokens that some of the wave's rows do not see; then they
      // are hidden.  Token of score element e of block tb: t0 + tok + 32 tb + 8 (e / 4) + 4 h
      // + e % 4.
      auto get_marks = [&](uint32_t(&x)[NB]) __attribute__((always_inline)) {  // m1's
#pragma unroll
        for (int tb = 0; tb < NB; ++tb) x[tb] = marks[m1][tok / 32 + tb];
      };
      auto hide = [&](int i, const uint32_t(&marked)[NB]) __attribute__((always_inline)) {
        const int t0 = t_lo + i * BT;
        uint32_t bad[NB], any = 0;
#pragma unroll
        for (int tb = 0; tb < NB; ++tb)
          any |= bad[tb] = __builtin_amdgcn_readfirstlane(marked[tb]);
        if (t0 + BT <= t_hi && t0 + BT - 1 <= pos0 + wave_first && !any) {
          seen = true;
          return false;
        }
        const int left = last - t0 - tok - 4 * h;
        bad_seen |= any != 0;
#pragma unroll
        for (int tb = 0; tb < NB; ++tb) {
          const uint32_t gone = opaque(bad[tb] >> (4 * h));  // no masks kept over the loop
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int t = 32 * tb + 8 * (e >> 2) + (e & 3);
            const bool hidden = t > left || (gone >> (t % 32) & 1);
            s[tb][e] = hidden ? -INFINITY : s[tb][e];
            seen |= !hidden;
          }
        }
        return true;
      };
      auto largest = [&]() __attribute__((always_inline)) {
        float x = -INFINITY;
#pragma unroll
        for (int tb = 0; tb < NB; ++tb)
#pragma unroll
          for (int e = 0; e < 16; ++e) x = fmaxf(x, s[tb][e]);
        return x;
      };
      auto scaled = [&](float x) { return max_of_halves(x) * c2 - weight_shift<VT>(); };
      float mx = -INFINITY;
      if (n > 0) {
        if constexpr (Move::kInRegisters) mv.template next<KEEP>(t_lo);
        for (int i = -2; i < (wave_on ? 0 : n); ++i) {
          move(i);
#pragma unroll
          for (int p = 0; p < 24; ++p) load(p);
          if (wave_on && i == -1) {
            // q is waited for here, not before the first product of every tile, where that
            // would be for the next tiles' loads as well
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qb[ks]));
#pragma unroll
            for (int tb = 0; tb < NB; ++tb) {
#pragma unroll
              for (int e = 0; e < 16; ++e) s[tb][e] = 0.0f;
#pragma unroll
              for (int ks = 0; ks < KS; ++ks)
                s[tb] = mfma32<QT>(read_k(k_wave, tb * KS + ks), qb[ks], s[tb]);
            }
            uint32_t marked[NB];
            get_marks(marked);
            hide(0, marked);
            mx = scaled(largest());
          }
          mv.settle(marks[3]);
          __syncthreads();
        }
        // The inner loop changes the accumulators by products alone: with a branch in it that
        // scales them they were held, and moved, twice.  A wave that meets scores too
        // large for its maximum leaves it.
        for (int i = 0; wave_on && i < n;) {
          const float m_new = fmaxf(m_run, mx);
          // a row with every score so far -inf keeps l = 0 and acc = 0
          const float m_use = m_new == -INFINITY ? 0.0f : m_new;
          const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
          l_run *= alpha;
#pragma unroll
          for (int d = 0; d < DN; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[d][e] *= alpha;
          m_run = m_new;
          bool over;
          do {
            move(i);
            uint32_t marked[NB];
            get_marks(marked);
            const uint32_t k_rd = k_wave + (~i & 1) * TB, v_rd = v_wave + (i & 1) * TB;
            // weights of 16 tokens each, 8 per lane: both terms
            u32x4 pb[2][2 * NB];
            float l2 = 0.0f;
            // weights of elements 2 e, 2 e + 1 of block tb
            auto weigh = [&](int tb, int e) __attribute__((always_inline)) {
              const float p0 = __builtin_amdgcn_exp2f(s[tb][2 * e] * c2 - m_use);
              const float p1 = __builtin_amdgcn_exp2f(s[tb][2 * e + 1] * c2 - m_use);
              l_run += p0;
              l2 += p1;
              const auto [hi, lo] = two_terms<VT>(p0, p1);
              pb[0][2 * tb + e / 4][e % 4] = hi;
              pb[1][2 * tb + e / 4][e % 4] = lo;
            };
            // The order of the products and of what is done in their shadow: weights of the
            // first 32 tokens; scores of the next tile's first 32 over them, beside the
            // other weights; the other scores, beside the first reads of V; then V's
            // products, beside the maximum.  Reads are four products and more ahead.
            constexpr int AHEAD = 4, VR = DN > 2 ? DN : 2, VW = DN > 1 ? 2 : 1;
            // V fragment p of the tile: 16 tokens p / DN, dims 32 (p % DN) ..
            auto read_v_of = [&](int p) __attribute__((always_inline)) {
              return read_v((v_rd ^ (64 * (p % DN))) + 16 * (p / DN) * RB);
            };
            u32x4 kf[AHEAD], vf[VR];
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) kf[q] = read_k(k_rd, q);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              load(e);
              weigh(0, e);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int q = 0; q < QN; ++q) {
              const int tb = q / KS, ks = q % KS;
              if (ks == 0)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[tb][e] = 0.0f;
              s[tb] = mfma32<QT>(kf[q % AHEAD], qb[ks], s[tb]);
              if (q + AHEAD < QN) kf[q % AHEAD] = read_k(k_rd, q + AHEAD);
              load(8 + q);
              if (tb + 1 < NB)
#pragma unroll
                for (int e = ks * 8 / KS; e < (ks + 1) * 8 / KS; ++e) weigh(tb + 1, e);
              else if (ks < VR)
                vf[ks] = read_v_of(ks);
              __builtin_amdgcn_sched_barrier(0);
            }
            float big = -INFINITY;
#pragma unroll
            for (int q = 0; q < 2 * PN; ++q) {
              // both terms of VW fragments in turn: no product waits for the one before it
              const int p = q / (2 * VW) * VW + q % VW, st = p / DN, d = p % DN, term = q / VW % 2;
              acc[d] = mfma32<VT>(vf[p % VR], pb[term][st], acc[d]);
              if (term == 1 && p + VR < PN) vf[p % VR] = read_v_of(p + VR);
#pragma unroll
              for (int e = q * (8 * NB) / PN; e < (q + 1) * (8 * NB) / PN; ++e)
                big = fmaxf(big, s[e / 16][e % 16]);
              __builtin_amdgcn_sched_barrier(0);
            }
            // (not put off to where they are used: the scores would be held twice)
            asm volatile("" : "+v"(big), "+v"(l_run), "+v"(l2));
            l_run += l2;
            // (behind the last tile the scores are of what lies in LDS, and not used)
            ++i;
            over = false;
            if (i < n) {
              if (hide(i, marked)) big = largest();
              mx = scaled(big);
              over = __any(mx > m_run + kSlack);
            }
            mv.settle(marks[3]);
            __syncthreads();
          } while (i < n && !over);
        }
      }
      const bool wild_seen = n > 0 && marks[3][0] != 0;

      float l = l_run + __shfl_xor(l_run, 32);
      seen |= __shfl_xor((int)seen, 32) != 0;
      if constexpr (TS > 1) {  // the tokens' parts become one in the first of their waves
        static_assert(TS == 2, "two parts");
        f32x4* x = reinterpret_cast<f32x4*>(k_lds) + (cg + dim / 32 / DN * CG) * (DN * 256) + lane;
        float* y = reinterpret_cast<float*>(v_lds) + (cg + dim / 32 / DN * CG) * 192 + lane;
        if (tok) {
#pragma unroll
          for (int i = 0; i < 4 * DN; ++i)
            x[64 * i] = f32x4{acc[i / 4][4 * (i % 4)], acc[i / 4][4 * (i % 4) + 1],
                              acc[i / 4][4 * (i % 4) + 2], acc[i / 4][4 * (i % 4) + 3]};
          y[0] = m_run;
          y[64] = l;
          y[128] = seen;
        }
        __syncthreads();
        if (!tok) {
          const float m = fmaxf(m_run, y[0]), m_use = m == -INFINITY ? 0.0f : m;
          const float f0 = __builtin_amdgcn_exp2f(m_run - m_use);
          const float f1 = __builtin_amdgcn_exp2f(y[0] - m_use);
          l = l * f0 + y[64] * f1;
          seen |= y[128] != 0.0f;
          m_run = m;
#pragma unroll
          for (int i = 0; i < 4 * DN; ++i) {
            const f32x4 o = x[64 * i];
#pragma unroll
            for (int n = 0; n < 4; ++n)
              acc[i / 4][4 * (i % 4) + n] = acc[i / 4][4 * (i % 4) + n] * f0 + o[n] * f1;
          }
        }
      }
      const bool whole = begins && t_hi == e;
      if (!whole && begins) {
        const int64_t reach = start + (int64_t)(e + BT - 1) / BT * unit - 1;
        cut.more = (int32_t)(reach / sh.length - sh.index);
        cut.share = (int32_t)sh.index;
        cut.row0 = sq.row0 + row_lo;
        cut.cols = cols;
        cut.head = head;
      }
      if (col < cols && tok == 0) {
        if (whole) {
          // no token: zeros; every score -inf: 0 / 0 = NaN, as softmax gives
          const float f = seen ? a.v_scale / l : 0.0f;
          const int64_t o = ((int64_t)qrow * a.num_q_heads + qh) * D + dim;
#pragma unroll
          for (int d = 0; d < DN; ++d)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              f32x4 x = {acc[d][4 * n], acc[d][4 * n + 1], acc[d][4 * n + 2], acc[d][4 * n + 3]};
              store4(a.out, QT, o + 32 * d + 8 * n + 4 * h, x * f);
            }
        } else {
          float* p = a.part + ((sh.index * 2 + begins) * kRows + col) * (D + kPartPad) + dim;
#pragma unroll
          for (int d = 0; d < DN; ++d)
#pragma unroll
            for (int n = 0; n < 4; ++n)
              *reinterpret_cast<f32x4*>(p + 32 * d + 8 * n + 4 * h) =
                  f32x4{acc[d][4 * n], acc[d][4 * n + 1], acc[d][4 * n + 2], acc[d][4 * n + 3]};
          if (h == 0 && dim == 0) {
            p[D] = m_run;
            p[D + 1] = seen && l == 0.0f ? -1.0f : l;  // -1: tokens, all of them -inf
          }
        }
        if (wild_seen) {
          // V elements that are not finite were multiplied as 0: what they make of the rows
          // that see their tokens.  (Of those in unchecked tiles nothing changes.)
          const uint8_t* q = a.q + (int64_t)qrow * a.q_row + qh * a.q_head;
          for (int t = max(t_lo, pos0 + 1 - BT); t <= last; ++t) {
            if (!mv.there(t)) continue;
            float p = 0.0f;
            bool known = false;
            for (int i = 0; i < 16 * DN; ++i) {  // the dims that this lane has stored
              const int d = dim + i / 4 * 8 + 4 * h + i % 4;
              const float v = mv.v_elem(t, d);
              if (fabsf(v) < INFINITY) continue;
              if (!known) {
                float x = 0.0f;
                for (int n = 0; n < D; ++n) x += kv_elem<QT>(q + 2 * n) * mv.k_elem(t, n);
                p = __builtin_amdgcn_exp2f(x * c2 - m_run);
                known = true;
              }
              if (whole) {
                uint16_t* o = a.out + ((int64_t)qrow * a.num_q_heads + qh) * D + d;
                const float x = kv_elem<QT>(reinterpret_cast<const uint8_t*>(o));
                *o = (uint16_t)pair16<QT>(x + p * v * a.v_scale, 0.0f);
              } else {
                float* o = a.part + ((sh.index * 2 + begins) * kRows + col) * (D + kPartPad) + d;
                *o += p * v;
              }
            }
          }
        }
      }
    };
    if (begins || t_lo < e) {
      const int used = __builtin_amdgcn_readfirstlane(cols);
      if (used > 64)
        piece(std::integral_constant<int, 4>{});
      else if (used > 32)
        piece(std::integral_constant<int, 2>{});
      else
        piece(std::integral_constant<int, 1>{});
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
  if (bad_seen && lane == 0 && a.err_flag) atomicOr(a.err_flag, AMF_ERRFLAG_BLOCK_RANGE);
}

// out = v_scale sum_k f_k acc_k / sum_k f_k l_k, f_k = 2^(m_k - M), over the pieces of a
// cut tile; D / 4 lanes a column, kMergeParts workgroups a tile.  Bound by the pieces' bytes,
// up to 69 MB: 15 to 22 us at 128 columns, 6 at few (eight parts, and accumulators loaded
// with the statistics, gained nothing).
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
// 256, caches or outputs that are not 16-byte aligned and groups of more than kRows heads;
// every K and V element is read again for each row and head, and a wave's tokens follow each
// other: 32 / 8 heads of 96, prompt of 2048 rows 3.9 ms (INT4 7.8; of 128 on the tiles 0.09), 16
// single rows of 2048 tokens 1.2 ms (0.05); fp32 heads of 128 7.4 and 1.4.
template <int KV, int QT>
__global__ __launch_bounds__(kThreads) void rows_general_kernel(RowsArgs a) {
  __shared__ float q_lds[kWaves][kMaxDim];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, D = a.head_dim;
  const int64_t block = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int64_t id = block * kWaves + wave;
  const int64_t row = id / a.num_q_heads;
  const int qh = (int)(id - row * a.num_q_heads), head = qh / a.group;
  int seq = -1;
  int64_t ctx = 0, pos = -1;
  int flags = 0;
  if (block == 0 && a.err_flag) {  // what only the sequences show
    for (int s = threadIdx.x; s < a.num_seqs; s += kThreads) get_seq(a, s, &flags);
    if (flags) atomicOr(a.err_flag, flags);
    flags = 0;
  }
  if (row < a.n_rows && a.num_seqs > 0) {
    auto holds = [&](int s) {
      const int64_t first = a.query_start[s], end = a.query_start[s + 1];
      return first >= 0 && first <= row && row < end && end <= a.n_rows;
    };
    int lo = 0, hi = a.num_seqs;  // the last sequence that starts at or before the row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.query_start[mid] <= row) lo = mid; else hi = mid;
    }
    if (holds(lo)) seq = lo;
    // a row of nobody, or of a sequence beside a malformed one
    for (int s0 = 0; seq < 0 && s0 < a.num_seqs; s0 += 64) {
      const uint64_t on = __ballot(s0 + lane < a.num_seqs && holds(s0 + lane));
      if (on) seq = s0 + __ffsll((unsigned long long)on) - 1;
    }
    if (seq >= 0) {
      ctx = max(a.context_lens[seq], 0);
      pos = ctx - (a.query_start[seq + 1] - row);
    }
  }
  if (seq >= 0) {
    const uint8_t* q = a.q + row * a.q_row + qh * a.q_head;
    for (int d = lane; d < D; d += 64) q_lds[wave][d] = kv_elem<QT>(q + d * elem_bytes<QT>());
  }
  __syncthreads();
  if (seq < 0) return;
  const int64_t cap = (int64_t)a.table_pages * a.block_size;
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
#define AMF_ROWS(DD)                                                                  \
  if constexpr (KV == kInt4) {                                                        \
    rows_kernel<QT, KV, DD, true><<<grid, kThreads, 0, st>>>(a);                      \
  } else {                                                                            \
    a.by16 ? rows_kernel<QT, KV, DD, true><<<grid, kThreads, 0, st>>>(a)              \
           : rows_kernel<QT, KV, DD, false><<<grid, kThreads, 0, st>>>(a);            \
  }                                                                                   \
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
  // (2^26 rows of one head are 2^32 threads, one more than a dimension of a grid holds)
  const int64_t blocks = (a.n_rows * a.num_q_heads + kWaves - 1) / kWaves;
  const int64_t x = std::min<int64_t>(blocks, 1 << 20);
  rows_general_kernel<KV, QT>
      <<<dim3((unsigned)x, (unsigned)((blocks + x - 1) / x)), kThreads, 0, st>>>(a);
}

// Shares of a call: of kMinShare, that the longest contexts of the tables could fill.
int call_shares(int64_t n_rows, int num_seqs, int table_pages, int block_size, int num_q_heads,
                int num_kv_heads, int D) {
  const int tile_rows = std::max(1, kRows / (num_q_heads / num_kv_heads));
  const int64_t tiles = n_rows / tile_rows + std::min<int64_t>(num_seqs, n_rows);
  const int64_t cap = kWide * ((int64_t)table_pages * block_size + tile_rows) + kTileCost;
  // a workgroup's registers and LDS: two to a CU, at the largest head_dim one
  const int64_t fit = D == 256 ? kMaxShares / 2 : kMaxShares;
  const int64_t most = (tiles * num_kv_heads * cap + kMinShare - 1) / kMinShare;
  // whole rounds of the XCDs
  return (int)std::min<int64_t>(fit, (most + kXcds - 1) / kXcds * kXcds);
}

int64_t share_bytes(int D) {
  return (int64_t)sizeof(Cut) + part_floats(D) * (int64_t)sizeof(float);
}

int check(const char* who, const RowsArgs& a, int32_t q_dtype, const void* workspace,
          int64_t workspace_bytes) {
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
  const int64_t need = amf_paged_attn_rows_call_bytes(a.n_rows, a.num_seqs, a.table_pages,
                                                      a.block_size, a.num_q_heads, a.num_kv_heads,
                                                      a.head_dim);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)
    return fail(AMF_ERR_WORKSPACE, "%s: workspace of %lld bytes (16-byte aligned) needed, got %lld",
                who, (long long)need, (long long)workspace_bytes);
  return AMF_OK;
}

void finish_args(RowsArgs* a, void* workspace, float softmax_scale, float k_scale) {
  a->group = a->num_q_heads / a->num_kv_heads;
  a->tile_rows = std::max(1, kRows / a->group);
  const int b = a->block_size;
  a->block_shift = __builtin_ctz((unsigned)b);
  a->by16 = b % 16 == 0 && (b & (b - 1)) == 0 && a->page_stride >= 0 && a->token_stride >= 0 &&
            a->page_stride % 16 == 0 && a->token_stride % 16 == 0 &&
            a->token_stride < ((int64_t)1 << 27) && a->page_stride < ((int64_t)1 << 35) &&
            (a->pool_pages - 1) * (a->page_stride / 16) + b * (a->token_stride / 16) <
                ((int64_t)1 << 32);
  a->page_units = (uint32_t)(a->page_stride / 16);
  a->token_units = (uint32_t)(a->token_stride / 16);
  const float scale =
      softmax_scale > 0.0f ? softmax_scale : 1.0f / __builtin_sqrtf((float)a->head_dim);
  a->score_scale = scale * k_scale * kLog2e;
  a->shares = call_shares(a->n_rows, a->num_seqs, a->table_pages, b, a->num_q_heads,
                          a->num_kv_heads, a->head_dim);
  a->cuts = static_cast<Cut*>(workspace);
  a->part = reinterpret_cast<float*>(a->cuts + a->shares);
}

}  // namespace

extern "C" int64_t amf_paged_attn_rows_workspace_bytes(int32_t num_q_heads, int32_t num_kv_heads,
                                                       int32_t head_dim) {
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || head_dim <= 0 ||
      head_dim > kMaxDim)
    return 0;
  if (!matrix_dim(head_dim)) return 16;
  return kMaxShares * share_bytes(head_dim);
}

extern "C" int64_t amf_paged_attn_rows_call_bytes(int64_t n_rows, int32_t num_seqs,
                                                  int32_t table_pages, int32_t block_size,
                                                  int32_t num_q_heads, int32_t num_kv_heads,
                                                  int32_t head_dim) {
  const int64_t most =
      amf_paged_attn_rows_workspace_bytes(num_q_heads, num_kv_heads, head_dim);
  if (most <= 16 || n_rows < 0 || num_seqs < 0 || table_pages < 0 || block_size <= 0 ||
      n_rows > ((int64_t)1 << 26) / num_q_heads ||
      (int64_t)table_pages * block_size > kMaxContext)
    return most;
  return std::max<int64_t>(16, call_shares(n_rows, num_seqs, table_pages, block_size, num_q_heads,
                                           num_kv_heads, head_dim) *
                                   share_bytes(head_dim));
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
  a.pages = (uint32_t)std::min<int64_t>(std::max<int64_t>(pool_pages, 0), 1ll << 31);
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
  const int rc = check(who, a, q_dtype, workspace, workspace_bytes);
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
  a.pages = (uint32_t)std::min<int64_t>(std::max<int64_t>(pool_pages, 0), 1ll << 31);
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
  const int rc = check(who, a, q_dtype, workspace, workspace_bytes);
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

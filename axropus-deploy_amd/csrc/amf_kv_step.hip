// amf_kv_step.hip - the rows of a step: rotary positions of queries and keys,
// keys and values written at their slots into a cache (16-bit, fp32, FP8) or an
// INT4 pool, and rows read back by their slots.
//
// Rotation.  Pair i of a head turns by the angle p f_i (p the row's position):
//   (a, b) -> factor * (a cos - b sin, b cos + a sin).
// Positions reach 10^6 and more, where an angle in fp32 is off by 0.03 and more,
// so angle, sine and cosine are 64-bit, once per (row, pair) into LDS, and the
// heads of the row share them.  The products are 64-bit too (three operations a
// value, hidden behind the loads) and rounded to fp32 and from there to the
// type: a key that is quantised afterwards then has the bits that an unquantised
// cache of its type would hold, and the same codes as a page saved from there.
//
// All kernels move bytes: each value is read once and written once, in chunks of
// 8 elements where addresses allow (else one at a time), and the rest is hidden.  Steps of
// many rows are bound by HBM (10500 rows of 18 heads of 256, 64 dims rotated: 40 us, 4.9
// TB/s; 11000 rows of 64 + 8 heads of 128, rotated, K and V written as FP8: 86 us, 4.9; 6700
// rows into an INT4 pool 44 us, 52000 rows read from one 64, 4.4; 24000 FP8 rows read 27,
// 5.5), steps of one row a sequence by the latency of a launch (4 to 10 us).  The angles of a
// tile of rows are one set-up (a load, a sine, a barrier): with four times as many
// workgroups, of a quarter of the items each, the 10500 rows took 54 us.
#include <algorithm>

#include "amf_int4_asym.h"
#include "amf_internal.h"
#include "amf_kernel_util.h"
#include "amf_paged.h"

namespace {

using namespace amf;

constexpr int kThreads = 256;

// Division by a number that a launch has once: the quotient from floor((2^32 - 1) / d) is
// one too small at most (n below 2^31).
struct Div {
  uint32_t d, m;
  Div() = default;
  explicit Div(uint32_t x) : d(x), m(x ? 0xFFFFFFFFu / x : 0) {}
  __device__ __forceinline__ uint32_t operator()(uint32_t n, uint32_t& rest) const {
    uint32_t q = __umulhi(n, m);
    rest = n - q * d;
    if (rest >= d) {
      ++q;
      rest -= d;
    }
    return q;
  }
};

struct alignas(16) Turn {
  double c, s;
};

// Rows [row][head][dim], strides in bytes, dims contiguous.
struct Rows {
  uint8_t* p;
  int64_t row, head;
  int heads;
};

struct RotaryArgs {
  const int64_t* positions;
  const double* freqs;
  double factor;
  int pairs;  // 0: nothing is rotated
  bool interleaved;
};

// Where slots lie in a cache, strides in bytes.
struct CacheAt {
  uint8_t* k;
  uint8_t* v;
  int64_t page, token, head;
  int64_t pool_slots;
  int block;
  float k_scale, v_scale;
};

__device__ __forceinline__ void fill_turns(const RotaryArgs& a, int64_t row0, int rows, Turn* tab) {
  for (int i = threadIdx.x; i < rows * a.pairs; i += kThreads) {
    const int r = i / a.pairs, p = i - r * a.pairs;
    double s, c;
    sincos((double)a.positions[row0 + r] * a.freqs[p], &s, &c);
    tab[i] = {c * a.factor, s * a.factor};
  }
}

__device__ __forceinline__ void turn(const Turn& t, float& a, float& b) {
  const double x = a, y = b;
  a = (float)__builtin_fma(x, t.c, -(y * t.s));
  b = (float)__builtin_fma(y, t.c, x * t.s);
}

// One element of type DT.
template <int DT>
__device__ __forceinline__ void put_elem(uint8_t* p, float x) {
  if constexpr (DT == AMF_DTYPE_F32)
    *reinterpret_cast<float*>(p) = x;
  else
    *reinterpret_cast<uint16_t*>(p) = (uint16_t)pack2<DT == AMF_DTYPE_BF16>(x, 0.0f);
}

template <int DT>
__device__ __forceinline__ float round_to(float x) {
  if constexpr (DT == AMF_DTYPE_F32) return x;
  constexpr bool B = DT == AMF_DTYPE_BF16;
  return half_lo<B>(pack2<B>(x, 0.0f));
}

// Eight elements of type DT at p, which are read again soon (cached stores).
template <int DT>
__device__ __forceinline__ void put8(uint8_t* p, const float* x) {
  if constexpr (DT == AMF_DTYPE_F32) {
    reinterpret_cast<f32x4*>(p)[0] = f32x4{x[0], x[1], x[2], x[3]};
    reinterpret_cast<f32x4*>(p)[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    *reinterpret_cast<u32x4*>(p) = pack8<DT == AMF_DTYPE_BF16>(x);
  }
}

// x / scale on e4m3's range; a NaN stays one.
__device__ __forceinline__ float on_e4m3(float x, float scale) {
  const float y = x / scale;
  return y != y ? y : fminf(fmaxf(y, -448.0f), 448.0f);
}

// N elements (8, or 1 of x) rounded to DT, to p: of type DT, or as FP8 codes.
template <int DT, bool FP8, bool VEC>
__device__ __forceinline__ void emit(uint8_t* p, const float* x, float scale) {
  if constexpr (!FP8) {
    if constexpr (VEC)
      put8<DT>(p, x);
    else
      put_elem<DT>(p, x[0]);
  } else if constexpr (VEC) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = on_e4m3(round_to<DT>(x[i]), scale);
    *reinterpret_cast<u32x2*>(p) = u32x2{f32x4_to_e4m3(y), f32x4_to_e4m3(y + 4)};
  } else {
    const float y[4] = {on_e4m3(round_to<DT>(x[0]), scale), 0.0f, 0.0f, 0.0f};
    *p = (uint8_t)f32x4_to_e4m3(y);
  }
}

// Items of a head: pairs (VEC: 8 pairs, else one), and what is not rotated (VEC: 8
// elements, else one).  A kernel takes the pairs of all heads first, so that the lanes of a
// wave do the same (rotating 64 of 256 dims, a third of the time went to waves that did
// both).
struct Items {
  Div rot, rest;
  Items() = default;
  Items(int dim, int pairs, bool vec)
      : rot(pairs / (vec ? 8 : 1)), rest((dim - 2 * pairs) / (vec ? 8 : 1)) {}
};

// A chunk of a row as it lies in memory: 8 elements (VEC) or one.
template <int DT, bool VEC>
struct Chunk {
  u32x4 w[VEC && DT == AMF_DTYPE_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (!VEC) {
      w[0][0] = f2u(kv_elem<DT>(p));
    } else {
      w[0] = reinterpret_cast<const u32x4*>(p)[0];
      if constexpr (DT == AMF_DTYPE_F32) w[1] = reinterpret_cast<const u32x4*>(p)[1];
    }
  }
  __device__ __forceinline__ void get(float* x) const {
    if constexpr (!VEC) {
      x[0] = u2f(w[0][0]);
    } else if constexpr (DT == AMF_DTYPE_F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = u2f(w[i / 4][i % 4]);
    } else {
      unpack8<DT == AMF_DTYPE_BF16>(w[0], x);
    }
  }
};

// A head of a row; kind: of q (0), k (1) or v (2), or a number of the caller's.
struct Head {
  int kind;
  uint32_t r, h;
  const uint8_t* p;
};

// Chunks are loaded kAhead, or pairs of them kAhead / 2, at a time before the first is stored
// (stores may be to what is read, for all that the compiler knows; one at a time, too few
// bytes are on their way).
constexpr int kAhead = 4;

// The pairs of n heads: find(head) gives its Head, put(Head, dim, values) takes the results.
template <int DT, bool VEC, class Find, class Put>
__device__ __forceinline__ void each_pair(const RotaryArgs& rot, const Items& items, uint32_t n,
                                          uint32_t at, uint32_t step, const Turn* turns,
                                          Find find, Put put) {
  constexpr int B = kAhead / 2, N = VEC ? 8 : 1, ES = elem_bytes<DT>();
  const uint32_t all = n * items.rot.d;
  const int second = rot.interleaved ? N : rot.pairs;
  for (uint32_t i0 = at; i0 < all; i0 += B * step) {
    Chunk<DT, VEC> x[B], y[B];
    Head head[B];
    uint32_t it[B];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      if (i0 - threadIdx.x + j * step >= all) break;
      head[j] = find(items.rot(min(i0 + j * step, all - 1), it[j]));
      const uint8_t* p = head[j].p + it[j] * (rot.interleaved ? 2 * N : N) * ES;
      x[j].load(p);
      y[j].load(p + second * ES);
    }
#pragma unroll
    for (int j = 0; j < B; ++j) {
      if (i0 + j * step >= all) break;
      const Turn* t = turns + head[j].r * rot.pairs + it[j] * N;
      float a[8], b[8];
      x[j].get(a);
      y[j].get(b);
      if (VEC && rot.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          turn(t[i], a[2 * i], a[2 * i + 1]);
          turn(t[4 + i], b[2 * i], b[2 * i + 1]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) turn(t[i], a[i], b[i]);
      }
      const int dim = it[j] * (rot.interleaved ? 2 * N : N);
      put(head[j], dim, a);
      put(head[j], dim + second, b);
    }
  }
}

// `all` chunks that are not rotated: find(i, dim) gives chunk i's head and first dim.
template <int DT, bool VEC, class Find, class Put>
__device__ __forceinline__ void each_chunk(uint32_t all, uint32_t at, uint32_t step, Find find,
                                           Put put) {
  for (uint32_t i0 = at; i0 < all; i0 += kAhead * step) {
    Chunk<DT, VEC> x[kAhead];
    Head head[kAhead];
    uint32_t dim[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 - threadIdx.x + j * step >= all) break;
      head[j] = find(min(i0 + j * step, all - 1), dim[j]);
      x[j].load(head[j].p + dim[j] * elem_bytes<DT>());
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + j * step >= all) break;
      float a[8];
      x[j].get(a);
      put(head[j], dim[j], a);
    }
  }
}

struct StepArgs {
  Rows q, k, v;       // read
  Rows q_out, k_out;  // written (k_out where there is no cache)
  CacheAt cache;
  RotaryArgs rot;
  const int64_t* slots;
  int32_t* err_flag;
  int64_t n_rows;
  int dim;
  int tile;  // rows of a workgroup, at most kTile
  Items items, v_items;  // of heads of q and k, and of v
  Div q_heads, k_heads, v_heads;
};
constexpr int kTile = 8;

enum { TO_ROWS, TO_CACHE, TO_FP8 };

// Workgroup (x, y): rows tile x .. of the step, every gridDim.y-th of their items.
template <int DT, int TO, bool VEC>
__global__ __launch_bounds__(kThreads) void step_kernel(StepArgs a) {
  extern __shared__ __attribute__((aligned(16))) Turn turns[];
  __shared__ int64_t at[kTile];  // the rows' places in the cache, -1: none
  const int64_t row0 = (int64_t)blockIdx.x * a.tile;
  const int rows = (int)min((int64_t)a.tile, a.n_rows - row0);
  fill_turns(a.rot, row0, rows, turns);
  if (TO != TO_ROWS && (int)threadIdx.x < rows) {
    const int64_t s = a.slots[row0 + threadIdx.x];
    const bool in = s >= 0 && s < a.cache.pool_slots;
    at[threadIdx.x] = in ? s / a.cache.block * a.cache.page + s % a.cache.block * a.cache.token
                         : -1;
    if (s >= a.cache.pool_slots && a.err_flag && blockIdx.y == 0)
      atomicOr(a.err_flag, AMF_ERRFLAG_BLOCK_RANGE);
  }
  __syncthreads();
  constexpr int ES = elem_bytes<DT>(), OS = TO == TO_FP8 ? 1 : ES, N = VEC ? 8 : 1;
  const int pairs = a.rot.pairs;
  const uint32_t hq = rows * a.q.heads, hk = rows * a.k.heads;
  const uint32_t first = blockIdx.y * kThreads + threadIdx.x, step = gridDim.y * kThreads;
  auto find = [&](uint32_t n) {  // heads of q, then of k
    Head x;
    x.kind = n >= hq;
    const Div heads = x.kind ? a.k_heads : a.q_heads;
    x.r = heads(x.kind ? n - hq : n, x.h);
    const Rows& from = x.kind ? a.k : a.q;
    x.p = from.p + (row0 + x.r) * from.row + x.h * from.head;
    return x;
  };
  auto put = [&](const Head& x, int dim, const float* v) {
    if (TO != TO_ROWS && x.kind) {
      if (at[x.r] < 0) return;
      uint8_t* o = (x.kind == 1 ? a.cache.k : a.cache.v) + at[x.r] + x.h * a.cache.head;
      emit<DT, TO == TO_FP8, VEC>(o + dim * OS, v, x.kind == 1 ? a.cache.k_scale : a.cache.v_scale);
    } else {
      const Rows& to = x.kind ? a.k_out : a.q_out;
      emit<DT, false, VEC>(to.p + (row0 + x.r) * to.row + x.h * to.head + dim * ES, v, 1.0f);
    }
  };
  each_pair<DT, VEC>(a.rot, a.items, hq + hk, first, step, turns, find, put);
  const uint32_t rest = (hq + hk) * a.items.rest.d;
  const uint32_t nv = TO == TO_ROWS ? 0 : rows * a.v.heads * a.v_items.rest.d;
  each_chunk<DT, VEC>(
      rest + nv, first, step,
      [&](uint32_t i, uint32_t& dim) {
        uint32_t c;
        Head x;
        if (i < rest) {
          x = find(a.items.rest(i, c));
          dim = 2 * pairs + c * N;
        } else {
          const uint32_t n = a.v_items.rest(i - rest, c);
          x.kind = 2;
          x.r = a.v_heads(n, x.h);
          x.p = a.v.p + (row0 + x.r) * a.v.row + x.h * a.v.head;
          dim = c * N;
        }
        return x;
      },
      put);
}

// ------------------------------------------------------------ INT4 pools ----

struct PoolAt {
  uint8_t* kc;
  uint32_t* kp;
  uint8_t* vc;
  uint32_t* vp;
  int64_t pool_slots;
};

// The V codes of a pool keep the eight tokens of half a page in one word per
// dim.  Rows of a step that follow each other in such a half are a run, which
// one wave takes: the tokens in the low three bits of the lane, chunks of 8 dims
// in the others.  A workgroup serves the runs that begin in its kTile rows (they
// end at most 7 rows later).
struct Runs {
  uint32_t starts, cont;  // bit e: row row0 - 1 + e starts / goes on with a run
  __device__ __forceinline__ int count() const { return __popc(starts); }
  // The entry at which run n starts.
  __device__ __forceinline__ int entry(int n) const {
    uint32_t m = starts;
    for (; n > 0; --n) m &= m - 1;
    return __ffs(m) - 1;
  }
  __device__ __forceinline__ int length(int e) const { return __ffs(~(cont >> (e + 1))); }
};
constexpr int kEntries = 2 * kTile;

// Slots of rows row0 - 1 .. row0 + 14 into `slot` (-1: none); wave 0 flags.
__device__ __forceinline__ void load_slots(const int64_t* slots, int64_t row0, int64_t n_rows,
                                           int64_t pool_slots, int64_t* slot, int32_t* err) {
  if (threadIdx.x >= kEntries) return;
  const int64_t row = row0 - 1 + threadIdx.x;
  int64_t s = row >= 0 && row < n_rows ? slots[row] : -1;
  if (s >= pool_slots) {
    s = -1;
    if (err) atomicOr(err, AMF_ERRFLAG_BLOCK_RANGE);
  }
  slot[threadIdx.x] = s < 0 ? -1 : s;
}

__device__ __forceinline__ Runs find_runs(const int64_t* slot, int64_t row0) {
  const int e = threadIdx.x & 63;
  bool cont = false, start = false;
  if (e > 0 && e < kEntries && slot[e] >= 0) {
    cont = slot[e] == slot[e - 1] + 1 && slot[e] % 8 != 0;
    start = e <= kTile && !cont;
  }
  Runs r;
  r.starts = (uint32_t)__ballot(start);
  r.cont = (uint32_t)__ballot(cont);
  return r;
}

// w of the eight lanes that differ in their low three bits, as an 8 x 8 matrix
// of nibbles, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t w) {
  const int t = threadIdx.x & 7;
#pragma unroll
  for (int b = 1; b < 8; b <<= 1) {
    const uint32_t m = b == 1 ? 0x0F0F0F0Fu : b == 2 ? 0x00FF00FFu : 0x0000FFFFu;
    const uint32_t p = __shfl_xor(w, b);
    w = t & b ? (w & ~m) | ((p >> (4 * b)) & m) : (w & m) | ((p & m) << (4 * b));
  }
  return w;
}

struct PoolStepArgs {
  Rows q, k, v, q_out;
  PoolAt pool;
  RotaryArgs rot;
  const int64_t* slots;
  int32_t* err_flag;
  int64_t n_rows;
  int dim;
  int kv_blocks;   // workgroups of a row tile that take KV heads (the others take q)
  int head_block;  // KV heads of such a workgroup
  Items items;     // of a head
  Div q_heads;
};

// Codes of 8 of a group's values, from the group's extremes.
__device__ __forceinline__ uint32_t asym_codes8(const float* x, float mn, float mx,
                                                uint32_t* param) {
  AsymParams p;
  p.mn = mn;
  p.scale = fmaxf(mx - mn, 1e-8f) / kAsymLevels;
  p.rscale = 1.0f / p.scale;
  *param = asym_param_word(p);
  uint32_t w = 0;
#pragma unroll
  for (int n = 0; n < 8; ++n) w = asym_insert<64>(w, n, x[n], p);
  return w;
}

__device__ __forceinline__ void min_max8(const float* x, float& mn, float& mx) {
  mn = mx = x[0];
#pragma unroll
  for (int n = 1; n < 8; ++n) {
    mn = fminf(mn, x[n]);
    mx = fmaxf(mx, x[n]);
  }
}

template <int DT, bool VEC>
__global__ __launch_bounds__(kThreads) void int4_step_kernel(PoolStepArgs a) {
  extern __shared__ __attribute__((aligned(16))) Turn turns[];
  __shared__ int64_t slot[kEntries];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row0 = (int64_t)blockIdx.x * kTile;
  const int rows = (int)min((int64_t)kTile, a.n_rows - row0);
  const int D = a.dim, pairs = a.rot.pairs;
  constexpr int ES = elem_bytes<DT>();
  fill_turns(a.rot, row0, rows, turns);
  if ((int)blockIdx.y >= a.kv_blocks) {
    __syncthreads();
    const uint32_t hq = rows * a.q.heads;
    const uint32_t first = (blockIdx.y - a.kv_blocks) * kThreads + tid;
    const uint32_t step = (gridDim.y - a.kv_blocks) * kThreads;
    auto find = [&](uint32_t n) {
      Head x;
      x.kind = 0;
      x.r = a.q_heads(n, x.h);
      x.p = a.q.p + (row0 + x.r) * a.q.row + x.h * a.q.head;
      return x;
    };
    auto put = [&](const Head& x, int dim, const float* v) {
      uint8_t* o = a.q_out.p + (row0 + x.r) * a.q_out.row + x.h * a.q_out.head;
      emit<DT, false, VEC>(o + dim * ES, v, 1.0f);
    };
    each_pair<DT, VEC>(a.rot, a.items, hq, first, step, turns, find, put);
    each_chunk<DT, VEC>(
        hq * a.items.rest.d, first, step,
        [&](uint32_t i, uint32_t& dim) {
          const uint32_t n = a.items.rest(i, dim);
          dim = 2 * pairs + dim * (VEC ? 8 : 1);
          return find(n);
        },
        put);
    return;
  }
  float* kx = reinterpret_cast<float*>(turns + kTile * pairs);  // [rows][heads][dim]
  load_slots(a.slots, row0, a.n_rows, a.pool.pool_slots, slot,
             blockIdx.y == 0 ? a.err_flag : nullptr);
  __syncthreads();
  const int H = a.k.heads, h0 = blockIdx.y * a.head_block, nh = min(a.head_block, H - h0);
  const int G = D / 32, C = D / 8;
  auto find = [&](uint32_t n) {
    Head x;
    x.kind = (int)n;
    x.r = n / nh;
    x.h = h0 + (n - x.r * nh);
    x.p = a.k.p + (row0 + x.r) * a.k.row + x.h * a.k.head;
    return x;
  };
  auto put = [&](const Head& x, int dim, const float* v) {
#pragma unroll
    for (int n = 0; n < (VEC ? 8 : 1); ++n) kx[x.kind * D + dim + n] = round_to<DT>(v[n]);
  };
  each_pair<DT, VEC>(a.rot, a.items, rows * nh, tid, kThreads, turns, find, put);
  each_chunk<DT, VEC>(
      rows * nh * a.items.rest.d, tid, kThreads,
      [&](uint32_t i, uint32_t& dim) {
        const uint32_t n = a.items.rest(i, dim);
        dim = 2 * pairs + dim * (VEC ? 8 : 1);
        return find(n);
      },
      put);
  __syncthreads();
  // K: a chunk of 8 dims per lane, four lanes a group
  for (uint32_t i = tid; i < rows * nh * C; i += kThreads) {
    const uint32_t hr = i / C, c = i - hr * C;
    const uint32_t r = hr / nh, h = h0 + (hr - r * nh);
    float x[8], mn, mx;
#pragma unroll
    for (int n = 0; n < 8; ++n) x[n] = kx[hr * D + 8 * c + n];
    min_max8(x, mn, mx);
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      mn = fminf(mn, __shfl_xor(mn, o));
      mx = fmaxf(mx, __shfl_xor(mx, o));
    }
    uint32_t param;
    const uint32_t w = asym_codes8(x, mn, mx, &param);
    const int64_t s = slot[r + 1];
    if (s < 0) continue;
    const int64_t line = (s / 16 * H + h) * 16 + s % 16;
    *reinterpret_cast<uint32_t*>(a.pool.kc + line * (D / 2) + 4 * c) = w;
    if (c % 4 == 0) a.pool.kp[line * G + c / 4] = param;
  }
  // V: runs, 64 dims a wave
  const Runs runs = find_runs(slot, row0);
  const int XB = (D + 63) / 64, t = lane & 7;
  const int n = runs.count() * nh * XB;
  for (int i = wave; i < n; i += kThreads / 64) {
    const int xb = i % XB, hr = i / XB, h = h0 + hr % nh, e = runs.entry(hr / nh);
    const int len = runs.length(e), c = xb * 8 + (lane >> 3);
    const int64_t s0 = slot[e];
    const int t0 = (int)(s0 % 8), half = (int)(s0 % 16) / 8;
    const bool mine = t >= t0 && t < t0 + len && c < C;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0}, mn, mx;
    if (mine) {
      const uint8_t* p = a.v.p + (row0 - 1 + e + t - t0) * a.v.row + h * a.v.head + 8 * c * ES;
      if constexpr (VEC) {
        load8<DT>(p, x);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = kv_elem<DT>(p + k * ES);
      }
    }
    min_max8(x, mn, mx);
#pragma unroll
    for (int o = 8; o < 32; o <<= 1) {
      mn = fminf(mn, __shfl_xor(mn, o));
      mx = fmaxf(mx, __shfl_xor(mx, o));
    }
    uint32_t param;
    const uint32_t w = transpose8(asym_codes8(x, mn, mx, &param));
    const int64_t head = s0 / 16 * H + h;
    if (c < C) {
      uint32_t* p =
          reinterpret_cast<uint32_t*>(a.pool.vc + head * 8 * D + 64 * c + 32 * half + 4 * t);
      if (len == 8) {
        *p = w;
      } else {
        // the word's other tokens belong to earlier steps, or to another run
        const uint32_t m = (uint32_t)(((1ull << (4 * len)) - 1) << (4 * t0));
        atomicAnd(p, ~m);
        atomicOr(p, w & m);
      }
    }
    if (mine && c % 4 == 0) a.pool.vp[(head * G + c / 4) * 16 + 8 * half + t] = param;
  }
}

// ----------------------------------------------------------------- reads ----

struct ReadArgs {
  Rows k_out, v_out;
  CacheAt cache;
  PoolAt pool;
  const int64_t* slots;
  int32_t* err_flag;
  int64_t n_rows;
  int dim;
  Div heads, chunks;  // of a row, of a head (of 8 elements, or one)
};

// Elements of rows, 8 (VEC) or one a lane; rows without a slot become zeros.
template <int KV, int DT, bool VEC>
__global__ __launch_bounds__(kThreads) void read_kernel(ReadArgs a) {
  __shared__ int64_t at[kTile];
  const int64_t row0 = (int64_t)blockIdx.x * kTile;
  const int rows = (int)min((int64_t)kTile, a.n_rows - row0);
  if ((int)threadIdx.x < rows) {
    const int64_t s = a.slots[row0 + threadIdx.x];
    const bool in = s >= 0 && s < a.cache.pool_slots;
    at[threadIdx.x] = in ? s / a.cache.block * a.cache.page + s % a.cache.block * a.cache.token
                         : -1;
    if (s >= a.cache.pool_slots && a.err_flag && blockIdx.y == 0)
      atomicOr(a.err_flag, AMF_ERRFLAG_BLOCK_RANGE);
  }
  __syncthreads();
  constexpr bool FP8 = KV == AMF_DTYPE_E4M3;
  constexpr int N = VEC ? 8 : 1, IS = FP8 ? 1 : elem_bytes<KV>(), ES = elem_bytes<DT>();
  const uint32_t n = rows * a.heads.d * a.chunks.d;
  // kAhead chunks are loaded before the first of them is stored (stores may be to what is
  // read, for all that the compiler knows)
  constexpr int B = VEC ? kAhead : 1;
  for (uint32_t i0 = blockIdx.y * kThreads + threadIdx.x; i0 < 2 * n;
       i0 += B * gridDim.y * kThreads) {
    float x[B][8];
    uint32_t r[B], h[B], c[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const uint32_t i = min(i0 + b * gridDim.y * kThreads, 2 * n - 1);
      const bool value = i >= n;
      const uint32_t hr = a.chunks(value ? i - n : i, c[b]);
      r[b] = a.heads(hr, h[b]);
      const uint8_t* p = (value ? a.cache.v : a.cache.k) + max(at[r[b]], (int64_t)0) +
                         h[b] * a.cache.head + c[b] * N * IS;
      if constexpr (!VEC) {
        x[b][0] = kv_elem<KV>(p);
      } else if constexpr (FP8) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(p);
        e4m3x4_to_f32(w[0], x[b]);
        e4m3x4_to_f32(w[1], x[b] + 4);
      } else {
        load8<KV>(p, x[b]);
      }
    }
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const uint32_t i = i0 + b * gridDim.y * kThreads;
      if (i >= 2 * n) break;
      const bool value = i >= n, there = at[r[b]] >= 0;
      const float scale = !FP8 ? 1.0f : value ? a.cache.v_scale : a.cache.k_scale;
#pragma unroll
      for (int k = 0; k < N; ++k) x[b][k] = there ? x[b][k] * scale : 0.0f;
      const Rows& to = value ? a.v_out : a.k_out;
      emit<DT, false, VEC>(to.p + (row0 + r[b]) * to.row + h[b] * to.head + c[b] * N * ES, x[b],
                           1.0f);
    }
  }
}

// u * s + z of 8 codes (the product is exact: 4 bits by 11).
__device__ __forceinline__ void asym_values8(uint32_t w, uint32_t param, float* x) {
  const float s = param_scale(param), z = param_zero(param);
#pragma unroll
  for (int n = 0; n < 8; ++n) x[n] = nib(w, n) * s + z;
}

template <int DT, bool VEC>
__device__ __forceinline__ void put_chunk(uint8_t* p, const float* x) {
  if constexpr (VEC) {
    put8<DT>(p, x);
  } else {
#pragma unroll
    for (int n = 0; n < 8; ++n) put_elem<DT>(p + n * elem_bytes<DT>(), x[n]);
  }
}

template <int DT, bool VEC>
__global__ __launch_bounds__(kThreads) void int4_read_kernel(ReadArgs a, int head_block) {
  __shared__ int64_t slot[kEntries];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row0 = (int64_t)blockIdx.x * kTile;
  const int rows = (int)min((int64_t)kTile, a.n_rows - row0);
  load_slots(a.slots, row0, a.n_rows, a.pool.pool_slots, slot,
             blockIdx.y == 0 ? a.err_flag : nullptr);
  __syncthreads();
  const int D = a.dim, H = a.k_out.heads, G = D / 32, C = D / 8;
  constexpr int ES = elem_bytes<DT>();
  const int h0 = blockIdx.y * head_block, nh = min(head_block, H - h0);
  const Runs runs = find_runs(slot, row0);
  // (kAhead chunks loaded before the first is stored, as above: 52000 rows 66 us, so 62)
  const uint32_t nk = rows * nh * C;
  for (uint32_t i0 = tid; i0 < nk; i0 += kAhead * kThreads) {
    uint32_t w[kAhead], param[kAhead], r[kAhead], h[kAhead], c[kAhead];
#pragma unroll
    for (int b = 0; b < kAhead; ++b) {
      if (i0 - tid + b * kThreads >= nk) break;
      const uint32_t hr = a.chunks(min(i0 + b * kThreads, nk - 1), c[b]);
      r[b] = hr / nh;
      h[b] = h0 + (hr - r[b] * nh);
      const int64_t s = max(slot[r[b] + 1], (int64_t)0);
      const int64_t line = (s / 16 * H + h[b]) * 16 + s % 16;
      w[b] = *reinterpret_cast<const uint32_t*>(a.pool.kc + line * (D / 2) + 4 * c[b]);
      param[b] = a.pool.kp[line * G + c[b] / 4];
    }
#pragma unroll
    for (int b = 0; b < kAhead; ++b) {
      if (i0 + b * kThreads >= nk) break;
      const int64_t row = row0 + r[b];
      float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (slot[r[b] + 1] >= 0)
        asym_values8(w[b], param[b], x);
      else
        put_chunk<DT, VEC>(a.v_out.p + row * a.v_out.row + h[b] * a.v_out.head + 8 * c[b] * ES, x);
      put_chunk<DT, VEC>(a.k_out.p + row * a.k_out.row + h[b] * a.k_out.head + 8 * c[b] * ES, x);
    }
  }
  const int XB = (D + 63) / 64, t = lane & 7;
  const int n = runs.count() * nh * XB;
  constexpr int W = kThreads / 64;
  for (int i0 = wave; i0 < n; i0 += kAhead * W) {
    uint32_t w[kAhead], param[kAhead];
    int h[kAhead], e[kAhead], c[kAhead];
#pragma unroll
    for (int b = 0; b < kAhead; ++b) {
      if (i0 + b * W >= n) break;
      const int i = i0 + b * W, xb = i % XB, hr = i / XB;
      h[b] = h0 + hr % nh;
      e[b] = runs.entry(hr / nh);
      c[b] = xb * 8 + (lane >> 3);
      const int64_t s0 = slot[e[b]], head = s0 / 16 * H + h[b];
      const int half = (int)(s0 % 16) / 8, at = min(c[b], C - 1);
      w[b] = *reinterpret_cast<const uint32_t*>(a.pool.vc + head * 8 * D + 64 * at + 32 * half +
                                                4 * t);
      param[b] = a.pool.vp[(head * G + at / 4) * 16 + 8 * half + t];
    }
#pragma unroll
    for (int b = 0; b < kAhead; ++b) {
      if (i0 + b * W >= n) break;
      float x[8];
      asym_values8(transpose8(w[b]), param[b], x);
      const int t0 = (int)(slot[e[b]] % 8), len = runs.length(e[b]);
      if (t >= t0 && t < t0 + len && c[b] < C) {
        const int64_t row = row0 - 1 + e[b] + t - t0;
        put_chunk<DT, VEC>(a.v_out.p + row * a.v_out.row + h[b] * a.v_out.head + 8 * c[b] * ES, x);
      }
    }
  }
}

// ------------------------------------------------------------------ host ----

// Whether rows of `es`-byte elements allow 16-byte chunks of 8 elements (32 for fp32).
bool chunks(const Rows& r, int es) {
  const int64_t a = 8 * es < 16 ? 8 : 16;
  return ((int64_t)(uintptr_t)r.p | r.row | r.head) % a == 0;
}
bool chunks(const CacheAt& c, int es) {
  const int64_t a = 8 * es < 16 ? 8 : 16;
  return ((int64_t)(uintptr_t)c.k | (int64_t)(uintptr_t)c.v | c.page | c.token | c.head) % a == 0;
}

Rows rows_of(const void* p, int64_t row_stride, int64_t head_stride, int heads, int es) {
  return Rows{static_cast<uint8_t*>(const_cast<void*>(p)), row_stride * es,
              heads > 1 ? head_stride * es : 0, heads};
}

int check_rotary(const char* who, const int64_t* positions, const double* freqs, int32_t pairs,
                 int32_t dim, int64_t n_rows) {
  if (pairs < 0 || 2 * (int64_t)pairs > dim ||
      (pairs > 0 && n_rows > 0 && (!positions || !freqs)))
    return fail(AMF_ERR_INVALID_ARG, "%s: %d pairs of a head of %d dims, or null pointer", who,
                pairs, dim);
  return AMF_OK;
}

// Angles and rotated keys of a row tile fit the LDS; a grid has below 2^32 threads.
constexpr int kMaxDim = 512;
constexpr int64_t kMaxRows = 1 << 25;

int check_rows(const char* who, int32_t dtype, int64_t n_rows, int32_t dim, int32_t heads,
               int32_t q_heads) {
  if (!cache_elem_bytes(dtype) || n_rows < 0 || dim <= 0 || heads <= 0 || q_heads < 0)
    return fail(AMF_ERR_INVALID_ARG, "%s: bad dtype=%d n_rows=%lld head_dim=%d heads=%d/%d", who,
                dtype, (long long)n_rows, dim, heads, q_heads);
  if (dim > kMaxDim || heads > 65536 || q_heads > 65536 || n_rows > kMaxRows)
    return fail(AMF_ERR_UNSUPPORTED, "%s: head_dim=%d heads=%d/%d n_rows=%lld", who, dim, heads,
                q_heads, (long long)n_rows);
  return AMF_OK;
}

// Workgroups of `items` items a row tile: as many as fill the chip, each with
// an item at least for every thread.  (Of FP8 rows of 8 heads of 128 read, 8192 take 9.5 us with
// 2048 workgroups, 10.1 with 1024, 11.5 with 4096; 4096 rows 6.9, 6.2, 9.0; 16384 are more tiles
// than that, one each.)
unsigned splits(int64_t tiles, int64_t items) {
  const int64_t most = std::max<int64_t>(1, items / kThreads), want = (2048 + tiles - 1) / tiles;
  return (unsigned)std::min<int64_t>({most, want, 65535});
}

bool pairs_in_chunks(int pairs, int dim) { return pairs % 8 == 0 && dim % 8 == 0; }

template <int TO>
void launch_step(StepArgs a, int32_t dtype, bool vec, hipStream_t st) {
  a.items = Items(a.dim, a.rot.pairs, vec);
  a.v_items = Items(a.dim, 0, vec);
  a.q_heads = Div(a.q.heads);
  a.k_heads = Div(a.k.heads);
  a.v_heads = Div(a.v.heads);
  const int64_t tiles = (a.n_rows + a.tile - 1) / a.tile;
  const int64_t heads = a.q.heads + a.k.heads + (TO == TO_ROWS ? 0 : a.v.heads);
  const int64_t items = a.tile * heads * (a.dim - a.rot.pairs) / (vec ? 8 : 1);
  const dim3 grid((unsigned)tiles, splits(tiles, items));
  const size_t lds = (size_t)a.tile * a.rot.pairs * sizeof(Turn);
  AMF_WITH_DTYPE(dtype, vec ? step_kernel<DT, TO, true><<<grid, kThreads, lds, st>>>(a)
                            : step_kernel<DT, TO, false><<<grid, kThreads, lds, st>>>(a));
}

// Rows of a workgroup: one while rows are few (latency), else as many as share
// its set-up.  (8 + 1 heads of 128 rotated, one row a workgroup against four: 256 rows 3.1 us,
// 3.8; 1000 rows 3.7, 4.0; 2048 rows 5.9, 4.8.  Of 16384 rows into FP8, one, two, four, eight:
// 53, 33, 24, 21 us; of 32 + 8 heads 99, 82, 75, 77.  Where rows are wide as well, four suit
// few rows too: 64 rows of 32 + 8 heads into FP8 5.2 us, 4.2.)
int tile_rows(int64_t n_rows) { return n_rows < 1024 ? 1 : 4; }

}  // namespace

extern "C" int amf_rotary_embedding(
    const void* q, int64_t q_row_stride, int64_t q_head_stride, void* q_out,
    int64_t qo_row_stride, int64_t qo_head_stride, int32_t num_q_heads, const void* k,
    int64_t k_row_stride, int64_t k_head_stride, void* k_out, int64_t ko_row_stride,
    int64_t ko_head_stride, int32_t num_kv_heads, int32_t dtype, int64_t n_rows, int32_t head_dim,
    const int64_t* positions, const double* freqs, int32_t n_pairs, int32_t interleaved,
    double factor, void* stream) {
  const char* who = "amf_rotary_embedding";
  if (num_kv_heads < 0 || num_q_heads + num_kv_heads <= 0)
    return fail(AMF_ERR_INVALID_ARG, "%s: bad heads=%d/%d", who, num_q_heads, num_kv_heads);
  int rc = check_rows(who, dtype, n_rows, head_dim, std::max(num_kv_heads, 1), num_q_heads);
  if (rc) return rc;
  if ((rc = check_rotary(who, positions, freqs, n_pairs, head_dim, n_rows))) return rc;
  if (n_rows == 0) return ok();
  if ((num_q_heads > 0 && (!q || !q_out)) || (num_kv_heads > 0 && (!k || !k_out)))
    return fail(AMF_ERR_INVALID_ARG, "%s: null pointer", who);
  const int es = cache_elem_bytes(dtype);
  StepArgs a{};
  a.q = rows_of(q, q_row_stride, q_head_stride, num_q_heads, es);
  a.q_out = rows_of(q_out, qo_row_stride, qo_head_stride, num_q_heads, es);
  a.k = rows_of(k, k_row_stride, k_head_stride, num_kv_heads, es);
  a.k_out = rows_of(k_out, ko_row_stride, ko_head_stride, num_kv_heads, es);
  a.rot = RotaryArgs{positions, freqs, factor, n_pairs, interleaved != 0};
  a.n_rows = n_rows;
  a.dim = head_dim;
  a.tile = tile_rows(n_rows);
  const bool vec = pairs_in_chunks(n_pairs, head_dim) &&
                   (num_q_heads == 0 || (chunks(a.q, es) && chunks(a.q_out, es))) &&
                   (num_kv_heads == 0 || (chunks(a.k, es) && chunks(a.k_out, es)));
  launch_step<TO_ROWS>(a, dtype, vec, as_stream(stream));
  return check_launch(who);
}

extern "C" int amf_kv_write(
    const void* k, int64_t k_row_stride, int64_t k_head_stride, const void* v,
    int64_t v_row_stride, int64_t v_head_stride, int32_t dtype, int64_t n_rows,
    int32_t num_kv_heads, int32_t head_dim, const int64_t* slot_mapping, void* k_cache,
    void* v_cache, int32_t kv_dtype, int64_t page_stride, int64_t token_stride,
    int64_t head_stride, int64_t pool_pages, int32_t block_size, float k_scale, float v_scale,
    const int64_t* positions, const double* freqs, int32_t n_pairs, int32_t interleaved,
    double factor, const void* q, int64_t q_row_stride, int64_t q_head_stride, void* q_out,
    int64_t qo_row_stride, int64_t qo_head_stride, int32_t num_q_heads, int32_t* err_flag,
    void* stream) {
  const char* who = "amf_kv_write";
  int rc = check_rows(who, dtype, n_rows, head_dim, num_kv_heads, num_q_heads);
  if (rc) return rc;
  if ((rc = check_rotary(who, positions, freqs, n_pairs, head_dim, n_rows))) return rc;
  if (pool_pages <= 0 || block_size <= 0)
    return fail(AMF_ERR_INVALID_ARG, "%s: bad pool_pages=%lld block_size=%d", who,
                (long long)pool_pages, block_size);
  if (kv_dtype != dtype && kv_dtype != AMF_DTYPE_E4M3)
    return fail(AMF_ERR_UNSUPPORTED, "%s: rows of type %d into a cache of type %d", who, dtype,
                kv_dtype);
  if (!(k_scale > 0.0f) || !(v_scale > 0.0f))
    return fail(AMF_ERR_INVALID_ARG, "%s: scales must be positive", who);
  if (n_rows == 0) return ok();
  if (!k || !v || !slot_mapping || !k_cache || !v_cache || (num_q_heads > 0 && (!q || !q_out)))
    return fail(AMF_ERR_INVALID_ARG, "%s: null pointer", who);
  const int es = cache_elem_bytes(dtype), cs = kv_elem_bytes(kv_dtype);
  StepArgs a{};
  a.q = rows_of(q, q_row_stride, q_head_stride, num_q_heads, es);
  a.q_out = rows_of(q_out, qo_row_stride, qo_head_stride, num_q_heads, es);
  a.k = rows_of(k, k_row_stride, k_head_stride, num_kv_heads, es);
  a.v = rows_of(v, v_row_stride, v_head_stride, num_kv_heads, es);
  a.cache = CacheAt{static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache),
                    page_stride * cs, token_stride * cs, head_stride * cs,
                    pool_pages * block_size, block_size, k_scale, v_scale};
  a.rot = RotaryArgs{positions, freqs, factor, n_pairs, interleaved != 0};
  a.slots = slot_mapping;
  a.err_flag = err_flag;
  a.n_rows = n_rows;
  a.dim = head_dim;
  a.tile = tile_rows(n_rows);
  const bool vec = pairs_in_chunks(n_pairs, head_dim) && chunks(a.k, es) && chunks(a.v, es) &&
                   chunks(a.cache, cs) &&
                   (num_q_heads == 0 || (chunks(a.q, es) && chunks(a.q_out, es)));
  if (kv_dtype == AMF_DTYPE_E4M3)
    launch_step<TO_FP8>(a, dtype, vec, as_stream(stream));
  else
    launch_step<TO_CACHE>(a, dtype, vec, as_stream(stream));
  return check_launch(who);
}

extern "C" int amf_int4_kv_write(
    const void* k, int64_t k_row_stride, int64_t k_head_stride, const void* v,
    int64_t v_row_stride, int64_t v_head_stride, int32_t dtype, int64_t n_rows,
    int32_t num_kv_heads, int32_t head_dim, const int64_t* slot_mapping, void* k_codes,
    void* k_params, void* v_codes, void* v_params, int64_t pool_pages, const int64_t* positions,
    const double* freqs, int32_t n_pairs, int32_t interleaved, double factor, const void* q,
    int64_t q_row_stride, int64_t q_head_stride, void* q_out, int64_t qo_row_stride,
    int64_t qo_head_stride, int32_t num_q_heads, int32_t* err_flag, void* stream) {
  const char* who = "amf_int4_kv_write";
  int rc = check_rows(who, dtype, n_rows, head_dim, num_kv_heads, num_q_heads);
  if (rc) return rc;
  if ((rc = check_rotary(who, positions, freqs, n_pairs, head_dim, n_rows))) return rc;
  if (pool_pages <= 0)
    return fail(AMF_ERR_INVALID_ARG, "%s: bad pool_pages=%lld", who, (long long)pool_pages);
  if (head_dim % 32)
    return fail(AMF_ERR_UNSUPPORTED, "%s: head_dim %d is not a multiple of 32", who, head_dim);
  if (n_rows == 0) return ok();
  if (!k || !v || !slot_mapping || !k_codes || !k_params || !v_codes || !v_params ||
      (num_q_heads > 0 && (!q || !q_out)))
    return fail(AMF_ERR_INVALID_ARG, "%s: null pointer", who);
  if (((uintptr_t)k_codes | (uintptr_t)k_params | (uintptr_t)v_codes | (uintptr_t)v_params) & 15)
    return fail(AMF_ERR_INVALID_ARG, "%s: the pool's planes must be 16-byte aligned", who);
  const int es = cache_elem_bytes(dtype);
  PoolStepArgs a{};
  a.q = rows_of(q, q_row_stride, q_head_stride, num_q_heads, es);
  a.q_out = rows_of(q_out, qo_row_stride, qo_head_stride, num_q_heads, es);
  a.k = rows_of(k, k_row_stride, k_head_stride, num_kv_heads, es);
  a.v = rows_of(v, v_row_stride, v_head_stride, num_kv_heads, es);
  a.pool = PoolAt{static_cast<uint8_t*>(k_codes), static_cast<uint32_t*>(k_params),
                  static_cast<uint8_t*>(v_codes), static_cast<uint32_t*>(v_params),
                  pool_pages * 16};
  a.rot = RotaryArgs{positions, freqs, factor, n_pairs, interleaved != 0};
  a.slots = slot_mapping;
  a.err_flag = err_flag;
  a.n_rows = n_rows;
  a.dim = head_dim;
  const bool vec = pairs_in_chunks(n_pairs, head_dim) && chunks(a.k, es) && chunks(a.v, es) &&
                   (num_q_heads == 0 || (chunks(a.q, es) && chunks(a.q_out, es)));
  a.items = Items(head_dim, n_pairs, vec);
  a.q_heads = Div(num_q_heads);
  const int64_t tiles = (n_rows + kTile - 1) / kTile;
  // rotated keys of a workgroup's heads in 32 KB of LDS at most
  const int most = std::max(1, (32 << 10) / (kTile * head_dim * 4));
  // all of them once the row tiles alone are two workgroups a CU (8 KV heads, 2048 rows 15.2 us;
  // from 256 tiles on 17.0, from 1024 17.0, from 2048 19.2; 512 rows 7.3, 6.8, 7.2, 7.2)
  const int few = tiles >= 512 ? most : std::max(1, (int)(num_kv_heads * tiles / 512));
  a.head_block = std::min({most, few, num_kv_heads});
  a.kv_blocks = (num_kv_heads + a.head_block - 1) / a.head_block;
  const int64_t q_items = (int64_t)kTile * num_q_heads * (head_dim - n_pairs) / (vec ? 8 : 1);
  const unsigned q_blocks = num_q_heads > 0 ? splits(tiles, q_items) : 0;
  if (a.kv_blocks + (int64_t)q_blocks > 65535)
    return fail(AMF_ERR_UNSUPPORTED, "%s: %d / %d heads of %d dims", who, num_q_heads,
                num_kv_heads, head_dim);
  const dim3 grid((unsigned)tiles, a.kv_blocks + q_blocks);
  const size_t lds = (size_t)kTile * n_pairs * sizeof(Turn) +
                     (size_t)kTile * a.head_block * head_dim * sizeof(float);
  AMF_WITH_DTYPE(dtype,
                 vec ? int4_step_kernel<DT, true><<<grid, kThreads, lds, as_stream(stream)>>>(a)
                     : int4_step_kernel<DT, false><<<grid, kThreads, lds, as_stream(stream)>>>(a));
  return check_launch(who);
}

extern "C" int amf_kv_read(const void* k_cache, const void* v_cache, int32_t kv_dtype,
                           int64_t page_stride, int64_t token_stride, int64_t head_stride,
                           int64_t pool_pages, int32_t block_size, float k_scale, float v_scale,
                           const int64_t* slot_mapping, void* k, int64_t k_row_stride,
                           int64_t k_head_stride, void* v, int64_t v_row_stride,
                           int64_t v_head_stride, int32_t dtype, int64_t n_rows,
                           int32_t num_kv_heads, int32_t head_dim, int32_t* err_flag,
                           void* stream) {
  const char* who = "amf_kv_read";
  int rc = check_rows(who, dtype, n_rows, head_dim, num_kv_heads, 0);
  if (rc) return rc;
  if (pool_pages <= 0 || block_size <= 0)
    return fail(AMF_ERR_INVALID_ARG, "%s: bad pool_pages=%lld block_size=%d", who,
                (long long)pool_pages, block_size);
  if (kv_dtype != dtype && kv_dtype != AMF_DTYPE_E4M3)
    return fail(AMF_ERR_UNSUPPORTED, "%s: rows of type %d from a cache of type %d", who, dtype,
                kv_dtype);
  if (n_rows == 0) return ok();
  if (!k || !v || !slot_mapping || !k_cache || !v_cache)
    return fail(AMF_ERR_INVALID_ARG, "%s: null pointer", who);
  const int es = cache_elem_bytes(dtype), cs = kv_elem_bytes(kv_dtype);
  ReadArgs a{};
  a.k_out = rows_of(k, k_row_stride, k_head_stride, num_kv_heads, es);
  a.v_out = rows_of(v, v_row_stride, v_head_stride, num_kv_heads, es);
  a.cache = CacheAt{static_cast<uint8_t*>(const_cast<void*>(k_cache)),
                    static_cast<uint8_t*>(const_cast<void*>(v_cache)), page_stride * cs,
                    token_stride * cs, head_stride * cs, pool_pages * block_size, block_size,
                    k_scale, v_scale};
  a.slots = slot_mapping;
  a.err_flag = err_flag;
  a.n_rows = n_rows;
  a.dim = head_dim;
  const bool vec = head_dim % 8 == 0 && chunks(a.k_out, es) && chunks(a.v_out, es) &&
                   chunks(a.cache, cs);
  a.heads = Div(num_kv_heads);
  a.chunks = Div(head_dim / (vec ? 8 : 1));
  const int64_t tiles = (n_rows + kTile - 1) / kTile;
  const int64_t items = (int64_t)2 * kTile * num_kv_heads * head_dim / (vec ? 8 : 1);
  const dim3 grid((unsigned)tiles, splits(tiles, items));
  hipStream_t st = as_stream(stream);
  AMF_WITH_DTYPE(dtype, {
    if (kv_dtype == AMF_DTYPE_E4M3)
      vec ? read_kernel<AMF_DTYPE_E4M3, DT, true><<<grid, kThreads, 0, st>>>(a)
          : read_kernel<AMF_DTYPE_E4M3, DT, false><<<grid, kThreads, 0, st>>>(a);
    else
      vec ? read_kernel<DT, DT, true><<<grid, kThreads, 0, st>>>(a)
          : read_kernel<DT, DT, false><<<grid, kThreads, 0, st>>>(a);
  });
  return check_launch(who);
}

extern "C" int amf_int4_kv_read(const void* k_codes, const void* k_params, const void* v_codes,
                                const void* v_params, int64_t pool_pages,
                                const int64_t* slot_mapping, void* k, int64_t k_row_stride,
                                int64_t k_head_stride, void* v, int64_t v_row_stride,
                                int64_t v_head_stride, int32_t dtype, int64_t n_rows,
                                int32_t num_kv_heads, int32_t head_dim, int32_t* err_flag,
                                void* stream) {
  const char* who = "amf_int4_kv_read";
  int rc = check_rows(who, dtype, n_rows, head_dim, num_kv_heads, 0);
  if (rc) return rc;
  if (pool_pages <= 0)
    return fail(AMF_ERR_INVALID_ARG, "%s: bad pool_pages=%lld", who, (long long)pool_pages);
  if (head_dim % 32)
    return fail(AMF_ERR_UNSUPPORTED, "%s: head_dim %d is not a multiple of 32", who, head_dim);
  if (n_rows == 0) return ok();
  if (!k || !v || !slot_mapping || !k_codes || !k_params || !v_codes || !v_params)
    return fail(AMF_ERR_INVALID_ARG, "%s: null pointer", who);
  if (((uintptr_t)k_codes | (uintptr_t)k_params | (uintptr_t)v_codes | (uintptr_t)v_params) & 15)
    return fail(AMF_ERR_INVALID_ARG, "%s: the pool's planes must be 16-byte aligned", who);
  const int es = cache_elem_bytes(dtype);
  ReadArgs a{};
  a.k_out = rows_of(k, k_row_stride, k_head_stride, num_kv_heads, es);
  a.v_out = rows_of(v, v_row_stride, v_head_stride, num_kv_heads, es);
  a.pool = PoolAt{static_cast<uint8_t*>(const_cast<void*>(k_codes)),
                  static_cast<uint32_t*>(const_cast<void*>(k_params)),
                  static_cast<uint8_t*>(const_cast<void*>(v_codes)),
                  static_cast<uint32_t*>(const_cast<void*>(v_params)), pool_pages * 16};
  a.slots = slot_mapping;
  a.err_flag = err_flag;
  a.n_rows = n_rows;
  a.dim = head_dim;
  const bool vec = chunks(a.k_out, es) && chunks(a.v_out, es);
  a.chunks = Div(head_dim / 8);
  const int64_t tiles = (n_rows + kTile - 1) / kTile;
  // KV heads of a workgroup: 2048 workgroups while there are so many (8 heads, 8192 rows 14.0 us;
  // 512 or 1024 workgroups 14.1, 8192 18.0; 4096 rows 9.1, 9.2 or 8.8, 10.7)
  const int head_block = (int)std::max<int64_t>(
      (num_kv_heads + 65534) / 65535, std::min<int64_t>(num_kv_heads, num_kv_heads * tiles / 2048));
  const dim3 grid((unsigned)tiles, (num_kv_heads + head_block - 1) / head_block);
  hipStream_t st = as_stream(stream);
  AMF_WITH_DTYPE(dtype, vec ? int4_read_kernel<DT, true><<<grid, kThreads, 0, st>>>(a, head_block)
                            : int4_read_kernel<DT, false><<<grid, kThreads, 0, st>>>(a, head_block));
  return check_launch(who);
}

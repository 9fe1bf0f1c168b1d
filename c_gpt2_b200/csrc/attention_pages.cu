// Attention over cache pages with a shared prefix (w8a8_attention_pages).
//
//   O_r = sum_j w_rj V_j / sum_j w_rj,  w_rj = exp(q_r.k_j / 8 - m_r),  j < end_r
//
// formed in one pass over the keys (running maximum and sum; base-2
// exponentials of scores scaled by log2(e) / 8), with fp32 scores, maxima, sums
// and accumulators. The weights are rounded to bf16 for the tensor cores: half a
// step at most, 2^-8 of a weight and of either sign, which an average over keys
// shrinks below the rounding of the output; their sum is taken before it.
//
// Rows and keys are cut up so that shared keys are read once for many rows:
//   tensor-core items (tcgen05)  up to 256 rows: of all sequences over the shared
//                                prefix, or of one over prefix and tail
//   16-row groups (mma.sync)     the few rows of one sequence and key head over
//                                its tail, or over a prefix that few rows share
// Both leave parts (maximum, sum, unnormalised O) of their rows in the workspace,
// which a last kernel joins; a call whose every row is one item's or one group's
// writes O at once. make_plan has the choice. Lengths are known on the device
// only, so the kernels cut the keys themselves.
#include "common.cuh"
#include "kernels.cuh"
#include "runtime.cuh"

#include <math.h>

namespace w8a8 {

namespace {

constexpr int kSms = 148;            // the plan below is made for this many SMs
constexpr float kMaxSlack = 8.0f;    // see grown()
constexpr float kScale2 = 0.125f * 1.44269504088896340736f;  // log2(e) / sqrt(64)
constexpr int kErrEntry = 0x1601;    // a table entry outside the pool
constexpr int kErrWaitFull = 0x1602;

constexpr int kStageKeys = 64;
constexpr int kStages = 2;                         // of each warp
constexpr uint32_t kTileBytes = kStageKeys * 128;  // keys or values of a stage
constexpr int kMmaWarps = 7;                       // of a CTA, one an SM
constexpr int kRows = 16;                          // query rows of an item
// A prefix of more 16-row stages than this goes to the tensor-core kernel, if it takes several
// row tiles. That kernel has a fixed cost of some 8 us; the 16-row kernel, whose re-reads hit
// L2, gets through about 500 stages a microsecond (64 rows of 4 key heads over 16384 positions,
// 4096 stages: 25.0 us with it, 20.6 with the other; a single row tile is read once: 8 rows of
// 16 key heads over 16384 positions, as many stages: 28.6 and 33.0).
constexpr int kMinTcStages = 4000;

// Division of 0 <= n < 2^31 by a fixed d >= 1: for d > 1 with 2^s < d <= 2^(s+1), the
// quotient is the high word of n * ceil(2^(32+s) / d), shifted by s (Granlund and
// Montgomery's division by invariant integers).
struct Div {
  uint32_t mul, shift;
};
Div make_div(uint32_t d) {
  if (d <= 1) return {0, 0};
  uint32_t s = 0;
  while ((2ull << s) < d) ++s;
  return {(uint32_t)(((1ull << (32 + s)) + d - 1) / d), s};
}
__device__ __forceinline__ int quot(int n, const Div &d) {
  return d.mul ? (int)(__umulhi((uint32_t)n, d.mul) >> d.shift) : n;
}

constexpr int kTileRows = 128, kPairRows = 256;  // tensor-core row tiles
constexpr int kTcKeys = 128;                     // and keys of a block

// The tensor-core items of a key head over the shared prefix: the rows that hold a query,
// packed, in pairs of tiles and perhaps a last single one, the keys of a pair in s2 chunks of
// c2, a single tile's in s1 of c1. A CTA's time goes by its blocks, and a single tile's take
// half as long, so its chunks are twice as long.
constexpr int kMostCost = 1 << 25;
struct Across {
  int rows, pairs, s2, c2, s1, c1;  // s1 = 0: no single tile
  int cost;                         // rounds of CTAs times blocks of one
};
// With a pair's keys in about `splits` chunks; of at most max_items in all, if there is a
// choice. What a CTA does besides its blocks takes the time of three.
__host__ __device__ inline Across across_of(int rows, int n_kv, int n_shared, int splits,
                                            int max_items) {
  Across p = {};
  const int tiles = (rows + kTileRows - 1) / kTileRows, single = tiles & 1;
  const int blocks = (n_shared + kTcKeys - 1) / kTcKeys;
  p.rows = rows;
  p.pairs = tiles >> 1;
  const int b2 = (blocks + splits - 1) / splits;
  const int b1 = p.pairs && 2 * b2 < blocks ? 2 * b2 : p.pairs ? blocks : b2;
  p.c2 = b2 * kTcKeys;
  p.c1 = b1 * kTcKeys;
  p.s2 = p.pairs ? (blocks + b2 - 1) / b2 : 0;
  p.s1 = single ? (blocks + b1 - 1) / b1 : 0;
  const int items = n_kv * (p.pairs * p.s2 + p.s1);
  const int64_t cost = (int64_t)((items + kSms - 1) / kSms) * (p.pairs ? b2 + 3 : (b1 + 1) / 2 + 3);
  p.cost = cost < kMostCost && (splits == 1 || items <= max_items) ? (int)cost : kMostCost;
  return p;
}

struct ApArgs {
  const uint16_t *Q;
  int64_t ldq;
  uint16_t *O;
  int64_t ldo;
  const int32_t *table, *n_ctx, *n_new, *shared;
  int max_pages, n_pages, page_shift;
  int n_seq, T, g, n_kv, max_ctx, n_shared;
  // groups of the 16-row kernel (a row tile of a key head, and the keys it sees, in
  // 64-key stages): of the prefix [n_kv][p_tiles] with p_stages each, then of every
  // sequence [n_kv][its row tiles] over its tail (see Walk)
  int p_tiles, p_stages;
  int base;            // where a sequence's groups begin: n_shared, or 0 if nothing is shared out
  int whole;           // stages given to every sequence's groups, none split; 0: as many as it has
  // tensor-core items: rows of one sequence over all its keys, [pairs][n_seq][n_kv][splits]
  // of `chunk` keys; or of all sequences over the prefix, as `across` has them (if every row
  // holds a query) or plan_across finds them
  int by_seq, pairs, splits, chunk;
  Across across;
  int tc;              // CTAs of the tensor-core kernel
  int behind;          // the 16-row kernel runs behind the tensor-core kernel
  int direct;          // every row is one item's or group's, which writes O itself
  int64_t rows;        // n_seq * T * n_head
  Div by_g, by_T, by_head;
  // Parts of rows: 256 of each tensor-core item; then, of the 16-row groups, one a row over the
  // prefix (at part_p) and one over the tail (part_t); and, of groups that several warps share,
  // [warps][2][16] (part_f): a warp's rows of the group it joined, and of the one it began.
  int64_t part_p, part_t, part_f, parts;
  float *Op;           // [part][64]
  float2 *ml;          // [part] maximum (base 2), sum
  // [3][rows]: first part (tensor-core items) or first warp of the row's parts over the prefix,
  // their number, and for the tail first warp * 2^16 + number
  int *shares;
  int *err;
};

// Positions up to the one that the last row sees: where more are new than there are rows, the
// rows are the first of them.
__device__ __forceinline__ int seq_len(const ApArgs &a, int b) {
  const int len = min(max(a.n_ctx[b], 0), a.max_ctx);
  return a.n_new ? max(len - max(a.n_new[b] - a.T, 0), 0) : len;
}
__device__ __forceinline__ int seq_new(const ApArgs &a, int b) {
  return a.n_new ? min(max(a.n_new[b], 0), a.T) : a.T;
}

struct Row {
  int m;  // token row, -1: none
  int h, end;
};
// (volatile: the exponentials stay between the barriers of a turn at them)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Pairs of fp32 (one instruction for two results).
typedef unsigned long long F2;
__device__ __forceinline__ F2 f2(float x, float y) {
  F2 v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  return v;
}
__device__ __forceinline__ void f2_split(F2 v, float &x, float &y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
  F2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// A maximum to subtract: 0 where nothing has been seen yet.
__device__ __forceinline__ float safe_max(float m) { return m == -INFINITY ? 0.0f : m; }

// The running maximum that a row's weights refer to moves only when the row's
// maximum has grown by more than 2^8 in the weights: the sums stay far from the
// ends of fp32's range, and O is rescaled rarely.
__device__ __forceinline__ bool grown(float top, float m) {
  return top > m && !((top - m) * kScale2 <= kMaxSlack);
}

// A load after which nothing is read from L1 that was there before it.
__device__ __forceinline__ void load_acquire(const int *p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
}

struct MmaSmem {
  uint64_t full[kMmaWarps][kStages];
};

// A warp's part of a group.
struct Item {
  int b, nn;    // sequence of a tail and its new rows; -1: prefix
  int kvh, r0;  // key head; first row of the tile among the (m, g) rows of b or of all
  int k0, k1;   // positions
  int n_valid;  // positions that hold anything, of a prefix: that some query sees
  int warps;    // where `begins`: warps that share the group
  bool begins, ends;
};

// All groups' stages in a row, of which every warp takes an equal stretch: the
// kernel has no stragglers whatever the sequences' lengths. A walk passes over the
// sequences 32 at a time, a lane each.
struct Walk {
  int left, per_warp, me;         // stages to go, of a stretch; this warp
  int b, kvh, tile, s0;           // the next group, and its stages already taken
  int st, tiles, n_valid, nn;     // its stages; its sequence's row tiles, length, new rows
  int base;                       // sequence of lane 0
  uint32_t more;                  // lanes with sequences still to come
  int l_st, l_tiles, l_valid, l_nn;  // this lane's sequence
};

__device__ __forceinline__ int tail_stages(const ApArgs &a, int n_valid) {
  if (a.whole) return a.whole;
  return n_valid > a.base ? (n_valid - a.base + kStageKeys - 1) / kStageKeys : 0;
}
__device__ __forceinline__ int row_tiles(const ApArgs &a, int nn) {
  return (nn * a.g + kRows - 1) / kRows;
}

// All groups' stages; *prefix: the shared positions that some query sees. (Those behind may hold
// anything: their values are kept out of the products, where 0 * NaN would not stay 0.)
__device__ __forceinline__ int all_stages(const ApArgs &a, int lane, int *prefix) {
  int v = 0, seen = 0;
#pragma unroll 4
  for (int b = lane; b < a.n_seq; b += 32) {
    const int len = seq_len(a, b), nn = seq_new(a, b);
    v += tail_stages(a, len) * row_tiles(a, nn);
    if (nn > 0) seen = max(seen, len);
  }
  *prefix = min(__reduce_max_sync(~0u, seen), a.n_shared);
  return (a.p_tiles * a.p_stages + __reduce_add_sync(~0u, v)) * a.n_kv;
}

// The next 32 sequences; returns this lane's stages.
__device__ __forceinline__ int walk_batch(const ApArgs &a, Walk &w, int lane) {
  const int b = w.base + lane;
  w.l_valid = w.l_nn = w.l_st = 0;
  if (b < a.n_seq) {
    w.l_valid = seq_len(a, b);
    w.l_nn = seq_new(a, b);
    w.l_st = tail_stages(a, w.l_valid);
  }
  w.l_tiles = row_tiles(a, w.l_nn);
  const int v = w.l_st * w.l_tiles * a.n_kv;
  w.more = __ballot_sync(~0u, v > 0);
  return v;
}
__device__ __forceinline__ void walk_take_lane(Walk &w, int l) {
  w.b = w.base + l;
  w.more &= ~1u << l;
  w.st = __shfl_sync(~0u, w.l_st, l);
  w.tiles = __shfl_sync(~0u, w.l_tiles, l);
  w.n_valid = __shfl_sync(~0u, w.l_valid, l);
  w.nn = __shfl_sync(~0u, w.l_nn, l);
}
// The first sequence from the batch at w.base on; there is one while w.left > 0.
__device__ __forceinline__ void walk_next_seq(const ApArgs &a, Walk &w, int lane) {
  while (w.more == 0) {
    w.base += 32;
    walk_batch(a, w, lane);
  }
  walk_take_lane(w, __ffs(w.more) - 1);
}

__device__ __forceinline__ Walk walk_begin(const ApArgs &a, int me, int per_warp, int all,
                                           int prefix, int lane) {
  Walk w = {};
  w.me = me;
  w.per_warp = per_warp;
  int x = min((int64_t)me * per_warp, (int64_t)all);
  w.left = min(per_warp, all - x);
  if (w.left <= 0) return w;
  const int pre = a.n_kv * a.p_tiles * a.p_stages;
  int v = walk_batch(a, w, lane);
  if (x < pre) {
    w.b = -1;
    w.st = a.p_stages;
    w.tiles = a.p_tiles;
    w.n_valid = prefix;
  } else {
    x -= pre;
    int l;
    for (;;) {
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(~0u, v, d);
        if (lane >= d) v += y;
      }
      const uint32_t past = __ballot_sync(~0u, x < v);
      if (past) {
        l = __ffs(past) - 1;
        break;
      }
      x -= __shfl_sync(~0u, v, 31);
      w.base += 32;
      v = walk_batch(a, w, lane);
    }
    const int before = __shfl_sync(~0u, v, max(l - 1, 0));
    if (l > 0) x -= before;
    walk_take_lane(w, l);
  }
  const int group = x / w.st;
  w.s0 = x - group * w.st;
  w.kvh = group / w.tiles;
  w.tile = group - w.kvh * w.tiles;
  return w;
}

// The part of the next group that lies in the warp's stretch; w.left > 0.
__device__ __forceinline__ Item walk_next(const ApArgs &a, Walk &w, int lane) {
  Item it;
  const int n = min(w.st - w.s0, w.left);
  it.b = w.b;
  it.nn = w.nn;
  it.kvh = w.kvh;
  it.r0 = w.tile * kRows;
  it.n_valid = w.n_valid;
  it.begins = w.s0 == 0;
  it.ends = w.s0 + n == w.st;
  it.warps = w.st <= w.left ? 1 : 1 + (w.st - w.left + w.per_warp - 1) / w.per_warp;
  it.k0 = w.s0 * kStageKeys;
  it.k1 = it.k0 + n * kStageKeys;
  if (it.b < 0) {
    it.k1 = min(it.k1, it.n_valid);
  } else {
    it.k0 += a.base;
    // the last row of the tile sees furthest
    const int t_last = min(quot(it.r0 + kRows - 1, a.by_g), w.nn - 1);
    it.k1 = min(it.k1 + a.base, it.n_valid - w.nn + t_last + 1);
  }
  w.left -= n;
  w.s0 += n;
  if (it.ends && w.left > 0) {
    w.s0 = 0;
    if (++w.tile == w.tiles) {
      w.tile = 0;
      if (++w.kvh == a.n_kv) {
        w.kvh = 0;
        walk_next_seq(a, w, lane);
      }
    }
  }
  return it;
}

// Row R of an item's (m, g) rows; for those of one sequence nothing is read.
__device__ __forceinline__ Row get_row(const ApArgs &a, const Item &it, int R) {
  Row w;
  const int j = quot(R, a.by_g);
  w.h = it.kvh * a.g + (R - j * a.g);
  int b = it.b, t = j, nn = it.nn, len = it.n_valid;
  if (b < 0) {
    b = quot(j, a.by_T);
    t = j - b * a.T;
    nn = b < a.n_seq ? seq_new(a, b) : 0;
    len = b < a.n_seq ? seq_len(a, b) : 0;
  }
  w.m = t < nn ? b * a.T + t : -1;
  w.end = t < nn ? len - nn + t + 1 : 0;
  return w;
}

__device__ __forceinline__ int item_stages(const Item &it) {
  return it.k1 > it.k0 ? (it.k1 - it.k0 + kStageKeys - 1) / kStageKeys : 0;
}

}  // namespace

// What a warp holds of an item: rows lane / 4 and lane / 4 + 8 of 16.
struct MmaState {
  uint32_t q[4][4];       // Q, by 16 dims
  float o[8][4];          // O, by 8 dims
  float m[2], l[2];       // reference of the weights (a score), this lane's sums
};

// 64 keys: S = Q K^T, weights, O += P V. HI: rows 8..15 hold anything.
// lim: keys of this stage that the rows see.
template <bool HI>
__device__ __forceinline__ void mma_stage(MmaState &w, uint32_t kb, uint32_t vb,
                                          const int (&lim)[2], int lane) {
  constexpr int R = HI ? 2 : 1;
  const int lm = lane >> 3, lr = lane & 7;
  const uint32_t krow = kb + ((lm >> 1) * 8 + lr) * 128;  // K: matrices (key half, dim half)
  const uint32_t vrow = vb + ((lm & 1) * 8 + lr) * 128;   // V: matrices (dim half, key half)
  float c[8][4] = {};
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    const uint32_t at = krow + (((ks * 2 + (lm & 1)) ^ lr) << 4);
#pragma unroll
    for (int h = 0; h < 4; ++h) {  // 16 keys
      uint32_t b[4];
      ldsm4(at + h * 2048, b);
      mma16816(c[2 * h], w.q[ks], b[0], b[1]);
      mma16816(c[2 * h + 1], w.q[ks], b[2], b[3]);
    }
  }
  if (__any_sync(~0u, lim[0] < kStageKeys || (HI && lim[1] < kStageKeys))) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if ((j >> 1) * 8 + (j & 1) + (lane & 3) * 2 >= lim[r])
          c[j >> 1][2 * r + (j & 1)] = -INFINITY;
  }
  bool up[2] = {};
  float f[2] = {1.0f, 1.0f};
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float t0 = fmaxf(c[0][2 * r], c[0][2 * r + 1]), t1 = fmaxf(c[1][2 * r], c[1][2 * r + 1]);
#pragma unroll
    for (int j = 2; j < 8; j += 2) {
      t0 = fmaxf(t0, fmaxf(c[j][2 * r], c[j][2 * r + 1]));
      t1 = fmaxf(t1, fmaxf(c[j + 1][2 * r], c[j + 1][2 * r + 1]));
    }
    float t = fmaxf(t0, t1);
    t = fmaxf(t, __shfl_xor_sync(~0u, t, 1));
    t = fmaxf(t, __shfl_xor_sync(~0u, t, 2));
    up[r] = grown(t, w.m[r]);
    if (up[r]) {
      f[r] = ex2((w.m[r] - t) * kScale2);
      w.m[r] = t;
    }
  }
  if (__any_sync(~0u, up[0] || up[1])) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      w.l[r] *= f[r];
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        w.o[d][2 * r] *= f[r];
        w.o[d][2 * r + 1] *= f[r];
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float ms = safe_max(w.m[r]) * kScale2;
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = ex2(fmaf(c[j][2 * r], kScale2, -ms));
      const float y = ex2(fmaf(c[j][2 * r + 1], kScale2, -ms));
      s0 += x;
      s1 += y;
      c[j][2 * r] = __uint_as_float(pack_bf2(x, y));
    }
    w.l[r] += s0 + s1;
  }
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const uint32_t pa[4] = {__float_as_uint(c[2 * h][0]), HI ? __float_as_uint(c[2 * h][2]) : 0u,
                            __float_as_uint(c[2 * h + 1][0]),
                            HI ? __float_as_uint(c[2 * h + 1][2]) : 0u};
#pragma unroll
    for (int d2 = 0; d2 < 4; ++d2) {
      uint32_t b[4];
      ldsm4t(vrow + h * 2048 + (((d2 * 2 + (lm >> 1)) ^ lr) << 4), b);
      mma16816(w.o[2 * d2], pa, b[0], b[1]);
      mma16816(w.o[2 * d2 + 1], pa, b[2], b[3]);
    }
  }
}

// ---------------------------------------------------------------------------
// Items of 16 rows on mma.sync, a warp each: for the tails, whose row tile holds
// the few rows of one sequence and key head, and for a prefix that few rows
// share. Bound by HBM: 64 keys of a head, 16 KB, in 700 cycles of an SM at the
// copy rate. The warps work alone, with no barrier between them, each with two
// 64-key stages that it fills itself by TMA (128-byte swizzle), one ahead, across
// the ends of items (four warps with three stages: 31 us where six with two take
// 25.5, seven 24.5). Measured, 64 sequences of 20 heads, nothing shared: 5.7 TB/s
// with up to 4096 positions each (645 to 726 MB by the lengths drawn, 114 to 128 us;
// 6 % less without the arithmetic), but 28 to 30 us with up to 512 (81 to 91 MB):
// some 4 us until the first keys arrive, 4 for the join, and SMs that get their
// bytes up to a quarter later than the average.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kMmaWarps * 32, 1)
    attention_pages_mma_kernel(const __grid_constant__ CUtensorMap tmK,
                               const __grid_constant__ CUtensorMap tmV,
                               const __grid_constant__ ApArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  uint8_t *ring = smem + warp * (kStages * 2 * kTileBytes);
  MmaSmem *ctl = reinterpret_cast<MmaSmem *>(smem + kMmaWarps * kStages * 2 * kTileBytes);
  uint64_t *full = ctl->full[warp];
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
    if (warp == 0) {
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
    }
  }
  __syncwarp();
  // Behind the tensor-core kernel there is nothing to wait for before the end: both only write
  // parts of rows, and a CTA here starts as an SM is free. What came before that kernel is
  // complete, with its writes in memory: each of its CTAs waited for that before it let this
  // kernel start. TMA reads from there; for the plain loads, the acquire drops what this SM's L1
  // may hold of older contents (0.1 us a call; a full fence 1.2).
  pdl_launch_dependents();
  if (a.behind) load_acquire(a.n_ctx);
  else pdl_wait();

  // neighbouring stretches on different SMs: they share keys in L2, and few stages spread out
  const int me = warp * gridDim.x + blockIdx.x;
  int prefix;
  const int all = all_stages(a, lane, &prefix), unit = max(a.whole, 1);
  const int warps = gridDim.x * kMmaWarps;
  const int per_warp = max((all / unit + warps - 1) / warps, 1) * unit;
  Walk walk = walk_begin(a, me, per_warp, all, prefix, lane);

  // ---- loading: lane i < 2 * boxes brings one box (16 to 64 rows) of a stage ----
  const int box = min(1 << a.page_shift, kStageKeys);
  const int boxes = kStageKeys / box;
  const bool act = lane < 2 * boxes, is_v = lane >= boxes;
  const int bx = is_v ? lane - boxes : lane;
  Walk ahead = walk;  // of the loads
  Item coming;        // the item that is being loaded
  int at_stage = 0, of_stages = 0;
  auto next_item = [&]() {  // one with keys
    at_stage = of_stages = 0;
    while (of_stages == 0 && ahead.left > 0) {
      coming = walk_next(a, ahead, lane);
      of_stages = item_stages(coming);
    }
  };
  auto entry = [&]() -> int {  // page of this lane's box, n_pages: reads as zeros
    const int pos = coming.k0 + at_stage * kStageKeys + bx * box;
    if (!act || of_stages == 0 || pos >= coming.k1) return a.n_pages;
    const int k = pos >> a.page_shift;
    int p = -1;
    if (pos < a.n_shared) p = a.shared[k];
    else if (k < a.max_pages) p = a.table[(int64_t)coming.b * a.max_pages + k];
    if (p < 0 || p >= a.n_pages) {
      report_error(a.err, kErrEntry);
      p = a.n_pages;
    }
    return p;
  };
  next_item();
  int page = entry();
  uint32_t loaded = 0;
  auto load = [&]() {
    if (of_stages == 0) return;
    const int st = loaded % kStages;
    if (lane == 0) mbar_arrive_expect_tx(&full[st], 2 * kTileBytes);
    __syncwarp();
    if (act) {
      const int pos = coming.k0 + at_stage * kStageKeys + bx * box;
      const int y = (coming.kvh << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
      tma_load_3d(ring + (st * 2 + is_v) * kTileBytes + bx * box * 128, is_v ? &tmV : &tmK,
                  &full[st], 0, y, page);
    }
    ++loaded;
    if (++at_stage == of_stages) next_item();
    page = entry();
  };
#pragma unroll 1
  for (int i = 0; i < kStages - 1; ++i) load();

  // an item with its rows and Q, which are fetched while the one before is worked on
  struct Ready {
    Item it;
    Row row[2];
    uint32_t q[4][4];
  };
  auto prepare = [&]() {
    Ready y;
    y.it = walk_next(a, walk, lane);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      y.row[r] = get_row(a, y.it, y.it.r0 + (lane >> 2) + 8 * r);
      const Row &w = y.row[r];
      const uint32_t *src = reinterpret_cast<const uint32_t *>(a.Q + (int64_t)w.m * a.ldq +
                                                               w.h * kPageHd) + (lane & 3);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        y.q[ks][r] = w.m < 0 ? 0u : src[ks * 8];
        y.q[ks][r + 2] = w.m < 0 ? 0u : src[ks * 8 + 4];
      }
    }
    return y;
  };
  uint32_t n = 0;
  bool more = walk.left > 0;
  Ready ready;
  if (more) ready = prepare();
  while (more) {
    const Ready cur = ready;
    const Item &it = cur.it;
    const Row(&row)[2] = cur.row;
    more = walk.left > 0;
    if (more) ready = prepare();
    const int stages = item_stages(it);
    const bool hi = __any_sync(~0u, row[1].m >= 0);
    MmaState w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        w.q[i][k] = cur.q[i][k];
        w.o[i][k] = w.o[i + 4][k] = 0.0f;
      }
    w.m[0] = w.m[1] = -INFINITY;
    w.l[0] = w.l[1] = 0.0f;
    bool late = false;  // a copy that did not arrive: the warp has no more to do, but ends below
    for (int s = 0; s < stages; ++s, ++n) {
      load();  // into the stage that was read last
      const int st = n % kStages;
      if (!__all_sync(~0u, mbar_wait(&full[st], (n / kStages) & 1, nullptr, a.err, kErrWaitFull))) {
        // no copy may still be writing shared memory when the warp exits
        for (uint32_t i = n + 1; i < loaded; ++i)
          mbar_wait(&full[i % kStages], (i / kStages) & 1, nullptr, a.err, kErrWaitFull);
        late = true;
        break;
      }
      const int key0 = it.k0 + s * kStageKeys;
      uint8_t *sK = ring + st * 2 * kTileBytes, *sV = sK + kTileBytes;
      if (key0 + kStageKeys > it.n_valid) {
        // rows of the last page that hold nothing yet: 0 * V must stay 0
        for (int u = max(it.n_valid - key0, 0) * 8 + lane; u < kStageKeys * 8; u += 32)
          *reinterpret_cast<uint4 *>(sV + u * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();  // before the next copy into this stage
        __syncwarp();
      }
      const int lim[2] = {min(row[0].end, it.k1) - key0, min(row[1].end, it.k1) - key0};
      if (hi) mma_stage<true>(w, smem_u32(sK), smem_u32(sV), lim, lane);
      else mma_stage<false>(w, smem_u32(sK), smem_u32(sV), lim, lane);
      __syncwarp();  // reads of this stage, then the copy that the next load() starts into it
    }
    if (late) break;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float l = w.l[r];
      l += __shfl_xor_sync(~0u, l, 1);
      l += __shfl_xor_sync(~0u, l, 2);
      if (row[r].m < 0) continue;
      if (a.direct) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint32_t *dst = reinterpret_cast<uint32_t *>(a.O + (int64_t)row[r].m * a.ldo +
                                                     row[r].h * kPageHd + (lane & 3) * 2);
#pragma unroll
        for (int d = 0; d < 8; ++d)
          dst[4 * d] = pack_bf2(w.o[d][2 * r] * inv, w.o[d][2 * r + 1] * inv);
      } else {
        const int64_t id = (int64_t)row[r].m * (a.n_kv * a.g) + row[r].h;
        if (it.begins && (lane & 3) == 0) {
          if (it.b < 0) {
            a.shares[id] = me;
            a.shares[a.rows + id] = it.warps;
          } else {
            a.shares[2 * a.rows + id] = me << 16 | it.warps;
          }
        }
        const int64_t at = it.begins && it.ends
                               ? (it.b < 0 ? a.part_p : a.part_t) + id
                               : a.part_f + (me * 2 + it.begins) * kRows + (lane >> 2) + 8 * r;
        float2 *dst = reinterpret_cast<float2 *>(a.Op + at * kPageHd + (lane & 3) * 2);
#pragma unroll
        for (int d = 0; d < 8; ++d) dst[4 * d] = make_float2(w.o[d][2 * r], w.o[d][2 * r + 1]);
        if ((lane & 3) == 0) a.ml[at] = make_float2(w.m[r] * kScale2, l);
      }
    }
  }
  // This kernel's end is to mean the other's too, for which one CTA waits; the rest make room
  // for CTAs that have not run yet (all waiting: 76.0 instead of 75.3 us for 96 rows behind
  // 32832 keys, 68 instead of 64 for 8 padded prompts behind 4000).
  if (a.behind && blockIdx.x == gridDim.x - 1) pdl_wait();
}

// ---------------------------------------------------------------------------
// Items of up to 256 rows on tcgen05 (kind::f16): a CTA holds a pair of 128-row
// Q tiles and streams 128-key blocks of K and V past both, so a block is read
// from memory once for 256 rows. Warps:
//   0-3, 4-7  softmax of group 0 and 1: a thread a row (TMEM lane), the row's
//             128 scores of a block in registers
//   8         TMA (a box a page, or 64 rows of a larger one)
//   9, 10     issue the MMAs of group 0 and 1: S = Q K^T (128 columns), then
//             O += P V with P read from TMEM, where the softmax left it as bf16,
//             so that neither P nor its re-reads pass through shared memory
//             (one thread for both groups was late for each: S and O came 400
//             cycles after they were wanted, of 3400 a block); 9 owns TMEM
// Each group has S (128 columns), P (64) and O (64): all 512 columns. S is free
// once a group holds it in registers, so S of the next block is formed while
// the exponentials of this one run, and the groups' MMAs overlap each other's
// softmax. A single tile (the last rows, or few of them) is worked on by both
// groups, a block each in turn, which are joined at the end.
// Bound by the exponentials and what goes with them: a pair of tiles takes some
// 2900-3200 cycles a block; 2 x 128 x 128 exponentials alone take 2400 (9.4 cycles a
// warp's instruction, measured), the MMAs 1530. Tried and slower: a fourth or more
// of the exponentials as polynomials on the multiply-add units (77 us with 1/8, 83
// with 3/8, as without: 77, of which this kernel is 47); two warps a quarter-tile,
// half a row each (67 against 49 us); scores read from TMEM twice in rolled loops
// (58 against 47); no turns (52 against 47). A CTA spends some 14000 cycles outside
// its blocks (plan, rows, Q, first scores, output), which across_of counts.
// ---------------------------------------------------------------------------
namespace {

constexpr int kBoxRows = 64;  // at most, of a TMA box
constexpr int kTcStages = 5;
constexpr uint32_t kTcTile = kTcKeys * 128;  // Q tile, or K or V of a block: 16 KB
constexpr int kTcTmaWarp = 8, kTcMmaWarp = 9;
constexpr int kTcThreads = 12 * 32;  // three warpgroups; the last warp only passes registers
constexpr int kTcSoftThreads = 8 * 32;
constexpr uint32_t kColS = 0, kColP = 128, kColO = 192, kColGroup = 256;
constexpr int kErrTc = 0x1610;

struct TcCtl {
  uint64_t q_full;
  uint64_t kv_full[kTcStages], kv_empty[kTcStages];
  uint64_t s_full[2], s_free[2], p_full[2], o_done[2];
  uint64_t turn[2][4];  // group g's, of a quarter
  uint64_t v_ready, drain;
  uint32_t tmem_base;
  int abort_flag;
  int cut;  // the block inside which the positions end that some query sees, -1: none
  int idle[8];
  float2 ml[kTileRows];  // group 1's, where both groups work on one tile
};

struct TcItem {
  int b, kvh;      // sequence, -1: rows of all
  int r0, r1;      // rows among the (m, g) rows of b, or of all that hold a query
  int k0, k1, n_valid;
  int split, splits;  // of the rows' items over their keys
};

// The items over the prefix; how many rows of a padded batch hold a query is known here only.
__device__ __forceinline__ Across plan_across(const ApArgs &a, int lane) {
  if (!a.n_new) return a.across;
  int valid = 0;
#pragma unroll 4
  for (int b = lane; b < a.n_seq; b += 32) valid += seq_new(a, b);
  valid = __reduce_add_sync(~0u, valid);
  Across p = across_of(valid * a.g, a.n_kv, a.n_shared, lane + 1, a.tc);
  int best = p.cost << 5 | lane;  // a lane a choice
#pragma unroll
  for (int d = 16; d; d >>= 1) best = min(best, __shfl_xor_sync(~0u, best, d));
  p.c2 = __shfl_sync(~0u, p.c2, best & 31);
  p.s2 = __shfl_sync(~0u, p.s2, best & 31);
  p.c1 = __shfl_sync(~0u, p.c1, best & 31);
  p.s1 = __shfl_sync(~0u, p.s1, best & 31);
  return p;
}

__device__ __forceinline__ TcItem get_tc_item(const ApArgs &a, int idx, int lane) {
  TcItem it;
  it.split = 0;
  if (a.by_seq) {
    // the last rows of a sequence see furthest: those items first
    int q = idx / a.splits;
    it.split = idx - q * a.splits;
    it.kvh = q % a.n_kv;
    q /= a.n_kv;
    it.b = q % a.n_seq;
    const int pair = a.pairs - 1 - q / a.n_seq;
    const int nn = seq_new(a, it.b);
    it.n_valid = seq_len(a, it.b);
    it.r0 = pair * kPairRows;
    it.r1 = min(it.r0 + kPairRows, nn * a.g);
    const int end = it.r1 > it.r0 ? max(it.n_valid - nn + (it.r1 - 1) / a.g + 1, 0) : 0;
    it.splits = (end + a.chunk - 1) / a.chunk;
    it.k0 = it.split * a.chunk;
    it.k1 = min(it.k0 + a.chunk, end);
    return it;
  }
  const Across p = plan_across(a, lane);
  const int full = p.pairs * p.s2, each = full + p.s1;
  it.b = -1;
  it.kvh = each ? idx / each : a.n_kv;
  it.r0 = it.r1 = it.k0 = it.k1 = it.splits = 0;
  it.n_valid = a.n_shared;
  if (it.kvh >= a.n_kv) return it;  // one CTA too many
  const int q = idx - it.kvh * each;
  const bool one = q >= full;
  const int pair = one ? p.pairs : q / p.s2;
  const int chunk = one ? p.c1 : p.c2;
  it.split = one ? q - full : q - pair * p.s2;
  it.splits = one ? p.s1 : p.s2;
  it.r0 = pair * kPairRows;
  it.r1 = min(it.r0 + kPairRows, p.rows);
  it.k0 = it.split * chunk;
  it.k1 = min(it.k0 + chunk, a.n_shared);
  return it;
}

// Row R of the item, for a lane of a converged warp. Among the packed rows of a padded batch the
// sequence is searched for, 32 at a time.
__device__ __forceinline__ Row get_tc_row(const ApArgs &a, const TcItem &it, int R, int lane) {
  Row w;
  w.m = -1;
  w.h = w.end = 0;
  const int j = quot(R, a.by_g);  // query among it.b's, or among all
  int b = it.b, t = j;
  if (b < 0 && !a.n_new) {
    b = quot(j, a.by_T);
    t = j - b * a.T;
  } else if (b < 0) {
    int start = 0;
    for (int base = 0; base < a.n_seq; base += 32) {
      int upto = base + lane < a.n_seq ? seq_new(a, base + lane) : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(~0u, upto, d);
        if (lane >= d) upto += y;
      }
      const int in = __shfl_sync(~0u, upto, 31);
      const bool mine = j >= start && j < start + in;
      if (__any_sync(~0u, mine)) {
        int l = 0, before = 0;  // lanes whose sequences end at or before j
#pragma unroll
        for (int d = 16; d; d >>= 1) {
          const int y = __shfl_sync(~0u, upto, l + d - 1);
          if (y <= j - start) {
            l += d;
            before = y;
          }
        }
        if (mine) {
          b = base + l;
          t = j - start - before;
        }
      }
      start += in;
      if (__all_sync(~0u, j < start || R >= it.r1)) break;
    }
  }
  if (R < it.r1) {
    w.h = it.kvh * a.g + (R - j * a.g);
    w.m = b * a.T + t;
    w.end = seq_len(a, b) - seq_new(a, b) + t + 1;
  }
  return w;
}

}  // namespace

__global__ void __launch_bounds__(kTcThreads, 1)
    attention_pages_tc_kernel(const __grid_constant__ CUtensorMap tmK,
                              const __grid_constant__ CUtensorMap tmV,
                              const __grid_constant__ ApArgs a) {
  // (an address known when this is compiled: no register holds it; 96 rows of 32 heads behind
  // 32832 keys: 77.5 -> 75.9 us a call)
  extern __shared__ __align__(1024) uint8_t smem_tc[];
  uint8_t *smem = smem_tc;
  if (smem_u32(smem) & 1023) {
    if (threadIdx.x == 0) report_error(a.err, kErrTc + 12);
    return;
  }
  uint8_t *sQ = smem;                       // [2] tiles
  uint8_t *sKV = smem + 2 * kTcTile;        // [stages] K, V
  TcCtl *ctl = reinterpret_cast<TcCtl *>(sKV + kTcStages * 2 * kTcTile);
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();  // (after the wait: see attention_pages_mma_kernel)
  const TcItem it = get_tc_item(a, blockIdx.x, lane);
  const int n_rows = it.r1 - it.r0;
  const int blocks = it.k1 > it.k0 ? (it.k1 - it.k0 + kTcKeys - 1) / kTcKeys : 0;
  if (n_rows <= 0) return;
  const bool one = n_rows <= kTileRows;      // both groups on one tile
  // an item without keys leaves no part, unless rows get their zeros here
  if (blocks == 0 && !a.direct && it.split > 0) return;
  const int units = one ? blocks : 2 * blocks;  // unit u: group u & 1
  if (threadIdx.x == 0) {
    mbar_init(&ctl->q_full, 8);
    for (int i = 0; i < kTcStages; ++i) {
      mbar_init(&ctl->kv_full[i], 1);
      mbar_init(&ctl->kv_empty[i], 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->s_full[i], 1);
      mbar_init(&ctl->s_free[i], 4);
      mbar_init(&ctl->p_full[i], 4);
      mbar_init(&ctl->o_done[i], 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(&ctl->turn[i >> 2][i & 3], 1);
    mbar_init(&ctl->v_ready, 1);
    mbar_init(&ctl->drain, 2);
    ctl->abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (warp == kTcMmaWarp) {
    tmem_alloc(&ctl->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem_base;
  volatile int *abort_flag = &ctl->abort_flag;

  if (warp < 8) {
    reg_alloc<208>();  // 256 x 208 + 128 x 88 are the launch's 384 x 168
    // ---------------- softmax ----------------
    const int g = warp >> 2, qd = warp & 3;
    const int r = qd * 32 + lane;  // TMEM lane
    const Row row = get_tc_row(a, it, it.r0 + (one ? 0 : g) * kTileRows + r, lane);
    const bool idle = __all_sync(~0u, row.m < 0);  // no rows in this warp
    const uint32_t trow = tmem + g * kColGroup + ((uint32_t)(qd * 32) << 16);
    // Q row into its swizzled place
    if (!one || g == 0) {
      uint8_t *dst = sQ + g * kTcTile + r * 128;
      const uint4 *src = reinterpret_cast<const uint4 *>(a.Q + (int64_t)row.m * a.ldq + row.h * kPageHd);
      uint4 v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = row.m >= 0 ? src[i] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4 *>(dst + ((i ^ (r & 7)) * 16)) = v[i];
      fence_proxy_async_smem();
    }
    __syncwarp();
    if (lane == 0) {
      ctl->idle[warp] = idle;
      mbar_arrive(&ctl->q_full);
    }
    named_barrier_sync(1, kTcSoftThreads);
    // The two warps of an SM quarter take turns at the exponentials, so that one's fill the
    // other's loads, maxima and hand-overs; a warp without rows needs no turn.
    const bool turns = !idle && !ctl->idle[warp ^ 4];

    float m = -INFINITY, l = 0.0f;  // m: score that weights refer to, unscaled
    const int mine = g < units ? (units - g + 1) / 2 : 0;  // this group's units
    bool ok = true;
    for (int i = 0; i < mine && ok; ++i) {
      const int key0 = it.k0 + (one ? 2 * i + g : i) * kTcKeys;
      // P of the last unit has been read, and O is complete up to it
      auto last_done = [&]() {
        return i == 0 || __all_sync(~0u, mbar_wait(&ctl->o_done[g], (i - 1) & 1, abort_flag, a.err,
                                                   kErrTc + 8));
      };
      ok = __all_sync(~0u, mbar_wait(&ctl->s_full[g], i & 1, abort_flag, a.err, kErrTc + 7));
      if (!ok) break;
      if (idle) {
        if (lane == 0) mbar_arrive(&ctl->s_free[g]);
        ok = last_done();  // (p_full's phases must not run into one another)
        if (lane == 0 && ok) mbar_arrive(&ctl->p_full[g]);
        continue;
      }
      tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(trow + kColS + 32 * c, s[c]);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->s_free[g]);
      // keys of this block that the row sees
      const int lim = min(row.end, it.k1) - key0;
      if (__any_sync(~0u, lim < kTcKeys)) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (32 * c + k >= lim) s[c][k] = 0xff800000u;  // -inf
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        mx[c] = fmaxf(__uint_as_float(s[c][0]), __uint_as_float(s[c][1]));
#pragma unroll
      for (int k = 2; k < 32; k += 2)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          mx[c] = max3(mx[c], __uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1]));
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const bool up = grown(top, m);
      float f = 1.0f;
      if (up) {
        f = ex2((m - top) * kScale2);  // 0 at the first key (m = -inf)
        m = top;
        l *= f;
      }
      const bool rescale = i > 0 && __any_sync(~0u, up);
      const float ms = safe_max(m) * kScale2;
      ok = last_done();
      if (!ok) break;
      tc_fence_after();
      if (rescale) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(trow + kColO + 32 * c, o);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
          tmem_st_32x32b_x32(trow + kColO + 32 * c, o);
        }
      }
      if (turns && (g == 1 || i > 0)) {
        ok = __all_sync(~0u, mbar_wait(&ctl->turn[g][qd], (i - 1 + g) & 1, abort_flag, a.err,
                                       kErrTc + 11));
        if (!ok) break;
      }
      // Weights, 32 keys at a time: the exponentials of a chunk are issued between the scaling of
      // the next chunk and the sums and packing of the last, whose results have arrived by then
      // (a warp issues in order and would otherwise wait for each). Scaling and sums work on
      // pairs (f32x2).
      const F2 scale2 = f2(kScale2, kScale2), minus = f2(-ms, -ms);
      F2 sum[4] = {0, 0, 0, 0};  // (of zeros)
      uint32_t p[2][32];
      auto pair = [&](int c, int k) {
        return f2(__uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1]));
      };
      auto put = [&](int c, int k, F2 v) {
        float x, y;
        f2_split(v, x, y);
        s[c][k] = __float_as_uint(x);
        s[c][k + 1] = __float_as_uint(y);
      };
      auto scale = [&](int c, int k) { put(c, k, f2_fma(pair(c, k), scale2, minus)); };
      auto take = [&](int c, int k) {  // keys k, k + 1
        sum[(k >> 1) & 3] = f2_add(sum[(k >> 1) & 3], pair(c, k));
        p[c >> 1][16 * (c & 1) + k / 2] =
            pack_bf2(__uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1]));
      };
#pragma unroll
      for (int k = 0; k < 32; k += 2) scale(0, k);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          s[c][k] = __float_as_uint(ex2(__uint_as_float(s[c][k])));
          s[c][k + 1] = __float_as_uint(ex2(__uint_as_float(s[c][k + 1])));
          if (c < 3) scale(c + 1, k);
          if (c > 0) take(c - 1, k);
        }
        if (c == 2) tmem_st_32x32b_x32(trow + kColP, p[0]);
      }
      if (turns && lane == 0) mbar_arrive(&ctl->turn[g ^ 1][qd]);
#pragma unroll
      for (int k = 0; k < 32; k += 2) take(3, k);
      tmem_st_32x32b_x32(trow + kColP + 32, p[1]);
      {
        float x, y;
        f2_split(f2_add(f2_add(sum[0], sum[1]), f2_add(sum[2], sum[3])), x, y);
        l += x + y;
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->p_full[g]);
    }
    if (mine > 0 && ok)
      ok = __all_sync(~0u, mbar_wait(&ctl->o_done[g], (mine - 1) & 1, abort_flag, a.err,
                                     kErrTc + 9));
    tc_fence_after();
    // ---- output: m in base 2 from here on ----
    m *= kScale2;
    if (one) {
      if (g == 1) ctl->ml[r] = make_float2(m, l);
      tc_fence_before();
      named_barrier_sync(1, kTcSoftThreads);
      tc_fence_after();
    }
    if ((!one || g == 0) && !idle && ok && !*abort_flag) {
      float f0 = 1.0f, f1 = 0.0f, l_all = l, m_all = m;
      const bool second = one && units > 1;  // group 1 has a share
      if (second) {
        const float2 w = ctl->ml[r];
        m_all = fmaxf(m, w.x);
        const float ms = safe_max(m_all);
        f0 = ex2(m - ms);
        f1 = ex2(w.x - ms);
        l_all = f0 * l + f1 * w.y;
      }
      const float inv = l_all == 0.0f ? 0.0f : 1.0f / l_all;
      const int at = blockIdx.x * kPairRows + g * kTileRows + r;
      // Rows leave through this warp's share of its Q tile, which no product reads any more, 32
      // dims at a time: a lane's row in, eight lanes a row out, four lines a store (a lane a row
      // would touch 32 lines with each).
      uint8_t *buf = sQ + g * kTcTile + qd * 32 * 128;
      const int sub = lane >> 3, chunk = lane & 7;
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        float x[32];
        {
          uint32_t o[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0u;
          if (mine > 0) tmem_ld_32x32b_x32(trow + kColO + 32 * half, o);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 32; ++k) x[k] = __uint_as_float(o[k]);
        }
        if (second) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(trow + kColGroup + kColO + 32 * half, o);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 32; ++k) x[k] = f0 * x[k] + f1 * __uint_as_float(o[k]);
        }
        const float scale = a.direct ? inv : 1.0f;
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          *reinterpret_cast<float4 *>(buf + lane * 128 + ((k ^ (lane & 7)) * 16)) =
              make_float4(x[4 * k] * scale, x[4 * k + 1] * scale, x[4 * k + 2] * scale,
                          x[4 * k + 3] * scale);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int q = 4 * i + sub;
          const float4 y =
              *reinterpret_cast<const float4 *>(buf + q * 128 + ((chunk ^ (q & 7)) * 16));
          const int m = __shfl_sync(~0u, row.m, q), h = __shfl_sync(~0u, row.h, q);
          if (m < 0) continue;
          const int d0 = 32 * half + 4 * chunk;
          if (a.direct) {
            uint32_t *dst =
                reinterpret_cast<uint32_t *>(a.O + (int64_t)m * a.ldo + h * kPageHd + d0);
            dst[0] = pack_bf2(y.x, y.y);
            dst[1] = pack_bf2(y.z, y.w);
          } else {
            *reinterpret_cast<float4 *>(a.Op + (int64_t)(at - lane + q) * kPageHd + d0) = y;
          }
        }
      }
      if (row.m >= 0 && !a.direct) {
        a.ml[at] = make_float2(m_all, l_all);
        if (it.split == 0) {
          const int64_t id = (int64_t)row.m * (a.n_kv * a.g) + row.h;
          a.shares[id] = at;
          a.shares[a.rows + id] = it.splits;
        }
      }
    }
  } else {
    reg_dealloc<88>();
  if (warp == kTcTmaWarp) {
    // ---------------- TMA: lane i < 2 * boxes issues one box of a block ----------------
    const int box = min(1 << a.page_shift, kBoxRows);
    const int boxes = kTcKeys / box;
    const bool act = lane < 2 * boxes;
    const bool is_v = lane >= boxes;
    const int bx = is_v ? lane - boxes : lane;
    // page of this lane's box of a block, as the lists have it (any value behind the item's keys)
    auto fetch = [&](int j) -> int {
      const int pos = it.k0 + j * kTcKeys + bx * box, k = pos >> a.page_shift;
      if (!act || pos >= it.k1) return -1;
      if (pos < a.n_shared) return a.shared[k];
      return k < a.max_pages ? a.table[(int64_t)it.b * a.max_pages + k] : -1;
    };
    int p = blocks ? fetch(0) : 0;
    // Positions that some query sees (see all_stages), counted while the first entries arrive;
    // no other warp waits for it (all of them: 75 -> 77 us for 96 rows behind 32832 keys). Boxes
    // behind read as zeros, and the rest of a block inside which they end is overwritten.
    int valid = it.n_valid;
    if (it.b < 0) {
      int seen = 0;
#pragma unroll 4
      for (int b = lane; b < a.n_seq; b += 32)
        if (seq_new(a, b) > 0) seen = max(seen, seq_len(a, b));
      valid = min(__reduce_max_sync(~0u, seen), a.n_shared);
    }
    const int k1 = min(it.k1, valid), rest = valid - it.k0;
    const int cut = rest > 0 && rest < blocks * kTcKeys && rest % kTcKeys ? rest / kTcKeys : -1;
    if (lane == 0) ctl->cut = cut;  // (released by the first arrival below)
    int n = 0;
    for (; n < blocks; ++n) {
      const int next = n + 1 < blocks ? fetch(n + 1) : 0;
      const int st = n % kTcStages;
      const int pos = it.k0 + n * kTcKeys + bx * box;
      if (!act || pos >= k1) {
        p = a.n_pages;  // reads as zeros
      } else if (p < 0 || p >= a.n_pages) {
        report_error(a.err, kErrEntry);
        p = a.n_pages;
      }
      bool ok = true;
      if (n >= kTcStages)
        ok = mbar_wait(&ctl->kv_empty[st], ((n / kTcStages) & 1) ^ 1, abort_flag, a.err, kErrTc);
      if (!__all_sync(~0u, ok)) break;
      if (lane == 0) mbar_arrive_expect_tx(&ctl->kv_full[st], 2 * kTcTile);
      __syncwarp();
      if (act) {
        const int y = (it.kvh << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
        tma_load_3d(sKV + (st * 2 + is_v) * kTcTile + bx * box * 128, is_v ? &tmV : &tmK,
                    &ctl->kv_full[st], 0, y, p);
      }
      p = next;
      if (n == cut && __all_sync(~0u, mbar_wait(&ctl->kv_full[st], (n / kTcStages) & 1, abort_flag,
                                                a.err, kErrTc + 1))) {
        uint8_t *v = sKV + (st * 2 + 1) * kTcTile;
        for (int x = rest % kTcKeys * 8 + lane; x < kTcKeys * 8; x += 32)
          *reinterpret_cast<uint4 *>(v + x * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->v_ready);
      }
    }
    if (*abort_flag)  // no copy may still be writing shared memory when the CTA exits
      for (int i = n > kTcStages ? n - kTcStages : 0; i < n; ++i)
        mbar_wait(&ctl->kv_full[i % kTcStages], (i / kTcStages) & 1, nullptr, a.err, kErrTc + 1);
  } else if (warp == kTcMmaWarp || warp == kTcMmaWarp + 1) {
    // ---------------- MMA of one group: one thread ----------------
    const int g = warp - kTcMmaWarp;
    if (elect_one()) {
      const uint32_t idS = make_idesc(1, 1, kTileRows, kTcKeys);
      const uint32_t idO = make_idesc_bmn(1, 1, kTileRows, kPageHd);
      const uint64_t q_desc = make_sw128_desc(smem_u32(sQ)) + (one ? 0 : g) * (kTcTile >> 4);
      const uint64_t k_desc = make_sw128_desc(smem_u32(sKV));
      const uint64_t v_desc = make_sw128_mn_desc(smem_u32(sKV) + kTcTile);
      const uint32_t base = tmem + g * kColGroup;
      const int mine = (units - g + 1) / 2;
      bool ok = mine > 0 && mbar_wait(&ctl->q_full, 0, abort_flag, a.err, kErrTc + 2);
      int seen = 0;  // blocks that have been in shared memory
      int cut = -1;
      auto issue_s = [&](int i) -> bool {
        const int j = one ? 2 * i + g : i;  // block
        if (i > 0 && !mbar_wait(&ctl->s_free[g], (i - 1) & 1, abort_flag, a.err, kErrTc + 3))
          return false;
        for (;; ++seen) {
          const int st = seen % kTcStages;
          if (!mbar_wait(&ctl->kv_full[st], (seen / kTcStages) & 1, abort_flag, a.err, kErrTc + 4))
            return false;
          if (seen == j) break;
          mbar_arrive(&ctl->kv_empty[st]);  // the other group's: a stage is freed by both
        }
        ++seen;
        tc_fence_after();
        tc_mma_bf16_x4(base + kColS, q_desc, k_desc + (j % kTcStages) * (2 * kTcTile >> 4), idS);
        tc_commit(&ctl->s_full[g]);
        return true;
      };
      auto issue_o = [&](int i) -> bool {
        const int j = one ? 2 * i + g : i;
        if (!mbar_wait(&ctl->p_full[g], i & 1, abort_flag, a.err, kErrTc + 5)) return false;
        if (j == cut && !mbar_wait(&ctl->v_ready, 0, abort_flag, a.err, kErrTc + 10)) return false;
        tc_fence_after();
        tc_mma_bf16_ta_x8(base + kColO, base + kColP, v_desc + (j % kTcStages) * (2 * kTcTile >> 4),
                          idO, i > 0);
        tc_commit(&ctl->o_done[g]);
        tc_commit(&ctl->kv_empty[j % kTcStages]);
        return true;
      };
      if (ok) ok = issue_s(0);
      if (ok) cut = *(volatile int *)&ctl->cut;  // written before the first block's arrival
      for (int i = 0; i < mine && ok; ++i) {
        if (i + 1 < mine) ok = issue_s(i + 1);
        if (ok) ok = issue_o(i);
      }
      // no MMA may still be writing TMEM when it is released
      tc_commit(&ctl->drain);
      mbar_wait(&ctl->drain, 0, nullptr, a.err, kErrTc + 6);
    }
    __syncwarp();
  }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kTcMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// The join of a row's parts: eight lanes, eight dims a lane, four parts' loads in
// flight; SUB = 4 such groups share a row's parts where there are few rows, since
// a row's chain of dependent reads (length, words of the row, parts) is the time
// of the kernel then.
// ---------------------------------------------------------------------------
template <int SUB>
__global__ void __launch_bounds__(256)
    attention_pages_join_kernel(const __grid_constant__ ApArgs a) {
  constexpr int kLanes = 8 * SUB;
  const int64_t row = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const int d0 = (threadIdx.x & 7) * 8, sub = threadIdx.x / 8 % SUB;
  pdl_launch_dependents();
  pdl_wait();
  if (row >= a.rows) return;
  const int m = quot((int)row, a.by_head), h = (int)row - m * (a.n_kv * a.g);
  const int b = quot(m, a.by_T), t = m - b * a.T;
  // words of a row are read before it is known which of them hold anything
  const int first = a.shares[row], n_first = a.shares[a.rows + row];
  const int tail_word = a.shares[2 * a.rows + row];
  if (t >= seq_new(a, b)) return;
  const int n1 = a.tc || a.p_stages ? min(max(n_first, 0), 0xffff) : 0;
  const int tail = !a.by_seq && tail_stages(a, seq_len(a, b)) > 0 ? tail_word : 0;
  const int n2 = n1 + (tail & 0xffff);
  const int gi = h - quot(h, a.by_g) * a.g;
  const int R = (m * a.g + gi) & (kRows - 1), Rt = (t * a.g + gi) & (kRows - 1);  // in their tiles
  // parts: of the prefix (or of all keys), then of the tail
  auto part = [&](int i) -> int64_t {
    if (i < n1 && a.tc) return (int64_t)first + i * kPairRows;
    if (i < n1)
      return n1 == 1 ? a.part_p + row
                     : a.part_f + (((int64_t)first + i) * 2 + (i == 0)) * kRows + R;
    i -= n1;
    return (tail & 0xffff) == 1 ? a.part_t + row
                                : a.part_f + (((tail >> 16) + i) * 2 + (i == 0)) * kRows + Rt;
  };
  float mx = -INFINITY, l = 0.0f, acc[8] = {};
  for (int i0 = 4 * sub; i0 < n2; i0 += 4 * SUB) {
    float2 v[4];
    float4 x[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int64_t at = i0 + i < n2 ? part(i0 + i) : -1;
      // (words that a kernel which gave up on a wait has not written may hold anything)
      const bool live = at >= 0 && at < a.parts;
      if (!live) at = 0;
      const float4 *src = reinterpret_cast<const float4 *>(a.Op + at * kPageHd + d0);
      v[i] = live ? a.ml[at] : make_float2(-INFINITY, 0.0f);
      x[i][0] = live ? src[0] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      x[i][1] = live ? src[1] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    const float top = fmaxf(fmaxf(fmaxf(v[0].x, v[1].x), fmaxf(v[2].x, v[3].x)), mx);
    const float ms = safe_max(top), f = ex2(mx - ms);
    mx = top;
    l *= f;
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[d] *= f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i0 + i >= n2) break;
      const float w = ex2(v[i].x - ms);
      l += w * v[i].y;
      const float y[8] = {x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w,
                          x[i][1].x, x[i][1].y, x[i][1].z, x[i][1].w};
#pragma unroll
      for (int d = 0; d < 8; ++d) acc[d] += w * y[d];
    }
  }
  if constexpr (SUB > 1) {  // (a row is left by all of a warp or by none)
    static_assert(kLanes == 32, "a warp a row");
#pragma unroll
    for (int x = 8; x < kLanes; x *= 2) {
      const float other = __shfl_xor_sync(~0u, mx, x), top = fmaxf(mx, other);
      const float f = ex2(mx - safe_max(top));
      mx = top;
      l *= f;
      l += __shfl_xor_sync(~0u, l, x);
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        acc[d] *= f;
        acc[d] += __shfl_xor_sync(~0u, acc[d], x);
      }
    }
    if (sub != 0) return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint32_t *dst = reinterpret_cast<uint32_t *>(a.O + m * a.ldo + h * kPageHd + d0);
#pragma unroll
  for (int d = 0; d < 4; ++d) dst[d] = pack_bf2(acc[2 * d] * inv, acc[2 * d + 1] * inv);
}

// ---------------------------------------------------------------------------
// plan and launch
// ---------------------------------------------------------------------------
namespace {

struct Plan {
  int tc_grid;     // CTAs of the tensor-core kernel, 0: not launched
  bool by_seq;     // they cover everything
  int pairs, splits, chunk;
  int grid;        // CTAs of the 16-row kernel, 0: not launched
  int p_tiles, p_stages, base, whole;
  bool direct;
  int64_t part_p, part_t, part_f, parts;
};

int64_t cdiv(int64_t x, int64_t y) { return (x + y - 1) / y; }

// W8A8_ERR_UNSUPPORTED: more items or stages than 32 bits count.
int make_plan(int n_seq, int T, int n_head, int n_kv, int max_ctx, int n_shared, Plan *out) {
  Plan p = {};
  const int g = n_head / n_kv;
  const int64_t own = (int64_t)T * g, all = own * n_seq;  // rows of a key head
  const int64_t rows = all * n_kv;
  const int tail = max_ctx - n_shared > 0 ? max_ctx - n_shared : 1;
  int64_t tc_grid = 0;
  // A sequence's rows over prefix and tail in one tensor-core item, or all rows over the prefix
  // and the tails to the 16-row kernel: by the time that one SM takes, where a 128 x 128 block
  // counts as 5.5 stages of 16 rows by 64 keys (1640 cycles, and some 300 with seven warps).
  const int64_t heads = (int64_t)n_seq * n_kv;
  const int64_t one_item = heads * cdiv(own, kTileRows) * cdiv(n_shared + tail, kTcKeys) * 11;
  const int64_t two_items = n_kv * cdiv(all, kTileRows) * cdiv(n_shared, kTcKeys) * 11 +
                            heads * cdiv(own, kRows) * cdiv(tail, kStageKeys) * 2;
  if (own > 2 * kRows && one_item < two_items) {
    // Chunks for two CTAs an SM, of eight blocks at least.
    p.by_seq = true;
    p.pairs = (int)cdiv(own, kPairRows);
    const int64_t groups = (int64_t)n_seq * n_kv * p.pairs;
    int64_t c = cdiv(cdiv(max_ctx, cdiv(2 * kSms, groups)), kTcKeys) * kTcKeys;
    p.chunk = (int)(c < 8 * kTcKeys ? 8 * kTcKeys : c);
    p.splits = (int)cdiv(max_ctx, p.chunk);
    tc_grid = groups * p.splits;
    p.direct = p.splits == 1;
  } else {
    const int64_t p_stages = cdiv(n_shared, kStageKeys), p_tiles = cdiv(all, kRows);
    const int64_t t_stages = cdiv(tail, kStageKeys), t_tiles = cdiv(own, kRows);
    const int64_t pre = n_kv * p_tiles * p_stages, groups = n_seq * t_tiles * n_kv;
    const int64_t a_stages = cdiv(max_ctx, kStageKeys);
    int64_t stages = groups * t_stages;
    p.base = n_shared;
    if (pre > kMinTcStages && all > kRows) {
      // a CTA for each pair at least, and room for two rounds of them
      tc_grid = n_kv * cdiv(all, kPairRows);
      if (tc_grid < 2 * kSms) tc_grid = 2 * kSms;
    } else if (a_stages <= 4 && (n_shared == 0 || groups <= kSms * kMmaWarps)) {
      // short sequences, a group a warp if they share anything: whole groups, which read what is
      // shared for themselves, and no join (2 sequences of 96, 64 shared: 14.0 -> 10.4 us a call)
      p.base = 0;
      p.whole = (int)a_stages;
      p.direct = true;
      stages = groups * a_stages;
    } else if (n_shared > 0) {
      p.p_tiles = (int)p_tiles;
      p.p_stages = (int)p_stages;
      stages += pre;
    }
    if (stages > 0x7fffffff - kSms * kMmaWarps) return W8A8_ERR_UNSUPPORTED;
    const int64_t work = p.whole ? stages / p.whole : stages;
    p.grid = (int)(work < kSms ? work : kSms);
    p.part_p = tc_grid * kPairRows;
    p.part_t = p.part_p + (p.p_stages ? rows : 0);
    p.part_f = p.part_t + rows;
    // warps with a stretch
    p.parts = p.part_f + (work < kSms * kMmaWarps ? work : kSms * kMmaWarps) * 2 * kRows;
  }
  if (tc_grid > 0x7fffffff / kPairRows) return W8A8_ERR_UNSUPPORTED;
  p.tc_grid = (int)tc_grid;
  if (p.by_seq) p.parts = tc_grid * kPairRows;
  if (p.direct) p.parts = 0;
  *out = p;
  return W8A8_OK;
}

// Shared-memory opt-in of a kernel on the current device, once.
template <typename K>
int opt_in_smem(K *kernel, size_t bytes, bool (&done)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return W8A8_ERR_CUDA;
  if (!done[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) !=
        cudaSuccess)
      return W8A8_ERR_CUDA;
    done[dev] = true;
  }
  return W8A8_OK;
}

}  // namespace

// Parts of rows (64 sums, a maximum and a sum of weights each), and three words a row.
int attention_pages_workspace(int n_seq, int T, int n_head, int n_kv, int max_ctx, int n_shared,
                              size_t *bytes) {
  Plan p;
  const int st = make_plan(n_seq, T, n_head, n_kv, max_ctx, n_shared, &p);
  if (st) return st;
  *bytes = p.direct ? 16
                    : (size_t)p.parts * (kPageHd * sizeof(float) + sizeof(float2)) +
                          3 * sizeof(int) * (size_t)n_seq * T * n_head;
  return W8A8_OK;
}

int launch_attention_pages(const PagesArgs &c, const AttnPagesCall &q, cudaStream_t s) {
  const int g = q.n_head / c.n_kv_head;
  Plan p;
  int st = make_plan(q.n_seq, q.T, q.n_head, c.n_kv_head, q.max_ctx, q.n_shared, &p);
  if (st) return st;
  ApArgs a = {};
  a.Q = q.Q;
  a.ldq = q.ldq;
  a.O = q.O;
  a.ldo = q.ldo;
  a.table = c.table;
  a.n_ctx = c.n_ctx;
  a.n_new = q.n_new;
  a.shared = q.shared;
  a.max_pages = c.max_pages;
  a.n_pages = c.n_pages;
  a.page_shift = __builtin_ctz((unsigned)c.page);
  a.n_seq = q.n_seq;
  a.T = q.T;
  a.g = g;
  a.n_kv = c.n_kv_head;
  a.max_ctx = q.max_ctx;
  a.n_shared = q.n_shared;
  a.p_tiles = p.p_tiles;
  a.p_stages = p.p_stages;
  a.base = p.base;
  a.whole = p.whole;
  a.by_seq = p.by_seq;
  a.pairs = p.pairs;
  a.splits = p.splits;
  a.chunk = p.chunk;
  a.direct = p.direct;
  a.tc = p.tc_grid;
  if (p.tc_grid && !p.by_seq && !q.n_new) {
    // every row holds a query: the items, and no CTA more, are known here
    a.across = across_of(q.n_seq * q.T * g, a.n_kv, a.n_shared, 1, a.tc);
    for (int i = 2; i <= 32; ++i) {
      const Across x = across_of(q.n_seq * q.T * g, a.n_kv, a.n_shared, i, a.tc);
      if (x.cost < a.across.cost) a.across = x;
    }
    p.tc_grid = a.n_kv * (a.across.pairs * a.across.s2 + a.across.s1);
  }
  a.behind = p.tc_grid > 0 && p.grid > 0;
  a.rows = (int64_t)q.n_seq * q.T * q.n_head;
  a.by_g = make_div(g);
  a.by_T = make_div(q.T);
  a.by_head = make_div(q.n_head);
  a.part_p = p.part_p;
  a.part_t = p.part_t;
  a.part_f = p.part_f;
  a.parts = p.parts;
  a.Op = reinterpret_cast<float *>(q.ws);
  a.ml = reinterpret_cast<float2 *>(a.Op + p.parts * kPageHd);
  a.shares = reinterpret_cast<int *>(a.ml + p.parts);
  DeviceCtx *ctx = device_ctx(&st);
  if (!ctx) return st;
  a.err = ctx->err;
  const int64_t off = (int64_t)q.layer * c.n_kv_head * c.page * kPageHd;
  const uint64_t rows = (uint64_t)c.n_kv_head * c.page;
  CUtensorMap tmK, tmV;
  auto maps = [&](int box) {  // of at most `box` rows
    const CUtensorMapDataType bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (c.page < box) box = c.page;
    int e = make_tmap_3d(&tmK, c.K + off, bf, (uint64_t)c.n_pages, rows, kPageHd, kPageHd * 2,
                         (uint64_t)c.page_stride * 2, kPageHd, box);
    return e ? e : make_tmap_3d(&tmV, c.V + off, bf, (uint64_t)c.n_pages, rows, kPageHd,
                                kPageHd * 2, (uint64_t)c.page_stride * 2, kPageHd, box);
  };
  static bool tc_ready[64], mma_ready[64];
  if (p.tc_grid) {
    const size_t smem = 1024 + (2 + 2 * kTcStages) * kTcTile + sizeof(TcCtl);
    st = opt_in_smem(attention_pages_tc_kernel, smem, tc_ready);
    if (st || (st = maps(kBoxRows))) return st;
    launch_pdl(attention_pages_tc_kernel, dim3((unsigned)p.tc_grid), dim3(kTcThreads), smem, s,
               tmK, tmV, a);
    st = check_launch("attention_pages_tc");
    if (st) return st;
  }
  if (p.grid) {
    const size_t smem = 1024 + kMmaWarps * kStages * 2 * kTileBytes + sizeof(MmaSmem);
    st = opt_in_smem(attention_pages_mma_kernel, smem, mma_ready);
    if (st || (st = maps(kStageKeys))) return st;
    launch_pdl(attention_pages_mma_kernel, dim3(p.grid), dim3(kMmaWarps * 32), smem, s, tmK, tmV, a);
    st = check_launch("attention_pages_mma");
    if (st) return st;
  }
  if (a.direct) return W8A8_OK;
  // four groups a row as long as they all run at once (eight CTAs an SM)
  if (a.rows <= (int64_t)kSms * 8 * 8)
    launch_pdl(attention_pages_join_kernel<4>, dim3((unsigned)cdiv(a.rows, 8)), dim3(256), 0, s, a);
  else
    launch_pdl(attention_pages_join_kernel<1>, dim3((unsigned)cdiv(a.rows, 32)), dim3(256), 0, s,
               a);
  return check_launch("attention_pages_join");
}

}  // namespace w8a8

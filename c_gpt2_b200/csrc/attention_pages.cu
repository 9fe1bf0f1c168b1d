// Attention over cache pages with a shared prefix (w8a8_attention_pages).
//
//   O_r = sum_j w_rj V_j / sum_j w_rj,  w_rj = exp(q_r.k_j / 8 - m_r),  j < end_r
//
// formed in one pass over the keys (running maximum and sum; base-2
// exponentials of scores scaled by log2(e) / 8), with fp32 scores, maxima, sums
// and accumulators. The weights are rounded to bf16 for the tensor cores: at
// most half a step, 2^-9 of each weight and of either sign, below the rounding
// of the output itself.
//
// The key axis of a row is cut into the shared prefix and the sequence's own
// tail, and each of those into chunks; every (rows, chunk) pair is an item of
// work that leaves (m, sum, unnormalised O) in the workspace, and a last kernel
// joins a row's items. The prefix items take rows of ALL sequences, so the
// shared pages are read once for 16 rows, not once a sequence.
#include "common.cuh"
#include "kernels.cuh"
#include "runtime.cuh"

#include <math.h>

namespace w8a8 {

namespace {

constexpr int kSms = 148;            // the plan below is made for this many SMs
constexpr float kScale2 = 0.125f * 1.44269504088896340736f;  // log2(e) / sqrt(64)
constexpr int kErrEntry = 0x1601;    // a table entry outside the pool
constexpr int kErrWaitFull = 0x1602, kErrWaitEmpty = 0x1603;

constexpr int kStageKeys = 64;
constexpr int kStages = 5;
constexpr uint32_t kTileBytes = kStageKeys * 128;  // keys or values of a stage
constexpr int kMmaWarps = 4;                       // 16 keys of a stage each
constexpr int kMmaThreads = kMmaWarps * 32 + 32;   // + the TMA warp
constexpr int kRows = 16;                          // query rows of an item
constexpr int kOPitch = 68;                        // floats a row of the join buffer

struct ApArgs {
  const uint16_t *Q;
  int64_t ldq;
  uint16_t *O;
  int64_t ldo;
  const int32_t *table, *n_ctx, *n_new, *shared;
  int max_pages, n_pages, page_shift;
  int n_seq, T, g, n_kv, max_ctx, n_shared;
  // 16-row items: prefix [n_kv][p_tiles][p_splits], then tails
  // [n_seq][n_kv][t_tiles][t_splits]; slots of a row: p_splits of the first kind
  // of item, whichever kernel runs it, then t_splits of tails
  int p_tiles, p_splits, p_chunk;
  int t_tiles, t_splits, t_chunk;
  // tensor-core items (see attention_pages_tc_kernel)
  int by_seq;          // rows of one sequence over all its keys, or of all over the prefix
  int pairs;           // pairs of 128-row tiles: of a sequence, or full ones of all rows
  int full_splits;     // items over the prefix of a full pair; p_splits: the larger number
  int one_splits, one_chunk;  // prefix items of a last single tile
  int p_end;           // the first kind's items cover positions below this
  int direct;      // one slot a row: the item writes O itself
  int64_t rows;    // n_seq * T * n_head
  float *Op;       // [slot][rows][64]
  float2 *ml;      // [slot][rows]  maximum (base 2), sum
  int *err;
};

constexpr int kTileRows = 128, kPairRows = 256;  // tensor-core row tiles

struct Item {
  int b;       // sequence of a tail, -1: prefix
  int kvh, r0; // key head; first row of the tile among the (m, g) rows of b or of all
  int slot;
  int k0, k1;  // positions
  int n_valid; // positions that hold anything
};

__device__ __forceinline__ int seq_len(const ApArgs &a, int b) {
  return min(max(a.n_ctx[b], 0), a.max_ctx);
}
__device__ __forceinline__ int seq_new(const ApArgs &a, int b) {
  return a.n_new ? min(max(a.n_new[b], 0), a.T) : a.T;
}

__device__ __forceinline__ Item get_item(const ApArgs &a, int64_t idx) {
  Item it;
  const int64_t n_pre = (int64_t)a.n_kv * a.p_tiles * a.p_splits;
  if (idx < n_pre) {
    const int s = (int)(idx % a.p_splits);
    const int64_t q = idx / a.p_splits;
    it.b = -1;
    it.r0 = (int)(q % a.p_tiles) * kRows;
    it.kvh = (int)(q / a.p_tiles);
    it.slot = s;
    it.k0 = s * a.p_chunk;
    it.k1 = min(it.k0 + a.p_chunk, a.n_shared);
    it.n_valid = a.n_shared;
    return it;
  }
  idx -= n_pre;
  const int s = (int)(idx % a.t_splits);
  int64_t q = idx / a.t_splits;
  const int rt = (int)(q % a.t_tiles);
  q /= a.t_tiles;
  it.kvh = (int)(q % a.n_kv);
  it.b = (int)(q / a.n_kv);
  it.r0 = rt * kRows;
  it.slot = a.p_splits + s;
  it.n_valid = seq_len(a, it.b);
  const int nn = seq_new(a, it.b);
  it.k0 = a.n_shared + s * a.t_chunk;
  // the last row of the tile sees furthest
  const int t_last = min((it.r0 + kRows - 1) / a.g, nn - 1);
  const int end = it.n_valid - nn + t_last + 1;
  it.k1 = it.r0 < nn * a.g ? min(it.k0 + a.t_chunk, end) : it.k0;
  return it;
}
__device__ __forceinline__ int item_stages(const Item &it) {
  return it.k1 > it.k0 ? (it.k1 - it.k0 + kStageKeys - 1) / kStageKeys : 0;
}

struct Row {
  int64_t m;  // token row, -1: none
  int h, end;
};
// Row R of the (m, g) rows of sequence `seq` (-1: of all) and one key head.
__device__ __forceinline__ Row get_row(const ApArgs &a, int seq, int kvh, int64_t R) {
  Row w;
  w.m = R / a.g;
  w.h = kvh * a.g + (int)(R - w.m * a.g);
  int b = seq, t = (int)w.m;
  if (b < 0) {
    b = (int)(w.m / a.T);
    t = (int)(w.m - (int64_t)b * a.T);
  } else {
    w.m += (int64_t)b * a.T;
  }
  w.end = 0;
  if (b >= a.n_seq) {
    w.m = -1;
    return w;
  }
  const int nn = seq_new(a, b);
  if (t >= nn) w.m = -1;
  else w.end = seq_len(a, b) - nn + t + 1;
  return w;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
// named_barrier_sync that also tells every thread whether any had `pred` set.
__device__ __forceinline__ bool named_barrier_or(int id, int n, bool pred) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)pred), "r"(id), "r"(n)
      : "memory");
  return any != 0;
}
// A maximum to subtract: 0 where nothing has been seen yet.
__device__ __forceinline__ float safe_max(float m) { return m == -INFINITY ? 0.0f : m; }

struct MmaSmem {
  uint64_t full[kStages], empty[kStages];
  int abort_flag;
  float m[kMmaWarps][kRows], l[kMmaWarps][kRows];
  alignas(16) float O[kMmaWarps][kRows][kOPitch];  // read and written in pairs
};

}  // namespace

// ---------------------------------------------------------------------------
// Items of 16 rows on mma.sync: four warps take 16 keys each of every 64-key
// stage (TMA, 128-byte swizzle), each with its own running maximum, sum and
// O, joined through shared memory at the item's end. For the tails a row tile
// holds the few rows of one sequence and key head, and the keys are read once:
// the kernel is bound by HBM, and five 16 KB stages on two CTAs an SM cover
// its latency. The CTAs are persistent, so the TMA warp fetches the next
// item's keys while the last one is joined.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kMmaThreads, 2)
    attention_pages_mma_kernel(const __grid_constant__ CUtensorMap tmK,
                               const __grid_constant__ CUtensorMap tmV, ApArgs a,
                               int64_t n_item) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t *sK = smem, *sV = smem + kStages * kTileBytes;
  MmaSmem *ctl = reinterpret_cast<MmaSmem *>(sV + kStages * kTileBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&ctl->full[i], 1);
      mbar_init(&ctl->empty[i], kMmaWarps);
    }
    ctl->abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  __syncthreads();
  volatile int *abort_flag = &ctl->abort_flag;
  pdl_launch_dependents();
  pdl_wait();

  if (warp == kMmaWarps) {
    // ---------------- TMA: lane i < 2 * boxes issues one box of a stage ----------------
    const int box = min(1 << a.page_shift, kStageKeys);  // rows
    const int boxes = kStageKeys / box;
    const bool act = lane < 2 * boxes;
    const bool is_v = lane >= boxes;
    const int bx = is_v ? lane - boxes : lane;
    uint32_t n = 0;  // stages issued
    for (int64_t idx = blockIdx.x; idx < n_item; idx += gridDim.x) {
      const Item it = get_item(a, idx);
      const int ns = item_stages(it);
      auto entry = [&](int s) -> int {  // page of this lane's box, n_pages: reads as zeros
        const int pos = it.k0 + s * kStageKeys + bx * box;
        if (!act || pos >= it.k1) return a.n_pages;
        const int k = pos >> a.page_shift;
        int p = -1;
        if (it.b < 0) p = a.shared[k];
        else if (k < a.max_pages) p = a.table[(int64_t)it.b * a.max_pages + k];
        if (p < 0 || p >= a.n_pages) {
          report_error(a.err, kErrEntry);
          p = a.n_pages;
        }
        return p;
      };
      int p = ns ? entry(0) : 0;
      for (int s = 0; s < ns; ++s, ++n) {
        const int next = s + 1 < ns ? entry(s + 1) : 0;
        const int st = n % kStages;
        bool ok = true;
        if (n >= kStages)
          ok = mbar_wait(&ctl->empty[st], ((n / kStages) & 1) ^ 1, abort_flag, a.err,
                         kErrWaitEmpty);
        if (!__all_sync(~0u, ok)) goto drain;
        if (lane == 0) mbar_arrive_expect_tx(&ctl->full[st], 2 * kTileBytes);
        __syncwarp();
        if (act) {
          const int pos = it.k0 + s * kStageKeys + bx * box;
          const int y = (it.kvh << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
          tma_load_3d((is_v ? sV : sK) + st * kTileBytes + bx * box * 128, is_v ? &tmV : &tmK,
                      &ctl->full[st], 0, y, p);
        }
        p = next;
      }
    }
  drain:
    if (*abort_flag) {
      // no copy may still be writing shared memory when the CTA exits
      for (uint32_t i = n > kStages ? n - kStages : 0; i < n; ++i)
        mbar_wait(&ctl->full[i % kStages], (i / kStages) & 1, nullptr, a.err, kErrWaitFull);
    }
    return;
  }

  // ---------------- the four mma warps ----------------
  const int kw = warp * 16;  // this warp's keys of a stage
  // shared-memory offsets of the ldmatrix rows (128-byte swizzle)
  const int lm = lane >> 3, lr = lane & 7;
  const int krow = kw + (lm >> 1) * 8 + lr;  // K: matrices (key half, dim half)
  const int vrow = kw + (lm & 1) * 8 + lr;   // V: matrices (dim half, key half)
  uint32_t n = 0;
  for (int64_t idx = blockIdx.x; idx < n_item; idx += gridDim.x) {
    const Item it = get_item(a, idx);
    const int ns = item_stages(it);
    if (ns == 0 && !a.direct) continue;
    const Row row[2] = {get_row(a, it.b, it.kvh, it.r0 + (lane >> 2)),
                        get_row(a, it.b, it.kvh, it.r0 + (lane >> 2) + 8)};
    uint32_t q[4][4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Row &w = row[i & 1];
        q[ks][i] = w.m < 0 ? 0u
                           : *reinterpret_cast<const uint32_t *>(
                                 a.Q + w.m * a.ldq + w.h * kPageHd + ks * 16 + (i >> 1) * 8 +
                                 (lane & 3) * 2);
      }
    float o[8][4] = {};
    float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
    bool ok = true;
    for (int s = 0; s < ns; ++s, ++n) {
      const int st = n % kStages;
      if (!mbar_wait(&ctl->full[st], (n / kStages) & 1, abort_flag, a.err, kErrWaitFull)) {
        ok = false;
        break;
      }
      const int key0 = it.k0 + s * kStageKeys + kw;
      const uint32_t kb = smem_u32(sK + st * kTileBytes), vb = smem_u32(sV + st * kTileBytes);
      if (key0 + 16 > it.n_valid) {
        // rows of the last page that hold nothing yet: 0 * V must stay 0
        const int first = max(it.n_valid - key0, 0);
        for (int u = first * 8 + lane; u < 16 * 8; u += 32)
          *reinterpret_cast<uint4 *>(sV + st * kTileBytes + (kw + (u >> 3)) * 128 +
                                     (u & 7) * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
      }
      float c[2][4] = {};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        uint32_t b[4];
        ldsm4(kb + krow * 128 + (((ks * 2 + (lm & 1)) ^ (krow & 7)) << 4), b);
        mma16816(c[0], q[ks], b[0], b[1]);
        mma16816(c[1], q[ks], b[2], b[3]);
      }
      float p[2][4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {  // rows lane/4 and lane/4 + 8
        float t = mx[r];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = key0 + (j >> 1) * 8 + (lane & 3) * 2 + (j & 1);
          float x = c[j >> 1][2 * r + (j & 1)] * kScale2;
          x = key < min(row[r].end, it.k1) ? x : -INFINITY;
          p[r][j] = x;
          t = fmaxf(t, x);
        }
        t = fmaxf(t, __shfl_xor_sync(~0u, t, 1));
        t = fmaxf(t, __shfl_xor_sync(~0u, t, 2));
        const float ms = safe_max(t), f = ex2(mx[r] - ms);
        mx[r] = t;
        sum[r] *= f;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          o[d][2 * r] *= f;
          o[d][2 * r + 1] *= f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[r][j] = ex2(p[r][j] - ms);
          sum[r] += p[r][j];
        }
      }
      const uint32_t pa[4] = {pack_bf2(p[0][0], p[0][1]), pack_bf2(p[1][0], p[1][1]),
                              pack_bf2(p[0][2], p[0][3]), pack_bf2(p[1][2], p[1][3])};
#pragma unroll
      for (int d2 = 0; d2 < 4; ++d2) {
        uint32_t b[4];
        ldsm4t(vb + vrow * 128 + (((d2 * 2 + (lm >> 1)) ^ (vrow & 7)) << 4), b);
        mma16816(o[2 * d2], pa, b[0], b[1]);
        mma16816(o[2 * d2 + 1], pa, b[2], b[3]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->empty[st]);
    }
    // ---- join the four warps ----
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      sum[r] += __shfl_xor_sync(~0u, sum[r], 1);
      sum[r] += __shfl_xor_sync(~0u, sum[r], 2);
      const int rr = (lane >> 2) + 8 * r;
      if ((lane & 3) == 0) {
        ctl->m[warp][rr] = mx[r];
        ctl->l[warp][rr] = sum[r];
      }
#pragma unroll
      for (int d = 0; d < 8; ++d)
        *reinterpret_cast<float2 *>(&ctl->O[warp][rr][d * 8 + (lane & 3) * 2]) =
            make_float2(o[d][2 * r], o[d][2 * r + 1]);
    }
    if (named_barrier_or(1, kMmaWarps * 32, !ok)) return;  // a wait ran out in some warp
    {
      const int r = threadIdx.x >> 3, d0 = (threadIdx.x & 7) * 8;
      const Row w = get_row(a, it.b, it.kvh, it.r0 + r);
      if (w.m >= 0) {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kMmaWarps; ++i) m = fmaxf(m, ctl->m[i][r]);
        const float ms = safe_max(m);
        float l = 0.0f, acc[8] = {};
#pragma unroll
        for (int i = 0; i < kMmaWarps; ++i) {
          const float f = ex2(ctl->m[i][r] - ms);
          l += f * ctl->l[i][r];
#pragma unroll
          for (int d = 0; d < 8; ++d) acc[d] += f * ctl->O[i][r][d0 + d];
        }
        if (a.direct) {
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
          uint32_t *dst = reinterpret_cast<uint32_t *>(a.O + w.m * a.ldo + w.h * kPageHd + d0);
#pragma unroll
          for (int d = 0; d < 4; ++d) dst[d] = pack_bf2(acc[2 * d] * inv, acc[2 * d + 1] * inv);
        } else {
          const int64_t at = (int64_t)it.slot * a.rows + w.m * (a.n_kv * a.g) + w.h;
          float4 *dst = reinterpret_cast<float4 *>(a.Op + at * kPageHd + d0);
          dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
          dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
          if (d0 == 0) a.ml[at] = make_float2(m, l);
        }
      }
    }
    named_barrier_sync(1, kMmaWarps * 32);
  }
}

// ---------------------------------------------------------------------------
// Items of up to 256 rows on tcgen05 (kind::f16): a CTA holds a pair of 128-row
// Q tiles and streams 128-key blocks of K and V past both, so a block is read
// from memory once for 256 rows. Warps:
//   0-3, 4-7  softmax of group 0 and 1: a thread a row (TMEM lane), the row's
//             128 scores of a block in registers
//   8         TMA (a box a page, or 64 rows of a larger one)
//   9         owns TMEM, issues the MMAs: S = Q K^T (128 columns), then
//             O += P V with P read from TMEM, where the softmax left it as bf16,
//             so that neither P nor its re-reads pass through shared memory
// Each group has S (128 columns), P (64) and O (64): all 512 columns. S is free
// once a group holds it in registers, so S of the next block is formed while
// the exponentials of this one run, and the groups' MMAs overlap each other's
// softmax. A single tile (the last rows, or few of them) is worked on by both
// groups, a block each in turn, which are joined at the end.
// The running maximum that weights refer to moves only when a row's maximum has
// grown by more than 2^8 (in the exponent): the sums stay far from the range of
// fp32, and O is rescaled rarely, by the group itself.
// Bound by the exponentials: 128 x 128 of them at 16 a cycle are 1024 cycles,
// the two products of a tile 512.
// ---------------------------------------------------------------------------
namespace {

constexpr int kTcKeys = 128;
constexpr int kTcStages = 5;
constexpr uint32_t kTcTile = kTcKeys * 128;  // Q tile, or K or V of a block: 16 KB
constexpr int kTcTmaWarp = 8, kTcMmaWarp = 9;
constexpr int kTcThreads = 12 * 32;  // three warpgroups; the last two warps only pass registers
constexpr int kTcSoftThreads = 8 * 32;
constexpr uint32_t kColS = 0, kColP = 128, kColO = 192, kColGroup = 256;
constexpr float kMaxSlack = 8.0f;  // base 2
constexpr int kErrTc = 0x1610;

struct TcCtl {
  uint64_t q_full;
  uint64_t kv_full[kTcStages], kv_empty[kTcStages];
  uint64_t s_full[2], s_free[2], p_full[2], o_done[2];
  uint64_t turn[2][4];  // group g's, of a quarter
  uint64_t v_ready, drain;
  uint32_t tmem_base;
  int abort_flag;
  int idle[8];
  float2 ml[kTileRows];  // group 1's, where both groups work on one tile
};

struct TcItem {
  int b, kvh;      // sequence, -1: rows of all
  int64_t r0, r1;  // rows among the (m, g) rows of b, or of all
  int slot, k0, k1, n_valid;
};

__device__ __forceinline__ TcItem get_tc_item(const ApArgs &a, int idx) {
  TcItem it;
  if (a.by_seq) {
    // the last rows of a sequence see furthest: those items first
    const int s = idx % a.p_splits;
    int q = idx / a.p_splits;
    it.kvh = q % a.n_kv;
    q /= a.n_kv;
    it.b = q % a.n_seq;
    const int pair = a.pairs - 1 - q / a.n_seq;
    const int nn = seq_new(a, it.b), n = seq_len(a, it.b);
    it.r0 = (int64_t)pair * kPairRows;
    it.r1 = min(it.r0 + kPairRows, (int64_t)nn * a.g);
    it.slot = s;
    it.k0 = s * a.p_chunk;
    it.n_valid = n;
    const int end = it.r1 > it.r0 ? n - nn + (int)((it.r1 - 1) / a.g) + 1 : 0;
    it.k1 = min(it.k0 + a.p_chunk, end);
    return it;
  }
  const int full = a.pairs * a.full_splits;
  it.b = -1;
  it.kvh = idx / (full + a.one_splits);
  const int q = idx - it.kvh * (full + a.one_splits);
  const bool one = q >= full;
  const int pair = one ? a.pairs : q / a.full_splits;
  it.slot = one ? q - full : q - pair * a.full_splits;
  it.r0 = (int64_t)pair * kPairRows;
  it.r1 = min(it.r0 + kPairRows, (int64_t)a.n_seq * a.T * a.g);
  const int chunk = one ? a.one_chunk : a.p_chunk;
  it.k0 = it.slot * chunk;
  it.k1 = min(it.k0 + chunk, a.n_shared);
  it.n_valid = a.n_shared;
  return it;
}

__device__ __forceinline__ Row get_tc_row(const ApArgs &a, const TcItem &it, int64_t R) {
  Row w = get_row(a, it.b, it.kvh, R);
  if (R >= it.r1) {
    w.m = -1;
    w.end = 0;
  }
  return w;
}

}  // namespace

__global__ void __launch_bounds__(kTcThreads, 1)
    attention_pages_tc_kernel(const __grid_constant__ CUtensorMap tmK,
                              const __grid_constant__ CUtensorMap tmV, ApArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t *sQ = smem;                       // [2] tiles
  uint8_t *sKV = smem + 2 * kTcTile;        // [stages] K, V
  TcCtl *ctl = reinterpret_cast<TcCtl *>(sKV + kTcStages * 2 * kTcTile);
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();
  const TcItem it = get_tc_item(a, blockIdx.x);
  const int n_rows = (int)(it.r1 - it.r0);
  const int blocks = it.k1 > it.k0 ? (it.k1 - it.k0 + kTcKeys - 1) / kTcKeys : 0;
  // an item without keys: its slot is not read, unless rows get their zeros here
  if (n_rows <= 0 || (blocks == 0 && !a.direct)) return;
  const bool one = n_rows <= kTileRows;      // both groups on one tile
  const int units = one ? blocks : 2 * blocks;  // unit u: group u & 1
  // the last block reaches behind the positions that hold anything
  const bool v_cut = it.k0 + blocks * kTcKeys > it.n_valid;
  if (threadIdx.x == 0) {
    mbar_init(&ctl->q_full, 8);
    for (int i = 0; i < kTcStages; ++i) {
      mbar_init(&ctl->kv_full[i], 1);
      mbar_init(&ctl->kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->s_full[i], 1);
      mbar_init(&ctl->s_free[i], 4);
      mbar_init(&ctl->p_full[i], 4);
      mbar_init(&ctl->o_done[i], 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(&ctl->turn[i >> 2][i & 3], 1);
    mbar_init(&ctl->v_ready, 1);
    mbar_init(&ctl->drain, 1);
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
    reg_alloc<208>();
    // ---------------- softmax ----------------
    const int g = warp >> 2, qd = warp & 3;
    const int r = qd * 32 + lane;  // TMEM lane
    const Row row = get_tc_row(a, it, it.r0 + (one ? 0 : g) * kTileRows + r);
    const bool idle = __all_sync(~0u, row.m < 0);  // no rows in this warp
    const uint32_t trow = tmem + g * kColGroup + ((uint32_t)(qd * 32) << 16);
    // Q row into its swizzled place
    if (!one || g == 0) {
      uint8_t *dst = sQ + g * kTcTile + r * 128;
      const uint4 *src = reinterpret_cast<const uint4 *>(a.Q + row.m * a.ldq + row.h * kPageHd);
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
      for (int c = 0; c < 4; ++c) {
        mx[c] = __uint_as_float(s[c][0]);
#pragma unroll
        for (int k = 1; k < 32; ++k) mx[c] = fmaxf(mx[c], __uint_as_float(s[c][k]));
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const bool grown = top > m && !((top - m) * kScale2 <= kMaxSlack);
      float f = 1.0f;
      if (grown) {
        f = ex2((m - top) * kScale2);  // 0 at the first key (m = -inf)
        m = top;
        l *= f;
      }
      const bool rescale = i > 0 && __any_sync(~0u, grown);
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
      // (a warp issues in order and would otherwise wait for each).
      float sum[4] = {};
      auto scale = [&](int c, int k) {
        s[c][k] = __float_as_uint(fmaf(__uint_as_float(s[c][k]), kScale2, -ms));
      };
      auto take = [&](int c, int k) {  // keys k, k + 1
        const float x = __uint_as_float(s[c][k]), y = __uint_as_float(s[c][k + 1]);
        sum[k & 2] += x;
        sum[(k & 2) + 1] += y;
        s[c][k / 2] = pack_bf2(x, y);
      };
      auto store = [&](int c) {  // chunks c - 1 and c
        uint32_t p[32];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          p[k] = s[c - 1][k];
          p[16 + k] = s[c][k];
        }
        tmem_st_32x32b_x32(trow + kColP + 16 * (c - 1), p);
      };
#pragma unroll
      for (int k = 0; k < 32; ++k) scale(0, k);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          s[c][k] = __float_as_uint(ex2(__uint_as_float(s[c][k])));
          s[c][k + 1] = __float_as_uint(ex2(__uint_as_float(s[c][k + 1])));
          if (c < 3) {
            scale(c + 1, k);
            scale(c + 1, k + 1);
          }
          if (c > 0) take(c - 1, k);
        }
        if (c == 2) store(1);
      }
      if (turns && lane == 0) mbar_arrive(&ctl->turn[g ^ 1][qd]);
#pragma unroll
      for (int k = 0; k < 32; k += 2) take(3, k);
      store(3);
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
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
      const int64_t at = (int64_t)it.slot * a.rows + row.m * (a.n_kv * a.g) + row.h;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t o[16], o1[16];
        if (mine > 0) {
          tmem_ld_32x32b_x16(trow + kColO + 16 * c, o);
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = 0u;
        }
        if (second) tmem_ld_32x32b_x16(trow + kColGroup + kColO + 16 * c, o1);
        tmem_ld_wait();
        float x[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          x[k] = __uint_as_float(o[k]);
          if (second) x[k] = f0 * x[k] + f1 * __uint_as_float(o1[k]);
        }
        if (row.m >= 0) {
          if (a.direct) {
            uint32_t *dst =
                reinterpret_cast<uint32_t *>(a.O + row.m * a.ldo + row.h * kPageHd + 16 * c);
#pragma unroll
            for (int k = 0; k < 8; ++k) dst[k] = pack_bf2(x[2 * k] * inv, x[2 * k + 1] * inv);
          } else {
            float4 *dst = reinterpret_cast<float4 *>(a.Op + at * kPageHd + 16 * c);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              dst[k] = make_float4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
          }
        }
      }
      if (row.m >= 0 && !a.direct) a.ml[at] = make_float2(m_all, l_all);
    }
  } else {
    reg_dealloc<88>();
  if (warp == kTcTmaWarp) {
    // ---------------- TMA: lane i < 2 * boxes issues one box of a block ----------------
    const int box = min(1 << a.page_shift, kStageKeys);  // rows
    const int boxes = kTcKeys / box;
    const bool act = lane < 2 * boxes;
    const bool is_v = lane >= boxes;
    const int bx = is_v ? lane - boxes : lane;
    auto entry = [&](int j) -> int {  // page of this lane's box, n_pages: reads as zeros
      const int pos = it.k0 + j * kTcKeys + bx * box;
      if (!act || pos >= it.k1) return a.n_pages;
      const int k = pos >> a.page_shift;
      int p = -1;
      if (pos < a.n_shared) p = a.shared[k];
      else if (k < a.max_pages) p = a.table[(int64_t)it.b * a.max_pages + k];
      if (p < 0 || p >= a.n_pages) {
        report_error(a.err, kErrEntry);
        p = a.n_pages;
      }
      return p;
    };
    int p = blocks ? entry(0) : 0;
    int n = 0;
    for (; n < blocks; ++n) {
      const int next = n + 1 < blocks ? entry(n + 1) : 0;
      const int st = n % kTcStages;
      bool ok = true;
      if (n >= kTcStages)
        ok = mbar_wait(&ctl->kv_empty[st], ((n / kTcStages) & 1) ^ 1, abort_flag, a.err, kErrTc);
      if (!__all_sync(~0u, ok)) break;
      if (lane == 0) mbar_arrive_expect_tx(&ctl->kv_full[st], 2 * kTcTile);
      __syncwarp();
      if (act) {
        const int pos = it.k0 + n * kTcKeys + bx * box;
        const int y = (it.kvh << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
        tma_load_3d(sKV + (st * 2 + is_v) * kTcTile + bx * box * 128, is_v ? &tmV : &tmK,
                    &ctl->kv_full[st], 0, y, p);
      }
      p = next;
    }
    if (n == blocks && v_cut) {
      // rows of the last page that hold nothing yet: 0 * V must stay 0
      const int j = blocks - 1, st = j % kTcStages;
      if (mbar_wait(&ctl->kv_full[st], (j / kTcStages) & 1, abort_flag, a.err, kErrTc + 1)) {
        uint8_t *v = sKV + (st * 2 + 1) * kTcTile;
        for (int x = (it.n_valid - it.k0 - j * kTcKeys) * 8 + lane; x < kTcKeys * 8; x += 32)
          *reinterpret_cast<uint4 *>(v + x * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->v_ready);
      }
    }
    if (*abort_flag)  // no copy may still be writing shared memory when the CTA exits
      for (int i = n > kTcStages ? n - kTcStages : 0; i < n; ++i)
        mbar_wait(&ctl->kv_full[i % kTcStages], (i / kTcStages) & 1, nullptr, a.err, kErrTc + 1);
  } else if (warp == kTcMmaWarp) {
    // ---------------- MMA: one thread ----------------
    if (elect_one()) {
      const uint32_t idS = make_idesc(1, 1, kTileRows, kTcKeys);
      const uint32_t idO = make_idesc_bmn(1, 1, kTileRows, kPageHd);
      const uint64_t q_desc = make_sw128_desc(smem_u32(sQ));
      const uint64_t k_desc = make_sw128_desc(smem_u32(sKV));
      const uint64_t v_desc = make_sw128_mn_desc(smem_u32(sKV) + kTcTile);
      bool ok = mbar_wait(&ctl->q_full, 0, abort_flag, a.err, kErrTc + 2);
      int seen = 0;  // blocks known to be in shared memory
      auto issue_s = [&](int u) -> bool {
        const int g = u & 1, i = u >> 1, j = one ? u : i;  // group, its unit, block
        if (i > 0 && !mbar_wait(&ctl->s_free[g], (i - 1) & 1, abort_flag, a.err, kErrTc + 3))
          return false;
        const int st = j % kTcStages;
        if (j >= seen) {
          if (!mbar_wait(&ctl->kv_full[st], (j / kTcStages) & 1, abort_flag, a.err, kErrTc + 4))
            return false;
          seen = j + 1;
        }
        tc_fence_after();
        tc_mma_bf16_x4(tmem + g * kColGroup + kColS, q_desc + (one ? 0 : g) * (kTcTile >> 4),
                       k_desc + st * (2 * kTcTile >> 4), idS);
        tc_commit(&ctl->s_full[g]);
        return true;
      };
      auto issue_o = [&](int u) -> bool {
        const int g = u & 1, i = u >> 1, j = one ? u : i;
        if (!mbar_wait(&ctl->p_full[g], i & 1, abort_flag, a.err, kErrTc + 5)) return false;
        if (v_cut && j == blocks - 1 &&
            !mbar_wait(&ctl->v_ready, 0, abort_flag, a.err, kErrTc + 10))
          return false;
        tc_fence_after();
        const uint32_t base = tmem + g * kColGroup;
        tc_mma_bf16_ta_x8(base + kColO, base + kColP, v_desc + (j % kTcStages) * (2 * kTcTile >> 4),
                          idO, i > 0);
        tc_commit(&ctl->o_done[g]);
        if (one || g == 1) tc_commit(&ctl->kv_empty[j % kTcStages]);
        return true;
      };
      for (int u = 0; u < 2 && u < units && ok; ++u) ok = issue_s(u);
      for (int u = 0; u < units && ok; u += 2) {
        for (int v = u + 2; v < u + 4 && v < units && ok; ++v) ok = issue_s(v);
        for (int v = u; v < u + 2 && v < units && ok; ++v) ok = issue_o(v);
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
// The join of a row's items, a warp a row (two dims a lane). An item without
// keys below the row's end was not run: its slot is not read.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) attention_pages_join_kernel(ApArgs a) {
  const int lane = threadIdx.x & 31;
  const int n_head = a.n_kv * a.g;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  pdl_launch_dependents();
  pdl_wait();
  if (row >= a.rows) return;
  const int64_t m = row / n_head;
  const int b = (int)(m / a.T), t = (int)(m - (int64_t)b * a.T);
  const int nn = seq_new(a, b);
  if (t >= nn) return;
  const int end = seq_len(a, b) - nn + t + 1;
  const int slots = a.p_splits + a.t_splits;
  // the row's place among the prefix rows of its key head tells its items' chunk
  const int64_t R = m * a.g + (int)(row - m * n_head) % a.g;
  const int p_chunk = a.one_splits && R >= (int64_t)a.pairs * kPairRows ? a.one_chunk : a.p_chunk;
  auto live = [&](int s) {
    return s < a.p_splits ? s * (int64_t)p_chunk < min(end, a.p_end)
                          : a.n_shared + (s - a.p_splits) * (int64_t)a.t_chunk < end;
  };
  float mx = -INFINITY;
  for (int s = lane; s < slots; s += 32)
    if (live(s)) mx = fmaxf(mx, a.ml[s * a.rows + row].x);
#pragma unroll
  for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, d));
  const float ms = safe_max(mx);
  float l = 0.0f;
  float2 acc = make_float2(0.0f, 0.0f);
  for (int s = 0; s < slots; ++s) {
    if (!live(s)) continue;
    const float2 v = a.ml[s * a.rows + row];
    const float2 x = reinterpret_cast<const float2 *>(a.Op + (s * a.rows + row) * kPageHd)[lane];
    const float f = ex2(v.x - ms);
    l += f * v.y;
    acc.x += f * x.x;
    acc.y += f * x.y;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  reinterpret_cast<uint32_t *>(a.O + m * a.ldo + (row - m * n_head) * kPageHd)[lane] =
      pack_bf2(acc.x * inv, acc.y * inv);
}

// ---------------------------------------------------------------------------
// plan and launch
// ---------------------------------------------------------------------------
namespace {

struct Plan {
  bool tc;         // a tensor-core launch
  bool by_seq;     // it covers everything
  int tc_items;
  int p_tiles, p_splits, p_chunk, t_tiles, t_splits, t_chunk;
  int pairs, full_splits, one_splits, one_chunk, p_end;
};

int64_t cdiv(int64_t x, int64_t y) { return (x + y - 1) / y; }

// Keys of a chunk when `groups` items share `keys` keys each: enough items for
// `want`, chunks of at least min_keys, a multiple of `step`.
int chunk_keys(int64_t keys, int64_t groups, int64_t want, int min_keys, int step) {
  const int64_t splits = cdiv(want, groups);
  const int64_t c = cdiv(cdiv(keys, splits), step) * step;
  return (int)(c < min_keys ? min_keys : c);
}

Plan make_plan(int n_seq, int T, int n_head, int n_kv, int max_ctx, int n_shared) {
  Plan p = {};
  const int g = n_head / n_kv;
  const int64_t want = kSms * 4;  // 16-row items: two waves of two CTAs an SM
  const int64_t own = (int64_t)T * g, all = own * n_seq;  // rows of a key head
  p.p_end = n_shared;
  if (own >= 64) {
    // enough rows a sequence to fill a tile: prefix and tail in one item
    p.tc = p.by_seq = true;
    p.pairs = (int)cdiv(own, kPairRows);
    const int64_t groups = (int64_t)n_seq * n_kv * p.pairs;
    p.p_chunk = chunk_keys(max_ctx, groups, groups >= kSms ? groups : kSms, 4 * kTcKeys, kTcKeys);
    p.p_splits = (int)cdiv(max_ctx, p.p_chunk);
    p.p_end = max_ctx;
    p.tc_items = (int)(groups * p.p_splits);
    return p;
  }
  if (n_shared > 0 && all > 32) {
    p.tc = true;
    // full pairs get twice the chunks of a last single tile, whose blocks take half the time;
    // one CTA an SM in all, if there are that few
    const int64_t tiles = cdiv(all, kTileRows);
    p.pairs = (int)(tiles / 2);
    const int single = (int)(tiles & 1);
    int64_t per = kSms / n_kv;  // CTAs a key head
    int64_t s1 = per / (2 * p.pairs + single);
    if (s1 < 1) s1 = 1;
    int64_t s2 = p.pairs ? (per - s1 * single) / p.pairs : 0;
    if (s2 < 1) s2 = 1;
    p.p_chunk = chunk_keys(n_shared, 1, s2, 2 * kTcKeys, kTcKeys);
    p.one_chunk = chunk_keys(n_shared, 1, s1, 2 * kTcKeys, kTcKeys);
    p.full_splits = p.pairs ? (int)cdiv(n_shared, p.p_chunk) : 0;
    p.one_splits = single ? (int)cdiv(n_shared, p.one_chunk) : 0;
    p.p_splits = p.full_splits > p.one_splits ? p.full_splits : p.one_splits;
    p.tc_items = n_kv * (p.pairs * p.full_splits + p.one_splits);
  } else if (n_shared > 0) {
    p.p_tiles = (int)cdiv(all, kRows);
    p.p_chunk = chunk_keys(n_shared, (int64_t)n_kv * p.p_tiles, want, 2 * kStageKeys, kStageKeys);
    p.p_splits = (int)cdiv(n_shared, p.p_chunk);
  }
  p.t_tiles = (int)cdiv(own, kRows);
  const int tail = max_ctx - n_shared > 0 ? max_ctx - n_shared : 1;
  p.t_chunk = chunk_keys(tail, (int64_t)n_seq * n_kv * p.t_tiles, want, 2 * kStageKeys, kStageKeys);
  p.t_splits = (int)cdiv(tail, p.t_chunk);
  return p;
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

size_t attention_pages_workspace_bytes(int n_seq, int T, int n_head, int n_kv, int max_ctx,
                                       int n_shared) {
  const Plan p = make_plan(n_seq, T, n_head, n_kv, max_ctx, n_shared);
  const int slots = p.p_splits + p.t_splits;
  const size_t rows = (size_t)n_seq * T * n_head;
  return slots <= 1 ? 16 : slots * rows * (kPageHd * sizeof(float) + sizeof(float2));
}

int launch_attention_pages(const PagesArgs &c, const AttnPagesCall &q, int sm_count,
                           cudaStream_t s) {
  const int g = q.n_head / c.n_kv_head;
  const Plan p = make_plan(q.n_seq, q.T, q.n_head, c.n_kv_head, q.max_ctx, q.n_shared);
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
  a.p_splits = p.p_splits;
  a.p_chunk = p.p_chunk;
  a.t_tiles = p.t_tiles;
  a.t_splits = p.t_splits;
  a.t_chunk = p.t_chunk;
  a.by_seq = p.by_seq;
  a.pairs = p.pairs;
  a.full_splits = p.full_splits;
  a.one_splits = p.one_splits;
  a.one_chunk = p.one_chunk;
  a.p_end = p.p_end;
  a.rows = (int64_t)q.n_seq * q.T * q.n_head;
  const int slots = p.p_splits + p.t_splits;
  a.direct = slots == 1;
  a.Op = reinterpret_cast<float *>(q.ws);
  a.ml = reinterpret_cast<float2 *>(a.Op + (size_t)slots * a.rows * kPageHd);
  int st;
  DeviceCtx *ctx = device_ctx(&st);
  if (!ctx) return st;
  a.err = ctx->err;
  const int box = c.page < kStageKeys ? c.page : kStageKeys;
  const int64_t off = (int64_t)q.layer * c.n_kv_head * c.page * kPageHd;
  const CUtensorMapDataType bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap tmK, tmV;
  const uint64_t rows = (uint64_t)c.n_kv_head * c.page;
  st = make_tmap_3d(&tmK, c.K + off, bf, (uint64_t)c.n_pages, rows, kPageHd, kPageHd * 2,
                    (uint64_t)c.page_stride * 2, kPageHd, box);
  if (st) return st;
  st = make_tmap_3d(&tmV, c.V + off, bf, (uint64_t)c.n_pages, rows, kPageHd, kPageHd * 2,
                    (uint64_t)c.page_stride * 2, kPageHd, box);
  if (st) return st;
  static bool tc_ready[64], mma_ready[64];
  if (p.tc) {
    const size_t smem = 1024 + (2 + 2 * kTcStages) * kTcTile + sizeof(TcCtl);
    st = opt_in_smem(attention_pages_tc_kernel, smem, tc_ready);
    if (st) return st;
    launch_pdl(attention_pages_tc_kernel, dim3((unsigned)p.tc_items), dim3(kTcThreads), smem, s,
               tmK, tmV, a);
    st = check_launch("attention_pages_tc");
    if (st) return st;
  }
  const int64_t items = (int64_t)a.n_kv * p.p_tiles * p.p_splits +
                        (int64_t)a.n_seq * a.n_kv * p.t_tiles * p.t_splits;
  if (items > 0) {
    const size_t smem = 1024 + 2 * kStages * kTileBytes + sizeof(MmaSmem);
    st = opt_in_smem(attention_pages_mma_kernel, smem, mma_ready);
    if (st) return st;
    const int64_t grid = items < 2 * sm_count ? items : 2 * sm_count;
    launch_pdl(attention_pages_mma_kernel, dim3((unsigned)grid), dim3(kMmaThreads), smem, s, tmK,
               tmV, a, items);
    st = check_launch("attention_pages_mma");
    if (st) return st;
  }
  if (a.direct) return W8A8_OK;
  launch_pdl(attention_pages_join_kernel, dim3((unsigned)cdiv(a.rows, 8)), dim3(256), 0, s, a);
  return check_launch("attention_pages_join");
}

}  // namespace w8a8

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
  // items: prefix [n_kv][p_tiles][p_splits], then tails [n_seq][n_kv][t_tiles][t_splits]
  int p_tiles, p_splits, p_chunk;
  int t_tiles, t_splits, t_chunk;
  int direct;      // one slot a row: the item writes O itself
  int64_t rows;    // n_seq * T * n_head
  float *Op;       // [slot][rows][64]
  float2 *ml;      // [slot][rows]  maximum (base 2), sum
  int *err;
};

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
__device__ __forceinline__ Row get_row(const ApArgs &a, const Item &it, int r) {
  Row w;
  const int64_t R = it.r0 + r;
  w.m = R / a.g;
  w.h = it.kvh * a.g + (int)(R - w.m * a.g);
  int b = it.b, t = (int)w.m;
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
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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
    const Row row[2] = {get_row(a, it, lane >> 2), get_row(a, it, (lane >> 2) + 8)};
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
      const Row w = get_row(a, it, r);
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
  auto live = [&](int s) {
    return s < a.p_splits ? s * a.p_chunk < min(end, a.n_shared)
                          : a.n_shared + (s - a.p_splits) * a.t_chunk < end;
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
  int p_tiles, p_splits, p_chunk, t_tiles, t_splits, t_chunk;
};

int64_t cdiv(int64_t x, int64_t y) { return (x + y - 1) / y; }

// Keys of a chunk when `groups` items share `keys` keys each: enough items for
// `want`, chunks of at least min_keys, a multiple of the stage.
int chunk_keys(int64_t keys, int64_t groups, int64_t want, int min_keys) {
  int64_t splits = cdiv(want, groups);
  int64_t c = cdiv(cdiv(keys, splits), kStageKeys) * kStageKeys;
  return (int)(c < min_keys ? min_keys : c);
}

Plan make_plan(int n_seq, int T, int n_head, int n_kv, int max_ctx, int n_shared) {
  Plan p = {};
  const int g = n_head / n_kv;
  const int64_t want = kSms * 4;  // items: two waves of two CTAs an SM
  if (n_shared > 0) {
    p.p_tiles = (int)cdiv((int64_t)n_seq * T * g, kRows);
    p.p_chunk = chunk_keys(n_shared, (int64_t)n_kv * p.p_tiles, want, 2 * kStageKeys);
    p.p_splits = (int)cdiv(n_shared, p.p_chunk);
  }
  p.t_tiles = (int)cdiv((int64_t)T * g, kRows);
  const int tail = max_ctx - n_shared > 0 ? max_ctx - n_shared : 1;
  p.t_chunk = chunk_keys(tail, (int64_t)n_seq * n_kv * p.t_tiles, want, 2 * kStageKeys);
  p.t_splits = (int)cdiv(tail, p.t_chunk);
  return p;
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
  static bool attr[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return W8A8_ERR_CUDA;
  const size_t smem = 1024 + 2 * kStages * kTileBytes + sizeof(MmaSmem);
  if (!attr[dev]) {
    if (cudaFuncSetAttribute(attention_pages_mma_kernel,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
        cudaSuccess)
      return W8A8_ERR_CUDA;
    attr[dev] = true;
  }
  const int64_t items = (int64_t)a.n_kv * p.p_tiles * p.p_splits +
                        (int64_t)a.n_seq * a.n_kv * p.t_tiles * p.t_splits;
  const int64_t grid = items < 2 * sm_count ? items : 2 * sm_count;
  launch_pdl(attention_pages_mma_kernel, dim3((unsigned)grid), dim3(kMmaThreads), smem, s, tmK,
             tmV, a, items);
  st = check_launch("attention_pages_mma");
  if (st || a.direct) return st;
  launch_pdl(attention_pages_join_kernel, dim3((unsigned)cdiv(a.rows, 8)), dim3(256), 0, s, a);
  return check_launch("attention_pages_join");
}

}  // namespace w8a8

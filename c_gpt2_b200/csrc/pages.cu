// Cache pages: appending to, forking, freeing, compacting and copying the
// pages that hold sequences' keys and values (include/gpt2_w8a8.h,
// w8a8_pages_*). No counterpart in the reference, whose cache is one
// contiguous run of ctx rows (gpt2.c:758-759).
//
// The page table, the lengths and the page counts live on the device and are
// updated there, so a decode step that grows its sequences replays from a
// CUDA graph. Each update that hands out pages runs in one CTA: which page
// goes to whom is a prefix sum over the requests met with a prefix sum over
// the free pages, lowest index first, so the result does not depend on any
// order of execution. What touches many bytes (rows of partly filled pages,
// whole pages) runs in a second, grid-wide kernel.
#include "common.cuh"
#include "kernels.cuh"
#include "runtime.cuh"

namespace w8a8 {

namespace {

constexpr int kBookThreads = 1024;
constexpr int kBookWarps = kBookThreads / 32;
constexpr int kScan = 8;  // pages a lane looks at per round of a scan: 8192 a CTA
constexpr int kRound = kBookThreads * kScan;

constexpr int kErrPage = 0x1501;  // a table entry outside the pool, or a count below zero
constexpr int kErrPos = 0x1502;   // a position outside the table

// Exclusive prefix of v over the warps' values (v equal in a warp's lanes),
// and the sum over all warps.
__device__ __forceinline__ int warps_prefix(int v, int *buf, int *sum) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();  // the previous use of buf
  if (lane == 0) buf[warp] = v;
  __syncthreads();
  int x = buf[lane];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(~0u, x, d);
    if (lane >= d) x += y;
  }
  *sum = __shfl_sync(~0u, x, 31);
  return warp ? __shfl_sync(~0u, x, (warp + 31) & 31) : 0;
}

// Inclusive prefix of one value a thread over the block, and the sum.
__device__ __forceinline__ int block_inclusive(int v, int *buf, int *sum) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(~0u, v, d);
    if (lane >= d) v += y;
  }
  return v + warps_prefix(__shfl_sync(~0u, v, 31), buf, sum);
}

// Calls give(rank, p) for the free pages p of rank 0 .. want - 1 (rank: how
// many free pages lie below p) and returns how many free pages there are, or
// any number >= want where there are at least that many.
template <typename F>
__device__ __forceinline__ int scan_free(const int32_t *refs, int n_pages, int want, int *buf,
                                         F give) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int seen = 0;
  for (int64_t base = 0; base < n_pages && seen < want; base += kRound) {
    uint32_t bal[kScan];
    int mine = 0;
    const int64_t p0 = base + warp * (32 * kScan) + lane;
    int32_t v[kScan];
#pragma unroll
    for (int k = 0; k < kScan; ++k) v[k] = p0 + 32 * k < n_pages ? refs[p0 + 32 * k] : 1;
#pragma unroll
    for (int k = 0; k < kScan; ++k) {
      bal[k] = __ballot_sync(~0u, v[k] == 0);
      mine += __popc(bal[k]);
    }
    int sum;
    int rank = seen + warps_prefix(mine, buf, &sum);
#pragma unroll
    for (int k = 0; k < kScan; ++k) {
      if ((bal[k] >> lane) & 1) {
        const int r = rank + __popc(bal[k] & ((1u << lane) - 1));
        if (r < want) give(r, (int)(p0 + 32 * k));
      }
      rank += __popc(bal[k]);
    }
    seen += sum;
  }
  return seen;
}

// First i in [0, n) with upto[i] > rank (upto ascending, upto[n - 1] > rank).
__device__ __forceinline__ int owner_of(const int *upto, int n, int rank) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (upto[mid] > rank) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(int n, int page) { return (n + page - 1) / page; }

// Positions that a slot may hold: those of its table row, and that 32 bits count.
__device__ __forceinline__ int64_t capacity(const PagesArgs &a) {
  return min((int64_t)a.max_pages * a.page, (int64_t)0x7fffff00);
}

}  // namespace

// ---------------------------------------------------------------------------
// extend: need_b = ceil((n + new) / page) - ceil(n / page) pages for sequence
// b; in order of b, b is served if the needs up to and with its own are at
// most the free pages. One CTA; latency-bound (a few dependent loads and a
// scan of refs, 4 bytes a page, ended as soon as enough free pages are found):
// 4.8 us for 64 sequences and 6000 pages.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kBookThreads)
    pages_extend_kernel(PagesArgs a, const int32_t *n_new, int32_t *pos0) {
  extern __shared__ int sh[];
  __shared__ int buf[kBookWarps];
  int *upto = sh;  // [n_slot]
  pdl_launch_dependents();
  pdl_wait();
  const int64_t cap = capacity(a);
  int total = 0;
  for (int base = 0; base < a.n_slot; base += kBookThreads) {
    const int i = base + threadIdx.x;
    int need = 0;
    if (i < a.n_slot) {
      const int n = a.n_ctx[i], add = n_new[i];
      if (add > 0 && n >= 0 && (int64_t)n + add <= cap)
        need = pages_of(n + add, a.page) - pages_of(n, a.page);
    }
    int sum;
    const int inc = block_inclusive(need, buf, &sum);
    if (i < a.n_slot) upto[i] = total + inc;
    total += sum;
  }
  __syncthreads();
  const int free = scan_free(a.refs, a.n_pages, total, buf, [&](int rank, int p) {
    const int i = owner_of(upto, a.n_slot, rank);
    const int k = rank - (i ? upto[i - 1] : 0) + pages_of(a.n_ctx[i], a.page);
    a.table[(int64_t)i * a.max_pages + k] = p;
    a.refs[p] = 1;
  });
  __syncthreads();
  for (int i = threadIdx.x; i < a.n_slot; i += kBookThreads) {
    const int n = a.n_ctx[i], add = n_new[i];
    const int before = i ? upto[i - 1] : 0, need = upto[i] - before;
    const bool ok = add > 0 && n >= 0 && (int64_t)n + add <= cap && (need == 0 || upto[i] <= free);
    // the one sequence that the free pages ended inside gives its share back
    if (!ok && need > 0 && before < free) {
      int32_t *row = a.table + (int64_t)i * a.max_pages + pages_of(n, a.page);
      for (int k = 0; k < free - before; ++k) {
        a.refs[row[k]] = 0;
        row[k] = -1;
      }
    }
    pos0[i] = ok ? n : (add > 0 ? W8A8_PAGES_REFUSED : W8A8_PAGES_NONE);
    if (ok) a.n_ctx[i] = n + add;
  }
}

// ---------------------------------------------------------------------------
// write: row t of sequence b at position pos0[b] + t of its pages. A warp takes a
// row's keys or its values, so that the place is worked out once a row (with four
// divisions a 16-byte unit instead, the kernel was bound by issue: 27 us for 16
// prompts of up to 1000 rows of 20 heads, whose bytes take 12.5); a head's segment
// is 128 contiguous bytes on both sides, and four units a lane are in flight.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
    pages_write_kernel(PagesArgs a, int64_t layer_off, const uint16_t *Kn, int64_t ldk,
                       const uint16_t *Vn, int64_t ldv, int n_seq, int T, const int32_t *n_new,
                       const int32_t *pos0) {
  const int64_t x = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int64_t m = x >> 1;
  const bool is_v = x & 1;
  pdl_launch_dependents();
  pdl_wait();
  if (m >= (int64_t)n_seq * T) return;
  const int b = (int)((uint32_t)m / (uint32_t)T), t = (int)m - b * T;
  const int p0 = pos0[b];
  if (p0 < 0 || (n_new && t >= n_new[b])) return;
  const int64_t pos = (int64_t)p0 + t;
  const int shift = __ffs(a.page) - 1;
  if (pos >> shift >= a.max_pages) {
    if (lane == 0) report_error(a.err, kErrPos);
    return;
  }
  const int p = a.table[(int64_t)b * a.max_pages + (pos >> shift)];
  if (p < 0 || p >= a.n_pages) {
    if (lane == 0) report_error(a.err, kErrPage);
    return;
  }
  const uint4 *from = reinterpret_cast<const uint4 *>(is_v ? Vn + m * ldv : Kn + m * ldk);
  uint4 *to = reinterpret_cast<uint4 *>((is_v ? a.V : a.K) + (int64_t)p * a.page_stride +
                                        layer_off + (pos & (a.page - 1)) * kPageHd);
  const int n = a.n_kv_head * 8;
  for (int w0 = lane; w0 < n; w0 += 128) {
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (w0 + 32 * j < n) v[j] = __ldcs(from + w0 + 32 * j);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int w = w0 + 32 * j;
      if (w < n) to[(int64_t)(w >> 3) * (a.page * 8) + (w & 7)] = v[j];
    }
  }
}

// ---------------------------------------------------------------------------
// fork, first kernel: which entries of the list hold, and a page for each
// whose source ends inside one.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kBookThreads)
    pages_fork_book_kernel(PagesArgs a, const int32_t *src, const int32_t *dst, int n,
                           int32_t *status) {
  extern __shared__ int sh[];
  __shared__ int buf[kBookWarps];
  int *claim = sh;               // [n_slot] the first entry of the list that names the slot
  int *upto = sh + a.n_slot;     // [n]
  int *len = upto + n;           // [n] the source's length at the call, -1: refused
  pdl_launch_dependents();
  pdl_wait();
  const int64_t cap = capacity(a);
  for (int i = threadIdx.x; i < a.n_slot; i += kBookThreads) claim[i] = n;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kBookThreads)
    if (dst[i] >= 0 && dst[i] < a.n_slot) atomicMin(&claim[dst[i]], i);
  __syncthreads();
  int total = 0;
  for (int base = 0; base < n; base += kBookThreads) {
    const int i = base + threadIdx.x;
    int need = 0;
    if (i < n) {
      const int s = src[i], d = dst[i];
      int l = -1;
      if (s >= 0 && s < a.n_slot && d >= 0 && d < a.n_slot && claim[d] == i && a.n_ctx[d] == 0) {
        l = a.n_ctx[s];
        if (l > cap) l = -1;
      }
      len[i] = l;
      need = l > 0 && l % a.page ? 1 : 0;
    }
    int sum;
    const int inc = block_inclusive(need, buf, &sum);
    if (i < n) upto[i] = total + inc;
    total += sum;
  }
  __syncthreads();
  const int free = scan_free(a.refs, a.n_pages, total, buf, [&](int rank, int p) {
    const int i = owner_of(upto, n, rank);
    a.table[(int64_t)dst[i] * a.max_pages + len[i] / a.page] = p;
    a.refs[p] = 1;
  });
  for (int i = threadIdx.x; i < n; i += kBookThreads) {
    const int need = upto[i] - (i ? upto[i - 1] : 0);
    const bool fits = need == 0 || upto[i] <= free;
    status[i] = len[i] < 0 ? W8A8_FORK_BAD : fits ? W8A8_FORK_OK : W8A8_FORK_FULL;
    if (len[i] > 0 && fits) a.n_ctx[dst[i]] = len[i];
  }
}

// The whole pages' entries and counts, an entry of the list a CTA; then the rows
// that the last pages hold: a CTA takes a piece of a page (four 16-byte
// units a thread, of both pools in turn) and copies it for its share of the list,
// keeping what it read while the source stays the same: for the forks of one
// sequence the writes are left, and the reads of each entry's status, length and
// pages, one after the other, which its stores wait for (63 forks of 19 rows, 36
// layers of 20 heads, 220 MB: 52 us, 4.2 TB/s; a plain fill of as much takes 34).
__global__ void __launch_bounds__(256)
    pages_fork_rows_kernel(PagesArgs a, const int32_t *src, const int32_t *dst, int n,
                           const int32_t *status) {
  pdl_launch_dependents();
  pdl_wait();
  for (int i = blockIdx.y * gridDim.x + blockIdx.x; i < n; i += gridDim.x * gridDim.y) {
    if (status[i] != W8A8_FORK_OK) continue;
    const int whole = a.n_ctx[dst[i]] / a.page;
    for (int k = threadIdx.x; k < whole; k += 256) {
      const int p = a.table[(int64_t)src[i] * a.max_pages + k];
      a.table[(int64_t)dst[i] * a.max_pages + k] = p;
      if (p >= 0 && p < a.n_pages) atomicAdd(&a.refs[p], 1);
      else report_error(a.err, kErrPage);
    }
  }
  const bool is_v = blockIdx.x & 1;
  uint4 *pool = reinterpret_cast<uint4 *>(is_v ? a.V : a.K);
  const int64_t stride = a.page_stride / 8;
  const int u0 = (blockIdx.x >> 1) * 1024 + threadIdx.x;
  int held = -1, held_rows = 0;  // page and rows in v
  uint4 v[4];
  int64_t at[4];
  bool live[4];
  for (int i = blockIdx.y; i < n; i += gridDim.y) {
    if (status[i] != W8A8_FORK_OK) continue;
    const int len = a.n_ctx[dst[i]], whole = len / a.page, rows = len % a.page;
    if (rows == 0) continue;
    const int pf = a.table[(int64_t)src[i] * a.max_pages + whole];
    const int pt = a.table[(int64_t)dst[i] * a.max_pages + whole];
    if (pf < 0 || pf >= a.n_pages || pt < 0 || pt >= a.n_pages) {
      if (threadIdx.x == 0) report_error(a.err, kErrPage);
      continue;
    }
    if (pf != held || rows != held_rows) {
      // rows * 8 units in each (layer, head) segment of the page
      const int seg_units = rows * 8, n_unit = a.n_layer * a.n_kv_head * seg_units;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int x = u0 + j * 256, seg = x / seg_units;
        live[j] = x < n_unit;
        at[j] = (int64_t)seg * a.page * 8 + (x - seg * seg_units);
        if (live[j]) v[j] = pool[pf * stride + at[j]];
      }
      held = pf;
      held_rows = rows;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (live[j]) __stcs(pool + pt * stride + at[j], v[j]);
  }
}

// ---------------------------------------------------------------------------
// free: a CTA per list entry. The exchange of n_ctx hands the slot to exactly
// one CTA, so a slot named twice is given back once.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
    pages_free_kernel(PagesArgs a, const int32_t *slots) {
  __shared__ int held;
  pdl_launch_dependents();
  pdl_wait();
  const int s = slots[blockIdx.x];
  if (s < 0 || s >= a.n_slot) return;
  if (threadIdx.x == 0) held = atomicExch(&a.n_ctx[s], 0);
  __syncthreads();
  const int n = pages_of((int)min((int64_t)max(held, 0), capacity(a)), a.page);
  int32_t *row = a.table + (int64_t)s * a.max_pages;
  for (int k = threadIdx.x; k < n; k += 256) {
    const int p = row[k];
    row[k] = -1;
    if (p < 0 || p >= a.n_pages) {
      report_error(a.err, kErrPage);
    } else if (atomicSub(&a.refs[p], 1) <= 0) {
      atomicAdd(&a.refs[p], 1);
      report_error(a.err, kErrPage);
    }
  }
}

// ---------------------------------------------------------------------------
// whole pages: 16 KB pieces of both pools, a CTA a piece at a time, four
// 16-byte loads in flight a thread. Bound by HBM: 301 pages of 2.9 MB a pool in
// 580 us, 0.94 of the rate of a plain copy.
// ---------------------------------------------------------------------------
namespace {

constexpr int kPieceUnits = 1024;  // 16-byte units

__device__ __forceinline__ void copy_piece(const uint16_t *from, uint16_t *to, int64_t units,
                                           int64_t piece) {
  const uint4 *f = reinterpret_cast<const uint4 *>(from);
  uint4 *d = reinterpret_cast<uint4 *>(to);
  const int64_t u0 = piece * kPieceUnits + threadIdx.x;
  uint4 v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (u0 + j * 256 < units) v[j] = __ldcs(f + u0 + j * 256);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (u0 + j * 256 < units) __stcs(d + u0 + j * 256, v[j]);
}

}  // namespace

__global__ void __launch_bounds__(256)
    pages_copy_kernel(const uint16_t *Ks, const uint16_t *Vs, int64_t src_stride, int n_src,
                      uint16_t *Kd, uint16_t *Vd, int64_t dst_stride, int n_dst, int64_t units,
                      const int32_t *src, const int32_t *dst, int n, int *err) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t pieces = (units + kPieceUnits - 1) / kPieceUnits;
  for (int64_t x = blockIdx.x; x < 2 * pieces * n; x += gridDim.x) {
    const int i = (int)(x / (2 * pieces));
    int64_t y = x - i * (2 * pieces);
    const bool v = y >= pieces;
    if (v) y -= pieces;
    const int s = src[i], d = dst[i];
    if (s < 0 || s >= n_src || d < 0 || d >= n_dst) {
      if (threadIdx.x == 0) report_error(err, kErrPage);
      continue;
    }
    copy_piece((v ? Vs : Ks) + s * src_stride, (v ? Vd : Kd) + d * dst_stride, units, y);
  }
}

// ---------------------------------------------------------------------------
// compact, first kernel: n_live, and the j-th page in use at or above it
// paired with the j-th free page below it (there are equally many). Second
// kernel: the pages' contents and the table's entries.
//   work: [0] moves, [1 ..] movers [n_pages], holes [n_pages], renamed [n_pages]
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kBookThreads)
    pages_compact_book_kernel(PagesArgs a, int32_t *n_live_out, int32_t *work) {
  __shared__ int buf[kBookWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int32_t *movers = work + 1, *holes = movers + a.n_pages, *renamed = holes + a.n_pages;
  pdl_launch_dependents();
  pdl_wait();
  int mine = 0;
  for (int64_t p = threadIdx.x; p < a.n_pages; p += kBookThreads) mine += a.refs[p] > 0;
  int n_live;
  block_inclusive(mine, buf, &n_live);
  int n_move = 0, n_hole = 0;
  for (int64_t base = 0; base < a.n_pages; base += kRound) {
    const int64_t p0 = base + warp * (32 * kScan) + lane;
    uint32_t mov[kScan], hol[kScan];
    int32_t v[kScan];
    int cm = 0, ch = 0;
#pragma unroll
    for (int k = 0; k < kScan; ++k) v[k] = p0 + 32 * k < a.n_pages ? a.refs[p0 + 32 * k] : 0;
#pragma unroll
    for (int k = 0; k < kScan; ++k) {
      const int64_t p = p0 + 32 * k;
      mov[k] = __ballot_sync(~0u, p < a.n_pages && p >= n_live && v[k] > 0);
      hol[k] = __ballot_sync(~0u, p < n_live && v[k] <= 0);
      cm += __popc(mov[k]);
      ch += __popc(hol[k]);
    }
    int sm, sh;
    int rm = n_move + warps_prefix(cm, buf, &sm);
    int rh = n_hole + warps_prefix(ch, buf, &sh);
    const uint32_t below = (1u << lane) - 1;
#pragma unroll
    for (int k = 0; k < kScan; ++k) {
      const int64_t p = p0 + 32 * k;
      if (p < a.n_pages) renamed[p] = (int)p;
      if ((mov[k] >> lane) & 1) movers[rm + __popc(mov[k] & below)] = (int)p;
      if ((hol[k] >> lane) & 1) holes[rh + __popc(hol[k] & below)] = (int)p;
      rm += __popc(mov[k]);
      rh += __popc(hol[k]);
    }
    n_move += sm;
    n_hole += sh;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < n_move; j += kBookThreads) {
    const int f = movers[j], t = holes[j];
    renamed[f] = t;
    a.refs[t] = a.refs[f];
    a.refs[f] = 0;
  }
  if (threadIdx.x == 0) {
    work[0] = n_move;
    *n_live_out = n_live;
  }
}

__global__ void __launch_bounds__(256)
    pages_compact_move_kernel(PagesArgs a, int64_t units, const int32_t *work) {
  const int32_t *movers = work + 1, *holes = movers + a.n_pages, *renamed = holes + a.n_pages;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t entries = (int64_t)a.n_slot * a.max_pages;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < entries;
       e += (int64_t)gridDim.x * 256) {
    const int p = a.table[e];
    if (p >= 0 && p < a.n_pages) {
      const int q = renamed[p];
      if (q != p) a.table[e] = q;
    }
  }
  const int64_t pieces = (units + kPieceUnits - 1) / kPieceUnits;
  const int64_t all = 2 * pieces * work[0];
  for (int64_t x = blockIdx.x; x < all; x += gridDim.x) {
    const int j = (int)(x / (2 * pieces));
    int64_t y = x - j * (2 * pieces);
    const bool v = y >= pieces;
    if (v) y -= pieces;
    uint16_t *pool = v ? a.V : a.K;
    copy_piece(pool + (int64_t)movers[j] * a.page_stride, pool + (int64_t)holes[j] * a.page_stride,
               units, y);
  }
}

// ---------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------
// The fork's lists at their longest, allowed once a device and never lowered: a call's own size
// would be for calls of other threads too, and the default 48 KB hold the kernel's static
// shared memory as well.
static int fork_book_opt_in() {
  static bool done[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return W8A8_ERR_CUDA;
  if (!done[dev]) {
    if (cudaFuncSetAttribute(pages_fork_book_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             3 * W8A8_PAGES_MAX_LIST * (int)sizeof(int)) != cudaSuccess)
      return W8A8_ERR_CUDA;
    done[dev] = true;
  }
  return W8A8_OK;
}

int launch_pages_extend(const PagesArgs &a, const int32_t *n_new, int32_t *pos0, cudaStream_t s) {
  launch_pdl(pages_extend_kernel, dim3(1), dim3(kBookThreads), (size_t)a.n_slot * 4, s, a, n_new,
             pos0);
  return check_launch("pages_extend");
}

int launch_pages_write(const PagesArgs &a, int layer, const uint16_t *Kn, int64_t ldk,
                       const uint16_t *Vn, int64_t ldv, int n_seq, int T, const int32_t *n_new,
                       const int32_t *pos0, cudaStream_t s) {
  const int64_t warps = 2 * (int64_t)n_seq * T;
  if (warps > 0x7fffffff) return W8A8_ERR_UNSUPPORTED;
  const int64_t blocks = (warps + 7) / 8;
  launch_pdl(pages_write_kernel, dim3((unsigned)blocks), dim3(256), 0, s, a,
             (int64_t)layer * a.n_kv_head * a.page * kPageHd, Kn, ldk, Vn, ldv, n_seq, T, n_new,
             pos0);
  return check_launch("pages_write");
}

int launch_pages_fork(const PagesArgs &a, const int32_t *src, const int32_t *dst, int n,
                      int32_t *status, int sm_count, cudaStream_t s) {
  const size_t smem = ((size_t)a.n_slot + 2 * (size_t)n) * 4;
  int st = fork_book_opt_in();
  if (st) return st;
  launch_pdl(pages_fork_book_kernel, dim3(1), dim3(kBookThreads), smem, s, a, src, dst, n, status);
  st = check_launch("pages_fork_book");
  if (st) return st;
  // a CTA for every piece of a page, and shares of the list for eight an SM
  const int64_t units = (int64_t)a.n_layer * a.n_kv_head * a.page * 8;
  const int64_t x = 2 * ((units + 1023) / 1024);
  int64_t y = ((int64_t)sm_count * 8 + x - 1) / x;
  if (y > n) y = n;
  launch_pdl(pages_fork_rows_kernel, dim3((unsigned)x, (unsigned)y), dim3(256), 0, s, a, src, dst,
             n, status);
  return check_launch("pages_fork_rows");
}

int launch_pages_free(const PagesArgs &a, const int32_t *slots, int n, cudaStream_t s) {
  launch_pdl(pages_free_kernel, dim3(n), dim3(256), 0, s, a, slots);
  return check_launch("pages_free");
}

int launch_pages_compact(const PagesArgs &a, int32_t *n_live, int32_t *work, int sm_count,
                         cudaStream_t s) {
  launch_pdl(pages_compact_book_kernel, dim3(1), dim3(kBookThreads), 0, s, a, n_live, work);
  int st = check_launch("pages_compact_book");
  if (st) return st;
  const int64_t units = (int64_t)a.n_layer * a.n_kv_head * a.page * 8;
  launch_pdl(pages_compact_move_kernel, dim3(sm_count * 8), dim3(256), 0, s, a, units, work);
  return check_launch("pages_compact_move");
}

int launch_pages_copy(const uint16_t *Ks, const uint16_t *Vs, int64_t src_stride, int n_src,
                      uint16_t *Kd, uint16_t *Vd, int64_t dst_stride, int n_dst, int64_t elems,
                      const int32_t *src, const int32_t *dst, int n, int *err, int sm_count,
                      cudaStream_t s) {
  const int64_t units = elems / 8;
  const int64_t all = 2 * ((units + kPieceUnits - 1) / kPieceUnits) * n;
  const int64_t grid = all < (int64_t)sm_count * 8 ? all : (int64_t)sm_count * 8;
  launch_pdl(pages_copy_kernel, dim3((unsigned)grid), dim3(256), 0, s, Ks, Vs, src_stride, n_src,
             Kd, Vd, dst_stride, n_dst, units, src, dst, n, err);
  return check_launch("pages_copy");
}

}  // namespace w8a8

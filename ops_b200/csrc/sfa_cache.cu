// sfa_cache.cu — pages of a kv cache: reserving, trimming, forking and copying
// them, moving the accepted rows of a drafted tree together, and compacting a
// pool.  The state is a reference count per page; a page is free when it is 0,
// and new pages are the free ones of lowest number in the order of the rows that
// ask.  So nothing depends on the order of atomics (counts only add up), and no
// free list has to be kept in order.
//
// Bookkeeping runs in one CTA (its cost is a few dependent passes over tables of
// some thousand entries; several CTAs would spend as long on meeting each other);
// pages and rows are then moved by as many CTAs as fill the SMs, from lists that
// the bookkeeping left in the workspace.  Measured: 2.35 GB read and written to
// move some 1100 pages of 128 KB in each of 8 pools in 394 us (0.91 of the measured copy
// rate); a beam step of 64 sequences (trim, fork, its 32 pages in 16 pools, reserve) in
// 37 us, 20.5 of them the pages' floor; acceptance and trim of 128 trees in 32 pools in
// 21 us, a chain of dependent reads (lengths, path, table, counts, rows) around 10 us of
// rows, and in 24 us where acceptance counts the table's entries itself (both with 6 us
// that restore the state between calls).
#include "sfa_common.cuh"
#include "sfa_internal.h"

#include <algorithm>
#include <string>

namespace sfa {
namespace cache {

constexpr int kPlan = 1024;       // threads of a bookkeeping CTA
constexpr int kMove = 256;        // threads of a moving CTA
constexpr int kMaxPools = 128;    // pools of one launch
constexpr int kChunk = 16384;     // bytes of a moving CTA's step
constexpr int kNone = 0x7f7f7f7f; // "no pair" in an owner table (a memset pattern, above every index)
constexpr int kRows = 64;         // accepted rows listed at a time

struct Pools {
  SfaCachePool t[kMaxPools];
};

struct Work {          // workspace, int32
  int* head;           // [16]: 0 pages in use, 1 pages to move
  int* off;            // [items] first new page of each item
  int* owner;          // [max(num_seqs, num_pages)]
  int* list;           // [num_pages] free pages, ascending (compact: holes)
  int* src;            // [max(count, num_pages)] page moves
  int* dst;
  int* remap;          // [num_pages]
};

static size_t carve(const SfaCacheParams& p, char* ws, Work* w) {
  const size_t items = (size_t)std::max(p.num_seqs, p.count), pages = (size_t)p.num_pages;
  size_t at = 0;
  auto take = [&](size_t n) {
    int* r = reinterpret_cast<int*>(ws) + at;
    at += (n + 63) / 64 * 64;
    return r;
  };
  Work r;
  r.head = take(16);
  r.off = take(items);
  r.owner = take(std::max((size_t)p.num_seqs, pages));
  r.list = take(pages);
  r.src = take(std::max((size_t)p.count, pages));
  r.dst = take(std::max((size_t)p.count, pages));
  r.remap = take(pages);
  if (w) *w = r;
  return at * sizeof(int);
}

__device__ __forceinline__ int pages_of(int rows, int page_size) { return rows > 0 ? (rows - 1) / page_size + 1 : 0; }

// Exclusive sum of v over the CTA's threads in order; *total: the sum.  A barrier before part[] is written and
// one after it, none once it has been read: what a thread wrote before or writes after the call is not yet
// there for the others.
template <typename N>
__device__ __forceinline__ N block_scan(N v, N* total) {
  __shared__ N part[kPlan / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  N run = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  __syncthreads();
  if (lane == 31) part[warp] = run;
  __syncthreads();
  N sums = part[lane];                                        // each warp scans the warps' sums for itself
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const N up = __shfl_up_sync(0xffffffffu, sums, o);
    if (lane >= o) sums += up;
  }
  *total = __shfl_sync(0xffffffffu, sums, 31);
  const N before = __shfl_sync(0xffffffffu, sums, max(warp - 1, 0));
  return (warp > 0 ? before : 0) + run - v;
}

// This thread's part of [0, n), the parts ascending with the thread.
__device__ __forceinline__ void strip(int n, int& i0, int& i1) {
  const int per = (n + kPlan - 1) / kPlan;
  i0 = min(n, (int)threadIdx.x * per);
  i1 = min(n, i0 + per);
}

// The first `want` free pages in ascending order into w.list; returns how many are free.
__device__ __forceinline__ int list_free(const SfaCacheParams& p, const Work& w, int want) {
  int i0, i1, mine = 0, all;
  strip(p.num_pages, i0, i1);
  for (int i = i0; i < i1; ++i) mine += p.refcounts[i] <= 0;
  int at = block_scan(mine, &all);
  for (int i = i0; i < i1 && at < want; ++i)
    if (p.refcounts[i] <= 0) w.list[at++] = i;
  __syncthreads();
  return all;
}

__global__ void __launch_bounds__(kPlan) reserve_kernel(const __grid_constant__ SfaCacheParams p, const __grid_constant__ Work w) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // pages that a row needs, -1 if it cannot get them at all
  auto need = [&](int s) {
    const int len = p.cache_seqlens[s], add = p.a[s];
    if (len < 0 || add < 0 || add > INT32_MAX - p.page_size - len) return -1;
    if (pages_of(len + add, p.page_size) > p.table_width) return -1;
    if (add > 0 && len % p.page_size) {
      const int pg = p.block_table[s * p.bt_stride + len / p.page_size];
      if (pg < 0 || pg >= p.num_pages || p.refcounts[pg] > 1) return -1;
    }
    const int n = pages_of(len + add, p.page_size) - pages_of(len, p.page_size);
    return n <= p.num_pages ? n : -1;
  };
  int s0, s1;
  long long mine = 0, want;
  strip(p.num_seqs, s0, s1);
  for (int s = s0; s < s1; ++s) mine += max(need(s), 0);
  long long at = block_scan(mine, &want);
  for (int s = s0; s < s1; ++s) {
    const int n = need(s);
    w.off[s] = n < 0 ? -1 : (int)min(at, (long long)p.num_pages);   // nothing is free from there on
    at += max(n, 0);
  }
  __syncthreads();
  const int have = want > 0 ? list_free(p, w, (int)min(want, (long long)p.num_pages)) : 0;
  for (int s = warp; s < p.num_seqs; s += kPlan / 32) {
    const int first = w.off[s];
    const int len = p.cache_seqlens[s], add = p.a[s];
    const int held = pages_of(len, p.page_size);
    const int n = first < 0 ? 0 : pages_of(len + add, p.page_size) - held;
    const bool ok = first >= 0 && (n == 0 || (int64_t)first + n <= have);
    __syncwarp();
    if (ok)
      for (int j = lane; j < n; j += 32) {
        const int pg = w.list[first + j];
        p.block_table[s * p.bt_stride + held + j] = pg;
        p.refcounts[pg] = 1;
      }
    if (lane == 0) {
      if (ok) p.cache_seqlens[s] = len + add;
      p.out[s] = ok ? 1 : 0;
    }
  }
}

__global__ void __launch_bounds__(kMove) trim_kernel(const __grid_constant__ SfaCacheParams p) {
  const int s = blockIdx.x, len = p.cache_seqlens[s], keep = p.a[s];
  if (keep < 0) return;
  const int left = min(len, keep);
  int32_t* row = p.block_table + s * p.bt_stride;
  for (int c = pages_of(left, p.page_size) + threadIdx.x; c < p.table_width; c += kMove) {
    const int pg = row[c];
    if (pg < 0) continue;
    if (pg < p.num_pages) atomicSub(p.refcounts + pg, 1);
    row[c] = -1;
  }
  __syncthreads();                       // every thread has read the length
  if (threadIdx.x == 0) p.cache_seqlens[s] = left;
}

__global__ void __launch_bounds__(kPlan) fork_kernel(const __grid_constant__ SfaCacheParams p, const __grid_constant__ Work w) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < p.num_seqs; i += kPlan) w.owner[i] = kNone;
  __syncthreads();
  for (int i = threadIdx.x; i < p.count; i += kPlan) {
    const int d = p.b[i];
    if (d >= 0 && d < p.num_seqs) atomicMin(w.owner + d, i);
  }
  __syncthreads();
  // the page to copy, -1: none, -2: the fork cannot be done
  auto partial = [&](int i) {
    const int s = p.a[i], d = p.b[i];
    if (s < 0 || s >= p.num_seqs || d < 0 || d >= p.num_seqs || s == d) return -2;
    if (w.owner[d] != i || p.cache_seqlens[d] != 0) return -2;
    const int len = p.cache_seqlens[s];
    if (len < 0 || pages_of(len, p.page_size) > p.table_width) return -2;
    if (len % p.page_size == 0) return -1;
    const int pg = p.block_table[s * p.bt_stride + len / p.page_size];
    return pg >= 0 && pg < p.num_pages ? pg : -2;
  };
  int i0, i1, mine = 0, want;
  strip(p.count, i0, i1);
  for (int i = i0; i < i1; ++i) mine += partial(i) >= 0;
  int at = block_scan(mine, &want);
  const int have = want > 0 ? list_free(p, w, want) : 0;
  for (int i = i0; i < i1; ++i) {
    const int pg = partial(i);
    const bool ok = pg == -1 || (pg >= 0 && at < have);
    w.src[i] = ok ? pg : -1;
    w.dst[i] = ok && pg >= 0 ? w.list[at] : -1;
    w.off[i] = ok ? p.cache_seqlens[p.a[i]] : -1;            // the target's length
    at += pg >= 0;
  }
  __syncthreads();                                           // sources are read, targets follow
  for (int i = warp; i < p.count; i += kPlan / 32) {
    const int len = w.off[i];
    if (lane == 0) p.out[i] = len >= 0 ? 1 : 0;
    if (len < 0) continue;
    const int d = p.b[i], whole = len / p.page_size;
    const int32_t* from = p.block_table + p.a[i] * p.bt_stride;
    int32_t* to = p.block_table + d * p.bt_stride;
    for (int c = lane; c < p.table_width; c += 32) {
      int pg = -1;
      if (c < whole) {
        pg = from[c];
        if (pg >= 0 && pg < p.num_pages) atomicAdd(p.refcounts + pg, 1);
      } else if (c == whole && w.dst[i] >= 0) {
        pg = w.dst[i];
        p.refcounts[pg] = 1;
      }
      to[c] = pg;
    }
    if (lane == 0) p.cache_seqlens[d] = len;
  }
}

// Pages in use and the moves that bring them to the lowest numbers: the k-th used
// page at or above their number goes to the k-th free page below it.
__global__ void __launch_bounds__(kPlan) compact_kernel(const __grid_constant__ SfaCacheParams p, const __grid_constant__ Work w) {
  int i0, i1, mine = 0, live, holes, moves;
  strip(p.num_pages, i0, i1);
  for (int i = i0; i < i1; ++i) mine += p.refcounts[i] > 0;
  block_scan(mine, &live);
  int free_low = 0, used_high = 0;
  for (int i = i0; i < i1; ++i) {
    const bool used = p.refcounts[i] > 0;
    free_low += !used && i < live;
    used_high += used && i >= live;
  }
  int h = block_scan(free_low, &holes), m = block_scan(used_high, &moves);
  for (int i = i0; i < i1; ++i) {
    const bool used = p.refcounts[i] > 0;
    if (!used && i < live) w.dst[h++] = i;
    if (used && i >= live) w.src[m++] = i;
    if (!used && i >= live) w.remap[i] = i;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < moves; k += kPlan) {
    const int from = w.src[k], to = w.dst[k];
    w.remap[from] = to;
    p.refcounts[to] = p.refcounts[from];
    p.refcounts[from] = 0;
  }
  if (threadIdx.x == 0) {
    w.head[0] = live;
    w.head[1] = moves;
    p.out[0] = live;
  }
}

__global__ void __launch_bounds__(kMove) claim_kernel(const __grid_constant__ SfaCacheParams p, const __grid_constant__ Work w) {
  const int i = blockIdx.x * kMove + threadIdx.x;
  if (i >= p.count) return;
  const int s = p.a[i], d = p.b[i];
  if (s >= 0 && s < p.num_pages && d >= 0 && d < p.num_pages) atomicMin(w.owner + d, i);
}

// n bytes (at most kChunk) by the whole CTA, in the widest units that fit.
template <typename V>
__device__ __forceinline__ void copy_units(const char* from, char* to, int n) {
  const V* f = reinterpret_cast<const V*>(from);
  V* t = reinterpret_cast<V*>(to);
  const int units = n / (int)sizeof(V);
  for (int i = threadIdx.x; i < units; i += kMove * 4) {
    V v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k * kMove < units) v[k] = f[i + k * kMove];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k * kMove < units) t[i + k * kMove] = v[k];
  }
}
__device__ __forceinline__ int unit_of(const SfaCachePool& t, int64_t extra) {
  const uint64_t all = reinterpret_cast<uint64_t>(t.base) | (uint64_t)t.page_stride | (uint64_t)t.page_bytes | (uint64_t)extra;
  return (all & 15) == 0 ? 16 : (all & 3) == 0 ? 4 : 1;
}

enum Moves { kFork, kCompact, kCopy };

// The pages of a list, every pool (gridDim.y).  Compaction also renumbers the table.
template <Moves KIND>
__global__ void __launch_bounds__(kMove) move_kernel(const __grid_constant__ SfaCacheParams p, const __grid_constant__ Work w,
                                                     const __grid_constant__ Pools pools, int first_launch) {
  const int moves = KIND == kCompact ? w.head[1] : p.count;
  if (KIND == kCompact && first_launch && blockIdx.y == 0) {
    const int live = w.head[0];
    const int64_t entries = (int64_t)p.num_seqs * p.table_width;
    for (int64_t i = (int64_t)blockIdx.x * kMove + threadIdx.x; i < entries; i += (int64_t)gridDim.x * kMove) {
      int32_t* e = p.block_table + i / p.table_width * p.bt_stride + i % p.table_width;
      const int pg = *e;
      if (pg >= live && pg < p.num_pages) *e = w.remap[pg];
    }
  }
  if (KIND == kCopy && first_launch && blockIdx.y == 0)
    for (int i = blockIdx.x * kMove + threadIdx.x; i < p.count; i += gridDim.x * kMove) {
      const int s = p.a[i], d = p.b[i];
      const bool in = s >= 0 && s < p.num_pages && d >= 0 && d < p.num_pages;
      p.out[i] = in && w.owner[d] == i && (s == d || w.owner[s] == kNone) ? 1 : 0;
    }
  if ((int)blockIdx.y >= p.num_pools) return;
  const SfaCachePool t = pools.t[blockIdx.y];
  const int unit = unit_of(t, 0);
  const int chunks = (int)((t.page_bytes + kChunk - 1) / kChunk);
  const int64_t steps = (int64_t)moves * chunks;
  for (int64_t k = blockIdx.x; k < steps; k += gridDim.x) {
    const int i = (int)(k / chunks);
    const int64_t at = (k - (int64_t)i * chunks) * kChunk;
    int s, d;
    if (KIND == kCopy) {
      s = p.a[i];
      d = p.b[i];
      const bool in = s >= 0 && s < p.num_pages && d >= 0 && d < p.num_pages;
      if (!in || s == d || w.owner[d] != i || w.owner[s] != kNone) continue;
    } else {
      s = w.src[i];
      d = w.dst[i];
      if (s < 0 || d < 0) continue;
    }
    const char* from = static_cast<const char*>(t.base) + s * t.page_stride + at;
    char* to = static_cast<char*>(t.base) + d * t.page_stride + at;
    const int n = (int)min((int64_t)kChunk, t.page_bytes - at);
    if (unit == 16) copy_units<uint4>(from, to, n);
    else if (unit == 4) copy_units<uint32_t>(from, to, n);
    else copy_units<uint8_t>(from, to, n);
  }
}

struct Rows {              // of one sequence, taken together: -1: stays where it is
  int page_from[kRows], row_from[kRows], page_to[kRows], row_to[kRows];
};

// Accepted rows i of a sequence: cache row prefix + a[i] to prefix + i.  A thread owns the same bytes of
// every row and takes the rows in order; a[i] >= i, so a row is read before a later one is written over it,
// eight at a time.
template <typename V>
__device__ __forceinline__ void move_rows(const SfaCachePool& t, const Rows& r, int n, int64_t row_bytes, int lane, int lanes) {
  char* base = static_cast<char*>(t.base);
  for (int64_t u = lane * sizeof(V); u < row_bytes; u += lanes * sizeof(V))
    for (int i = 0; i < n; i += 8) {
      V v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i + k < n && r.page_from[i + k] >= 0)
          v[k] = *reinterpret_cast<const V*>(base + r.page_from[i + k] * t.page_stride + r.row_from[i + k] * row_bytes + u);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i + k < n && r.page_from[i + k] >= 0)
          *reinterpret_cast<V*>(base + r.page_to[i + k] * t.page_stride + r.row_to[i + k] * row_bytes + u) = v[k];
    }
}

// A CTA finds the rows of its sequence once and moves them in several pools, `lanes` threads a pool.
// Nothing of a sequence moves if one of its rows would go into a page that others hold (a fork shares whole
// pages, those of drafted rows too): a path of several lists is looked through for that first.
__global__ void __launch_bounds__(kMove) accept_kernel(const __grid_constant__ SfaCacheParams p, const __grid_constant__ Pools pools,
                                                       int lanes, int first_launch) {
  __shared__ Rows rows;
  __shared__ int bad_at;
  const int s = blockIdx.x;
  const int len = p.cache_seqlens[s], m = p.b[s];
  const bool fine = m >= 0 && m <= len;
  const int prefix = len - m;
  int kept = 0;
  bool shared = false;
  for (int pass = p.refcounts && p.count > kRows ? 0 : 1; pass < 2 && !shared; ++pass) {
    bool more = fine;
    kept = 0;
    for (int i0 = 0; i0 < p.count && more; i0 += kRows) {
      const int i = i0 + threadIdx.x, n = min(kRows, p.count - i0);
      bool held = false;                                      // by another sequence too: the page this row goes to
      if (threadIdx.x == 0) bad_at = n;
      __syncthreads();
      if (threadIdx.x < n) {
        const int32_t* acc = p.a + s * p.a_stride;
        const int a = acc[i], before = i > 0 ? acc[i - 1] : -1;
        const bool ok = a >= 0 && a < m && a > before;
        if (!ok) atomicMin(&bad_at, (int)threadIdx.x);
        rows.page_from[threadIdx.x] = -1;
        if (ok && a != i) {
          const int x = prefix + a, y = prefix + i;
          const int cx = x / p.page_size, cy = y / p.page_size;
          if (cx < p.table_width && cy < p.table_width) {
            const int px = p.block_table[s * p.bt_stride + cx], py = p.block_table[s * p.bt_stride + cy];
            if (px >= 0 && px < p.num_pages && py >= 0 && py < p.num_pages) {
              held = p.refcounts && p.refcounts[py] > 1;
              rows.page_from[threadIdx.x] = px;
              rows.row_from[threadIdx.x] = x % p.page_size;
              rows.page_to[threadIdx.x] = py;
              rows.row_to[threadIdx.x] = y % p.page_size;
            }
          }
        }
      }
      __syncthreads();
      const int take = bad_at, together = kMove / lanes;
      shared = __syncthreads_or(held && (int)threadIdx.x < take);
      if (shared) break;
      more = take == n;
      kept += take;
      if (pass == 1)
        for (int q = blockIdx.y * together + threadIdx.x / lanes; q < p.num_pools; q += gridDim.y * together) {
          const SfaCachePool& t = pools.t[q];
          const int64_t row_bytes = t.page_bytes / p.page_size;
          const int unit = unit_of(t, row_bytes), lane = threadIdx.x % lanes;
          if (unit == 16) move_rows<uint4>(t, rows, take, row_bytes, lane, lanes);
          else if (unit == 4) move_rows<uint32_t>(t, rows, take, row_bytes, lane, lanes);
          else move_rows<uint8_t>(t, rows, take, row_bytes, lane, lanes);
        }
      __syncthreads();                                        // the rows have been read
    }
  }
  if (first_launch && blockIdx.y == 0 && threadIdx.x == 0) p.out[s] = fine && !shared ? prefix + kept : -1;
}

// How many entries of the table hold each page, into refcounts (zeroed before), a CTA a sequence.
__global__ void __launch_bounds__(kMove) count_kernel(const __grid_constant__ SfaCacheParams p) {
  const int s = blockIdx.x, n = min(p.table_width, pages_of(p.cache_seqlens[s], p.page_size));
  for (int c = threadIdx.x; c < n; c += kMove) {
    const int pg = p.block_table[s * p.bt_stride + c];
    if (pg >= 0 && pg < p.num_pages) atomicAdd(p.refcounts + pg, 1);
  }
}

static int bad(const char* what, const std::string& m) {
  return report_error(SFA_ERR_INVALID_ARGUMENT, std::string("cache ") + what + ": " + m);
}

static int check(const SfaCacheParams* p, const char* what, bool refs, bool table, bool pools, bool b, bool rows) {
  // which of the fields a call reads: reference counts, table and lengths, pools, the second argument
  // array; whether the arrays go by sequence (rows) or by count
  if (!p) return bad(what, "params is NULL");
  // strip() adds the threads to a size, and kNone is no index
  if (p->num_pools < 0 || p->num_seqs < 0 || p->num_pages < 0 || p->table_width < 0 || p->count < 0 || p->num_seqs >= kNone ||
      p->num_pages >= kNone || p->count >= kNone)
    return bad(what, "sizes must be >= 0 and below " + std::to_string(kNone));
  if (p->page_size < 1) return bad(what, "page_size must be positive");
  if (refs && p->num_pages > 0 && !p->refcounts) return bad(what, "refcounts must be non-NULL");
  if (table && p->num_seqs > 0 && (!p->cache_seqlens || (p->table_width > 0 && !p->block_table)))
    return bad(what, "block_table and cache_seqlens must be non-NULL");
  const int64_t items = rows ? p->num_seqs : p->count;
  if (items > 0 && (!p->a || !p->out || (b && !p->b))) return bad(what, "the argument and output arrays must be non-NULL");
  if (pools) {
    if (p->num_pools > 0 && !p->pools) return bad(what, "pools must be non-NULL");
    for (int i = 0; i < p->num_pools; ++i) {
      const SfaCachePool& t = p->pools[i];
      if (p->num_pages > 0 && !t.base && t.page_bytes > 0) return bad(what, "a pool's base must be non-NULL");
      if (t.page_bytes < 0 || t.page_bytes % p->page_size) return bad(what, "page_bytes must be a multiple of page_size");
      if (p->num_pages > 1 && t.page_stride < t.page_bytes) return bad(what, "page_stride must be at least page_bytes");
    }
  }
  return SFA_OK;
}

static int take_ws(const SfaCacheParams& p, const char* what, void* ws, size_t bytes, Work* w) {
  const size_t need = carve(p, static_cast<char*>(ws), w);
  if (!ws || bytes < need || (reinterpret_cast<uintptr_t>(ws) & 3))
    return report_error(SFA_ERR_WORKSPACE, std::string("cache ") + what + ": workspace missing, unaligned or too small: need " +
                                               std::to_string(need) + " bytes");
  return SFA_OK;
}

static int done(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SFA_OK : report_error(SFA_ERR_CUDA, std::string("cache ") + what + ": " + cudaGetErrorString(e));
}

// kMaxPools pools a launch; f(params with that many pools, pools, first launch).
template <typename F>
static void by_pools(const SfaCacheParams& p, bool at_least_one, F f) {
  for (int i = 0; i < p.num_pools || (i == 0 && at_least_one); i += kMaxPools) {
    SfaCacheParams q = p;
    Pools t{};
    q.num_pools = std::min(kMaxPools, p.num_pools - i);
    for (int k = 0; k < q.num_pools; ++k) t.t[k] = p.pools[i + k];
    f(q, t, i == 0 ? 1 : 0);
  }
}

// CTAs per pool: enough to fill the SMs eight deep together, no more than there are steps.
static unsigned move_ctas(const SfaCacheParams& q, const Pools& t, int64_t moves) {
  int64_t steps = 1;
  for (int k = 0; k < q.num_pools; ++k) steps = std::max(steps, moves * ((t.t[k].page_bytes + kChunk - 1) / kChunk));
  const int64_t fill = std::max<int64_t>(1, (int64_t)device_sm_count() * 8 / std::max(1, q.num_pools));
  return (unsigned)std::min(steps, fill);
}

}  // namespace cache
}  // namespace sfa

using namespace sfa;
using namespace sfa::cache;

extern "C" {

size_t sfa_cache_workspace_bytes(const SfaCacheParams* p) {
  if (!p || p->num_seqs < 0 || p->num_pages < 0 || p->count < 0) return 0;
  return carve(*p, nullptr, nullptr);
}

int sfa_cache_reserve(const SfaCacheParams* p, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(p, "reserve", true, true, false, false, true);
  if (rc || p->num_seqs == 0) return rc;
  Work w;
  if ((rc = take_ws(*p, "reserve", workspace, workspace_bytes, &w))) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  reserve_kernel<<<1, kPlan, 0, st>>>(*p, w);
  note_launch("cache_reserve", st);
  return done("reserve");
}

int sfa_cache_trim(const SfaCacheParams* p, void* stream) {
  SfaCacheParams q = p ? *p : SfaCacheParams{};
  q.out = q.out ? q.out : q.cache_seqlens;          // no output array
  const int rc = check(p ? &q : nullptr, "trim", true, true, false, false, true);
  if (rc || p->num_seqs == 0) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  trim_kernel<<<p->num_seqs, kMove, 0, st>>>(*p);
  note_launch("cache_trim", st);
  return done("trim");
}

int sfa_cache_fork(const SfaCacheParams* p, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(p, "fork", true, true, true, true, false);
  if (rc || p->count == 0) return rc;
  Work w;
  if ((rc = take_ws(*p, "fork", workspace, workspace_bytes, &w))) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  fork_kernel<<<1, kPlan, 0, st>>>(*p, w);
  note_launch("cache_fork", st);
  by_pools(*p, false, [&](const SfaCacheParams& q, const Pools& t, int first) {
    move_kernel<kFork><<<dim3(move_ctas(q, t, q.count), q.num_pools), kMove, 0, st>>>(q, w, t, first);
    note_launch("cache_fork_pages", st);
  });
  return done("fork");
}

int sfa_cache_accept(const SfaCacheParams* p, void* stream) {
  const int rc = check(p, "accept", false, true, true, true, true);
  if (rc || p->num_seqs == 0) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  by_pools(*p, true, [&](const SfaCacheParams& q, const Pools& t, int first) {
    // threads a pool: as many as the widest row has units; CTAs: one wave of eight per SM, each with
    // several pools (with a CTA for each sequence and pool, acceptance and trim of 128 sequences in 32 pools
    // took 11 us more)
    int lanes = 32;
    for (int k = 0; k < q.num_pools; ++k)
      while (lanes < kMove && t.t[k].page_bytes / q.page_size > 16 * (int64_t)lanes) lanes *= 2;
    const int most = std::max(1, (q.num_pools + kMove / lanes - 1) / (kMove / lanes));
    const int y = std::min(most, std::max(1, device_sm_count() * 8 / q.num_seqs));
    accept_kernel<<<dim3(q.num_seqs, y), kMove, 0, st>>>(q, t, lanes, first);
    note_launch("cache_accept", st);
  });
  return done("accept");
}

int sfa_cache_accept_table(const SfaCacheParams* p, void* stream) {
  const int rc = check(p, "accept", true, true, true, true, true);
  if (rc || p->num_seqs == 0) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p->num_pages > 0) {
    const cudaError_t e = cudaMemsetAsync(p->refcounts, 0, sizeof(int32_t) * (size_t)p->num_pages, st);
    if (e != cudaSuccess) return report_error(SFA_ERR_CUDA, std::string("cache accept: ") + cudaGetErrorString(e));
    note_memset("cache_count", st);
    count_kernel<<<p->num_seqs, kMove, 0, st>>>(*p);
    note_launch("cache_count", st);
  }
  return sfa_cache_accept(p, stream);
}

int sfa_cache_compact(const SfaCacheParams* p, void* workspace, size_t workspace_bytes, void* stream) {
  SfaCacheParams q0 = p ? *p : SfaCacheParams{};
  q0.cache_seqlens = q0.cache_seqlens ? q0.cache_seqlens : q0.out;   // no lengths, no argument arrays
  q0.a = q0.a ? q0.a : q0.out;
  int rc = check(p ? &q0 : nullptr, "compact", true, true, true, false, true);
  if (rc) return rc;
  if (!p->out) return bad("compact", "the output must be non-NULL");
  Work w;
  if ((rc = take_ws(*p, "compact", workspace, workspace_bytes, &w))) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  compact_kernel<<<1, kPlan, 0, st>>>(*p, w);
  note_launch("cache_compact", st);
  by_pools(*p, true, [&](const SfaCacheParams& q, const Pools& t, int first) {
    move_kernel<kCompact><<<dim3(std::max(8u, move_ctas(q, t, q.num_pages / 2)), std::max(1, q.num_pools)), kMove, 0, st>>>(q, w, t, first);
    note_launch("cache_compact_pages", st);
  });
  return done("compact");
}

int sfa_cache_copy(const SfaCacheParams* p, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(p, "copy", false, false, true, true, false);
  if (rc || p->count == 0) return rc;
  Work w;
  if ((rc = take_ws(*p, "copy", workspace, workspace_bytes, &w))) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = cudaMemsetAsync(w.owner, 0x7f, sizeof(int) * (size_t)std::max(p->num_pages, 1), st);
  if (e != cudaSuccess) return report_error(SFA_ERR_CUDA, std::string("cache copy: ") + cudaGetErrorString(e));
  note_memset("cache_copy_owner", st);
  claim_kernel<<<(p->count + kMove - 1) / kMove, kMove, 0, st>>>(*p, w);
  note_launch("cache_copy_claim", st);
  by_pools(*p, true, [&](const SfaCacheParams& q, const Pools& t, int first) {
    move_kernel<kCopy><<<dim3(move_ctas(q, t, q.count), std::max(1, q.num_pools)), kMove, 0, st>>>(q, w, t, first);
    note_launch("cache_copy_pages", st);
  });
  return done("copy");
}

}  // extern "C"

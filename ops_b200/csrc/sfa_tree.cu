// sfa_tree.cu — attention of drafted tokens (a tree, a chain, or one token) over
// a paged kv cache: the split of the work, the kernel that joins its pieces, and
// the host side.  sfa_tree_pair.cu and sfa_tree_wide.cu hold the attention.
//
//   o[r] = sum_t p[r,t] v[t] / sum_t p[r,t],  p = exp(scale q[r].k[t]) over the
//   cache rows r sees: all before the drafted ones, its ancestors and itself.
//
// Tile: the G query heads of a kv head times as many drafted rows as fit make the
// M = 128 rows of one MMA,
//     S[rows, keys] = Q . K^T,   O[rows, d_v] += P . V,
// so a key row read from the cache serves every head and every drafted row; a
// decode step is bound by those reads, a large tree by the MMAs and the softmax.
//
// Split: the (sequence, kv head, chunk of keys) space of all sequences is one line
// that gridDim.x CTAs cut into equal ranges, whatever the lengths of the caches; a CTA
// walks the units (sequence, kv head) its range touches.  A unit that lies in one range is
// finished there; pieces of the others go to a workspace as (m, l, O) and
// tree_combine_kernel joins them in range order.  The gridDim.y row tiles of a
// unit walk the same range at the same time and share its reads in L2.  The line does
// not count rows: gridDim.y comes from the longest sequence of drafted rows (max_q),
// gridDim.x is what is left of the SMs, and of a sequence with fewer rows only the CTAs
// of its own tiles work.  Rows of very different numbers therefore belong in calls of
// their own: 63 single tokens over 4096 to 32768 keys take 846 us and one chunk of 2048
// rows 706, both in one call 47.7 ms (64 tile pairs leave two ranges); 15 single tokens
// take 239 us and a chain of 64 rows 52, together 666.
//
// Keys come through the block table with TMA boxes of as many rows as divide both
// a page and a chunk, 128B-swizzled 64-dim slabs; a box without a page (a table
// entry outside the pool, or positions behind the cache) is read out of the
// tensor map's bounds, which fills zeros without touching memory.
//
// Softmax: one thread per row.  P = exp2(S c - m) in fp32, rounded once to the
// MMA operand's type (the row sum keeps the unrounded values).  m is not the
// maximum but a reference, set to it (fp16: 2^8 below it, see Reference): it is raised,
// and O rescaled in TMEM, only when a sum of P exceeds 2^14 (2^15), so the common pass
// takes no maximum.  P overwrites S's columns as the PV MMA's A operand.
#include "sfa_tree.cuh"

#include <algorithm>
#include <string>

namespace sfa {
namespace tree {

template <typename T>
__device__ __forceinline__ void store4(T* at, float4 v) {
  *reinterpret_cast<uint2*>(at) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
}

template <typename T>
__device__ __forceinline__ void empty_row(const SfaTreeParams& p, int64_t row, int head, int grp) {
  store4<T>(static_cast<T*>(p.o) + row * p.o_st + (int64_t)head * p.o_sh + grp * 4, make_float4(0.f, 0.f, 0.f, 0.f));
  if (grp == 0) p.lse[row * p.l_st + (int64_t)head * p.l_sh] = p.attn_sink ? __ldg(p.attn_sink + head) : -INFINITY;
}

// Rows before the first and behind the last sequence, then of each sequence past the tiles (max_q was too small).
template <typename T>
static __device__ __noinline__ void rows_of_no_tile(const Args& a, int first, int step) {
  const SfaTreeParams& p = a.p;
  const int n = p.num_seqs, groups = p.d_v / 4;
  const int begin = n > 0 && p.cu_seqlens ? min(p.total_q, max(0, __ldg(p.cu_seqlens))) : 0;
  const int end = n == 0 ? 0 : p.cu_seqlens ? max(begin, __ldg(p.cu_seqlens + n)) : n;
  const int64_t todo = (int64_t)(begin + max(0, p.total_q - end)) * p.h_q * groups;
#pragma unroll 1
  for (int64_t i = first; i < todo; i += step) {
    const int64_t row = i / (groups * p.h_q);
    empty_row<T>(p, row < begin ? row : end + (row - begin), (int)(i / groups % p.h_q), (int)(i % groups));
  }
  if (!p.cu_seqlens) return;
  const int covered = a.ntiles / a.n_hg * a.NT;
#pragma unroll 1
  for (int s = first; s < n; s += step) {
    const int q0 = __ldg(p.cu_seqlens + s), q1 = min(p.total_q, __ldg(p.cu_seqlens + s + 1));
#pragma unroll 1
    for (int row = q0 < 0 ? q1 : q0 + covered; row < q1; ++row)
#pragma unroll 1
      for (int i = 0; i < p.h_q * groups; ++i) empty_row<T>(p, row, i / groups, i % groups);
  }
}

// A row's pieces r0, r0 + step .. r1 of one tile, four dims: their maximum M (with the one given), sum and O.
__device__ __forceinline__ void join_pieces(const Args& a, int tile, int m, int grp, int first_piece, int r0, int r1, int step,
                                            float& M, float& lt, float4& o) {
  auto slot = [&](int r) { return part_slot(a, r, tile, r == first_piece); };
#pragma unroll 1
  for (int r = r0; r <= r1; r += 4 * step) {                  // four loads under way
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = r + k * step <= r1 ? a.part_ml[slot(r + k * step) * 128 + m].x : -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; ++k) M = fmaxf(M, v[k]);
  }
#pragma unroll 1
  for (int r = r0; r <= r1; r += 4 * step) {
    float2 ml[4];
    float4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t at = slot(r + k * step <= r1 ? r + k * step : r);
      ml[k] = a.part_ml[at * 128 + m];
      v[k] = reinterpret_cast<const float4*>(a.part_o)[(at * (a.dvp / 4) + grp) * 128 + m];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      // past the last piece, or a piece that holds no key of this row
      if (r + k * step > r1 || (ml[k].x == -INFINITY && ml[k].y == 0.f)) continue;
      const float w = ex2(ml[k].x - M);
      lt = fmaf(ml[k].y, w, lt);
      o.x = fmaf(v[k].x, w, o.x);
      o.y = fmaf(v[k].y, w, o.y);
      o.z = fmaf(v[k].z, w, o.z);
      o.w = fmaf(v[k].w, w, o.w);
    }
  }
}

// Joins the pieces of units that several ranges share, in a fixed order; also
// writes the rows nothing else does: of sequences without keys, outside all
// sequences, and past max_q.  Item = (row of a tile, four dims), a thread's work
// while a unit has few pieces.  From 32 on (a long cache with few kv heads) the eight
// warps of a CTA share the pieces of an item: with 74 pieces (256 dims, 131072 keys, two
// kv heads) a call takes 77 us instead of 87; with 19 (128 dims, eight heads) it would
// take 120 instead of 116.
constexpr int kJoinWarps = 8, kManyPieces = 32;
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) tree_combine_kernel(const __grid_constant__ Args a, int tile_rows) {
  __shared__ float4 part_o[kJoinWarps][32];
  __shared__ float2 part_ml[kJoinWarps][32];
  const SfaTreeParams& p = a.p;
  const int n = p.num_seqs, units = n * p.h_kv * a.ntiles;
  const int groups = p.d_v / 4;
  if ((int)blockIdx.x >= units)
    return rows_of_no_tile<T>(a, blockIdx.y * blockDim.x + threadIdx.x, gridDim.y * blockDim.x);
  const int tile = blockIdx.x % a.ntiles, h = blockIdx.x / a.ntiles % p.h_kv, s = blockIdx.x / a.ntiles / p.h_kv;
  const int c0 = a.cum[s], nch = a.cum[s + 1] - c0;
  const int line = a.cum[n] * p.h_kv, len = max(a.min_chunks, (line + a.ranges - 1) / a.ranges);
  const int u0 = c0 * p.h_kv + h * nch;
  const int r0 = u0 / len, r1 = nch > 0 ? (u0 + nch - 1) / len : r0;
  if (nch > 0 && r0 == r1) return;
  const Seq q = load_seq(a, s);
  const int node0 = tile / a.n_hg * a.NT;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool many = nch > 0 && r1 - r0 + 1 >= kManyPieces;
  const int blocks = (tile_rows + 31) / 32;                   // of 32 rows
  // many: a CTA an item of 32 rows and a group; else a warp
  const int step = many ? gridDim.y : gridDim.y * kJoinWarps;
#pragma unroll 1
  for (int i = many ? blockIdx.y : blockIdx.y * kJoinWarps + warp; i < blocks * groups; i += step) {
    const int m = i % blocks * 32 + lane, grp = i / blocks;
    const int node = node0 + (a.n_hg > 1 ? 0 : m / a.GB);
    const int hh = a.n_hg > 1 ? (tile % a.n_hg) * 128 + m : m % a.GB;
    const bool live = m < tile_rows && hh < a.G && node < q.rows && node - node0 < a.NT && q.q0 + node < p.total_q;
    const int head = h * a.G + hh;
    const int64_t row = q.q0 + node;
    if (nch == 0) {
      if (live) empty_row<T>(p, row, head, grp);
      continue;
    }
    const float s2 = p.attn_sink && live ? __ldg(p.attn_sink + head) * kLog2e : -INFINITY;
    float M = many ? -INFINITY : s2, lt = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) join_pieces(a, tile, m, grp, r0, many ? r0 + warp : r0, r1, many ? kJoinWarps : 1, M, lt, o);
    if (many) {
      __syncthreads();                                        // the item before has been read
      part_o[warp][lane] = o;
      part_ml[warp][lane] = make_float2(M, lt);
      __syncthreads();
      if (warp != 0) continue;
      M = s2;
#pragma unroll 1
      for (int k = 0; k < kJoinWarps; ++k) M = fmaxf(M, part_ml[k][lane].x);
      lt = 0.f;
      o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int k = 0; k < kJoinWarps; ++k) {
        const float2 ml = part_ml[k][lane];
        if (ml.x == -INFINITY && ml.y == 0.f) continue;
        const float w = ex2(ml.x - M);
        const float4 v = part_o[k][lane];
        lt = fmaf(ml.y, w, lt);
        o.x = fmaf(v.x, w, o.x);
        o.y = fmaf(v.y, w, o.y);
        o.z = fmaf(v.z, w, o.z);
        o.w = fmaf(v.w, w, o.w);
      }
    }
    if (!live) continue;
    if (s2 != -INFINITY) lt += ex2(s2 - M);
    const bool none = lt == 0.f;
    const float inv = none ? 0.f : 1.f / lt;
    if (none) o = make_float4(0.f, 0.f, 0.f, 0.f);
    store4<T>(static_cast<T*>(p.o) + row * p.o_st + (int64_t)head * p.o_sh + grp * 4,
              make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    if (grp == 0) p.lse[row * p.l_st + (int64_t)head * p.l_sh] = none ? -INFINITY : (M + lg2(lt)) * kLn2;
  }
}

struct Plan {
  Args a;
  size_t smem;
  size_t off_ml, off_cum, ws;
  int tile_rows;      // rows of a tile that can be live
  bool pair;          // the pair kernel
};

static int bad(const std::string& m) { return report_error(SFA_ERR_INVALID_ARGUMENT, "tree attention: " + m); }

static int check(const SfaTreeParams* p) {
  if (!p) return bad("params is NULL");
  if (p->num_seqs < 0 || p->total_q < 0 || p->max_q < 0 || p->max_k < 0 || p->num_pages < 0 || p->table_width < 0)
    return bad("sizes must be >= 0");
  if (p->page_size < 1) return bad("page_size must be positive");
  if (p->h_q < 1 || p->h_kv < 1 || p->h_q % p->h_kv) return bad("h_q must be a positive multiple of h_kv");
  if (p->d_qk < 8 || p->d_v < 8 || p->d_qk % 8 || p->d_v % 8 || p->d_qk > 256 || p->d_v > 256)
    return report_error(SFA_ERR_UNSUPPORTED, "tree attention: head dims must be multiples of 8 up to 256");
  if (p->dtype != SFA_DTYPE_BF16 && p->dtype != SFA_DTYPE_F16)
    return report_error(SFA_ERR_UNSUPPORTED, "tree attention: bf16 or fp16 only");
  if (!(p->scale > 0.f) || p->scale > 3.0e38f) return bad("scale must be positive and finite");
  if (p->parents && p->max_q > kMaxNodes) return bad("a tree has at most " + std::to_string(kMaxNodes) + " drafted rows a sequence");
  if ((int64_t)p->num_pages * p->page_size >= INT32_MAX)
    return report_error(SFA_ERR_UNSUPPORTED, "tree attention: a pool has fewer than 2^31 rows");
  // units first: their product with the tiles or chunks of one stays inside 64 bits, and a strip of
  // sequences inside 32
  if ((int64_t)p->num_seqs * p->h_kv >= (1 << 30)) return report_error(SFA_ERR_UNSUPPORTED, "tree attention: too many sequences and heads");
  const int64_t chunks = ((int64_t)p->table_width * p->page_size + 63) / 64;
  if (chunks * p->num_seqs * p->h_kv >= INT32_MAX || (int64_t)p->table_width * p->page_size >= INT32_MAX)
    return report_error(SFA_ERR_UNSUPPORTED, "tree attention: table too large");
  const int g = p->h_q / p->h_kv, per_tile = g > 128 ? 1 : 128 / g;         // rows and head tiles of a tile
  const int64_t tiles = ((int64_t)std::max(1, p->cu_seqlens ? p->max_q : 1) + per_tile - 1) / per_tile * ((g + 127) / 128);
  if (tiles > 65535 || tiles * p->num_seqs * p->h_kv >= INT32_MAX)
    return report_error(SFA_ERR_UNSUPPORTED, "tree attention: too many drafted rows a sequence for one call");
  if (p->total_q == 0) return SFA_OK;
  if (!p->q || !p->o || !p->lse) return bad("q, o and lse must be non-NULL");
  if (p->num_seqs > 0 && ((p->table_width > 0 && !p->block_table) || !p->cache_seqlens))
    return bad("block_table and cache_seqlens must be non-NULL");
  if (p->num_seqs > 0 && p->num_pages > 0 && (!p->k || !p->v)) return bad("k and v must be non-NULL");
  if (!p->cu_seqlens && p->total_q < p->num_seqs) return bad("without cu_seqlens q holds one row per sequence");
  // a stride is read only where its extent is above one
  auto strides_ok = [](const void* ptr, int64_t st, bool many, int64_t sh, bool heads) {
    return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && (!many || (st > 0 && st % 8 == 0)) &&
           (!heads || (sh > 0 && sh % 8 == 0));
  };
  const bool kv_rows = (int64_t)p->num_pages * p->page_size > 1;
  if (!strides_ok(p->q, p->q_st, p->total_q > 1, p->q_sh, p->h_q > 1) ||
      !strides_ok(p->k, p->k_st, kv_rows, p->k_sh, p->h_kv > 1) || !strides_ok(p->v, p->v_st, kv_rows, p->v_sh, p->h_kv > 1) ||
      !strides_ok(p->o, p->o_st, p->total_q > 1, p->o_sh, p->h_q > 1))
    return bad("q, k, v and o need 16-byte aligned bases and positive strides that are multiples of 8");
  return SFA_OK;
}

// Ring stages that fit `budget` bytes of shared memory, K first; false if two of each do not.
static bool fit_rings(Args& a, size_t budget, size_t fixed, size_t kb, size_t vb) {
  a.kst = a.vst = 2;
  if (fixed + 2 * kb + 2 * vb > budget) return false;
  while (a.kst < 4 || a.vst < 4) {
    const size_t now = fixed + a.kst * kb + a.vst * vb;
    if (a.kst <= a.vst && a.kst < 4 && now + kb <= budget) ++a.kst;
    else if (a.vst < 4 && now + vb <= budget) ++a.vst;
    else break;
  }
  return true;
}

// Shapes, kernel, shared memory and the split.  The pair kernel (128-key chunks, two softmax
// warpgroups) takes every shape whose O fits twice beside two 128-key S tiles in TMEM (d_v <= 128) and
// whose rings fit shared memory, the wide one the rest.  Forced on the wide kernel's predecessor (its
// 64-key chunks, one warpgroup), 128 rows a kv head of 128 dims over 131072 keys took 216 us against 123.
static Plan make_plan(const SfaTreeParams& p) {
  Plan pl{};
  Args& a = pl.a;
  a.p = p;
  a.G = p.h_q / p.h_kv;
  a.GB = std::min(a.G, 128);
  a.n_hg = (a.G + 127) / 128;
  a.NT = a.n_hg > 1 ? 1 : 128 / a.GB;
  const int max_q = p.cu_seqlens ? std::max(1, p.max_q) : 1;
  a.ntiles = (max_q + a.NT - 1) / a.NT * a.n_hg;
  pl.tile_rows = std::min(a.NT, max_q) * a.GB;
  a.nkq = (p.d_qk + 63) / 64;
  a.nkv = (p.d_v + 63) / 64;
  a.dvp = (p.d_v + 15) / 16 * 16;
  const size_t q = (size_t)a.nkq * kQSlab, full = 226 * 1024 - 1024;
  size_t sh = (pair_shared_bytes() + 127) / 128 * 128;
  int ctas_y = a.ntiles;
  if (a.dvp <= 128) {
    const size_t kb = (size_t)a.nkq * 128 * 128, vb = (size_t)a.nkv * 128 * 128;
    a.two = a.ntiles > 1 && fit_rings(a, full, 2 * q + sh, kb, vb);
    pl.pair = a.two || fit_rings(a, full, q + sh, kb, vb);
  }
  if (pl.pair) {
    a.keys = 128;
    a.keys_log = 7;
    a.off_k = (uint32_t)(a.two ? 2 * q : q);
    a.off_v = a.off_k + (uint32_t)(a.kst * a.nkq * 128 * 128);
    a.off_sh = a.off_v + (uint32_t)(a.vst * a.nkv * 128 * 128);
    a.tmem_cols = 512;
    a.min_chunks = 1;
    if (a.two) ctas_y = (a.ntiles + 1) / 2;
  } else {
    a.keys = 64;
    a.keys_log = 6;
    sh = (wide_shared_bytes() + 127) / 128 * 128;
    const size_t kb = (size_t)a.nkq * 64 * 128, vb = (size_t)a.nkv * 64 * 128;
    fit_rings(a, full, q + sh, kb, vb);           // 256 dims: 64 KB of Q, 32 KB a stage
    a.off_k = (uint32_t)q;
    a.off_v = a.off_k + (uint32_t)(a.kst * kb);
    a.off_sh = a.off_v + (uint32_t)(a.vst * vb);
    a.tmem_cols = 512;
    a.min_chunks = 2;
  }
  a.box = 1;
  while (a.box < a.keys && p.page_size % (a.box * 2) == 0) {
    a.box *= 2;
    ++a.box_log;
  }
  // all TMEM columns: one CTA per SM
  pl.smem = std::max(a.off_sh + sh + 1024, (size_t)116 * 1024);
  const int64_t covered = std::min<int64_t>((int64_t)p.table_width * p.page_size, std::max(1, p.max_k));
  const int64_t line = std::max<int64_t>(1, (int64_t)p.num_seqs * p.h_kv * ((covered + a.keys - 1) / a.keys));
  const int64_t slots = (int64_t)device_sm_count() / ctas_y;
  a.ranges = (int)std::max<int64_t>(1, std::min(slots, (line + a.min_chunks - 1) / a.min_chunks));
  const size_t pieces = a.ranges > 1 ? (size_t)a.ranges * a.ntiles * 2 : 0;
  size_t off = pieces * 128 * a.dvp * sizeof(float);
  pl.off_ml = off;
  off += pieces * 128 * sizeof(float2);
  pl.off_cum = off;
  off += ((size_t)p.num_seqs + 1) * sizeof(int32_t);
  pl.ws = (off + 255) & ~size_t(255);
  return pl;
}

template <typename T>
static cudaError_t launch(Plan& pl, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t st) {
  Args& a = pl.a;
  cudaError_t e = cudaSuccess;
  const bool keys = a.p.num_seqs > 0 && a.p.num_pages > 0 && a.p.table_width > 0;
  if (keys) {
    e = pl.pair ? launch_pair(a, pl.smem, tq, tk, tv, st) : launch_wide(a, pl.smem, tq, tk, tv, st);
    if (e != cudaSuccess) return e;
  } else {
    // no keys at all: every sequence has zero chunks
    if ((e = cudaMemsetAsync(a.cum, 0, ((size_t)a.p.num_seqs + 1) * sizeof(int32_t), st)) != cudaSuccess) return e;
    note_memset("tree_cum", st);
  }
  // a warp an item of 32 rows; as many CTAs as two per SM where units are few (eight each: 195 us for the
  // 74 pieces above)
  const int items = (pl.tile_rows + 31) / 32 * (a.p.d_v / 4);
  const int units = a.p.num_seqs * a.p.h_kv * a.ntiles, most = std::max(8, 2 * device_sm_count() / std::max(1, units));
  const int per = a.ranges >= kManyPieces ? 1 : kJoinWarps;   // items of a CTA at a time, where a unit can have many pieces
  const dim3 grid((unsigned)(units + 1), (unsigned)std::min(most, (items + per - 1) / per));
  tree_combine_kernel<T><<<grid, kJoinWarps * 32, 0, st>>>(a, pl.tile_rows);
  note_launch("tree_combine", st);
  return cudaGetLastError();
}

}  // namespace tree
}  // namespace sfa

using namespace sfa;

extern "C" {

size_t sfa_tree_workspace_bytes(const SfaTreeParams* p) {
  if (tree::check(p) || p->total_q == 0) return 0;
  return tree::make_plan(*p).ws;
}

int sfa_tree_attention(const SfaTreeParams* p, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = tree::check(p);
  if (rc) return rc;
  if (p->total_q == 0) return SFA_OK;
  tree::Plan pl = tree::make_plan(*p);
  if (!workspace || workspace_bytes < pl.ws || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return report_error(SFA_ERR_WORKSPACE, "tree attention: workspace missing, unaligned or too small: need " +
                                               std::to_string(pl.ws) + " bytes, 256-byte aligned");
  if (device_cc() != 100) return report_error(SFA_ERR_UNSUPPORTED, "tree attention needs an sm_100 device");
  tree::Args& a = pl.a;
  char* ws = static_cast<char*>(workspace);
  a.part_o = reinterpret_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + pl.off_ml);
  a.cum = reinterpret_cast<int32_t*>(ws + pl.off_cum);
  a.status = device_status_ptr();
  CUtensorMap tq{}, tk{}, tv{};
  cudaError_t e = cudaSuccess;
  if (p->num_seqs > 0 && p->num_pages > 0 && p->table_width > 0) {
    const uint64_t rows = (uint64_t)p->num_pages * p->page_size;
    e = make_tmap_bf16_4d(&tq, p->q, {(uint64_t)p->d_qk, (uint64_t)p->h_q, (uint64_t)p->total_q, 1}, {p->q_sh, p->q_st, 0},
                          {64u, (uint32_t)a.GB, (uint32_t)a.NT, 1u});
    if (e == cudaSuccess)
      e = make_tmap_bf16_4d(&tk, p->k, {(uint64_t)p->d_qk, rows, (uint64_t)p->h_kv, 1}, {p->k_st, p->k_sh, 0},
                            {64u, (uint32_t)a.box, 1u, 1u});
    if (e == cudaSuccess)
      e = make_tmap_bf16_4d(&tv, p->v, {(uint64_t)p->d_v, rows, (uint64_t)p->h_kv, 1}, {p->v_st, p->v_sh, 0},
                            {64u, (uint32_t)a.box, 1u, 1u});
    if (e != cudaSuccess) return report_error(SFA_ERR_CUDA, "tree attention: tensor maps");
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  e = p->dtype == SFA_DTYPE_F16 ? tree::launch<__half>(pl, tq, tk, tv, st) : tree::launch<__nv_bfloat16>(pl, tq, tk, tv, st);
  if (e != cudaSuccess) return report_error(SFA_ERR_CUDA, std::string("tree attention: ") + cudaGetErrorString(e));
  return SFA_OK;
}

}  // extern "C"

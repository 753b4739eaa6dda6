// sfa_tree.cuh — what the kernels of sfa_tree.cu, sfa_tree_pair.cu and sfa_tree_wide.cu share:
// the arguments, how the chunk line of all sequences is cut into ranges, and the
// walk of a CTA over the units its range touches.
#pragma once

#include <type_traits>

#include "sfa_common.cuh"
#include "sfa_internal.h"
#include "sfa_tc_common.cuh"
#include "sfa_tc_host.h"
#include "sfa_tok_common.cuh"

namespace sfa {
namespace tree {

using namespace tc;
using namespace tok;

constexpr int kQSlab = 128 * 128;               // bytes of a 128-row x 64-dim Q slab
constexpr int kMaxNodes = SFA_TREE_MAX_NODES;
constexpr int kAncWords = kMaxNodes / 32 + 3;   // + 2 zero words behind, odd row stride

struct Args {
  SfaTreeParams p;
  int G;             // query heads per kv head
  int GB, NT;        // heads and drafted rows of a tile
  int n_hg;          // head tiles (G above 128)
  int ntiles;        // row tiles
  int keys, keys_log; // keys per chunk, a power of two
  int two;           // pair kernel: a CTA takes two row tiles
  int ranges;        // gridDim.x
  int min_chunks;    // chunks of a range at least
  int nkq, nkv;      // 64-dim slabs of a key / value row
  int dvp;           // d_v rounded up to 16
  int box, box_log;  // rows of a K / V box, a power of two
  int kst, vst;      // ring stages
  uint32_t tmem_cols;
  uint32_t off_k, off_v, off_sh;
  float* part_o;     // [range][tile][2][dvp / 4][128][4]
  float2* part_ml;   // [range][tile][2][128]  (m, l)
  int32_t* cum;      // [num_seqs + 1] chunks before each sequence
  int32_t* status;
};

// A sequence: its drafted rows [q0, q0 + rows), cache rows before the drafted ones (negative when
// the cache is shorter), positions the table covers, chunks of those.
struct Seq {
  int q0, rows, prefix, kvc, nch;
};

static __device__ __noinline__ Seq load_seq(const Args& a, int s) {
  const SfaTreeParams& p = a.p;
  Seq r;
  const int len = __ldg(p.cache_seqlens + s);
  if (p.cu_seqlens) {
    r.q0 = __ldg(p.cu_seqlens + s);
    r.rows = r.q0 < 0 ? 0 : max(0, __ldg(p.cu_seqlens + s + 1) - r.q0);
  } else {
    r.q0 = s;
    r.rows = 1;
  }
  r.prefix = len - r.rows;
  const int64_t covered = (int64_t)p.table_width * p.page_size;
  r.kvc = (int)max((int64_t)0, min((int64_t)len, covered));
  r.nch = (r.kvc + a.keys - 1) >> a.keys_log;
  return r;
}

// This CTA's range of the chunk line.
struct Range {
  int s, h, c, left;
};

// Fills S.range (S.scan: an int per warp) by a block scan of the sequences' chunks, every thread a
// strip of sequences; CTA (0, 0) also writes a.cum.  The caller's barrier publishes it.
template <typename Shared>
static __device__ __noinline__ void find_range(const Args& a, Shared& S) {
  const SfaTreeParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, threads = blockDim.x, warps = threads >> 5;
  const int n = p.num_seqs, strip = (n + threads - 1) / threads;
  const int s0 = min(n, (int)threadIdx.x * strip), s1 = min(n, s0 + strip);
  int mine = 0;
#pragma unroll 1
  for (int s = s0; s < s1; ++s) mine += load_seq(a, s).nch;
  int run = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  if (lane == 31) S.scan[warp] = run;
  if (threadIdx.x == 0) S.range.left = 0;
  __syncthreads();
  int before = run - mine, all = 0;
  for (int i = 0; i < warps; ++i) {
    if (i < warp) before += S.scan[i];
    all += S.scan[i];
  }
  const int line = all * p.h_kv;
  const int len = max(a.min_chunks, (line + a.ranges - 1) / a.ranges);
  const int64_t x0 = (int64_t)blockIdx.x * len;
  const bool writer = blockIdx.x == 0 && blockIdx.y == 0;
#pragma unroll 1
  for (int s = s0; s < s1; ++s) {
    const int nch = load_seq(a, s).nch;
    if (writer) a.cum[s] = before;
    const int64_t u0 = (int64_t)before * p.h_kv;
    if (x0 >= u0 && x0 < u0 + (int64_t)nch * p.h_kv) {
      const int off = (int)(x0 - u0);
      S.range = Range{s, off / nch, off % nch, (int)min((int64_t)len, (int64_t)line - x0)};
    }
    before += nch;
  }
  if (writer && threadIdx.x == 0) a.cum[n] = all;
}

// A piece of this CTA's range: chunks [c0, c1) of unit (s, h); whole: the unit lies in this range.
struct Piece {
  int s, h, c0, c1;
  bool whole;
  Seq q;
};

struct Walk {
  const Args* a;
  int s, h, c, left;
  Seq q;
  __device__ __forceinline__ Walk(const Args& aa, const Range& r) : a(&aa), s(r.s), h(r.h), c(r.c), left(r.left) {
    if (left > 0) q = load_seq(aa, s);
  }
  __device__ __noinline__ bool next(Piece& g) {
    if (left <= 0) return false;
    const int n = min(q.nch - c, left);
    g.s = s; g.h = h; g.c0 = c; g.c1 = c + n;
    g.whole = n == q.nch;
    g.q = q;
    left -= n;
    c = 0;
    if (left > 0 && ++h == a->p.h_kv) {
      h = 0;
      do { q = load_seq(*a, ++s); } while (q.nch == 0 && s + 1 < a->p.num_seqs);   // left > 0: a later one has chunks
      if (q.nch == 0) left = 0;
    }
    return true;
  }
};

__device__ __forceinline__ int node_of_tile(const Args& a, int tile) {
  return (a.n_hg == 1 ? tile : tile / a.n_hg) * a.NT;
}

// End of the piece's chunks that hold a key one of the tile's rows can see (c0 if the tile has no rows).
__device__ __forceinline__ int tile_end(const Args& a, int tile, const Piece& g) {
  const int node0 = node_of_tile(a, tile);
  if (node0 >= g.q.rows) return g.c0;
  const int last = g.q.prefix + min(g.q.rows, node0 + a.NT);          // keys below it
  const int kend = max(0, min(g.q.kvc, last));
  return max(g.c0, min(g.c1, (kend + a.keys - 1) >> a.keys_log));
}

// A wait of at most ~2 s; on expiry the status word gets the kernel and the site.
// Its slow part is a function: the waits of a role loop would otherwise be most of its code.
static __device__ __noinline__ bool wait_on(uint64_t* bar, uint32_t parity, int32_t* status, int code) {
  if (mbar_wait(bar, parity)) return true;
  record_status(status, code);
  return false;
}
__device__ __forceinline__ bool bounded_wait(uint64_t* bar, uint32_t parity, int32_t* status, int kernel, int site) {
  return mbar_try_wait(bar, parity) || wait_on(bar, parity, status, (kernel << 16) | site);
}

// Pool row of the box at cache position pos, -1 if it holds no key.
static __device__ __noinline__ int box_row(const SfaTreeParams& p, const Piece& g, int pos) {
  if (pos >= g.q.kvc) return -1;
  const int pg = __ldg(p.block_table + (int64_t)g.s * p.bt_stride + pos / p.page_size);
  if (pg < 0 || pg >= p.num_pages) return -1;
  return pg * p.page_size + pos % p.page_size;
}

// Ancestors (and itself) of drafted row `node` as bits, from the sequence's parents in shared memory.
static __device__ __noinline__ void mark_ancestors(uint32_t* anc, const short* parent, int node, int rows) {
#pragma unroll 1
  for (int i = 0; i < kAncWords; ++i) anc[i] = 0;
  if (node >= rows) return;
  while (true) {                                      // ends: the number falls with every step
    anc[node >> 5] |= 1u << (node & 31);
    const int up = parent[node];
    if (up < 0 || up >= node) return;
    node = up;
  }
}

// Which of 32 keys drafted row `node` sees; d0: the first of them as a drafted row (negative: before them).
__device__ __forceinline__ uint32_t sees32(const uint32_t* anc, bool tree, int node, int d0) {
  if (!tree) {
    const int j = node - d0;
    return j < 0 ? 0u : j >= 31 ? ~0u : (2u << j) - 1;
  }
  if (d0 >= 0) {
    const int w = d0 >> 5;
    const uint32_t w0 = w < kAncWords ? anc[w] : 0, w1 = w + 1 < kAncWords ? anc[w + 1] : 0;
    return __funnelshift_r(w0, w1, d0 & 31);
  }
  return d0 <= -32 ? ~0u : (anc[0] << -d0) | ((1u << -d0) - 1);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16x2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// A mask of the two 16-bit values of w that are infinite or NaN.
template <typename T>
__device__ __forceinline__ uint32_t nonfinite2(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return ((w & e) == e ? 0xffffu : 0u) | ((w & (e << 16)) == (e << 16) ? 0xffff0000u : 0u);
}
// Whether one of them is: an exponent of all ones carries into the sign's place.
template <typename T>
__device__ __forceinline__ bool any_nonfinite2(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  constexpr uint32_t one = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
  return (((w & e) + one) & 0x80008000u) != 0;
}
__device__ __forceinline__ float as_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_f(__half x) { return __half2float(x); }

// Bits to flip in an instruction descriptor for bf16 operands when they are fp16 (format 0).
template <typename T>
constexpr uint32_t type_bits() {
  return std::is_same<T, __half>::value ? (1u << 7) | (1u << 10) : 0u;
}

// The tile's part slot of a range: 0 for a unit that began in an earlier range, 1 for one that goes on behind it.
__device__ __forceinline__ int64_t part_slot(const Args& a, int range, int tile, bool begins) {
  return ((int64_t)range * a.ntiles + tile) * 2 + (begins ? 1 : 0);
}

// sfa_tree_pair.cu and sfa_tree_wide.cu
size_t pair_shared_bytes();
size_t wide_shared_bytes();
cudaError_t launch_wide(const Args& a, size_t smem, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                        cudaStream_t st);
cudaError_t launch_pair(const Args& a, size_t smem, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                        cudaStream_t st);

}  // namespace tree
}  // namespace sfa

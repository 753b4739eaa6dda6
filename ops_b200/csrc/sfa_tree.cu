// sfa_tree.cu — attention of drafted tokens (a tree, a chain, or one token) over
// a paged kv cache, tensor cores (sm_100a).
//
//   o[r] = sum_t p[r,t] v[t] / sum_t p[r,t],  p = exp(scale q[r].k[t]) over the
//   cache rows r sees: all before the drafted ones, its ancestors and itself.
//
// Tile: the G query heads of a kv head times as many drafted rows as fit make the
// M = 128 rows of one MMA,
//     S[rows, 64 keys] = Q . K^T,   O[rows, d_v] += P . V,
// so a key row read from the cache serves every head and every drafted row; a
// decode step is bound by those reads, a large tree by the MMAs and the softmax.
//
// Split: the (sequence, kv head, 64-key chunk) space of all sequences is one line
// that gridDim.x CTAs cut into equal ranges, whatever the lengths; a CTA walks the
// units (sequence, kv head) its range touches.  A unit that lies in one range is
// finished there; pieces of the others go to a workspace as (m, l, O) and
// tree_combine_kernel joins them in range order.  The gridDim.y row tiles of a
// unit walk the same range at the same time and share its reads in L2.
//
// Keys come through the block table with TMA boxes of as many rows as divide both
// a page and a chunk, 128B-swizzled 64-dim slabs; a box without a page (a table
// entry outside the pool, or positions behind the cache) is read out of the
// tensor map's bounds, which fills zeros without touching memory.
//
// Softmax: one thread per row.  P = exp2(S c - m) in fp32, rounded once to the
// MMA operand's type (the row sum keeps the unrounded values); m is raised only
// when a chunk's maximum exceeds it by more than 8 in log2, so O is rescaled in
// TMEM rarely.  P overwrites S's columns as the PV MMA's A operand.
//
// Two CTAs per SM for d_qk, d_v <= 128 (256 TMEM columns, half the shared memory
// each): one's softmax latency is covered by the other's reads.
//
// Warps: 0 K (and Q, key masks), 1 V, 2 MMA issue (one thread), 4-7 softmax.
// Every wait is bounded (~2 s); on expiry the kernel records (7 << 16) | site in
// the status word and returns.
#include "sfa_tree.cuh"

#include <algorithm>
#include <string>

namespace sfa {
namespace tree {

constexpr int kThreads = 256;
constexpr int kKeys = 64;                       // keys per chunk
constexpr int kSlab = kKeys * 128;              // bytes of a 64-key x 64-dim slab
constexpr int kMasks = 8;                       // key-mask ring: more chunks than stages in flight

struct Shared {
  uint64_t q_full, q_empty;
  uint64_t k_full[8], k_empty[8], v_full[8], v_empty[8];
  uint64_t s_full[2], p_full[2];
  uint64_t pv_done;
  uint64_t sync;                       // softmax warps among themselves
  uint32_t tmem_base;
  uint32_t zeroed;                     // O of a piece was initialised by the softmax warps
  uint32_t bad[2];                     // keys of the chunk whose value row has a non-finite element
  uint2 mask[kMasks];                  // keys of the chunk that exist
  int scan[kThreads / 32];
  Range range;
  short parent[kMaxNodes];
  uint32_t anc[128][kAncWords];        // ancestors of each row of the tile
};

constexpr int kId = 7;                          // of this kernel in the status word
__device__ __forceinline__ bool wt(uint64_t* bar, uint32_t parity, int32_t* status, int site) {
  return bounded_wait(bar, parity, status, kId, site);
}
__device__ __forceinline__ bool wtw(uint64_t* bar, uint32_t parity, int32_t* status, int site) {
  return __all_sync(0xffffffffu, wt(bar, parity, status, site));
}

// Cuts the piece to the chunks of the tile's rows.
__device__ __forceinline__ void clip_to_tile(const Args& a, int tile, Piece& g, int& node0) {
  node0 = node_of_tile(a, tile);
  g.c1 = tile_end(a, tile, g);
}

// The chunks of the tile's pieces one after another.
struct Chunks {
  Walk w;
  Piece g;
  const Args* a;
  int c, node0;
  bool first;
  __device__ __forceinline__ Chunks(const Args& aa, const Shared& S) : w(aa, S.range), a(&aa), c(0), node0(0), first(false) {
    g.c0 = g.c1 = 0;
  }
  __device__ __forceinline__ bool next(int tile) {
    if (c + 1 < g.c1) {
      ++c;
      first = false;
      return true;
    }
    do {
      if (!w.next(g)) return false;
      clip_to_tile(*a, tile, g, node0);
    } while (g.c0 >= g.c1);
    c = g.c0;
    first = true;
    return true;
  }
  __device__ __forceinline__ bool last() const { return c + 1 == g.c1; }
};

// Producer of one ring (K or V): boxes of every chunk, in order.  The table
// entries of a chunk are read while the one before waits for its stage.
template <bool IS_K>
__device__ __forceinline__ void produce(const Args& a, Shared& S, uint8_t* ring, uint8_t* sq, const CUtensorMap* map,
                                        const CUtensorMap* tmq) {
  const int lane = threadIdx.x & 31, tile = blockIdx.y;
  const int slabs = IS_K ? a.nkq : a.nkv, stages = IS_K ? a.kst : a.vst;
  const int nb = kKeys / a.box, total = nb * slabs;
  const int outside = a.p.num_pages * a.p.page_size;       // a row past the pool: zeros
  const int b0 = (lane % nb) * a.box, b1 = ((lane + 32) % nb) * a.box;   // keys of this lane's boxes
  uint64_t* full = IS_K ? S.k_full : S.v_full;
  uint64_t* empty = IS_K ? S.k_empty : S.v_empty;
  Chunks it(a, S);
  bool ok = true, have = it.next(tile);
  int r0 = -1, r1 = -1;
  if (have) {
    r0 = box_row(a.p, it.g, it.c * kKeys + b0);
    r1 = nb > 32 ? box_row(a.p, it.g, it.c * kKeys + b1) : r0;
  }
  for (int ci = 0, qi = 0; have && ok; ++ci) {
    const int st = ci % stages;
    const int c = it.c, kvc = it.g.q.kvc, h = it.g.h, q0 = it.g.q.q0 + it.node0;
    const bool first = it.first;
    const int e0 = r0, e1 = r1;
    have = it.next(tile);
    if (have) {
      r0 = box_row(a.p, it.g, it.c * kKeys + b0);
      r1 = nb > 32 ? box_row(a.p, it.g, it.c * kKeys + b1) : r0;
    }
    if (IS_K && first) {
      if (lane == 0) {
        ok = wt(&S.q_empty, (qi & 1) ^ 1, a.status, 1);
        if (ok) {
          mbar_arrive_expect_tx(&S.q_full, (uint32_t)(a.nkq * a.GB * a.NT * 128));
          for (int s = 0; s < a.nkq; ++s)
            tma_load_4d(sq + s * kQSlab, tmq, &S.q_full, s * 64, h * a.G + (tile % a.n_hg) * 128, q0, 0);
        }
      }
      ++qi;
    }
    if (lane == 0 && ok) ok = wt(&empty[st], ((ci / stages) & 1) ^ 1, a.status, IS_K ? 2 : 3);
    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
    if (!ok) break;
    if (IS_K) {
      const uint32_t v0 = __ballot_sync(0xffffffffu, e0 >= 0), v1 = __ballot_sync(0xffffffffu, e1 >= 0);
      if (lane == 0) {
        uint64_t m = ~0ull;
        if ((v0 & v1) != 0xffffffffu || (c + 1) * kKeys > kvc) {
          const uint64_t one = a.box == 64 ? ~0ull : (1ull << a.box) - 1;
          m = 0;
          for (int b = 0; b < nb; ++b)
            if (((b < 32 ? v0 : v1) >> (b & 31)) & 1u) m |= one << (b * a.box);
          const int n = kvc - c * kKeys;                    // >= 1
          if (n < kKeys) m &= (1ull << n) - 1;
        }
        S.mask[ci % kMasks] = make_uint2((uint32_t)m, (uint32_t)(m >> 32));
      }
    }
    if (lane == 0) mbar_arrive_expect_tx(&full[st], (uint32_t)(slabs * kSlab));
    __syncwarp();
    uint8_t* dst = ring + (size_t)st * slabs * kSlab;
    for (int i = lane, j = 0; i < total; i += 32, ++j) {
      const int b = i % nb, s = i / nb;
      const int row = (nb > 32 && (j & 1)) ? e1 : e0;
      tma_load_4d(dst + s * kSlab + b * a.box * 128, map, &full[st], s * 64, row >= 0 ? row : outside, h, 0);
    }
  }
}

// The softmax warps' own barrier (bounded, unlike a named barrier).
__device__ __forceinline__ bool meet(Shared& S, int& n, int32_t* status) {
  warp_arrive(&S.sync);
  return wtw(&S.sync, (n++) & 1, status, 10);
}

template <typename T>
__device__ __forceinline__ void softmax_warps(const Args& a, Shared& S, uint8_t* sv, uint32_t tmem) {
  const SfaTreeParams& p = a.p;
  const int lane = threadIdx.x & 31, wq = (threadIdx.x >> 5) & 3, m = wq * 32 + lane, tile = blockIdx.y;
  const uint32_t tl = tmem + ((uint32_t)(wq * 32) << 16);
  const float c2 = p.scale * kLog2e;
  const int my_node = a.n_hg > 1 ? 0 : m / a.GB;              // drafted row of this thread in the tile
  const int my_head = a.n_hg > 1 ? (tile % a.n_hg) * 128 + m : m % a.GB;
  const bool in_tile = my_node < a.NT && my_head < a.G;
  Walk w(a, S.range);
  Piece g;
  int ci = 0, meets = 0, added = 0;
  bool ok = true;
  // Waits until PV of the first n chunks has completed.  Called with n growing by at most one: a
  // parity wait would take a phase two behind for the one it asks for.
  auto pv_through = [&](int n, int site) {
    if (added < n) {
      if (!wtw(&S.pv_done, added & 1, a.status, site)) return false;
      ++added;
    }
    return true;
  };
  while (ok && w.next(g)) {
    const bool split = !g.whole, begins = g.c0 == 0;
    int node0;
    clip_to_tile(a, tile, g, node0);
    const int node = node0 + my_node;
    const bool live = in_tile && node < g.q.rows && g.q.q0 + node < p.total_q;
    const bool any = __any_sync(0xffffffffu, live);
    const int prefix = g.q.prefix;
    // ancestors of the tile's rows, when the piece reaches the drafted keys
    const bool tree = p.parents != nullptr && g.c1 * kKeys > prefix && g.c0 < g.c1;
    if (tree) {
      const int rows = min(g.q.rows, min(kMaxNodes, p.total_q - g.q.q0));
      if (!(ok = meet(S, meets, a.status))) break;            // the piece before is done with both
      for (int i = m; i < rows; i += 128) S.parent[i] = (short)max(-1, min(__ldg(p.parents + g.q.q0 + i), i));
      if (!(ok = meet(S, meets, a.status))) break;
      if (m < a.NT) mark_ancestors(S.anc[m], S.parent, node0 + m, rows);
      if (!(ok = meet(S, meets, a.status))) break;
    }
    float mref = -INFINITY, l = 0.f;
    for (int c = g.c0; c < g.c1; ++c, ++ci) {
      const int sb = ci & 1;
      if (!(ok = wtw(&S.s_full[sb], (ci >> 1) & 1, a.status, 11))) break;
      tc_fence_after();
      const uint2 km = S.mask[ci % kMasks];
      const int k0 = c * kKeys, d0 = k0 - prefix;             // the chunk's first key, as a drafted row
      const bool drafted = k0 + kKeys > prefix;
      const bool whole = (km.x & km.y) == 0xffffffffu && !drafted;
      uint32_t lo = km.x, hi = km.y;
      if (drafted) {
        const bool by_tree = p.parents != nullptr;
        lo &= sees32(S.anc[my_node], by_tree, node, d0);
        hi &= sees32(S.anc[my_node], by_tree, node, d0 + 32);
      }
      if (!live) lo = hi = 0;
      const uint32_t ts = tl + a.col_s + sb * kKeys;
      float fac = 1.f, lc = 0.f;
      if (any) {
        float sc[64];
        {
          float (&s0)[32] = *reinterpret_cast<float(*)[32]>(sc);
          float (&s1)[32] = *reinterpret_cast<float(*)[32]>(sc + 32);
          tmem_ld32(ts, s0);
          tmem_ld32(ts + 32, s1);
          tmem_ld_wait();
        }
        float mc = -INFINITY;
        if (whole) {
#pragma unroll
          for (int i = 0; i < 64; ++i) mc = fmaxf(mc, sc[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            if (!(((i < 32 ? lo : hi) >> (i & 31)) & 1u)) sc[i] = -INFINITY;
            mc = fmaxf(mc, sc[i]);
          }
        }
        const float zc = mc * c2;
        if (live && (zc > mref + kRescaleLog2 || mref == -INFINITY)) {
          if (mref != -INFINITY) fac = ex2(mref - zc);
          mref = zc;
        }
        // nothing seen yet: any finite reference gives p = 0
        const float nm = mref == -INFINITY ? 0.f : -mref;
        float pk[32];
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          const float p0 = ex2(fmaf(sc[i], c2, nm)), p1 = ex2(fmaf(sc[i + 1], c2, nm));
          lc += p0 + p1;
          pk[i / 2] = __uint_as_float(pack2<T>(p0, p1));
        }
        tmem_st32(ts, pk);
        tmem_st_wait();
      }
      // the chunk before has been added (while this one's P was computed)
      if (!(ok = pv_through(ci, 12))) break;
      if (any) {
        if (c > g.c0 && __any_sync(0xffffffffu, fac != 1.f)) {
          // O to the raised maximum
          tc_fence_after();
          for (int x = 0; x < a.dvp; x += 16) {
            float o[16];
            tmem_ld16(tl + x, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= fac;
            tmem_st16(tl + x, o);
          }
          tmem_st_wait();
          l *= fac;
        }
        l += lc;
      }
      if (c == g.c0 && threadIdx.x == 128) S.zeroed = 0;
      const bool seen_by_some = drafted && g.q.rows > 1;      // drafted keys that some rows do not see
      if ((km.x & km.y) != 0xffffffffu || seen_by_some) {
        // value rows that must not enter the product: those that do not exist (stale rows of a
        // page would turn 0 * NaN into NaN) are cleared, and of drafted rows non-finite elements
        // are taken out here and added below to the rows that see them
        const int vs = ci % a.vst;
        if (seen_by_some) {
          if (threadIdx.x == 128) S.bad[0] = S.bad[1] = 0;
          if (!(ok = meet(S, meets, a.status))) break;
        }
        if (!(ok = wtw(&S.v_full[vs], (ci / a.vst) & 1, a.status, 13))) break;
        const int key = m & 63;
        const bool there = ((key < 32 ? km.x : km.y) >> (key & 31)) & 1u;
        const bool scan = seen_by_some && there && k0 + key >= prefix;
        if (!there || scan) {
          uint8_t* row = sv + (size_t)vs * a.nkv * kSlab + key * 128;
          uint32_t any_bad = 0;
          for (int s = m >> 6; s < a.nkv; s += 2) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              uint4* at = reinterpret_cast<uint4*>(row + s * kSlab + i * 16);
              if (!there) {
                *at = make_uint4(0, 0, 0, 0);
              } else {
                uint4 v = *at;
                const uint32_t b0 = nonfinite2<T>(v.x), b1 = nonfinite2<T>(v.y), b2 = nonfinite2<T>(v.z),
                               b3 = nonfinite2<T>(v.w);
                if (b0 | b1 | b2 | b3) {
                  any_bad = 1;
                  *at = make_uint4(v.x & ~b0, v.y & ~b1, v.z & ~b2, v.w & ~b3);
                }
              }
            }
          }
          if (any_bad) atomicOr(&S.bad[key >> 5], 1u << (key & 31));
        }
        fence_proxy_async_smem();
        if (seen_by_some) {
          if (!(ok = meet(S, meets, a.status))) break;
          const uint32_t blo = S.bad[0], bhi = S.bad[1];
          if (blo | bhi) {
            tc_fence_after();
            if (c == g.c0) {
              const float z[16] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
              for (int x = 0; x < a.dvp; x += 16) tmem_st16(tl + x, z);
              tmem_st_wait();
              if (threadIdx.x == 128) S.zeroed = 1;
            }
            tc_fence_after();
            for (int b = 0; b < 64; ++b) {
              if (!(((b < 32 ? blo : bhi) >> (b & 31)) & 1u)) continue;
              const bool sees = ((b < 32 ? lo : hi) >> (b & 31)) & 1u;
              const int vrow = box_row(p, g, k0 + b);
              const T* v = static_cast<const T*>(p.v) + (int64_t)max(vrow, 0) * p.v_st + (int64_t)g.h * p.v_sh;
              for (int x = 0; x < a.dvp; x += 16) {
                float o[16];
                tmem_ld16(tl + x, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const float e = sees && x + i < p.d_v ? as_f(v[x + i]) : 0.f;
                  if (!isfinite(e)) o[i] += e;
                }
                tmem_st16(tl + x, o);
              }
              tmem_st_wait();
            }
          }
        }
      }
      tc_fence_before();
      warp_arrive(&S.p_full[sb]);
    }
    if (!ok) break;
    // the piece's rows: finished, or (m, l, O) for tree_combine_kernel
    const bool ran = g.c0 < g.c1;
    if (!(ok = pv_through(ci, 14))) break;
    tc_fence_after();
    if (!any) continue;
    const int head = g.h * a.G + my_head;
    if (split) {
      const int64_t slot = part_slot(a, blockIdx.x, tile, begins);
      if (live) a.part_ml[slot * 128 + m] = make_float2(mref, l);
      if (ran) {
        float4* dst = reinterpret_cast<float4*>(a.part_o) + slot * (a.dvp / 4) * 128 + m;
        for (int x = 0; x < a.dvp; x += 16) {
          float o[16];
          tmem_ld16(tl + x, o);
          tmem_ld_wait();
          if (live) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              dst[(x / 4 + i) * 128] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        }
      }
    } else {
      const float sink = p.attn_sink && live ? __ldg(p.attn_sink + head) : -INFINITY;
      const float s2 = sink * kLog2e;
      const float M = fmaxf(mref, s2);
      const float wt_ = mref == -INFINITY ? 0.f : ex2(mref - M);
      const float lt = l * wt_ + (s2 == -INFINITY ? 0.f : ex2(s2 - M));
      const bool none = mref == -INFINITY && l == 0.f;
      const float inv = none ? 0.f : wt_ / lt;
      const int64_t row = g.q.q0 + node;
      T* orow = static_cast<T*>(p.o) + row * p.o_st + (int64_t)head * p.o_sh;
      for (int x = 0; x < a.dvp; x += 16) {
        float o[16];
        if (ran) {
          tmem_ld16(tl + x, o);
          tmem_ld_wait();
        }
        if (live) {
#pragma unroll
          for (int i = 0; i < 16; i += 8) {
            if (x + i >= p.d_v) break;
            uint4 r = make_uint4(0, 0, 0, 0);
            if (!none)
              r = make_uint4(pack2<T>(o[i] * inv, o[i + 1] * inv), pack2<T>(o[i + 2] * inv, o[i + 3] * inv),
                             pack2<T>(o[i + 4] * inv, o[i + 5] * inv), pack2<T>(o[i + 6] * inv, o[i + 7] * inv));
            *reinterpret_cast<uint4*>(orow + x + i) = r;
          }
        }
      }
      if (live) p.lse[row * p.l_st + (int64_t)head * p.l_sh] = none ? sink : (M + lg2(lt)) * kLn2;
    }
    tc_fence_before();
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
tree_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
            const __grid_constant__ CUtensorMap tmv) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = base;
  uint8_t* sk = base + a.off_k;
  uint8_t* sv = base + a.off_v;
  Shared& S = *reinterpret_cast<Shared*>(base + a.off_sh);
  const SfaTreeParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&S.q_full, 1);
    mbar_init(&S.q_empty, 1);
    for (int i = 0; i < 8; ++i) {
      mbar_init(&S.k_full[i], 1);
      mbar_init(&S.k_empty[i], 1);
      mbar_init(&S.v_full[i], 1);
      mbar_init(&S.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S.s_full[i], 1);
      mbar_init(&S.p_full[i], 4);
    }
    mbar_init(&S.pv_done, 1);
    mbar_init(&S.sync, 4);
    fence_barrier_init();
    prefetch_tmap(&tmq);
    prefetch_tmap(&tmk);
    prefetch_tmap(&tmv);
  }
  if (warp == 2) {
    tmem_alloc(&S.tmem_base, a.tmem_cols);
    tmem_relinquish();
  }
  find_range(a, S);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = S.tmem_base;
  const int tile = blockIdx.y;

  if (warp == 0) {
    produce<true>(a, S, sk, sq, &tmk, &tmq);
  } else if (warp == 1) {
    produce<false>(a, S, sv, sq, &tmv, &tmq);
  } else if (warp == 2) {
    if (lane == 0) {
      // S of a chunk is issued before PV of the one before; both run in issue order, so S may
      // overwrite the buffer whose P the PV before that reads
      const uint32_t id_s = idesc_bf16(128, kKeys, false, false) ^ type_bits<T>();
      const uint32_t id_o = idesc_bf16(128, a.dvp, false, true) ^ type_bits<T>();
      Chunks it(a, S);
      bool ok = true;
      int qi = 0;
      auto issue_s = [&](int ci) {
        if (it.first) {
          if (!(ok = wt(&S.q_full, qi & 1, a.status, 4))) return;
          ++qi;
        }
        const int ks = ci % a.kst;
        if (!(ok = wt(&S.k_full[ks], (ci / a.kst) & 1, a.status, 5))) return;
        tc_fence_after();
        const uint32_t d = tmem + a.col_s + (ci & 1) * kKeys;
        for (int s = 0; s < a.nkq; ++s) {
          const uint64_t qd = smem_desc(smem_u32(sq + s * kQSlab), 16, 1024, kSw128);
          const uint64_t kd = smem_desc(smem_u32(sk + ((size_t)ks * a.nkq + s) * kSlab), 16, 1024, kSw128);
          const int steps = min(4, (p.d_qk - s * 64 + 15) / 16);
          for (int k = 0; k < steps; ++k)
            mma_bf16_ss(d, qd + (uint64_t)((k * 32) >> 4), kd + (uint64_t)((k * 32) >> 4), id_s, (s + k) != 0);
        }
        mma_commit(&S.k_empty[ks]);
        mma_commit(&S.s_full[ci & 1]);
        if (it.last()) mma_commit(&S.q_empty);
      };
      bool cur = it.next(tile), first = it.first;
      if (cur) issue_s(0);
      for (int ci = 0; cur && ok; ++ci) {
        const bool more = it.next(tile), nfirst = it.first;
        if (more) {
          issue_s(ci + 1);
          if (!ok) break;
        }
        const int vs = ci % a.vst;
        if (!(ok = wt(&S.p_full[ci & 1], (ci >> 1) & 1, a.status, 6))) break;
        if (!(ok = wt(&S.v_full[vs], (ci / a.vst) & 1, a.status, 7))) break;
        tc_fence_after();
        const uint64_t vd = smem_desc(smem_u32(sv + (size_t)vs * a.nkv * kSlab), kSlab, 1024, kSw128);
        const uint32_t pa = tmem + a.col_s + (ci & 1) * kKeys;
        const bool add = !first || *(volatile uint32_t*)&S.zeroed != 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_bf16_ts(tmem, pa + k * 8, vd + (uint64_t)((k * 2048) >> 4), id_o, add || k != 0);
        mma_commit(&S.v_empty[vs]);
        mma_commit(&S.pv_done);
        cur = more;
        first = nfirst;
      }
    }
  } else if (warp >= 4) {
    softmax_warps<T>(a, S, sv, tmem);
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, a.tmem_cols);
}

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

// Joins the pieces of units that several ranges share, in range order; also
// writes the rows nothing else does: of sequences without keys, outside all
// sequences, and past max_q.  Item = (row of a tile, four dims).
template <typename T>
__global__ void __launch_bounds__(256) tree_combine_kernel(const __grid_constant__ Args a, int tile_rows) {
  const SfaTreeParams& p = a.p;
  const int n = p.num_seqs, units = n * p.h_kv * a.ntiles;
  const int groups = p.d_v / 4;
  T* out = static_cast<T*>(p.o);
  const int first = blockIdx.y * blockDim.x + threadIdx.x, step = gridDim.y * blockDim.x;
  if ((int)blockIdx.x >= units) return rows_of_no_tile<T>(a, first, step);
  const int tile = blockIdx.x % a.ntiles, h = blockIdx.x / a.ntiles % p.h_kv, s = blockIdx.x / a.ntiles / p.h_kv;
  const int c0 = a.cum[s], nch = a.cum[s + 1] - c0;
  const int line = a.cum[n] * p.h_kv, len = max(a.min_chunks, (line + a.ranges - 1) / a.ranges);
  const int u0 = c0 * p.h_kv + h * nch;
  const int r0 = u0 / len, r1 = nch > 0 ? (u0 + nch - 1) / len : r0;
  if (nch > 0 && r0 == r1) return;
  const Seq q = load_seq(a, s);
  const int node0 = tile / a.n_hg * a.NT;
#pragma unroll 1
  for (int i = first; i < tile_rows * groups; i += step) {
    const int m = i % tile_rows, grp = i / tile_rows;
    const int node = node0 + (a.n_hg > 1 ? 0 : m / a.GB);
    const int hh = a.n_hg > 1 ? (tile % a.n_hg) * 128 + m : m % a.GB;
    if (hh >= a.G || node >= q.rows || node - node0 >= a.NT || q.q0 + node >= p.total_q) continue;
    const int head = h * a.G + hh;
    const int64_t row = q.q0 + node;
    if (nch == 0) {
      empty_row<T>(p, row, head, grp);
      continue;
    }
    auto slot = [&](int r) { return part_slot(a, r, tile, r == r0); };
    const float s2 = p.attn_sink ? __ldg(p.attn_sink + head) * kLog2e : -INFINITY;
    float M = s2;
    for (int r = r0; r <= r1; ++r) M = fmaxf(M, a.part_ml[slot(r) * 128 + m].x);
    float lt = s2 == -INFINITY ? 0.f : ex2(s2 - M);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r = r0; r <= r1; ++r) {
      const float2 ml = a.part_ml[slot(r) * 128 + m];
      if (ml.x == -INFINITY && ml.y == 0.f) continue;        // the piece holds no key of this row
      const float w = ex2(ml.x - M);
      const float4 v = reinterpret_cast<const float4*>(a.part_o)[(slot(r) * (a.dvp / 4) + grp) * 128 + m];
      lt = fmaf(ml.y, w, lt);
      o.x = fmaf(v.x, w, o.x);
      o.y = fmaf(v.y, w, o.y);
      o.z = fmaf(v.z, w, o.z);
      o.w = fmaf(v.w, w, o.w);
    }
    const bool none = lt == 0.f;
    const float inv = none ? 0.f : 1.f / lt;
    if (none) o = make_float4(0.f, 0.f, 0.f, 0.f);
    store4<T>(out + row * p.o_st + (int64_t)head * p.o_sh + grp * 4,
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
  const int64_t chunks = ((int64_t)p->table_width * p->page_size + kKeys - 1) / kKeys;
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
// whose rings fit shared memory: 128 rows of d_qk = d_v = 128 over 131072 keys take 1.7 times as long
// in the single kernel, which keeps the wider heads.
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
    a.keys = kKeys;
    a.keys_log = 6;
    sh = (sizeof(Shared) + 127) / 128 * 128;
    const size_t kb = (size_t)a.nkq * kSlab, vb = (size_t)a.nkv * kSlab;
    fit_rings(a, full, q + sh, kb, vb);           // 256 dims: 64 KB of Q, 32 KB a stage
    a.off_k = (uint32_t)q;
    a.off_v = a.off_k + (uint32_t)(a.kst * kb);
    a.off_sh = a.off_v + (uint32_t)(a.vst * vb);
    a.col_s = a.dvp <= 128 ? 128 : 256;
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
    if (pl.pair) {
      if ((e = launch_pair(a, pl.smem, tq, tk, tv, st)) != cudaSuccess) return e;
    } else {
      e = cudaFuncSetAttribute(tree_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pl.smem);
    if (e != cudaSuccess) return e;
    tree_kernel<T><<<dim3(a.ranges, a.ntiles), kThreads, pl.smem, st>>>(a, tq, tk, tv);
    note_launch("tree_attention", st);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
  } else {
    // no keys at all: every sequence has zero chunks
    if ((e = cudaMemsetAsync(a.cum, 0, ((size_t)a.p.num_seqs + 1) * sizeof(int32_t), st)) != cudaSuccess) return e;
    note_memset("tree_cum", st);
  }
  const int items = pl.tile_rows * (a.p.d_v / 4);
  const dim3 grid((unsigned)(a.p.num_seqs * a.p.h_kv * a.ntiles + 1), (unsigned)std::min(8, (items + 255) / 256));
  tree_combine_kernel<T><<<grid, 256, 0, st>>>(a, pl.tile_rows);
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

// sfa_tree_wide.cu — the tree attention of sfa_tree.cu for values of 129 to 256 dims, and keys that are
// too wide for the pair kernel's rings.
//
// O takes up to 256 columns of TMEM, two S tiles of 64 keys another 128: one softmax warpgroup, and the
// S of the next chunk is computed while it works on this one's.  64 keys a chunk: Q of 256 dims takes
// 64 KB of shared memory, a stage of the K or V ring 32 KB.  Measured at 256 dims: one
// cache of 131072 keys, 2 kv heads of 8 query heads, 16 drafted rows, 78 us (3.5 TB/s,
// 17 of them the join of 148 pieces); 64-node trees on 8 sequences 132 us (732 TFLOP/s).
//
// Warps: 0 K, Q and key masks; 1 V; 2 MMA issue; 3 clears value rows that must not enter a product (see
// scrub); 4-7 softmax.  Every wait is bounded (~2 s); on expiry the kernel records (7 << 16) | site in
// the status word and returns.
#include "sfa_tree_roles.cuh"

namespace sfa {
namespace tree {
namespace wide {

using C = Kernel<64, 256, 7>;
using Shared = tree::Shared<C>;
constexpr int kKeys = C::kKeys, kSlab = C::kSlab;
constexpr uint32_t kColS = 256;      // S of even / odd chunks at 256 + 64 (n & 1), O at 0

// S of a chunk is issued before PV of the one before; MMAs run in issue order, so S may overwrite the
// buffer whose P the PV before that reads.  The warp stays converged around MMAs (see elect).
__device__ __forceinline__ void issue(const Args& a, Shared& S, uint8_t* sq, uint8_t* sk, uint8_t* sv, uint32_t tmem,
                                      uint32_t types) {
  const uint32_t id_s = idesc_bf16(128, kKeys, false, false) ^ types;
  const uint32_t id_o = idesc_bf16(128, a.dvp, false, true) ^ types;
  const uint32_t k_step = (uint32_t)(a.nkq * kSlab) >> 4, v_step = (uint32_t)(a.nkv * kSlab) >> 4;
  const uint64_t dq = smem_desc(smem_u32(sq), 16, 1024, kSw128), dk = smem_desc(smem_u32(sk), 16, 1024, kSw128);
  const uint64_t dv = smem_desc(smem_u32(sv), kSlab, 1024, kSw128);
  const uint32_t q0 = uniform((uint32_t)dq), k0 = uniform((uint32_t)dk), v0 = uniform((uint32_t)dv);
  const uint32_t hi_k = uniform((uint32_t)(dk >> 32)), hi_v = uniform((uint32_t)(dv >> 32));
  tmem = uniform(tmem);
  const int tail = (a.p.d_qk - (a.nkq - 1) * 64 + 15) / 16;      // 16-dim steps of the last slab
  uint32_t ks = 0, kph = 0, vs = 0, vph = 0, nq = 0, scrubs = 0, before = 0;
  for (uint32_t n = 0;; ++n) {
    if (!wtw<C>(&S.k_full[ks], kph, a.status, 5)) return;
    const uint32_t word = uniform(S.word[n % kRing]);
    const bool stop = (word & kStop) != 0;
    if (!stop) {
      if (word & kOpens) {
        if (!wtw<C>(&S.q_full, nq & 1u, a.status, 4)) return;
        ++nq;
      }
      tc_fence_after();
      const uint32_t d = tmem + kColS + kKeys * (n & 1u), kx = k0 + ks * k_step;
      if (elect()) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (x < a.nkq) {
            const uint32_t qy = q0 + x * (kQSlab >> 4), ky = kx + x * (kSlab >> 4);
            const int steps = x + 1 < a.nkq ? 4 : tail;
            mma_bf16_ss(d, desc(hi_k, qy), desc(hi_k, ky), id_s, x != 0);
            if (steps > 1) mma_bf16_ss(d, desc(hi_k, qy + 2), desc(hi_k, ky + 2), id_s, 1);
            if (steps > 2) mma_bf16_ss(d, desc(hi_k, qy + 4), desc(hi_k, ky + 4), id_s, 1);
            if (steps > 3) mma_bf16_ss(d, desc(hi_k, qy + 6), desc(hi_k, ky + 6), id_s, 1);
          }
        }
        mma_commit(&S.s_full[n & 1u]);
        mma_commit(&S.k_empty[ks]);
        if (word & kCloses) mma_commit(&S.q_empty);
      }
      __syncwarp();
      if (++ks == (uint32_t)a.kst) {
        ks = 0;
        kph ^= 1u;
      }
    }
    if (n > 0) {
      const uint32_t m = n - 1;
      if (!wtw<C>(&S.v_full[vs], vph, a.status, 7)) return;
      if (before & kScrubbed) {
        if (!wtw<C>(&S.v_ready[scrubs % kRing], (scrubs / kRing) & 1u, a.status, 8)) return;
        ++scrubs;
      }
      if (!wtw<C>(&S.p_full[m & 1u], (m >> 1) & 1u, a.status, 6)) return;
      tc_fence_after();
      const uint32_t add = !(before & kOpens) ? 1u : uniform(*(volatile uint32_t*)&S.zeroed[0]);
      const uint32_t pa = tmem + kColS + kKeys * (m & 1u), vl = v0 + vs * v_step;
      if (elect()) {
        mma_bf16_ts(tmem, pa, desc(hi_v, vl), id_o, add);
#pragma unroll
        for (int i = 1; i < kKeys / 16; ++i) mma_bf16_ts(tmem, pa + i * 8, desc(hi_v, vl + i * (2048 >> 4)), id_o, 1);
        mma_commit(&S.v_empty[vs]);
        mma_commit(&S.pv_done[0]);
      }
      __syncwarp();
      if (++vs == (uint32_t)a.vst) {
        vs = 0;
        vph ^= 1u;
      }
    }
    if (stop) return;
    before = word;
  }
}

template <typename T>
__device__ __forceinline__ void softmax(const Args& a, Shared& S, uint32_t tmem) {
  const SfaTreeParams& p = a.p;
  const int m = threadIdx.x & 127, wq = m >> 5, tile = blockIdx.y;
  const uint32_t to = tmem + ((uint32_t)(wq * 32) << 16);
  const float c2 = p.scale * kLog2e;
  const uint64_t c22 = two(c2, c2);
  const bool by_tree = p.parents != nullptr;
  const int node0 = node_of_tile(a, tile), my_node = a.n_hg > 1 ? 0 : m / a.GB, node = node0 + my_node;
  const int my_head = a.n_hg > 1 ? (tile % a.n_hg) * 128 + m : m - my_node * a.GB;
  Walk walk(a, S.range);
  Piece g;
  int n = 0, met = 0, scrubs = 0, added = 0;                  // chunks, meetings, scrubs before the job, PVs waited for
  bool ok = true;
  // Waits until PV of the first `until` chunks has completed.  Called with it growing by at most one: a
  // parity wait would take a phase two behind for the one it asks for.
  auto pv_through = [&](int until, int site) {
    if (added < until) {
      if (!wtw<C>(&S.pv_done[0], added & 1, a.status, site)) return false;
      ++added;
    }
    return true;
  };
  auto meet = [&](int site) {
    warp_arrive(&S.meet[0]);
    return wtw<C>(&S.meet[0], (met++) & 1, a.status, site);
  };
  while (ok && walk.next(g)) {
    const Job j = make_job<C>(a, g);
    const bool live = my_node < a.NT && my_head < a.G && node < g.q.rows && g.q.q0 + node < p.total_q;
    const bool any = __any_sync(0xffffffffu, live);
    const int prefix = g.q.prefix, rows_of = g.q.rows;
    const bool ran = j.c0 < j.end, tree = by_tree && rows_of > 1;   // a lone row sees the same either way
    if (tree && ran && j.end * kKeys > prefix) {
      // every warp has read the ancestors of the piece before (it waited for that piece's last PV)
      const int rows = min(rows_of, min(kMaxNodes, p.total_q - g.q.q0));
#pragma unroll 1
      for (int i = m; i < rows; i += 128) S.parent[0][i] = (short)max(-1, min(__ldg(p.parents + g.q.q0 + i), i));
      if (!(ok = meet(12))) break;
      if (m < a.NT) mark_ancestors(S.anc[0][m], S.parent[0], node0 + m, rows);
      if (!(ok = meet(13))) break;
    }
    float mref = -INFINITY, l = 0.f;
    for (int c = j.c0; c < j.end; ++c, ++n) {
      const bool first = c == j.c0;
      if (!(ok = wtw<C>(&S.s_full[n & 1], (n >> 1) & 1, a.status, 14))) break;
      tc_fence_after();
      const uint32_t ts = to + kColS + kKeys * (n & 1);
      const uint4 km = S.mask[n % kRing];
      const int d0 = c * kKeys - prefix;                      // the chunk's first key, as a drafted row
      const bool drafted = d0 + kKeys > 0;
      const bool whole = (km.x & km.y) == ~0u && !drafted;
      uint32_t v0 = km.x, v1 = km.y;
      if (any) {
        // loaded and waited for in one place: a load in flight across a call (a slow wait, a rescale)
        // would land in registers that the call has saved or given away
        float s0[32], s1[32];
        ld32(ts, s0);
        ld32(ts + 32, s1);
        ld_wait32(s0);
        ld_wait32(s1);
        if (drafted) {
          v0 &= sees32(S.anc[0][my_node], tree, node, d0);
          v1 &= sees32(S.anc[0][my_node], tree, node, d0 + 32);
        }
        if (!live) v0 = v1 = 0;
        if (!whole) {
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            if (!((v0 >> k) & 1u)) s0[k] = -INFINITY;
            if (!((v1 >> k) & 1u)) s1[k] = -INFINITY;
          }
        }
        // P against the reference maximum so far.  The maximum of these keys is not needed for that: if
        // their sum stays below `most`, so does every P (and an infinite or a first one does not), and
        // only otherwise is the reference raised and P done again.
        float part;
        for (bool again = false;; again = true) {
          const float nm = mref == -INFINITY ? 0.f : -mref;
          const uint64_t nm2 = two(nm, nm);
          uint64_t sum0 = 0, sum1 = 0;
          exps<T>(s0, c22, nm2, sum0, ts);
          exps<T>(s1, c22, nm2, sum1, ts + 16);
          float t0, t1;
          untwo(add2(sum0, sum1), t0, t1);
          part = t0 + t1;
          const bool up = live && (part > Reference<T>::most || mref == -INFINITY);
          if (again || !__any_sync(0xffffffffu, up)) break;
          float top = -INFINITY;
#pragma unroll
          for (int k = 0; k < 32; ++k) top = fmaxf(top, fmaxf(s0[k], s1[k]));
          top = top * c2 - Reference<T>::below;
          float fac = 1.f;
          if (up && top > mref) {
            if (mref != -INFINITY) fac = ex2(mref - top);
            mref = top;
          }
          if (__any_sync(0xffffffffu, fac != 1.f)) {
            l *= fac;
            if (!(ok = pv_through(n, 11))) break;             // O to the raised maximum: nothing is being added to it
            tc_fence_after();
            rescale<T>(to, first ? 0 : a.dvp, ts, 0, fac);
          }
        }
        l += part;                                            // zero where no key is seen
        tmem_st_wait();
      }
      // the chunk before has been added (while this one's P was computed)
      if (!ok || !(ok = pv_through(n, 12))) break;
      if (first && m == 0) S.zeroed[0] = 0;
      if (drafted && rows_of > 1) {
        const int k = scrubs + (c - j.scrub);
        if (!(ok = wtw<C>(&S.v_ready[k % kRing], (k / kRing) & 1, a.status, 16))) break;
        const uint4 bad = *reinterpret_cast<const uint4*>(S.bad[k % kRing]);
        if (bad.x | bad.y) {
          tc_fence_after();
          add_nonfinite<T>(a, g, c * kKeys, to, first, bad.x, live ? v0 : 0u);
          add_nonfinite<T>(a, g, c * kKeys + 32, to, false, bad.y, live ? v1 : 0u);
          if (first && m == 0) S.zeroed[0] = 1;
        }
      }
      tc_fence_before();
      warp_arrive(&S.p_full[n & 1]);
    }
    if (!ok || !(ok = pv_through(n, 17))) break;
    tc_fence_after();
    scrubs += max(0, j.end - j.scrub);
    if (!any) continue;
    const int head = g.h * a.G + my_head;
    const bool split = !g.whole, none = mref == -INFINITY && l == 0.f;
    float f = 1.f;
    float4* dst = nullptr;
    T* orow = nullptr;
    if (split) {
      const int64_t slot = part_slot(a, blockIdx.x, tile, g.c0 == 0);
      if (live) a.part_ml[slot * 128 + m] = make_float2(mref, l);
      dst = reinterpret_cast<float4*>(a.part_o) + slot * (a.dvp / 4) * 128 + m;
    } else {
      const float sink = p.attn_sink && live ? __ldg(p.attn_sink + head) : -INFINITY;
      const float s2 = sink * kLog2e, M = fmaxf(mref, s2);
      const float w = mref == -INFINITY ? 0.f : ex2(mref - M);
      const float lt = l * w + (s2 == -INFINITY ? 0.f : ex2(s2 - M));
      f = none ? 0.f : w / lt;
      const int64_t row = g.q.q0 + node;
      orow = static_cast<T*>(p.o) + row * p.o_st + (int64_t)head * p.o_sh;
      if (live) p.lse[row * p.l_st + (int64_t)head * p.l_sh] = none ? sink : (M + lg2(lt)) * kLn2;
    }
#pragma unroll 1
    for (int y = 0; y < a.dvp; y += 16) {
      float o[16] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (ran) {                                              // warp-uniform: the TMEM loads are the whole warp's
        tmem_ld16(to + y, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = none ? 0.f : o[i] * f;
      }
      if (!live) continue;
      if (split) {
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[(y / 4 + i) * 128] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; i += 8)
          if (y + i < p.d_v)
            *reinterpret_cast<uint4*>(orow + y + i) =
                make_uint4(pack2<T>(o[i], o[i + 1]), pack2<T>(o[i + 2], o[i + 3]), pack2<T>(o[i + 4], o[i + 5]),
                           pack2<T>(o[i + 6], o[i + 7]));
      }
    }
    tc_fence_before();
  }
}

template <typename T>
__global__ void __launch_bounds__(C::kThreads, 1)
tree_wide_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                 const __grid_constant__ CUtensorMap tmv) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sq = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sk = sq + a.off_k;
  uint8_t* sv = sq + a.off_v;
  Shared& S = *reinterpret_cast<Shared*>(sq + a.off_sh);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    mbar_init(&S.q_full, 1);
    mbar_init(&S.q_empty, 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&S.k_full[i], 1);
      mbar_init(&S.k_empty[i], 1);
      mbar_init(&S.v_full[i], 1);
      mbar_init(&S.v_empty[i], 1);
    }
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&S.scrub_go[i], 1);
      mbar_init(&S.v_ready[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S.s_full[i], 1);
      mbar_init(&S.p_full[i], 4);
    }
    mbar_init(&S.pv_done[0], 1);
    mbar_init(&S.meet[0], 4);
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
  if (warp < 2) {
    produce<C>(a, S, warp == 0, warp == 0 ? sk : sv, sq, warp == 0 ? &tmk : &tmv, &tmq);
  } else if (warp == 2) {
    issue(a, S, sq, sk, sv, tmem, type_bits<T>());
  } else if (warp == 3) {
    scrub<C, T>(a, S, sv);
  } else {
    softmax<T>(a, S, tmem);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, a.tmem_cols);
}

}  // namespace wide

size_t wide_shared_bytes() { return sizeof(wide::Shared); }

template <typename T>
static cudaError_t launch_wide_typed(const Args& a, size_t smem, const CUtensorMap& tq, const CUtensorMap& tk,
                                     const CUtensorMap& tv, cudaStream_t st) {
  const cudaError_t e =
      cudaFuncSetAttribute(wide::tree_wide_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  wide::tree_wide_kernel<T><<<dim3(a.ranges, a.ntiles), wide::C::kThreads, smem, st>>>(a, tq, tk, tv);
  note_launch("tree_attention", st);
  return cudaGetLastError();
}

cudaError_t launch_wide(const Args& a, size_t smem, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                        cudaStream_t st) {
  return a.p.dtype == SFA_DTYPE_F16 ? launch_wide_typed<__half>(a, smem, tq, tk, tv, st)
                                    : launch_wide_typed<__nv_bfloat16>(a, smem, tq, tk, tv, st);
}

}  // namespace tree
}  // namespace sfa

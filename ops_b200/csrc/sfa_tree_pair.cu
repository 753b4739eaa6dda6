// sfa_tree_pair.cu — the tree attention of sfa_tree.cu with two softmax
// warpgroups per CTA (d_v <= 128).
//
// A warpgroup's work between two MMAs (read S, exponentials, P back to TMEM)
// takes about as long as the MMAs and their hand-overs, so two of them take
// turns on the tensor core: each has its own S and O in TMEM (2 x 128 + 2 x 128
// columns) and works on chunks of 128 keys, the width at which the MMAs run at
// full rate.  What the two share depends on the rows:
//   rows: two row tiles (256 rows) against the same chunk, which is loaded once
//         for both: large trees, bound by the chain below;
//   keys: one row tile, alternate chunks; the two (m, l, O) are joined at the end
//         of the piece out of TMEM: decoding and small trees, bound by reads.
// A CTA goes by piece: it falls back to `keys` where its second tile is empty.
//
// Measured: one token for each of 16 sequences of 4096 to 32768 keys, 64 heads on
// 8, 179 us at 5.1 TB/s (0.79 of the measured copy rate); 64-node trees on 8
// sequences 244 us, 790 TFLOP/s (0.48 of the measured peak).  There a period of
// 4600 clocks covers 128 keys for both tiles: 2300 from S to P (1024 of them the
// exponentials' floor) and 2300 from P to the next S (1024 of them MMAs).  Not
// better: S in halves of 64 keys (half the MMA rate; 251 us), P handed over in
// halves (266), an issuing warp per warpgroup (281), softmax in steps of 32 keys
// (280).  The loops are rolled and the MMAs issued from a converged warp because
// the roles together have to fit the instruction cache: unrolled (148 KB of code)
// the first case took 408 us.
//
// Warps: 0 K, Q and key masks; 1 V; 2 MMA issue; 3 clears value rows that must not
// enter a product (see scrub); 4-7 and 8-11 softmax.
// Every wait is bounded (~2 s); on expiry the kernel records (8 << 16) | site in
// the status word and returns.
#include "sfa_tree_roles.cuh"

namespace sfa {
namespace tree {
namespace pair {

using C = Kernel<128, 384, 8>;
using Shared = tree::Shared<C>;
constexpr int kKeys = C::kKeys, kSlab = C::kSlab, kThreads = C::kThreads, kId = C::kId;
constexpr uint32_t kColS = 256;      // S of warpgroup w at 256 + 128 w, its O at 128 w

// Whether the phase has completed, without waiting; one answer for the warp.
__device__ __forceinline__ bool ready(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return __all_sync(0xffffffffu, ok != 0);
}

// The issuing warp takes what is ready: PV of the oldest task whose P is there, then S of the next
// chunk for a warpgroup that has no P outstanding (S overwrites the columns of P, and MMAs run in issue
// order, so it goes behind the PV that reads P, and right behind it: a warpgroup waits for both).
__device__ __forceinline__ void issue(const Args& a, Shared& S, uint8_t* sq, uint8_t* sk, uint8_t* sv, uint32_t tmem,
                                      uint32_t types) {
  const uint32_t id_s = idesc_bf16(128, kKeys, false, false) ^ types;
  const uint32_t id_o = idesc_bf16(128, a.dvp, false, true) ^ types;
  const uint32_t k_step = (uint32_t)(a.nkq * kSlab) >> 4, v_step = (uint32_t)(a.nkv * kSlab) >> 4;
  const uint32_t q_tile = (uint32_t)(a.nkq * kQSlab) >> 4;
  // descriptors: addresses advance in the low word, the high word holds layout only
  const uint64_t dq = smem_desc(smem_u32(sq), 16, 1024, kSw128), dk = smem_desc(smem_u32(sk), 16, 1024, kSw128);
  const uint64_t dv = smem_desc(smem_u32(sv), kSlab, 1024, kSw128);
  const uint32_t q0 = uniform((uint32_t)dq), k0 = uniform((uint32_t)dk), v0 = uniform((uint32_t)dv);
  const uint32_t hi_k = uniform((uint32_t)(dk >> 32)), hi_v = uniform((uint32_t)(dv >> 32));
  tmem = uniform(tmem);
  const int tail = (a.p.d_qk - (a.nkq - 1) * 64 + 15) / 16;      // 16-dim steps of the last slab
  uint32_t waiting = 0;                                          // warpgroups whose P is outstanding
  uint32_t sw = 0, rest_s = 0, pw = 0, rest_p = 0;               // words of the chunks at hand, warpgroups left of them
  uint32_t ks = 0, kph = 0, vs = 0, vph = 0, nq = 0, np0 = 0, np1 = 0;
  uint32_t cs = 0, cp = 0, scrubs = 0;                           // chunks begun by S / by PV, scrubbed ones passed
  bool stop = false, v_there = false;
  uint64_t idle_since = 0;
  uint32_t spins = 0;
  while (true) {
    bool moved = false;
    if (rest_p == 0 && cp < cs) {
      pw = uniform(S.word[cp++ % kRing]);
      rest_p = pw & kGroups;
      v_there = false;
    }
    if (rest_p != 0 && !v_there && ready(&S.v_full[vs], vph) &&
        (!(pw & kScrubbed) || ready(&S.v_ready[scrubs % kRing], (scrubs / kRing) & 1u))) {
      v_there = true;
      if (pw & kScrubbed) ++scrubs;
    }
    if (rest_p != 0 && v_there) {
      const uint32_t wg = (rest_p & 1u) ? 0u : 1u;
      if (((waiting >> wg) & 1u) && ready(&S.p_full[wg], (wg ? np1 : np0) & 1u)) {
        tc_fence_after();
        np0 += wg ^ 1u;
        np1 += wg;
        const uint32_t add = !(((pw & kBegins) >> 2 >> wg) & 1u) ? 1u : uniform(*(volatile uint32_t*)&S.zeroed[wg]);
        const uint32_t pa = tmem + kColS + 128 * wg, d = tmem + 128 * wg, vl = v0 + vs * v_step;
        const bool frees = rest_p == (1u << wg), ends = ((pw & kEnds) >> 4 >> wg) & 1u;
        if (elect()) {
          mma_bf16_ts(d, pa, desc(hi_v, vl), id_o, add);
#pragma unroll
          for (int i = 1; i < kKeys / 16; ++i) mma_bf16_ts(d, pa + i * 8, desc(hi_v, vl + i * (2048 >> 4)), id_o, 1);
          if (frees) mma_commit(&S.v_empty[vs]);
          if (ends) mma_commit(&S.pv_done[wg]);
        }
        __syncwarp();
        waiting &= ~(1u << wg);
        rest_p &= ~(1u << wg);
        if (frees && ++vs == (uint32_t)a.vst) {
          vs = 0;
          vph ^= 1u;
        }
        moved = true;
      }
    }
    if (rest_s != 0) {
      const uint32_t wg = (rest_s & 1u) ? 0u : 1u;
      const bool opens = (sw & kOpens) != 0 && rest_s == (sw & kGroups);
      if (!((waiting >> wg) & 1u) && (!opens || ready(&S.q_full, nq & 1u))) {
        tc_fence_after();
        nq += opens ? 1u : 0u;
        const uint32_t d = tmem + kColS + 128 * wg;
        const uint32_t qx = q0 + (((sw & kRows) && wg) ? q_tile : 0u), kx = k0 + ks * k_step;
        const bool frees = rest_s == (1u << wg);
        if (elect()) {
#pragma unroll
          for (int x = 0; x < 3; ++x) {                          // d_qk up to 192 fits this kernel's shared memory
            if (x < a.nkq) {
              const uint32_t qy = qx + x * (kQSlab >> 4), ky = kx + x * (kSlab >> 4);
              const int steps = x + 1 < a.nkq ? 4 : tail;
              mma_bf16_ss(d, desc(hi_k, qy), desc(hi_k, ky), id_s, x != 0);
              if (steps > 1) mma_bf16_ss(d, desc(hi_k, qy + 2), desc(hi_k, ky + 2), id_s, 1);
              if (steps > 2) mma_bf16_ss(d, desc(hi_k, qy + 4), desc(hi_k, ky + 4), id_s, 1);
              if (steps > 3) mma_bf16_ss(d, desc(hi_k, qy + 6), desc(hi_k, ky + 6), id_s, 1);
            }
          }
          mma_commit(&S.s_full[wg]);
          if (frees) mma_commit(&S.k_empty[ks]);
          if (frees && (sw & kCloses)) mma_commit(&S.q_empty);
        }
        __syncwarp();
        waiting |= 1u << wg;
        rest_s &= ~(1u << wg);
        if (frees && ++ks == (uint32_t)a.kst) {
          ks = 0;
          kph ^= 1u;
        }
        moved = true;
      }
    }
    if (!stop && rest_s == 0 && ready(&S.k_full[ks], kph)) {
      sw = uniform(S.word[cs % kRing]);
      stop = (sw & kStop) != 0;
      rest_s = stop ? 0u : sw & kGroups;
      cs += stop ? 0u : 1u;
      moved = true;
    }
    if (moved) {
      idle_since = 0;
      continue;
    }
    if (stop && rest_p == 0 && cp == cs) return;
    if ((++spins & 63) != 0) continue;
    const uint64_t now = __shfl_sync(0xffffffffu, global_timer_ns(), 0);
    if (idle_since == 0) {
      idle_since = now;
    } else if (now - idle_since > kWaitLimitNs) {
      record_status(a.status, (kId << 16) | 6);
      return;
    }
  }
}

template <typename T>
__device__ __forceinline__ void softmax(const Args& a, Shared& S, int wg, uint32_t tmem) {
  const SfaTreeParams& p = a.p;
  const int m = threadIdx.x & 127, wq = m >> 5;
  const uint32_t tl = tmem + ((uint32_t)(wq * 32) << 16), to = tl + 128 * wg, ts = tl + kColS + 128 * wg;
  const float c2 = p.scale * kLog2e;
  const uint64_t c22 = two(c2, c2);
  const bool by_tree = p.parents != nullptr;
  const int my_node = a.n_hg > 1 ? 0 : m / a.GB, m_head = m - my_node * a.GB;
  Walk walk(a, S.range);
  Piece g;
  int n = 0, jobs = 0, met = 0, joined = 0, base = 0, scrubs = 0;   // tasks, ended pieces, meetings, joins; chunks and scrubs before the job
  bool ok = true, owe = false;
  auto meet = [&](int site) {
    warp_arrive(&S.meet[wg]);
    return wtw<C>(&S.meet[wg], (met++) & 1, a.status, site);
  };
  while (ok && walk.next(g)) {
    const Job j = make_job<C>(a, g);
    const int tile = (a.two ? 2 * blockIdx.y : blockIdx.y) + (j.rows ? wg : 0);
    const int node0 = node_of_tile(a, tile);
    const int my_head = a.n_hg > 1 ? (tile % a.n_hg) * 128 + m : m_head;
    const int node = node0 + my_node;
    const bool live = my_node < a.NT && my_head < a.G && node < g.q.rows && g.q.q0 + node < p.total_q;
    const bool any = __any_sync(0xffffffffu, live);
    const int prefix = g.q.prefix, rows_of = g.q.rows, job_c0 = j.c0, job_scrub = j.scrub;
    const int c_first = j.rows ? j.c0 : j.c0 + wg, c_end = j.rows ? (wg ? j.end_b : j.end_a) : j.end, c_step = j.rows ? 1 : 2;
    const bool ran = c_first < c_end;
    const bool tree = by_tree && g.q.rows > 1;                // a lone row sees the same either way
    if (tree && ran && c_end * kKeys > prefix) {
      // every warp has read the ancestors of the piece before (it waited for that piece's last PV)
      const int rows = min(g.q.rows, min(kMaxNodes, p.total_q - g.q.q0));
#pragma unroll 1
      for (int i = m; i < rows; i += 128) S.parent[wg][i] = (short)max(-1, min(__ldg(p.parents + g.q.q0 + i), i));
      if (!(ok = meet(12))) break;
      if (m < a.NT) mark_ancestors(S.anc[wg][m], S.parent[wg], node0 + m, rows);
      if (!(ok = meet(13))) break;
    }
    float mref = -INFINITY, l = 0.f;
    for (int c = c_first; c < c_end; c += c_step, ++n) {
      const int cn = base + (c - job_c0);
      const bool first = c == c_first;
      if (!(ok = wtw<C>(&S.s_full[wg], n & 1, a.status, 14))) break;
      tc_fence_after();
      // S of this chunk was issued behind PV of the warpgroup's last one: O may be changed from here on
      const uint4 km = S.mask[cn % kRing];
      const int d0 = c * kKeys - prefix;                      // the chunk's first key, as a drafted row
      const bool drafted = d0 + kKeys > 0;
      const bool whole = (km.x & km.y & km.z & km.w) == ~0u && !drafted;
      uint32_t vis[4] = {km.x, km.y, km.z, km.w};
      if (any) {
        if (drafted) {
#pragma unroll
          for (int i = 0; i < 4; ++i) vis[i] &= sees32(S.anc[wg][my_node], tree, node, d0 + 32 * i);
        }
        // 64 keys at a time in a loop that is not unrolled, for the sake of the instruction cache
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          // loaded and waited for in one place: a load in flight across a call (a slow wait, a rescale)
          // would land in registers that the call has saved or given away
          float s0[32], s1[32];
          ld32(ts + 64 * i, s0);
          ld32(ts + 64 * i + 32, s1);
          ld_wait32(s0);
          ld_wait32(s1);
          if (!whole) {
            const uint32_t v0 = !live ? 0u : i ? vis[2] : vis[0], v1 = !live ? 0u : i ? vis[3] : vis[1];
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
            exps<T>(s0, c22, nm2, sum0, ts + 32 * i);         // over columns of S that have been read
            exps<T>(s1, c22, nm2, sum1, ts + 32 * i + 16);
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
              // O, the sum and P of the chunk's first half to the raised maximum
              l *= fac;
              rescale<T>(to, first ? 0 : a.dvp, ts, 32 * i, fac);
            }
          }
          l += part;                                          // zero where no key is seen
        }
        tmem_st_wait();
      }
      if (first) {
        if (m == 0) S.zeroed[wg] = 0;
        if (owe) {                                            // warpgroup A has taken O of the piece before
          if (!(ok = wtw<C>(&S.b_free, (joined - 1) & 1, a.status, 15))) break;
          owe = false;
        }
      }
      if (drafted && rows_of > 1) {
        const int k = scrubs + (c - job_scrub);
        if (!(ok = wtw<C>(&S.v_ready[k % kRing], (k / kRing) & 1, a.status, 16))) break;
        const uint4 bad = *reinterpret_cast<const uint4*>(S.bad[k % kRing]);
        if (bad.x | bad.y | bad.z | bad.w) {
          tc_fence_after();
          const bool mine = live && any;
          add_nonfinite<T>(a, g, c * kKeys, to, first, bad.x, mine ? vis[0] : 0u);
          add_nonfinite<T>(a, g, c * kKeys + 32, to, false, bad.y, mine ? vis[1] : 0u);
          add_nonfinite<T>(a, g, c * kKeys + 64, to, false, bad.z, mine ? vis[2] : 0u);
          add_nonfinite<T>(a, g, c * kKeys + 96, to, false, bad.w, mine ? vis[3] : 0u);
          if (first && m == 0) S.zeroed[wg] = 1;
        }
      }
      tc_fence_before();
      warp_arrive(&S.p_full[wg]);
    }
    if (!ok) break;
    base += j.end - j.c0;
    scrubs += max(0, j.end - j.scrub);
    if (ran) {
      if (!(ok = wtw<C>(&S.pv_done[wg], (jobs++) & 1, a.status, 17))) break;
      tc_fence_after();
    }
    float wa = 1.f, wb = 0.f;
    const bool join = !j.rows && j.end - j.c0 > 1;            // both warpgroups hold a part of the rows
    if (!j.rows && wg == 1) {
      if (join) {
        S.ml[m] = make_float2(mref, l);
        tc_fence_before();
        warp_arrive(&S.b_ready);
        owe = true;
        ++joined;
      }
      continue;
    }
    if (join) {
      if (!(ok = wtw<C>(&S.b_ready, (joined++) & 1, a.status, 18))) break;
      tc_fence_after();
      const float2 b = S.ml[m];
      const float M = fmaxf(mref, b.x);
      wa = mref == -INFINITY ? 0.f : ex2(mref - M);
      wb = b.x == -INFINITY ? 0.f : ex2(b.x - M);
      // a NaN sum has to survive a weight of zero
      l = (mref == -INFINITY ? l : l * wa) + (b.x == -INFINITY ? b.y : b.y * wb);
      mref = M;
    }
    if (any) {
      const int head = g.h * a.G + my_head;
      const bool split = !g.whole;
      const bool none = mref == -INFINITY && l == 0.f;
      float fa = wa, fb = wb;
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
        const float inv = none ? 0.f : w / lt;
        fa *= inv;
        fb *= inv;
        const int64_t row = g.q.q0 + node;
        orow = static_cast<T*>(p.o) + row * p.o_st + (int64_t)head * p.o_sh;
        if (live) p.lse[row * p.l_st + (int64_t)head * p.l_sh] = none ? sink : (M + lg2(lt)) * kLn2;
      }
#pragma unroll 1
      for (int y = 0; y < a.dvp; y += 16) {
        float o[16] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (ran) {                                            // warp-uniform: the TMEM loads are the whole warp's
          tmem_ld16(to + y, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] *= fa;
          if (join) {
            float ob[16];
            tmem_ld16(tl + 128 + y, ob);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = fmaf(ob[i], fb, o[i]);
          }
          if (none) {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = 0.f;
          }
        }
        if (live) {
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
      }
    }
    tc_fence_before();
    if (join) warp_arrive(&S.b_free);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
tree_pair_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
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
      mbar_init(&S.pv_done[i], 1);
      mbar_init(&S.meet[i], 4);
    }
    mbar_init(&S.b_ready, 4);
    mbar_init(&S.b_free, 4);
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
    softmax<T>(a, S, (warp - 4) >> 2, tmem);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, a.tmem_cols);
}

}  // namespace pair

size_t pair_shared_bytes() { return sizeof(pair::Shared); }

template <typename T>
static cudaError_t launch_pair_typed(const Args& a, size_t smem, const CUtensorMap& tq, const CUtensorMap& tk,
                                     const CUtensorMap& tv, cudaStream_t st) {
  const cudaError_t e =
      cudaFuncSetAttribute(pair::tree_pair_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const int y = a.two ? (a.ntiles + 1) / 2 : a.ntiles;
  pair::tree_pair_kernel<T><<<dim3(a.ranges, y), pair::kThreads, smem, st>>>(a, tq, tk, tv);
  note_launch("tree_attention_pair", st);
  return cudaGetLastError();
}

cudaError_t launch_pair(const Args& a, size_t smem, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                        cudaStream_t st) {
  return a.p.dtype == SFA_DTYPE_F16 ? launch_pair_typed<__half>(a, smem, tq, tk, tv, st)
                                    : launch_pair_typed<__nv_bfloat16>(a, smem, tq, tk, tv, st);
}

}  // namespace tree
}  // namespace sfa

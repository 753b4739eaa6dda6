// sfa_tree_roles.cuh — what the warps of the two attention kernels have in common: the chunks of a
// CTA one after another, the producers of the K and V rings, the scrub of value rows, and the
// arithmetic between the MMAs.  C: kKeys (a chunk's), kThreads, kId (of the kernel in the status word).
#pragma once

#include "sfa_tree.cuh"

namespace sfa {
namespace tree {

constexpr int kRing = 8;             // key masks and scrub results: more chunks than are in flight

// P is taken against a reference 2^below below the largest score seen when it was set, and the reference is
// raised when a sum of P passes `most`: so every P is far inside the type, and sums far inside fp32.  bf16
// has fp32's range.  In fp16, P below 2^-14 loses bits and below 2^-25 is gone while the row sum keeps it; with the
// reference at the maximum, one key that takes all left the others of a cache of 16384 up to 16 times the
// rounding of the rest off.  2^8 below, 64 keys as large as the largest still sum to half of `most`.
template <typename T>
struct Reference {
  static constexpr float most = 16384.f, below = 0.f;
};
template <>
struct Reference<__half> {
  static constexpr float most = 32768.f, below = 8.f;
};

template <int KEYS, int THREADS, int ID>
struct Kernel {
  static constexpr int kKeys = KEYS, kKeysLog = KEYS == 128 ? 7 : 6, kThreads = THREADS, kId = ID;
  static constexpr int kSlab = KEYS * 128;   // bytes of a 64-dim slab of a chunk
};

template <class C>
struct Shared {
  uint64_t q_full, q_empty;
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t scrub_go[kRing], v_ready[kRing];
  uint64_t s_full[2], p_full[2], pv_done[2], meet[2];
  uint64_t b_ready, b_free;            // keys: warpgroup B's piece is complete / has been taken
  uint32_t tmem_base;
  uint32_t zeroed[2];                  // O of a piece was initialised by the warpgroup
  alignas(16) uint32_t bad[kRing][4];              // keys whose value row has a non-finite element
  uint4 mask[kRing];                   // keys of the chunk that exist
  uint32_t word[kRing];                // chunk_word of the chunk
  float2 ml[128];                      // warpgroup B's (m, l)
  int scan[C::kThreads / 32];
  Range range;
  short parent[2][kMaxNodes];
  uint32_t anc[2][128][kAncWords];     // ancestors of each row of the warpgroup's tile
};

template <class C>
__device__ __forceinline__ bool wt(uint64_t* bar, uint32_t parity, int32_t* status, int site) {
  return bounded_wait(bar, parity, status, C::kId, site);
}
template <class C>
__device__ __forceinline__ bool wtw(uint64_t* bar, uint32_t parity, int32_t* status, int site) {
  return __all_sync(0xffffffffu, wt<C>(bar, parity, status, site));
}

// A piece as this CTA's two tiles see it: chunks [c0, end), of which tile A (rows: B) needs those
// before end_a (end_b), and those from `scrub` on hold value rows to clear.
struct Job {
  Piece g;
  int c0, end, end_a, end_b, scrub;
  bool rows;
};

template <class C>
static __device__ __noinline__ Job make_job(const Args& a, const Piece& g) {
  Job j;
  j.g = g;
  j.c0 = g.c0;
  const int ta = a.two ? 2 * blockIdx.y : blockIdx.y;
  j.end_a = tile_end(a, ta, g);
  j.rows = a.two && ta + 1 < a.ntiles && node_of_tile(a, ta + 1) < g.q.rows;
  j.end_b = j.rows ? tile_end(a, ta + 1, g) : g.c0;
  j.end = max(j.end_a, j.end_b);
  // the last, partly filled chunk; every chunk with drafted keys when some rows do not see some of them
  int f = g.q.kvc % C::kKeys ? g.q.nch - 1 : g.q.nch;
  if (g.q.rows > 1) f = min(f, max(0, g.q.prefix) / C::kKeys);
  j.scrub = max(f, g.c0);
  return j;
}

// The chunks of the CTA's jobs one after another; n counts them, k those that are scrubbed.
template <class C>
struct Chunks {
  Walk w;
  Job j;
  int c, n, k;
  __device__ __forceinline__ Chunks(const Args& a, const Shared<C>& S) : w(a, S.range), c(0), n(-1), k(-1) { j.c0 = j.end = 0; }
  __device__ __forceinline__ bool next() {
    if (c + 1 < j.end) {
      ++c;
    } else {
      do {
        Piece g;
        if (!w.next(g)) return false;
        j = make_job<C>(*w.a, g);
      } while (j.c0 >= j.end);
      c = j.c0;
    }
    ++n;
    k += scrubbed();
    return true;
  }
  __device__ __forceinline__ bool first() const { return c == j.c0; }
  __device__ __forceinline__ bool last() const { return c + 1 == j.end; }
  __device__ __forceinline__ bool scrubbed() const { return c >= j.scrub; }
  // the warpgroups that work on the chunk, as bits
  __device__ __forceinline__ int groups() const {
    return j.rows ? (c < j.end_a ? 1 : 0) | (c < j.end_b ? 2 : 0) : 1 << ((c - j.c0) & 1);
  }
};

// What the MMA issuer has to know of a chunk, in a word: the warpgroups that work on it, those for
// which it is the first / last of the job, whether it opens / ends the job (Q), is scrubbed, and reads
// Q's second tile; kStop ends the kernel.
enum : uint32_t {
  kGroups = 3u, kBegins = 3u << 2, kEnds = 3u << 4, kOpens = 1u << 6, kCloses = 1u << 7, kScrubbed = 1u << 8, kRows = 1u << 9,
  kStop = 1u << 31
};
template <class C>
__device__ __forceinline__ uint32_t chunk_word(const Chunks<C>& it) {
  const Job& j = it.j;
  const uint32_t groups = it.groups();
  uint32_t ends;
  if (j.rows) ends = (it.c + 1 == j.end_a ? 1u : 0u) | (it.c + 1 == j.end_b ? 2u : 0u);
  else ends = it.c + 2 >= j.end ? 3u : 0u;
  const uint32_t begins = (j.rows ? it.first() : it.c < j.c0 + 2) ? 3u : 0u;
  return groups | begins << 2 | ends << 4 | (it.first() ? kOpens : 0u) | (it.last() ? kCloses : 0u) |
         (it.scrubbed() ? kScrubbed : 0u) | (j.rows ? kRows : 0u);
}

// Producer of the K ring (which also loads Q and writes the key masks and chunk words) or of the V ring.
// One function for both, and no loop unrolled: what the warps of a CTA run has to stay in the
// instruction cache together.
template <class C>
__device__ __forceinline__ void produce(const Args& a, Shared<C>& S, bool is_k, uint8_t* ring, uint8_t* sq,
                                        const CUtensorMap* map, const CUtensorMap* tmq) {
  const SfaTreeParams& p = a.p;
  const int lane = threadIdx.x & 31;
  const int slabs = is_k ? a.nkq : a.nkv, stages = is_k ? a.kst : a.vst;
  const int nb_log = C::kKeysLog - a.box_log, nb = 1 << nb_log;      // boxes of a chunk, 1 .. 128
  const int outside = p.num_pages * p.page_size;           // a row past the pool: zeros
  uint64_t* full = is_k ? S.k_full : S.v_full;
  uint64_t* empty = is_k ? S.k_empty : S.v_empty;
  Chunks<C> it(a, S);
  bool ok = true;
  int qi = 0, st = 0, phase = 1;
  while (ok && it.next()) {
    const int n = it.n, h = it.j.g.h, k0 = it.c * C::kKeys, left = it.j.g.q.kvc - k0;
    // the lane's box (the first of its boxes when there are more than 32)
    int row = box_row(p, it.j.g, k0 + ((lane & (nb - 1)) << a.box_log));
    if (is_k && it.first()) {
      if (lane == 0 && (ok = wt<C>(&S.q_empty, (qi & 1) ^ 1, a.status, 1))) {
        const int tiles = it.j.rows ? 2 : 1;
        mbar_arrive_expect_tx(&S.q_full, (uint32_t)(tiles * a.nkq * a.GB * a.NT * 128));
        int tile = a.two ? 2 * blockIdx.y : blockIdx.y;
#pragma unroll 1
        for (int x = 0; x < tiles * a.nkq; ++x) {
          const int s = x < a.nkq ? x : x - a.nkq;
          if (x == a.nkq) ++tile;
          tma_load_4d(sq + x * kQSlab, tmq, &S.q_full, s * 64, h * a.G + (tile % a.n_hg) * 128,
                      it.j.g.q.q0 + node_of_tile(a, tile), 0);
        }
      }
      ++qi;
    }
    if (lane == 0 && ok) ok = wt<C>(&empty[st], phase, a.status, is_k ? 2 : 3);
    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
    if (!ok) break;
    uint4 mask = make_uint4(~0u, ~0u, ~0u, ~0u);
    const bool there = __all_sync(0xffffffffu, row >= 0) && left >= C::kKeys && nb <= 32;
    if (is_k) {
      if (!there) {
        uint32_t m[4] = {0, 0, 0, 0};
#pragma unroll 1
        for (int i = 0; i < C::kKeys / 32; ++i) {
          const int key = 32 * i + lane;
          const uint32_t w = __ballot_sync(0xffffffffu, key < left && box_row(p, it.j.g, k0 + (key >> a.box_log << a.box_log)) >= 0);
          if (i == 0) m[0] = w;
          else if (i == 1) m[1] = w;
          else if (i == 2) m[2] = w;
          else m[3] = w;
        }
        mask = make_uint4(m[0], m[1], m[2], m[3]);
      }
      if (lane == 0) {
        S.mask[n % kRing] = mask;
        S.word[n % kRing] = chunk_word(it);
      }
    }
    if (lane == 0) mbar_arrive_expect_tx(&full[st], (uint32_t)(slabs * C::kSlab));
    __syncwarp();
    uint8_t* dst = ring + (size_t)st * slabs * C::kSlab;
#pragma unroll 1
    for (int i = lane; i < nb * slabs; i += 32) {
      const int b = i & (nb - 1), s = i >> nb_log;
      if (nb > 32) row = box_row(p, it.j.g, k0 + (b << a.box_log));
      tma_load_4d(dst + s * C::kSlab + (b << a.box_log) * 128, map, &full[st], s * 64, row >= 0 ? row : outside, h, 0);
    }
    if (!is_k && it.scrubbed() && lane == 0) mbar_arrive(&S.scrub_go[it.k % kRing]);
    if (++st == stages) {
      st = 0;
      phase ^= 1;
    }
  }
  if (is_k && ok && lane == 0 && wt<C>(&empty[st], phase, a.status, 2)) {
    S.word[(it.n + 1) % kRing] = kStop;
    mbar_arrive(&full[st]);
  }
}

// Value rows that must not enter a product.  Rows behind the cache are cleared (a stale row's NaN
// would turn 0 * NaN into NaN); of drafted rows, which not all query rows see, non-finite elements
// are cleared and noted, and the softmax warps add them to the rows that see them.
template <class C, typename T>
__device__ __forceinline__ void scrub(const Args& a, Shared<C>& S, uint8_t* sv) {
  const int lane = threadIdx.x & 31;
  Chunks<C> it(a, S);
  bool ok = true;
  while (ok && it.next()) {
    if (!it.scrubbed()) continue;
    const int slot = it.k % kRing, vs = it.n % a.vst;
    // the producer has passed the stage's use before: its barrier is in this use's phase
    if (!(ok = wtw<C>(&S.scrub_go[slot], (it.k / kRing) & 1, a.status, 4))) break;
    if (!(ok = wtw<C>(&S.v_full[vs], (it.n / a.vst) & 1, a.status, 5))) break;
    const int k0 = it.c * C::kKeys, left = it.j.g.q.kvc - k0, drafted = it.j.g.q.rows > 1 ? it.j.g.q.prefix - k0 : C::kKeys;
    if (lane < 4) S.bad[slot][lane] = 0;
    __syncwarp();
    // four rows at a time, eight lanes a row (a 16-byte group each)
    uint8_t* at = sv + (size_t)vs * a.nkv * C::kSlab + (lane & 7) * 16;
#pragma unroll 1
    for (int r = max(0, min(left, drafted)) & ~3; r < C::kKeys; r += 4) {
      const int key = r + (lane >> 3);
      bool found = false;
#pragma unroll 2
      for (int s = 0; s < a.nkv; ++s) {
        uint4* x = reinterpret_cast<uint4*>(at + s * C::kSlab + key * 128);
        if (key >= left) {
          *x = make_uint4(0, 0, 0, 0);
        } else if (key >= drafted) {
          const uint4 v = *x;
          if (any_nonfinite2<T>(v.x) | any_nonfinite2<T>(v.y) | any_nonfinite2<T>(v.z) | any_nonfinite2<T>(v.w)) {
            found = true;
            *x = make_uint4(v.x & ~nonfinite2<T>(v.x), v.y & ~nonfinite2<T>(v.y), v.z & ~nonfinite2<T>(v.z),
                            v.w & ~nonfinite2<T>(v.w));
          }
        }
      }
      const uint32_t f = __ballot_sync(0xffffffffu, found);
      if (f != 0 && lane == 0)
        S.bad[slot][r >> 5] |= ((f & 0xffu ? 1u : 0u) | (f & 0xff00u ? 2u : 0u) | (f & 0xff0000u ? 4u : 0u) |
                                (f & 0xff000000u ? 8u : 0u)) << (r & 31);
    }
    fence_proxy_async_smem();
    warp_arrive(&S.v_ready[slot]);
  }
}

// One lane of the converged warp.  Around MMAs the warp stays converged and their operands are uniform,
// so that they sit in uniform registers: an MMA issued from a branch on the lane number takes three
// times the code (the compiler makes every operand uniform first), and the kernel lives or dies by
// its instruction cache.
__device__ __forceinline__ bool elect() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ uint64_t desc(uint32_t hi, uint32_t lo) { return (uint64_t)hi << 32 | lo; }

// 32 lanes x 32 columns; the registers hold them after ld_wait32.
__device__ __forceinline__ void ld32(uint32_t taddr, float (&v)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
               : "r"(taddr));
}

// Waits for this thread's TMEM loads and makes their registers depend on it.
__device__ __forceinline__ void ld_wait32(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                 "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]),
                 "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]),
                 "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}

// Two fp32 lanes in one instruction.
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void untwo(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <typename T>
__device__ __forceinline__ void scale_packed(float& word, float f);
template <>
__device__ __forceinline__ void scale_packed<__nv_bfloat16>(float& word, float f) {
  const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&word));
  word = __uint_as_float(pack2<__nv_bfloat16>(v.x * f, v.y * f));
}
template <>
__device__ __forceinline__ void scale_packed<__half>(float& word, float f) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&word));
  word = __uint_as_float(pack2<__half>(v.x * f, v.y * f));
}

// O (o_cols columns) and P (p_cols columns of packed pairs) times fac, in TMEM.
template <typename T>
__device__ __noinline__ void rescale(uint32_t to, int o_cols, uint32_t tp, int p_cols, float fac) {
  tmem_st_wait();
#pragma unroll 1
  for (int y = 0; y < o_cols; y += 16) {
    float o[16];
    tmem_ld16(to + y, o);
    tmem_ld_wait();
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] *= fac;
    tmem_st16(to + y, o);
  }
#pragma unroll 1
  for (int y = 0; y < p_cols; y += 16) {
    float o[16];
    tmem_ld16(tp + y, o);
    tmem_ld_wait();
#pragma unroll
    for (int k = 0; k < 16; ++k) scale_packed<T>(o[k], fac);
    tmem_st16(tp + y, o);
  }
  tmem_st_wait();
}

// Non-finite elements that the scrub took out of V (rows `bad` of the 32 keys from k0 on), added to the
// query row if it sees them; `zero`: O holds nothing yet.
template <typename T>
__device__ __noinline__ void add_nonfinite(const Args& a, const Piece& g, int k0, uint32_t to, bool zero, uint32_t bad,
                                           uint32_t vis) {
  const SfaTreeParams& p = a.p;
  if (zero) {
    const float z[16] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int y = 0; y < a.dvp; y += 16) tmem_st16(to + y, z);
    tmem_st_wait();
  }
#pragma unroll 1
  for (; bad; bad &= bad - 1) {
    const int b = __ffs(bad) - 1;
    const bool sees = (vis >> b) & 1u;
    const int row = box_row(p, g, k0 + b);
    const T* v = static_cast<const T*>(p.v) + (int64_t)max(row, 0) * p.v_st + (int64_t)g.h * p.v_sh;
#pragma unroll 1
    for (int y = 0; y < a.dvp; y += 16) {
      float o[16];
      tmem_ld16(to + y, o);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = sees && y + i < p.d_v ? as_f(v[y + i]) : 0.f;
        if (!isfinite(e)) o[i] += e;
      }
      tmem_st16(to + y, o);
    }
    tmem_st_wait();
  }
}

// P of 32 keys, exp2(s c2 - m) with m in nm2's lanes negated, packed into 16 columns; their sum into `sum`.
template <typename T>
__device__ __forceinline__ void exps(const float (&s)[32], uint64_t c22, uint64_t nm2, uint64_t& sum, uint32_t tp) {
  float pk[16];
#pragma unroll
  for (int k = 0; k < 32; k += 2) {
    float p0, p1;
    untwo(fma2(two(s[k], s[k + 1]), c22, nm2), p0, p1);
    p0 = ex2(p0);
    p1 = ex2(p1);
    sum = add2(sum, two(p0, p1));
    pk[k / 2] = __uint_as_float(pack2<T>(p0, p1));
  }
  tmem_st16(tp, pk);
}

}  // namespace tree
}  // namespace sfa

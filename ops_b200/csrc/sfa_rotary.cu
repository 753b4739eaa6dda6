// sfa_rotary.cu — RMS norm of each head and rotary positions in one pass, forward
// and backward, and the same step stored straight into a paged kv cache.
//
//   n = x * rsqrt(mean(x^2) + eps) * w,   y = R(position) n
//   dn = R^T dy,  dx = r (dn w - x r^2 mean(dn w x)),  dw = sum_rows dn x r
//
// The angle of a pair is position * frequency.  The frequency is held as a
// 64-bit fraction of a turn, and what that leaves over as 63 bits more, so the
// product modulo one turn is taken in whole numbers (no table, no range reduction
// in floating point): positions of any size keep the accuracy of sincospif.
//
// Memory-bound: every row is read once and written once, in fp32 registers
// between.  A row is spread over L lanes, each with two runs of P elements, so
// that both members of its P pairs are in the lane (half layout: P of the lower
// and P of the upper half; interleaved: 2P neighbours).  P = 8 where 16-byte
// accesses allow it, else 4.  32/L rows of one token go through a warp at a time;
// the token's cosines and sines are computed once, a pair per lane, and handed
// around in shared memory.  Arithmetic is on pairs of fp32 (f32x2).
#include "sfa_common.cuh"
#include "sfa_internal.h"

#include <algorithm>
#include <string>

namespace sfa {
namespace rotary {

constexpr int kWarps = 8;
constexpr int kMaxDim = 1024;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// A frequency (radians per position) as a fraction of a turn: units of 2^-64, and the rest in units of 2^-127.
struct Step {
  uint64_t units;
  int64_t rest;
};
__device__ __forceinline__ Step turn_step(double f) {
  // f / 2 pi as hi + lo; 1 / 2 pi rounded to a double, and what that leaves over
  constexpr double k1 = 0.15915494309189535, k2 = -9.839338337591243e-18;
  const double g = fabs(f), hi = g * k1, lo = fma(g, k2, fma(g, k1, -hi));
  const double u = (hi - floor(hi)) * 18446744073709551616.0;               // exact, below 2^64
  const double whole = floor(u), v = (u - whole) + lo * 18446744073709551616.0, n = rint(v);
  Step s{__double2ull_rz(whole) + (uint64_t)__double2ll_rn(n), __double2ll_rn((v - n) * 9223372036854775808.0)};
  if (f < 0.0) s = Step{0 - s.units, -s.rest};
  return s;
}

// `far`: 64-bit positions, for which the rest counts (2^31 positions of half a unit are 2^-34 of a turn).
__device__ __forceinline__ void turn(Step step, int64_t pos, bool far, float amplitude, float& c, float& s) {
  uint64_t units = step.units * (uint64_t)pos;
  if (far) units += 2 * (uint64_t)__mul64hi(step.rest, pos);
  const int32_t hi = (int32_t)(units >> 32);
  sincospif((float)hi * 4.656612873077393e-10f, &s, &c);   // hi / 2^31 half turns
  c *= amplitude;
  s *= amplitude;
}

struct Grid {
  int ctas[3];        // CTAs of each tensor
  int heads_per[3];   // heads of one work item
  int chunks[3];      // items of one token
  float* partial;     // [CTAs][dim] sums of dweight, backward
};

__device__ __forceinline__ int64_t position_of(const SfaRotaryParams& p, int b, int t) {
  const int64_t o = b * p.p_sb + t * p.p_st;
  return p.pos64 ? __ldg(static_cast<const long long*>(p.positions) + o)
                 : (int64_t)__ldg(static_cast<const int32_t*>(p.positions) + o);
}

// Pool row of new token `t` of a paged tensor, -1 if it is not stored.  Called by a whole warp.
__device__ __forceinline__ int64_t pool_row(const SfaRotaryParams& p, int t) {
  int s = t, i = 0, n = 1;
  if (p.cu_seqlens) {
    // last sequence that starts at or before t: 32 bounds at a time
    const int lane = threadIdx.x & 31;
    int lo = 0, span = p.num_seqs;
#pragma unroll 1
    while (span > 1) {
      const int step = (span + 31) >> 5, at = lo + lane * step;
      const bool in = lane * step < span && __ldg(p.cu_seqlens + at) <= t;
      const int c = __popc(__ballot_sync(0xffffffffu, in));
      const int skip = c > 0 ? (c - 1) * step : 0;
      lo += skip;
      span = min(step, span - skip);
    }
    s = lo;
    if (p.num_seqs <= 0) return -1;
    const int q0 = __ldg(p.cu_seqlens + s);
    i = t - q0;
    n = __ldg(p.cu_seqlens + s + 1) - q0;
  }
  if (s >= p.num_seqs || i < 0 || i >= n) return -1;
  const int64_t at = (int64_t)__ldg(p.cache_seqlens + s) - n + i;
  if (at < 0) return -1;
  const int64_t col = at / p.page_size;
  if (col >= p.table_width) return -1;
  const int pg = __ldg(p.block_table + s * p.bt_stride + col);
  if (pg < 0 || pg >= p.num_pages) return -1;
  return (int64_t)pg * p.page_size + at % p.page_size;
}

// Two fp32 lanes in one register pair.
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 untwo(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t neg2(uint64_t a) { return a ^ 0x8000000080000000ull; }

// P consecutive elements, as they lie in memory.
template <typename T, int P>
struct Run {
  static constexpr int W = P * (int)sizeof(T) / 4;
  uint32_t w[W];
  __device__ __forceinline__ void read(const uint8_t* p) {   // from shared memory
    if (W == 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x; w[1] = v.y; w[W - 2] = v.z; w[W - 1] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x; w[1] = v.y;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if (W == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[W - 2], w[W - 1]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
};

// Asynchronous copy of N bytes (8 or 16) into shared memory.
template <int N>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  if (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d), "l"(src) : "memory");
}

template <typename T> __device__ __forceinline__ uint64_t widen(uint32_t w);
template <> __device__ __forceinline__ uint64_t widen<__nv_bfloat16>(uint32_t w) {
  return two(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ uint64_t widen<__half>(uint32_t w) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return two(f.x, f.y);
}
template <typename T> __device__ __forceinline__ uint32_t narrow(uint64_t v);
template <> __device__ __forceinline__ uint32_t narrow<__nv_bfloat16>(uint64_t v) {
  const float2 f = untwo(v);
  return pack_bf16x2_rn(f.x, f.y);
}
template <> __device__ __forceinline__ uint32_t narrow<__half>(uint64_t v) {
  const float2 f = untwo(v);
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The lane's pairs as (first members, second members), two pairs to a register pair: j holds pairs
// (2j, 2j+1) of the lane in the half layout and (j, j + P/2) interleaved, where it swaps the words'
// halves (its own inverse).
template <typename T, int P>
__device__ __forceinline__ void take(const Run<T, P>& lo, const Run<T, P>& hi, bool inter, uint64_t (&a)[P / 2],
                                     uint64_t (&b)[P / 2]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < P / 2; ++j) {
      const float x0 = __uint_as_float(lo.w[2 * j]), x1 = __uint_as_float(lo.w[2 * j + 1]);
      const float y0 = __uint_as_float(hi.w[2 * j]), y1 = __uint_as_float(hi.w[2 * j + 1]);
      a[j] = inter ? two(x0, y0) : two(x0, x1);
      b[j] = inter ? two(x1, y1) : two(y0, y1);
    }
  } else {
    const uint32_t sa = inter ? 0x5410u : 0x3210u, sb = inter ? 0x7632u : 0x7654u;
#pragma unroll
    for (int j = 0; j < P / 2; ++j) {
      a[j] = widen<T>(__byte_perm(lo.w[j], hi.w[j], sa));
      b[j] = widen<T>(__byte_perm(lo.w[j], hi.w[j], sb));
    }
  }
}
template <typename T, int P>
__device__ __forceinline__ void give(const uint64_t (&a)[P / 2], const uint64_t (&b)[P / 2], bool inter, Run<T, P>& lo,
                                     Run<T, P>& hi) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < P / 2; ++j) {
      const float2 x = untwo(a[j]), y = untwo(b[j]);
      lo.w[2 * j] = __float_as_uint(x.x);
      lo.w[2 * j + 1] = __float_as_uint(inter ? y.x : x.y);
      hi.w[2 * j] = __float_as_uint(inter ? x.y : y.x);
      hi.w[2 * j + 1] = __float_as_uint(y.y);
    }
  } else {
    const uint32_t sa = inter ? 0x5410u : 0x3210u, sb = inter ? 0x7632u : 0x7654u;
#pragma unroll
    for (int j = 0; j < P / 2; ++j) {
      const uint32_t x = narrow<T>(a[j]), y = narrow<T>(b[j]);
      lo.w[j] = __byte_perm(x, y, sa);
      hi.w[j] = __byte_perm(x, y, sb);
    }
  }
}

template <int L>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Row elements of a lane's unit: runs of P at lo and hi; the unit's first pair, -1 if it is not turned.
struct Unit {
  int lo, hi, pair;
};
template <int P>
__device__ __forceinline__ Unit unit_of(const SfaRotaryParams& p, bool turned, int u) {
  const int first = p.start / (2 * P), n = p.rot / (2 * P);
  Unit r{2 * P * u, 2 * P * u + P, -1};
  if (turned && u >= first && u < first + n) {
    r.pair = P * (u - first);
    if (!p.interleaved) {
      r.lo = p.start + r.pair;
      r.hi = r.lo + (p.rot >> 1);
    }
  }
  return r;
}

// Steps of a warp whose rows are under way at a time.
template <int NS>
constexpr int stages() {
  return NS == 1 ? 4 : 2;
}
// Bytes of the ring: every thread copies its own runs and reads them back, so it needs no barrier.
template <typename T, int P, int NS, bool BWD>
constexpr int ring_bytes() {
  return stages<NS>() * NS * (BWD ? 4 : 2) * P * (int)sizeof(T) * kWarps * 32;
}

// The steps of a warp: 32 / L heads of a token at a time, item by item.
struct Steps {
  uint32_t item, items, stride;
  int chunks, per, heads, b, tt, h, h1;
  int len, batch;
  __device__ __forceinline__ bool open() {
    if (item >= items) return false;
    const uint32_t tok = item / (uint32_t)chunks;
    h = (int)(item - tok * chunks) * per;
    h1 = min(h + per, heads);
    b = batch == 1 ? 0 : (int)(tok / (uint32_t)len);
    tt = (int)tok - b * len;
    return true;
  }
  // to the next step; `fresh`: of another item
  __device__ __forceinline__ bool next(int rpw, bool& fresh) {
    h += rpw;
    fresh = h >= h1;
    if (!fresh) return true;
    item += stride;
    return open();
  }
};

// L lanes per row, NS units per lane (unit s * L + lane).  The rows of the next steps are on their way
// into shared memory while one is worked on.  Loaded into registers instead, a step's rows leave nothing
// in flight while they are worked on: 763 us for norm, rotary and gradients of 4 x 8192 tokens of 64 + 4
// heads of 128, against 507 us here (436 us would be the five passes over q and k at copy rate; instruction
// issue is 74 % busy in the forward, 62 % in the backward).  Forward: 3 CTAs per SM (20 us more with 2; the
// backward's registers allow 2).
// Two units a lane (above 512 dims of 16 bits, 256 of fp32) do not fit: the backward spills 510 to 550 bytes a
// thread, the forward 44 to 72, and 28 of the 64 lane slots idle at 576 dims.  8192 tokens of 16 + 1 heads of 576:
// forward 119 us for 49 of bytes, the step with gradients 682 for 123; of 512: 76 for 44, 213 for 109.
// Dynamic shared memory: the ring, the turn steps of the rot / 2 pairs, their (cos, sin) for each warp's token.
template <typename T, int P, int L, int NS, bool BWD, bool INTER>
__global__ void __launch_bounds__(kWarps * 32, BWD || NS > 1 ? 2 : 3)
rotary_kernel(const __grid_constant__ SfaRotaryParams p, const __grid_constant__ Grid g) {
  constexpr int RPW = 32 / L, H = P / 2, R = P * (int)sizeof(T), S = stages<NS>(), K = NS * (BWD ? 4 : 2);
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = lane % L, sub = lane / L, pairs = p.rot >> 1;
  uint8_t* ring = smem + threadIdx.x * R;                      // run k of stage s at (s * K + k) * kWarps * 32 * R
  Step* steps = reinterpret_cast<Step*>(smem + ring_bytes<T, P, NS, BWD>());
  float2* cs = reinterpret_cast<float2*>(steps + pairs) + warp * pairs;
  int ti = 0, cta = blockIdx.x;
  while (cta >= g.ctas[ti]) cta -= g.ctas[ti++];
  const SfaRotaryTensor& t = p.t[ti];
  const bool turned = (t.flags & SFA_ROTARY_TURN) && p.rot > 0;
  constexpr bool inter = INTER;
  const bool norm = t.weight != nullptr;
  const bool paged = !BWD && (t.flags & SFA_ROTARY_PAGED);
  const int units = p.dim / (2 * P);

  Unit un[NS];
  bool has[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int u = s * L + col;
    has[s] = u < units;
    un[s] = unit_of<P>(p, turned, has[s] ? u : 0);
  }
  Steps at;
  at.items = (uint32_t)(p.batch * p.len) * g.chunks[ti];
  at.item = cta * kWarps + warp;
  at.stride = g.ctas[ti] * kWarps;
  at.chunks = g.chunks[ti];
  at.per = g.heads_per[ti];
  at.heads = t.heads;
  at.len = p.len;
  at.batch = p.batch;
  Steps ahead = at;
  bool more = ahead.open(), fresh = true, moved = true;
  const T* ax = nullptr;                                       // the lane's row at `ahead`
  const T* ady = nullptr;
  // a lane without a unit reads zeros: nobody copies into its part of the ring
#pragma unroll
  for (int s = 0; s < NS; ++s)
    if (!has[s])
#pragma unroll 1
      for (int i = 0; i < S * (K / NS); ++i)
        for (int b = 0; b < R; b += 4)
          *reinterpret_cast<uint32_t*>(ring + ((i / (K / NS)) * K + s * (K / NS) + i % (K / NS)) * kWarps * 32 * R + b) = 0;
  // asks for the rows of the step at `ahead`, into `stage`
  auto ask = [&](int stage) {
    if (more) {
      if (moved) {
        ax = static_cast<const T*>(t.x) + ahead.b * t.x_sb + ahead.tt * t.x_st + (ahead.h + sub) * t.x_sh;
        if (BWD) ady = static_cast<const T*>(t.dy) + ahead.b * t.dy_sb + ahead.tt * t.dy_st + (ahead.h + sub) * t.dy_sh;
      }
      const bool row = ahead.h + sub < ahead.h1;
      uint8_t* dst = ring + stage * K * kWarps * 32 * R;
#pragma unroll
      for (int s = 0; s < NS; ++s)
        if (row && has[s]) {
          copy_async<R>(dst + (s * (K / NS)) * kWarps * 32 * R, ax + un[s].lo);
          copy_async<R>(dst + (s * (K / NS) + 1) * kWarps * 32 * R, ax + un[s].hi);
          if (BWD) {
            copy_async<R>(dst + (s * (K / NS) + 2) * kWarps * 32 * R, ady + un[s].lo);
            copy_async<R>(dst + (s * (K / NS) + 3) * kWarps * 32 * R, ady + un[s].hi);
          }
        }
      more = ahead.next(RPW, moved);
      ax += RPW * t.x_sh;
      if (BWD) ady += RPW * t.dy_sh;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int i = 0; i < S - 1; ++i) ask(i);

  if (turned) {
#pragma unroll 1
    for (int i = threadIdx.x; i < pairs; i += kWarps * 32) steps[i] = turn_step(__ldg(p.frequencies + i));
    __syncthreads();
  }
  uint64_t wa[NS][H], wb[NS][H], da[NS][H], db[NS][H];         // weights and their gradients, as take() orders pairs
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int j = 0; j < H; ++j) {
      // the elements of the two pairs of register j
      const int a0 = un[s].lo + 2 * j, b0 = inter ? un[s].lo + 2 * j + 1 : un[s].hi + 2 * j;
      const int a1 = inter ? un[s].hi + 2 * j : un[s].lo + 2 * j + 1, b1 = un[s].hi + 2 * j + 1;
      da[s][j] = db[s][j] = 0;
      wa[s][j] = norm ? two(__ldg(t.weight + a0), __ldg(t.weight + a1)) : two(1.f, 1.f);
      wb[s][j] = norm ? two(__ldg(t.weight + b0), __ldg(t.weight + b1)) : two(1.f, 1.f);
    }

  const float inv_dim = 1.f / (float)p.dim;
  const int64_t y_sh = BWD ? t.dx_sh : t.y_sh;
  T* y = nullptr;
  bool stored = true;
  uint64_t c[NS][H], sn[NS][H];
  int stage = 0;
  bool have = at.open();
  int64_t pos_next = have && turned ? position_of(p, at.b, at.tt) : 0;
#pragma unroll 1
  while (have) {
    if (fresh) {
      const int b = at.b, tt = at.tt;
      const int64_t pos = pos_next;
      int64_t yo;
      if (BWD) {
        yo = b * t.dx_sb + tt * t.dx_st;
      } else if (paged) {
        const int64_t row = pool_row(p, tt);
        stored = row >= 0;
        yo = stored ? row * t.y_st : 0;
      } else {
        yo = b * t.y_sb + tt * t.y_st;
      }
      y = static_cast<T*>(BWD ? t.dx : t.y) + yo;
      if (turned) {
        __syncwarp();
#pragma unroll 1
        for (int i = lane; i < pairs; i += 32) {
          float cc, ss;
          turn(steps[i], pos, p.pos64, p.amplitude, cc, ss);
          cs[i] = make_float2(cc, ss);
        }
        __syncwarp();
        Steps then = at;                                       // the next item's position, on its way meanwhile
        then.item += then.stride;
        if (then.open()) pos_next = position_of(p, then.b, then.tt);
      }
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int j = 0; j < H; ++j) {
          c[s][j] = two(1.f, 1.f);
          sn[s][j] = 0;
          if (un[s].pair >= 0) {
            const float2 u = cs[un[s].pair + (inter ? j : 2 * j)], v = cs[un[s].pair + (inter ? j + H : 2 * j + 1)];
            c[s][j] = two(u.x, v.x);
            sn[s][j] = two(u.y, v.y);
          }
        }
    }
    const int ask_at = stage == 0 ? S - 1 : stage - 1;         // the stage that the step before has left
    ask(ask_at);
    asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
    const uint8_t* src = ring + stage * K * kWarps * 32 * R;
    const int h = at.h + sub;
    uint64_t va[NS][H], vb[NS][H], ga[NS][H], gb[NS][H];
    uint64_t sq = 0, sd = 0;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      // rows past the heads are worked on too (what lies in the ring), and not stored
      Run<T, P> lo, hi;
      lo.read(src + (s * (K / NS)) * kWarps * 32 * R);
      hi.read(src + (s * (K / NS) + 1) * kWarps * 32 * R);
      take<T, P>(lo, hi, inter, va[s], vb[s]);
      if (BWD) {
        lo.read(src + (s * (K / NS) + 2) * kWarps * 32 * R);
        hi.read(src + (s * (K / NS) + 3) * kWarps * 32 * R);
        take<T, P>(lo, hi, inter, ga[s], gb[s]);
        if (un[s].pair >= 0) {
#pragma unroll
          for (int j = 0; j < H; ++j) {
            const uint64_t u = fma2(gb[s][j], sn[s][j], mul2(ga[s][j], c[s][j]));
            gb[s][j] = fma2(neg2(ga[s][j]), sn[s][j], mul2(gb[s][j], c[s][j]));
            ga[s][j] = u;
          }
        }
      }
      if (norm) {
#pragma unroll
        for (int j = 0; j < H; ++j) {
          sq = fma2(va[s][j], va[s][j], sq);
          sq = fma2(vb[s][j], vb[s][j], sq);
          if (BWD) {
            sd = fma2(mul2(ga[s][j], wa[s][j]), va[s][j], sd);
            sd = fma2(mul2(gb[s][j], wb[s][j]), vb[s][j], sd);
          }
        }
      }
    }
    float rn = 1.f, k = 0.f;
    if (norm) {
      const float2 q2 = untwo(sq), d2 = untwo(sd);
      rn = rsqrtf(row_sum<L>(q2.x + q2.y) * inv_dim + p.eps);
      if (BWD) k = row_sum<L>(d2.x + d2.y) * inv_dim * rn * rn * rn;
    }
    const uint64_t rn2 = two(rn, rn), k2 = two(-k, -k);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      if (!(h < at.h1 && has[s])) continue;
      uint64_t oa[H], ob[H];
#pragma unroll
      for (int j = 0; j < H; ++j) {
        if (BWD && norm) {
          da[s][j] = fma2(ga[s][j], mul2(va[s][j], rn2), da[s][j]);
          db[s][j] = fma2(gb[s][j], mul2(vb[s][j], rn2), db[s][j]);
          oa[j] = fma2(va[s][j], k2, mul2(mul2(ga[s][j], wa[s][j]), rn2));
          ob[j] = fma2(vb[s][j], k2, mul2(mul2(gb[s][j], wb[s][j]), rn2));
        } else if (BWD) {
          oa[j] = ga[s][j];
          ob[j] = gb[s][j];
        } else {
          oa[j] = norm ? mul2(mul2(va[s][j], rn2), wa[s][j]) : va[s][j];
          ob[j] = norm ? mul2(mul2(vb[s][j], rn2), wb[s][j]) : vb[s][j];
        }
      }
      if (!BWD && un[s].pair >= 0) {
#pragma unroll
        for (int j = 0; j < H; ++j) {
          const uint64_t u = fma2(neg2(ob[j]), sn[s][j], mul2(oa[j], c[s][j]));
          ob[j] = fma2(oa[j], sn[s][j], mul2(ob[j], c[s][j]));
          oa[j] = u;
        }
      }
      if (stored) {
        Run<T, P> lo, hi;
        give<T, P>(oa, ob, inter, lo, hi);
        lo.store(y + h * y_sh + un[s].lo);
        hi.store(y + h * y_sh + un[s].hi);
      }
    }
    if (++stage == S) stage = 0;
    have = at.next(RPW, fresh);
  }

  if (BWD && t.dweight != nullptr) {
    // the CTA's sum of each column, rows in a fixed order
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    float* part = reinterpret_cast<float*>(smem);              // [kWarps][dim], over the ring
    __syncthreads();
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int j = 0; j < H; ++j) {
        const int a0 = un[s].lo + 2 * j, b0 = inter ? un[s].lo + 2 * j + 1 : un[s].hi + 2 * j;
        const int a1 = inter ? un[s].hi + 2 * j : un[s].lo + 2 * j + 1, b1 = un[s].hi + 2 * j + 1;
        const float2 va = untwo(da[s][j]), vb = untwo(db[s][j]);
        float v[4] = {va.x, va.y, vb.x, vb.y};
        const int at[4] = {a0, a1, b0, b1};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int o = L; o < 32; o <<= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
          if (sub == 0 && has[s]) part[warp * p.dim + at[i]] = v[i];
        }
      }
    __syncthreads();
    for (int i = threadIdx.x; i < p.dim; i += kWarps * 32) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v += part[w * p.dim + i];
      g.partial[(int64_t)blockIdx.x * p.dim + i] = v;
    }
  }
}

// Any head size, offset, stride and alignment: one warp per row, one element at
// a time, a pair in one lane, the angle of every pair anew for every head.  Bound by
// that: 16384 tokens of 16 + 4 heads of 80 with 20 dims turned take 205 us forward and
// 562 with gradients, with 32 turned (the kernel above) 43 and 110.
template <typename T, bool BWD>
__global__ void __launch_bounds__(kWarps * 32)
rotary_any_kernel(const __grid_constant__ SfaRotaryParams p, const __grid_constant__ Grid g) {
  extern __shared__ float part[];   // [kWarps][dim], backward
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int ti = 0, cta = blockIdx.x;
  while (cta >= g.ctas[ti]) cta -= g.ctas[ti++];
  const SfaRotaryTensor& t = p.t[ti];
  const bool norm = t.weight != nullptr;
  const bool paged = !BWD && (t.flags & SFA_ROTARY_PAGED);
  const int rot = (t.flags & SFA_ROTARY_TURN) ? p.rot : 0;
  const int half = rot / 2, plain = p.dim - rot;
  float* mine = part + warp * p.dim;
  if (BWD)
    for (int i = lane; i < p.dim; i += 32) mine[i] = 0.f;
  __syncwarp();
  const int64_t items = (int64_t)p.batch * p.len * t.heads;
  for (int64_t item = (int64_t)cta * kWarps + warp; item < items; item += (int64_t)g.ctas[ti] * kWarps) {
    const int64_t tok = item / t.heads;
    const int h = (int)(item - tok * t.heads);
    const int b = (int)(tok / p.len), tt = (int)(tok - (int64_t)b * p.len);
    const T* x = static_cast<const T*>(t.x) + b * t.x_sb + tt * t.x_st + h * t.x_sh;
    const T* dy = BWD ? static_cast<const T*>(t.dy) + b * t.dy_sb + tt * t.dy_st + h * t.dy_sh : nullptr;
    T* y;
    if (BWD) {
      y = static_cast<T*>(t.dx) + b * t.dx_sb + tt * t.dx_st + h * t.dx_sh;
    } else if (paged) {
      const int64_t row = pool_row(p, tt);
      if (row < 0) continue;
      y = static_cast<T*>(t.y) + row * t.y_st + h * t.y_sh;
    } else {
      y = static_cast<T*>(t.y) + b * t.y_sb + tt * t.y_st + h * t.y_sh;
    }
    const int64_t pos = half ? position_of(p, b, tt) : 0;
    // element i of pair or plain slot j: pairs first, then the dims that are not turned
    auto cols = [&](int j, int& a, int& bb) {
      if (j < half) {
        a = p.start + (p.interleaved ? 2 * j : j);
        bb = a + (p.interleaved ? 1 : half);
      } else {
        a = j - half < p.start ? j - half : j - half + rot;
        bb = -1;
      }
    };
    auto grad = [&](int j, int a, int bb, float& da, float& db) {
      da = to_f(dy[a]);
      db = bb >= 0 ? to_f(dy[bb]) : 0.f;
      if (j < half) {
        float c, s;
        turn(turn_step(__ldg(p.frequencies + j)), pos, p.pos64, p.amplitude, c, s);
        const float u = da * c + db * s, v = db * c - da * s;
        da = u;
        db = v;
      }
    };
    float rn = 1.f, k = 0.f;
    if (norm) {
      float sq = 0.f, sd = 0.f;
      for (int j = lane; j < half + plain; j += 32) {
        int a, bb;
        cols(j, a, bb);
        const float xa = to_f(x[a]), xb = bb >= 0 ? to_f(x[bb]) : 0.f;
        sq += xa * xa + xb * xb;
        if (BWD) {
          float da, db;
          grad(j, a, bb, da, db);
          sd += da * __ldg(t.weight + a) * xa + (bb >= 0 ? db * __ldg(t.weight + bb) * xb : 0.f);
        }
      }
      rn = rsqrtf(row_sum<32>(sq) / (float)p.dim + p.eps);
      if (BWD) k = row_sum<32>(sd) / (float)p.dim * rn * rn;
    }
    for (int j = lane; j < half + plain; j += 32) {
      int a, bb;
      cols(j, a, bb);
      const float wa = norm ? __ldg(t.weight + a) : 1.f, wb = norm && bb >= 0 ? __ldg(t.weight + bb) : 1.f;
      const float xa = to_f(x[a]), xb = bb >= 0 ? to_f(x[bb]) : 0.f;
      float oa, ob;
      if (BWD) {
        float da, db;
        grad(j, a, bb, da, db);
        oa = norm ? rn * (da * wa - xa * k) : da;
        ob = norm ? rn * (db * wb - xb * k) : db;
        mine[a] += da * xa * rn;
        if (bb >= 0) mine[bb] += db * xb * rn;
      } else {
        const float na = xa * rn * wa, nb = xb * rn * wb;
        oa = na;
        ob = nb;
        if (j < half) {
          float c, s;
          turn(turn_step(__ldg(p.frequencies + j)), pos, p.pos64, p.amplitude, c, s);
          oa = na * c - nb * s;
          ob = nb * c + na * s;
        }
      }
      y[a] = from_f<T>(oa);
      if (bb >= 0) y[bb] = from_f<T>(ob);
    }
  }
  if (BWD && t.dweight != nullptr) {
    __syncthreads();
    for (int i = threadIdx.x; i < p.dim; i += kWarps * 32) {
      float v = 0.f;
      for (int k = 0; k < kWarps; ++k) v += part[k * p.dim + i];
      g.partial[(int64_t)blockIdx.x * p.dim + i] = v;
    }
  }
}

// dweight = the CTAs' partial sums, added in CTA order.  One CTA per tensor and 32 columns.
__global__ void rotary_dweight_kernel(const __grid_constant__ SfaRotaryParams p, const __grid_constant__ Grid g) {
  __shared__ float part[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x, ti = blockIdx.y;
  float* dw = p.t[ti].dweight;
  if (dw == nullptr) return;
  int first = 0;
  for (int i = 0; i < ti; ++i) first += g.ctas[i];
  float v = 0.f;
  if (col < p.dim)
    for (int r = threadIdx.y; r < g.ctas[ti]; r += 32) v += g.partial[(int64_t)(first + r) * p.dim + col];
  part[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && col < p.dim) {
    v = 0.f;
    for (int r = 0; r < 32; ++r) v += part[r][threadIdx.x];
    dw[col] = v;
  }
}

// How a call runs: P elements a run (0: the kernel for any shape), L lanes a row, NS units a lane.
struct Shape {
  int p, lanes, units;
};

// The widest runs that sizes and alignment allow: every run of P elements starts at a multiple of P, so head
// size, rotated part and its start are multiples of 8 at least, in every tensor of the call.
static Shape shape_of(const SfaRotaryParams& p, bool bwd) {
  const int size = p.dtype == SFA_DTYPE_F32 ? 4 : 2;
  auto fits = [&](int n) {
    if (p.dim % (2 * n) || p.rot % (2 * n) || p.start % (2 * n)) return false;
    auto ok = [&](const void* ptr, int64_t sb, int64_t st, int64_t sh) {
      return reinterpret_cast<uintptr_t>(ptr) % (n * size) == 0 && sb % n == 0 && st % n == 0 && sh % n == 0;
    };
    for (int i = 0; i < p.num_tensors; ++i) {
      const SfaRotaryTensor& t = p.t[i];
      if (!ok(t.x, t.x_sb, t.x_st, t.x_sh)) return false;
      if (!bwd && !ok(t.y, t.y_sb, t.y_st, t.y_sh)) return false;
      if (bwd && (!ok(t.dy, t.dy_sb, t.dy_st, t.dy_sh) || !ok(t.dx, t.dx_sb, t.dx_st, t.dx_sh))) return false;
    }
    return true;
  };
  Shape s{0, 32, 1};
  if (size == 2 && fits(8)) s.p = 8;
  else if (fits(4)) s.p = 4;
  if (!s.p) return s;
  const int units = p.dim / (2 * s.p);
  s.lanes = units <= 4 ? 4 : units <= 8 ? 8 : units <= 16 ? 16 : 32;
  s.units = (units + 31) / 32;
  if (s.p == 4 && s.units > 1) s.units = 4;        // P 4: up to 128 units
  return s;
}

// Items of up to 32 warp steps share one token's cosines; fewer when there would
// be too few items to fill the SMs (a decode step), down to one step each.
// The CTAs are shared out by work, an item's cosines counted as four steps: by heads alone, the few CTAs of
// a lone kv head ran 100 us behind the others.  Two CTAs per SM where each warp has few items (5003 tokens of
// 10 + 2 heads: 41 us, against 47 with eight), up to eight where that leaves it four (86 us less than with
// three for 32768 tokens), so that the SMs finish together.
static Grid make_grid(const SfaRotaryParams& p, const Shape& s) {
  Grid g{};
  const int sms = device_sm_count(), rpw = s.p ? 32 / s.lanes : 1;
  const int64_t tokens = (int64_t)p.batch * p.len;
  int64_t heads = 0;
  for (int i = 0; i < p.num_tensors; ++i) heads += p.t[i].heads;
  const int64_t steps = std::max<int64_t>(1, tokens * ((heads + rpw - 1) / rpw));
  const int per = (int)std::min<int64_t>(32, std::max<int64_t>(1, steps / ((int64_t)sms * 8)));
  int64_t cost[3], total = 0;
  for (int i = 0; i < p.num_tensors; ++i) {
    g.heads_per[i] = s.p ? std::min(p.t[i].heads, per * rpw) : 1;
    g.chunks[i] = (p.t[i].heads + g.heads_per[i] - 1) / g.heads_per[i];
    cost[i] = (p.t[i].heads + rpw - 1) / rpw + 4 * g.chunks[i];
    total += cost[i];
  }
  int64_t items = 0;
  for (int i = 0; i < p.num_tensors; ++i) items += tokens * g.chunks[i];
  const int64_t most =
      sms * std::min<int64_t>(8, std::max<int64_t>(2, items / ((int64_t)sms * kWarps * 4)));
  for (int i = 0; i < p.num_tensors; ++i) {
    const int64_t ctas = (tokens * g.chunks[i] + kWarps - 1) / kWarps;
    const int64_t share = std::max<int64_t>(1, most * cost[i] / total);
    g.ctas[i] = (int)std::min(ctas, share);
  }
  return g;
}

static int total_ctas(const SfaRotaryParams& p, const Grid& g) {
  int n = 0;
  for (int i = 0; i < p.num_tensors; ++i) n += g.ctas[i];
  return n;
}

template <typename T, int P, int L, int NS, bool BWD, bool INTER>
static void launch_layout(const SfaRotaryParams& p, const Grid& g, cudaStream_t st) {
  const size_t turns = (size_t)(p.rot / 2) * (sizeof(Step) + kWarps * sizeof(float2));   // at most 40 KB
  const size_t smem = std::max(ring_bytes<T, P, NS, BWD>() + turns, BWD ? kWarps * sizeof(float) * p.dim : (size_t)0);
  if (smem > 48 * 1024)
    cudaFuncSetAttribute(rotary_kernel<T, P, L, NS, BWD, INTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  rotary_kernel<T, P, L, NS, BWD, INTER><<<total_ctas(p, g), kWarps * 32, smem, st>>>(p, g);
}

template <typename T, int P, int L, int NS, bool BWD>
static void launch_shape(const SfaRotaryParams& p, const Grid& g, cudaStream_t st) {
  if (p.interleaved) launch_layout<T, P, L, NS, BWD, true>(p, g, st);
  else launch_layout<T, P, L, NS, BWD, false>(p, g, st);
}

template <typename T, int P, bool BWD>
static void launch_runs(const SfaRotaryParams& p, const Grid& g, const Shape& s, cudaStream_t st) {
  if (s.units > 1) return launch_shape<T, P, 32, P == 8 ? 2 : 4, BWD>(p, g, st);   // above 512 (256) dims
  if (s.lanes == 4) return launch_shape<T, P, 4, 1, BWD>(p, g, st);
  if (s.lanes == 8) return launch_shape<T, P, 8, 1, BWD>(p, g, st);
  if (s.lanes == 16) return launch_shape<T, P, 16, 1, BWD>(p, g, st);
  launch_shape<T, P, 32, 1, BWD>(p, g, st);
}

template <typename T, bool BWD>
static void launch_typed(const SfaRotaryParams& p, const Grid& g, const Shape& s, cudaStream_t st) {
  if (s.p == 0) {
    rotary_any_kernel<T, BWD><<<total_ctas(p, g), kWarps * 32, BWD ? sizeof(float) * kWarps * p.dim : 0, st>>>(p, g);
    return;
  }
  if constexpr (sizeof(T) == 2) {
    if (s.p == 8) return launch_runs<T, 8, BWD>(p, g, s, st);
  }
  launch_runs<T, 4, BWD>(p, g, s, st);
}

template <bool BWD>
static void launch(const SfaRotaryParams& p, const Grid& g, const Shape& s, cudaStream_t st) {
  if (p.dtype == SFA_DTYPE_BF16) launch_typed<__nv_bfloat16, BWD>(p, g, s, st);
  else if (p.dtype == SFA_DTYPE_F16) launch_typed<__half, BWD>(p, g, s, st);
  else launch_typed<float, BWD>(p, g, s, st);
}

static int bad(const std::string& m) { return report_error(SFA_ERR_INVALID_ARGUMENT, "rotary: " + m); }

static int check(const SfaRotaryParams* p, bool bwd) {
  if (!p) return bad("params is NULL");
  if (p->num_tensors < 1 || p->num_tensors > 3) return bad("num_tensors must be 1, 2 or 3");
  if (p->batch < 0 || p->len < 0) return bad("batch and len must be >= 0");
  if (p->dim < 1 || p->dim > kMaxDim) return bad("dim must be in [1, " + std::to_string(kMaxDim) + "]");
  if (p->rot < 0 || p->rot % 2 || p->rot > p->dim || p->start < 0 || p->start > p->dim - p->rot)
    return bad("rot must be even and [start, start + rot) within the head");
  if (p->dtype != SFA_DTYPE_BF16 && p->dtype != SFA_DTYPE_F16 && p->dtype != SFA_DTYPE_F32) return bad("unknown dtype");
  const bool empty = p->batch == 0 || p->len == 0;
  for (int i = 0; i < p->num_tensors; ++i) {
    const SfaRotaryTensor& t = p->t[i];
    if (t.heads < 1) return bad("heads must be positive");
    if (!empty && (int64_t)p->batch * p->len >= INT32_MAX / t.heads) return bad("a tensor must have fewer than 2^31 rows");
    const bool no_pool = (t.flags & SFA_ROTARY_PAGED) && p->num_pages == 0;
    if (!empty && (!t.x || (bwd ? !t.dy || !t.dx : !t.y && !no_pool))) return bad("tensor pointers must be non-NULL");
    if (!empty && (t.flags & SFA_ROTARY_TURN) && p->rot && (!p->positions || !p->frequencies))
      return bad("positions and frequencies must be non-NULL");
    if (bwd && t.dweight && !t.weight) return bad("dweight needs a weight");
    if (t.flags & SFA_ROTARY_PAGED) {
      if (bwd) return report_error(SFA_ERR_UNSUPPORTED, "rotary: a paged tensor is a forward format: no backward");
      if (p->batch != 1 && !empty) return bad("a paged tensor needs batch 1");
      if (p->page_size < 1 || p->num_pages < 0 || p->table_width < 0 || p->num_seqs < 0)
        return bad("page_size must be positive and num_pages, table_width, num_seqs >= 0");
      if (!empty && p->num_seqs > 0 && ((p->table_width > 0 && !p->block_table) || !p->cache_seqlens))
        return bad("a paged tensor needs block_table and cache_seqlens");
    }
  }
  return SFA_OK;
}

}  // namespace rotary
}  // namespace sfa

using namespace sfa;

extern "C" {

int sfa_rotary_fwd(const SfaRotaryParams* p, void* stream) {
  const int rc = rotary::check(p, false);
  if (rc) return rc;
  if (p->batch == 0 || p->len == 0) return SFA_OK;
  const rotary::Shape shape = rotary::shape_of(*p, false);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  rotary::launch<false>(*p, rotary::make_grid(*p, shape), shape, st);
  note_launch("rotary_fwd", st);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return report_error(SFA_ERR_CUDA, std::string("rotary forward: ") + cudaGetErrorString(e));
  return SFA_OK;
}

size_t sfa_rotary_bwd_workspace_bytes(const SfaRotaryParams* p) {
  if (rotary::check(p, true) || p->batch == 0 || p->len == 0) return 0;
  const rotary::Grid g = rotary::make_grid(*p, rotary::shape_of(*p, true));
  return sizeof(float) * (size_t)rotary::total_ctas(*p, g) * p->dim;
}

int sfa_rotary_bwd(const SfaRotaryParams* p, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = rotary::check(p, true);
  if (rc) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  bool dw = false;
  for (int i = 0; i < p->num_tensors; ++i) dw = dw || p->t[i].dweight;
  if (p->batch == 0 || p->len == 0) {
    for (int i = 0; i < p->num_tensors && e == cudaSuccess; ++i)
      if (p->t[i].dweight) e = cudaMemsetAsync(p->t[i].dweight, 0, sizeof(float) * p->dim, st);
  } else {
    const rotary::Shape shape = rotary::shape_of(*p, true);
    rotary::Grid g = rotary::make_grid(*p, shape);
    if (dw && (!workspace || workspace_bytes < sizeof(float) * (size_t)rotary::total_ctas(*p, g) * p->dim))
      return report_error(SFA_ERR_WORKSPACE, "rotary: workspace missing or too small");
    g.partial = static_cast<float*>(workspace);
    rotary::launch<true>(*p, g, shape, st);
    note_launch("rotary_bwd", st);
    e = cudaGetLastError();
    if (dw && e == cudaSuccess) {
      rotary::rotary_dweight_kernel<<<dim3((p->dim + 31) / 32, p->num_tensors), dim3(32, 32), 0, st>>>(*p, g);
      note_launch("rotary_dweight", st);
      e = cudaGetLastError();
    }
  }
  if (e != cudaSuccess) return report_error(SFA_ERR_CUDA, std::string("rotary backward: ") + cudaGetErrorString(e));
  return SFA_OK;
}

}  // extern "C"

// sfa_rotary.cu — RMS norm of each head and rotary positions in one pass, forward
// and backward, and the same step stored straight into a paged kv cache.
//
//   n = x * rsqrt(mean(x^2) + eps) * w,   y = R(position) n
//   dn = R^T dy,  dx = r (dn w - x r^2 mean(dn w x)),  dw = sum_rows dn x r
//
// The angle of a pair is position * frequency.  The frequency is held as a
// 64-bit fraction of a turn, so the product modulo 2^64 is the exact fraction
// of the turn (no table, no range reduction in floating point): positions of
// any size keep the accuracy of sincospif.
//
// Memory-bound: every row is read once and written once, in fp32 registers
// between.  A row is spread over L lanes (8 elements each: four of the lower
// and four of the upper half of the rotated part, so that both members of a
// pair are in one lane); 32/L rows of one token go through a warp at a time and
// share the token's cosines, several of them in flight.
#include "sfa_common.cuh"
#include "sfa_internal.h"

#include <algorithm>
#include <string>

namespace sfa {
namespace rotary {

constexpr int kWarps = 8;
constexpr int kMaxDim = 1024;

// Four consecutive elements as fp32.
template <typename T>
struct Quad;
template <>
struct Quad<float> {
  float4 r;
  __device__ __forceinline__ void load(const float* p) { r = __ldg(reinterpret_cast<const float4*>(p)); }
  __device__ __forceinline__ void get(float* v) const { v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w; }
  static __device__ __forceinline__ void store(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <>
struct Quad<__nv_bfloat16> {
  uint2 r;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { r = __ldg(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ void get(float* v) const {
    v[0] = __uint_as_float(r.x << 16); v[1] = __uint_as_float(r.x & 0xffff0000u);
    v[2] = __uint_as_float(r.y << 16); v[3] = __uint_as_float(r.y & 0xffff0000u);
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float* v) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2_rn(v[0], v[1]), pack_bf16x2_rn(v[2], v[3]));
  }
};
template <>
struct Quad<__half> {
  uint2 r;
  __device__ __forceinline__ void load(const __half* p) { r = __ldg(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ void get(float* v) const {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  }
  static __device__ __forceinline__ void store(__half* p, const float* v) {
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// A frequency (radians per position) as a 64-bit fraction of a turn.
__device__ __forceinline__ uint64_t turn_step(double f) {
  double t = f * 0.15915494309189533577;
  t -= floor(t);
  return __double2ull_rn(t * 18446744073709551616.0);
}

__device__ __forceinline__ void turn(uint64_t step, int64_t pos, float amplitude, float& c, float& s) {
  const int32_t hi = (int32_t)((step * (uint64_t)pos) >> 32);
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

// The eight elements (lo .. lo+3, hi .. hi+3) of unit u and its first pair (-1: not turned).
struct Unit {
  int lo, hi, pair;
};
__device__ __forceinline__ Unit unit_of(const SfaRotaryParams& p, bool turned, int u) {
  const int first = p.start >> 3, n = p.rot >> 3;
  Unit r{8 * u, 8 * u + 4, -1};
  if (turned && u >= first && u < first + n) {
    r.pair = 4 * (u - first);
    if (!p.interleaved) {
      r.lo = p.start + r.pair;
      r.hi = r.lo + (p.rot >> 1);
    }
  }
  return r;
}

// Turn the unit's four pairs by (c, sgn * s).
__device__ __forceinline__ void turn_unit(float (&v)[8], const float (&c)[4], const float (&s)[4], float sgn,
                                          bool interleaved) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float sn = sgn * s[i];
    const float a = interleaved ? v[2 * i] : v[i], b = interleaved ? v[2 * i + 1] : v[i + 4];
    const float x = a * c[i] - b * sn, y = b * c[i] + a * sn;
    if (interleaved) { v[2 * i] = x; v[2 * i + 1] = y; }
    else { v[i] = x; v[i + 4] = y; }
  }
}

template <int L>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// L lanes per row, NS units of eight elements per lane (unit s * L + lane).
template <typename T, int L, int NS, bool BWD>
__global__ void __launch_bounds__(kWarps * 32)
rotary_kernel(const __grid_constant__ SfaRotaryParams p, const __grid_constant__ Grid g) {
  constexpr int RPW = 32 / L;
  constexpr int U = NS == 1 ? (sizeof(T) == 2 ? 4 : 2) : 1;   // rows of a lane in flight
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = lane % L, sub = lane / L;
  int ti = 0, cta = blockIdx.x;
  while (cta >= g.ctas[ti]) cta -= g.ctas[ti++];
  const SfaRotaryTensor& t = p.t[ti];
  const bool turned = (t.flags & SFA_ROTARY_TURN) && p.rot > 0;
  const bool norm = t.weight != nullptr;
  const bool paged = !BWD && (t.flags & SFA_ROTARY_PAGED);
  const int units = p.dim >> 3;

  Unit un[NS];
  bool has[NS];
  float w[NS][8], acc[NS][8];
  uint64_t step[NS][4];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int u = s * L + col;
    has[s] = u < units;
    un[s] = unit_of(p, turned, has[s] ? u : 0);
    if (!has[s]) un[s].pair = -1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      acc[s][i] = 0.f;
      w[s][i] = norm ? __ldg(t.weight + (i < 4 ? un[s].lo + i : un[s].hi + i - 4)) : 1.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) step[s][i] = un[s].pair >= 0 ? turn_step(__ldg(p.frequencies + un[s].pair + i)) : 0;
  }

  const float inv_dim = 1.f / (float)p.dim;
  const int64_t items = (int64_t)p.batch * p.len * g.chunks[ti];
  const int64_t stride = (int64_t)g.ctas[ti] * kWarps;
  for (int64_t item = (int64_t)cta * kWarps + warp; item < items; item += stride) {
    const int64_t tok = item / g.chunks[ti];
    const int h0 = (int)(item - tok * g.chunks[ti]) * g.heads_per[ti];
    const int h1 = min(h0 + g.heads_per[ti], t.heads);
    const int b = (int)(tok / p.len), tt = (int)(tok - (int64_t)b * p.len);
    const T* x = static_cast<const T*>(t.x) + b * t.x_sb + tt * t.x_st;
    int64_t yo;
    bool stored = true;
    if (BWD) {
      yo = b * t.dx_sb + tt * t.dx_st;
    } else if (paged) {
      const int64_t row = pool_row(p, tt);
      stored = row >= 0;
      yo = stored ? row * t.y_st : 0;
    } else {
      yo = b * t.y_sb + tt * t.y_st;
    }
    T* y = static_cast<T*>(BWD ? t.dx : t.y) + yo;
    const T* dy = BWD ? static_cast<const T*>(t.dy) + b * t.dy_sb + tt * t.dy_st : nullptr;
    const int64_t y_sh = BWD ? t.dx_sh : t.y_sh;
    float c[NS][4], sn[NS][4];
    const int64_t pos = turned ? position_of(p, b, tt) : 0;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[s][i] = 1.f;
        sn[s][i] = 0.f;
        if (un[s].pair >= 0) turn(step[s][i], pos, p.amplitude, c[s][i], sn[s][i]);
      }
    for (int hb = h0; hb < h1; hb += RPW * U) {
      Quad<T> xl[U][NS], xh[U][NS], gl[U][NS], gh[U][NS];
#pragma unroll
      for (int r = 0; r < U; ++r) {
        const int h = hb + r * RPW + sub;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          if (h < h1 && has[s]) {
            xl[r][s].load(x + h * t.x_sh + un[s].lo);
            xh[r][s].load(x + h * t.x_sh + un[s].hi);
            if (BWD) {
              gl[r][s].load(dy + h * t.dy_sh + un[s].lo);
              gh[r][s].load(dy + h * t.dy_sh + un[s].hi);
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < U; ++r) {
        const int h = hb + r * RPW + sub;
        float v[NS][8], d[NS][8];
        float sq = 0.f, sd = 0.f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const bool on = h < h1 && has[s];
#pragma unroll
          for (int i = 0; i < 8; ++i) { v[s][i] = 0.f; d[s][i] = 0.f; }
          if (on) {
            xl[r][s].get(v[s]);
            xh[r][s].get(v[s] + 4);
            if (BWD) {
              gl[r][s].get(d[s]);
              gh[r][s].get(d[s] + 4);
              if (un[s].pair >= 0) turn_unit(d[s], c[s], sn[s], -1.f, p.interleaved);
            }
          }
          if (norm) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              sq = fmaf(v[s][i], v[s][i], sq);
              if (BWD) sd = fmaf(d[s][i] * w[s][i], v[s][i], sd);
            }
          }
        }
        float rn = 1.f, k = 0.f;
        if (norm) {
          sq = row_sum<L>(sq);
          rn = rsqrtf(sq * inv_dim + p.eps);
          if (BWD) k = row_sum<L>(sd) * inv_dim * rn * rn;
        }
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          if (!(h < h1 && has[s])) continue;
          float o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (BWD) {
              if (norm) {
                acc[s][i] = fmaf(d[s][i], v[s][i] * rn, acc[s][i]);
                o[i] = rn * (d[s][i] * w[s][i] - v[s][i] * k);
              } else {
                o[i] = d[s][i];
              }
            } else {
              o[i] = v[s][i] * rn * w[s][i];
            }
          }
          if (!BWD && un[s].pair >= 0) turn_unit(o, c[s], sn[s], 1.f, p.interleaved);
          if (stored) {
            Quad<T>::store(y + h * y_sh + un[s].lo, o);
            Quad<T>::store(y + h * y_sh + un[s].hi, o + 4);
          }
        }
      }
    }
  }

  if (BWD && t.dweight != nullptr) {
    // the CTA's sum of each column, rows in a fixed order
    __shared__ float part[kWarps][NS * L * 8];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v = acc[s][i];
#pragma unroll
        for (int o = L; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (sub == 0 && has[s]) part[warp][i < 4 ? un[s].lo + i : un[s].hi + i - 4] = v;
      }
    __syncthreads();
    for (int i = threadIdx.x; i < p.dim; i += kWarps * 32) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) v += part[k][i];
      g.partial[(int64_t)blockIdx.x * p.dim + i] = v;
    }
  }
}

// Any head size, offset, stride and alignment: one warp per row, one element at
// a time, a pair in one lane.
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
        turn(turn_step(__ldg(p.frequencies + j)), pos, p.amplitude, c, s);
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
          turn(turn_step(__ldg(p.frequencies + j)), pos, p.amplitude, c, s);
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

static bool vector_ok(const SfaRotaryParams& p, bool bwd) {
  if (p.dim % 8 || p.rot % 8 || p.start % 8) return false;
  const uintptr_t bytes = p.dtype == SFA_DTYPE_F32 ? 16 : 8;   // four elements
  auto ok = [&](const void* ptr, int64_t sb, int64_t st, int64_t sh) {
    return reinterpret_cast<uintptr_t>(ptr) % bytes == 0 && sb % 4 == 0 && st % 4 == 0 && sh % 4 == 0;
  };
  for (int i = 0; i < p.num_tensors; ++i) {
    const SfaRotaryTensor& t = p.t[i];
    if (!ok(t.x, t.x_sb, t.x_st, t.x_sh)) return false;
    if (!bwd && !ok(t.y, t.y_sb, t.y_st, t.y_sh)) return false;
    if (bwd && (!ok(t.dy, t.dy_sb, t.dy_st, t.dy_sh) || !ok(t.dx, t.dx_sb, t.dx_st, t.dx_sh))) return false;
  }
  return true;
}

static int lanes_per_row(int dim) {
  int l = 2;
  while (l < 32 && l * 8 < dim) l *= 2;
  return l;
}

// Items of up to 32 warp steps share one token's cosines; fewer when there would
// be too few items to fill the SMs (a decode step), down to one step each.
static Grid make_grid(const SfaRotaryParams& p, bool vec) {
  Grid g{};
  const int sms = device_sm_count(), rpw = vec ? 32 / lanes_per_row(p.dim) : 1;
  const int64_t tokens = (int64_t)p.batch * p.len;
  int64_t heads = 0;
  for (int i = 0; i < p.num_tensors; ++i) heads += p.t[i].heads;
  const int64_t steps = std::max<int64_t>(1, tokens * ((heads + rpw - 1) / rpw));
  const int per = (int)std::min<int64_t>(32, std::max<int64_t>(1, steps / ((int64_t)sms * 32)));
  const int most = sms * 8;
  for (int i = 0; i < p.num_tensors; ++i) {
    g.heads_per[i] = vec ? std::min(p.t[i].heads, per * rpw) : 1;
    g.chunks[i] = (p.t[i].heads + g.heads_per[i] - 1) / g.heads_per[i];
    const int64_t ctas = (tokens * g.chunks[i] + kWarps - 1) / kWarps;
    const int64_t share = std::max<int64_t>(1, most * (int64_t)p.t[i].heads / heads);
    g.ctas[i] = (int)std::min(ctas, share);
  }
  return g;
}

static int total_ctas(const SfaRotaryParams& p, const Grid& g) {
  int n = 0;
  for (int i = 0; i < p.num_tensors; ++i) n += g.ctas[i];
  return n;
}

template <typename T, bool BWD>
static void launch_typed(const SfaRotaryParams& p, const Grid& g, bool vec, cudaStream_t st) {
  const int n = total_ctas(p, g);
  const int threads = kWarps * 32;
  if (!vec) {
    rotary_any_kernel<T, BWD><<<n, threads, BWD ? sizeof(float) * kWarps * p.dim : 0, st>>>(p, g);
    return;
  }
  const int l = lanes_per_row(p.dim);
  if (l == 2) rotary_kernel<T, 2, 1, BWD><<<n, threads, 0, st>>>(p, g);
  else if (l == 4) rotary_kernel<T, 4, 1, BWD><<<n, threads, 0, st>>>(p, g);
  else if (l == 8) rotary_kernel<T, 8, 1, BWD><<<n, threads, 0, st>>>(p, g);
  else if (l == 16) rotary_kernel<T, 16, 1, BWD><<<n, threads, 0, st>>>(p, g);
  else if (p.dim <= 256) rotary_kernel<T, 32, 1, BWD><<<n, threads, 0, st>>>(p, g);
  else if (p.dim <= 512) rotary_kernel<T, 32, 2, BWD><<<n, threads, 0, st>>>(p, g);
  else rotary_kernel<T, 32, 4, BWD><<<n, threads, 0, st>>>(p, g);
}

template <bool BWD>
static void launch(const SfaRotaryParams& p, const Grid& g, bool vec, cudaStream_t st) {
  if (p.dtype == SFA_DTYPE_BF16) launch_typed<__nv_bfloat16, BWD>(p, g, vec, st);
  else if (p.dtype == SFA_DTYPE_F16) launch_typed<__half, BWD>(p, g, vec, st);
  else launch_typed<float, BWD>(p, g, vec, st);
}

static int bad(const std::string& m) { return report_error(SFA_ERR_INVALID_ARGUMENT, "rotary: " + m); }

static int check(const SfaRotaryParams* p, bool bwd) {
  if (!p) return bad("params is NULL");
  if (p->num_tensors < 1 || p->num_tensors > 3) return bad("num_tensors must be 1, 2 or 3");
  if (p->batch < 0 || p->len < 0) return bad("batch and len must be >= 0");
  if (p->dim < 1 || p->dim > kMaxDim) return bad("dim must be in [1, " + std::to_string(kMaxDim) + "]");
  if (p->rot < 0 || p->rot % 2 || p->start < 0 || p->start + p->rot > p->dim)
    return bad("rot must be even and [start, start + rot) within the head");
  if (p->dtype != SFA_DTYPE_BF16 && p->dtype != SFA_DTYPE_F16 && p->dtype != SFA_DTYPE_F32) return bad("unknown dtype");
  const bool empty = p->batch == 0 || p->len == 0;
  for (int i = 0; i < p->num_tensors; ++i) {
    const SfaRotaryTensor& t = p->t[i];
    if (t.heads < 1) return bad("heads must be positive");
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
  const bool vec = rotary::vector_ok(*p, false);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  rotary::launch<false>(*p, rotary::make_grid(*p, vec), vec, st);
  note_launch("rotary_fwd", st);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return report_error(SFA_ERR_CUDA, std::string("rotary forward: ") + cudaGetErrorString(e));
  return SFA_OK;
}

size_t sfa_rotary_bwd_workspace_bytes(const SfaRotaryParams* p) {
  if (rotary::check(p, true) || p->batch == 0 || p->len == 0) return 0;
  const rotary::Grid g = rotary::make_grid(*p, rotary::vector_ok(*p, true));
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
    const bool vec = rotary::vector_ok(*p, true);
    rotary::Grid g = rotary::make_grid(*p, vec);
    if (dw && (!workspace || workspace_bytes < sizeof(float) * (size_t)rotary::total_ctas(*p, g) * p->dim))
      return report_error(SFA_ERR_WORKSPACE, "rotary: workspace missing or too small");
    g.partial = static_cast<float*>(workspace);
    rotary::launch<true>(*p, g, vec, st);
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

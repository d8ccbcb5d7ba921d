// Rotary positions with several axes, and the norms of queries and keys for each head with the rotation in the same pass.
//
//   theta[n, i] = positions[n, axis(i)] * inv_freq[i]                 (double: positions may be far)
//   rotation of pair i:  a' = a cos - b sin,  b' = a sin + b cos      (a, b) = channels (2i, 2i+1) or (i, i + P); the rest passes
//   norm of a head:      xh = x * rsqrt(mean_c x^2 + eps),  y = rotate(gain * xh)
//   its gradient, with dz = rotate^-1(dy), t = gain * dz, r = rsqrt(mean_c x^2 + eps):
//                        dgain = sum_n dz * xh,   dx = r (t - x r^2 mean_c(t x))
//
// Bound: HBM.  One read and one write of the rows (the backward of the norm: two reads, one write); statistics, angles and the gain
// gradient in float32, the angle's product and reduction in float64, one rounding where a row is stored.
//
// A workgroup takes a tile of tokens, four rows a lane.  All of them are requested first; while they are on their way the tile's cos / sin
// table is computed in LDS -- once per (token, pair), not once per head: 16 heads share it.  A lane owns 8 channels of one head (16-byte
// accesses in bf16), the lanes of a head are adjacent, and a lane keeps its head from token to token, so that its gains and its share of
// the gain gradient stay in registers.
//
// 375 k tokens of 16 heads of 16 in bf16 (192 MB): rotation 75 us (5.1 TB/s; 97 us with the table first and the rows after it), with the
// norm 72 us (5.4 TB/s; 91), gradient 117 us (4.9 TB/s; 139), where a large copy runs at 5.9 TB/s.
#include "common.h"
#include <type_traits>

namespace {

constexpr int MAX_AXES = 4;
constexpr int TABLE_PAIRS = 2048;          // cos / sin pairs of a tile: 16 KB of LDS

// how the pairs lie: (2i, 2i+1) or (i, i + P); P a multiple of 4 or any (the selects that another P takes cost 5 % where they are not needed)
enum { MODE_ADJACENT = 0, MODE_SPLIT = 1, MODE_SPLIT_ANY = 2, MODE_ADJACENT_ANY = 3 };

struct RotaryArgs {
  const void* x; int64_t ldx, hpx;         // [n, h, dh]: row pitch and head pitch in elements, channels contiguous
  const void* dy;                          // contiguous [n, h, dh] (backward)
  void* y;                                 // contiguous [n, h, dh] (dx in the backward)
  int64_t n; int h, q_heads, dh;
  const void* pos; int64_t ldpos; int pos_kind;                     // 0 int32, 1 int64, 2 float32
  const double* inv_freq; int P, PT;       // PT: pairs of a table row, P rounded up to 4
  int sec_end[MAX_AXES];                   // pairs [sec_end[a-1], sec_end[a]) turn by axis a
  float sign;                              // -1: the inverse rotation
  const float* q_gain; const float* k_gain; int gain_pitch;         // 0: one gain for all heads
  float eps;
  int U, lgG, HB, R, TB;                   // units (8 channels) of a head, log2 of its lanes, heads and token rows of a pass, tile
  float* part;                             // backward: partial rows of the gain gradient
};

// 2 / pi, the 32 bits before the binary point and 1120 behind it
__constant__ uint32_t TWO_OVER_PI[36] = {
    0x00000000u, 0xa2f9836eu, 0x4e441529u, 0xfc2757d1u, 0xf534ddc0u, 0xdb629599u, 0x3c439041u, 0xfe5163abu, 0xdebbc561u,
    0xb7246e3au, 0x424dd2e0u, 0x06492eeau, 0x09d1921cu, 0xfe1deb1cu, 0xb129a73eu, 0xe88235f5u, 0x2ebb4484u, 0xe99c7026u,
    0xb45f7e41u, 0x3991d639u, 0x835339f4u, 0x9c845f8bu, 0xbdf9283bu, 0x1ff897ffu, 0xde05980fu, 0xef2f118bu, 0x5a0a6d1fu,
    0x6d367ecfu, 0x27cb09b7u, 0x4f463f66u, 0x9e5fea2du, 0x7527bac7u, 0xebe5f17bu, 0x3d0739f7u, 0x8a5292eau, 0x6bfb5fb1u};
// theta = m 2^e in multiples of pi/2, for 2^22 <= |theta| (Payne and Hanek's reduction): bits of 2 / pi that make multiples of 4 with m 2^e are
// left out, the 128 behind them hold the multiple's last two bits and, after the product with m, 70 bits and more of its fraction.  Sets
// k to the multiple modulo 4 and returns the rest as an angle; no angle for infinities and NaN.
__device__ __forceinline__ double far_angle(double theta, int& k) {
  const uint64_t bits = (uint64_t)__double_as_longlong(theta);
  const int exponent = (int)(bits >> 52) & 0x7ff;
  if (exponent == 0x7ff) return __longlong_as_double(0x7ff8000000000000ll);
  const uint64_t m = (bits & 0xfffffffffffffull) | 0x10000000000000ull;
  const int first = exponent - 1075 + 30, word = first >> 5, shift = first & 31;       // the first bit that counts: at most 1001
  uint64_t hi = (uint64_t)TWO_OVER_PI[word] << 32 | TWO_OVER_PI[word + 1], lo = (uint64_t)TWO_OVER_PI[word + 2] << 32 | TWO_OVER_PI[word + 3];
  const uint64_t next = (uint64_t)TWO_OVER_PI[word + 4] << 32;
  if (shift) {
    hi = hi << shift | lo >> (64 - shift);
    lo = lo << shift | next >> (64 - shift);
  }
  hi = __umul64hi(m, lo) + m * hi;
  lo = m * lo;
  const int64_t fraction = (int64_t)(hi << 2 | lo >> 62);                            // above a half: the next multiple, and back from it
  const int n = (int)(hi >> 62) + (fraction < 0 ? 1 : 0);
  const double angle = (double)fraction * (1.57079632679489661923 * 0x1p-64);
  k = (theta < 0 ? -n : n) & 3;
  return theta < 0 ? -angle : angle;
}

// cos and sin of the float64 product pos * w to float32 accuracy, Taylor series on [-pi/4, pi/4] (first dropped terms 2e-9 and 1e-10).  Up to
// 2^45: k = the nearest multiple of pi/2 (near enough: the remainder leaves that interval by less than 0.01), the remainder by two fused
// multiply-adds with the two halves of pi/2, of which 2^-108 is missing.  Beyond, a double has no place for k.
__device__ __forceinline__ float2 cos_sin(double pos, double w) {
  const double theta = pos * w;
  double rem;
  int q = 0;
  if (fabs(theta) <= 0x1p45) {
    const double k = rint(theta * 0.63661977236758134308);
    rem = fma(-k, 1.57079632679489661923, theta);
    rem = fma(-k, 6.12323399573676603587e-17, rem);
    q = (int)(k - 4.0 * floor(k * 0.25));
  } else {
    rem = far_angle(theta, q);
  }
  const float x = (float)rem, x2 = x * x;
  float s = fmaf(x2, 2.755731922e-6f, -1.984126984e-4f);
  s = fmaf(x2, s, 8.333333333e-3f);
  s = fmaf(x2, s, -1.666666667e-1f);
  s = fmaf(x * x2, s, x);
  float c = fmaf(x2, -2.755731922e-7f, 2.480158730e-5f);
  c = fmaf(x2, c, -1.388888889e-3f);
  c = fmaf(x2, c, 4.166666667e-2f);
  c = fmaf(x2 * x2, c, fmaf(x2, -0.5f, 1.0f));
  const float cc = (q & 1) ? s : c, ss = (q & 1) ? c : s;
  return make_float2((q == 1 || q == 2) ? -cc : cc, (q >= 2) ? -ss : ss);
}

__device__ __forceinline__ void fill_table(const RotaryArgs& a, int64_t t0, int tokens, float2* table) {
  const int total = tokens * a.PT;
  for (int e = threadIdx.x; e < total; e += 256) {
    const int t = e / a.PT, i = e - t * a.PT;
    float2 cs = make_float2(1.f, 0.f);
    if (i < a.P) {
      int axis = 0;
#pragma unroll
      for (int k = 0; k + 1 < MAX_AXES; ++k) axis += (i >= a.sec_end[k]) ? 1 : 0;
      const int64_t at = (t0 + t) * a.ldpos + axis;
      const double p = a.pos_kind == 0 ? (double)reinterpret_cast<const int32_t*>(a.pos)[at]
                     : a.pos_kind == 1 ? (double)reinterpret_cast<const int64_t*>(a.pos)[at]
                                       : (double)reinterpret_cast<const float*>(a.pos)[at];
      cs = cos_sin(p, a.inv_freq[i]);
      cs.y *= a.sign;
    }
    table[e] = cs;
  }
}

// sum over the 2^lg adjacent lanes that hold a head (the branches are uniform)
__device__ __forceinline__ float lanes_sum(float v, int lg) {
  for (int k = 0; k < lg; ++k) v += __shfl_xor(v, 1 << k, 64);
  return v;
}

template <class T> __device__ __forceinline__ void store4(T* p, const float* v);
template <> __device__ __forceinline__ void store4<float>(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <> __device__ __forceinline__ void store4<__hip_bfloat16>(__hip_bfloat16* p, const float* v) {
  __hip_bfloat16 t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = __float2bfloat16(v[i]);
  *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(t);
}

// Where the 8 channels of unit u of a head lie.  MODE_SPLIT (pairs (i, i + P), P a multiple of 4): a unit below P / 4 owns four whole
// pairs -- channels 4u.. and P + 4u.. -- and the exchange between the halves needs no other lane.  Otherwise 8u .. 8u + 7.
template <int MODE> __device__ __forceinline__ bool turned_unit(const RotaryArgs& a, int u) { return MODE == MODE_SPLIT ? 4 * u < a.P : true; }
template <int MODE> __device__ __forceinline__ int first_channel(const RotaryArgs& a, int u) {
  return (MODE == MODE_SPLIT && 4 * u < a.P) ? 4 * u : 8 * u;
}
template <int MODE> __device__ __forceinline__ int channel_of(const RotaryArgs& a, int u, int e) {
  if (MODE == MODE_SPLIT && 4 * u < a.P) return 4 * u + (e & 3) + (e >> 2) * a.P;
  return 8 * u + e;
}

// a unit as it lies in memory: requested early, unpacked where it is used
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
template <class T, bool VEC> struct Raw { float v[8]; };
template <> struct Raw<float, true> { f32x4 lo, hi; };
template <> struct Raw<__hip_bfloat16, true> { u32x4 v; };
template <class T, int MODE, bool VEC>
__device__ __forceinline__ Raw<T, VEC> request_unit(const T* row, const RotaryArgs& a, int u) {
  Raw<T, VEC> r;
  if constexpr (VEC && sizeof(T) == 4) {
    const bool turned = MODE == MODE_SPLIT && 4 * u < a.P;
    const T* lo = row + (turned ? 4 * u : 8 * u);
    r.lo = *reinterpret_cast<const f32x4*>(lo);
    r.hi = *reinterpret_cast<const f32x4*>(lo + (turned ? a.P : 4));
  } else if constexpr (VEC) {
    if constexpr (MODE == MODE_SPLIT) {
      const bool turned = 4 * u < a.P;
      const T* lo = row + (turned ? 4 * u : 8 * u);
      const uint2 l = *reinterpret_cast<const uint2*>(lo), h = *reinterpret_cast<const uint2*>(lo + (turned ? a.P : 4));
      r.v = u32x4{l.x, l.y, h.x, h.y};
    } else {
      r.v = *reinterpret_cast<const u32x4*>(row + 8 * u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = 8 * u + e < a.dh ? ld_f<T>(row + 8 * u + e) : 0.f;
  }
  return r;
}
template <class T, bool VEC> __device__ __forceinline__ void unpack(const Raw<T, VEC>& r, float* v) {
  if constexpr (VEC && sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = r.lo[e]; v[4 + e] = r.hi[e]; }
  } else if constexpr (VEC) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[2 * e] = __uint_as_float(r.v[e] << 16); v[2 * e + 1] = __uint_as_float(r.v[e] & 0xFFFF0000u); }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = r.v[e];
  }
}
template <class T, int MODE, bool VEC>
__device__ __forceinline__ void store_unit(T* row, const RotaryArgs& a, int u, const float* v) {
  if constexpr (VEC) {
    if (MODE == MODE_SPLIT && 4 * u < a.P) {
      store4<T>(row + 4 * u, v);
      store4<T>(row + 4 * u + a.P, v + 4);
    } else {
      store8<T>(row + 8 * u, v);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (8 * u + e < a.dh) st_f<T>(row + 8 * u + e, v[e]);
  }
}

// the same operations in the same order whatever the layout: the layouts agree bit for bit
__device__ __forceinline__ float turned_first(float p, float q, float2 w) { return fmaf(p, w.x, -(q * w.y)); }
__device__ __forceinline__ float turned_second(float p, float q, float2 w) { return fmaf(p, w.y, q * w.x); }

// turns the unit's channels in place; cs: the token's row of the table, xch: the 8 floats of every lane of the wave (MODE_SPLIT_ANY)
template <int MODE>
__device__ __forceinline__ void turn_unit(const RotaryArgs& a, int u, const float2* cs, float* v, float* xch) {
  if constexpr (MODE == MODE_ADJACENT || MODE == MODE_ADJACENT_ANY) {
    if (4 * u < a.P) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 w = cs[4 * u + j];
        const float p = v[2 * j], q = v[2 * j + 1];
        const bool turns = MODE == MODE_ADJACENT || 4 * u + j < a.P;          // the padding turns by 0: no way past an infinity
        v[2 * j] = turns ? turned_first(p, q, w) : p;
        v[2 * j + 1] = turns ? turned_second(p, q, w) : q;
      }
    }
  } else if constexpr (MODE == MODE_SPLIT) {
    if (4 * u < a.P) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 w = cs[4 * u + j];
        const float p = v[j], q = v[4 + j];
        v[j] = turned_first(p, q, w);
        v[4 + j] = turned_second(p, q, w);
      }
    }
  } else {
    // the halves meet at no multiple of 4: every lane lays its channels out in LDS (a head's lanes are one contiguous piece of its
    // wave) and picks each partner there.  LDS operations of a wave execute in order; the fences keep the compiler to it.
    const int lane = threadIdx.x & 63, G = 1 << a.lgG;
    float* mine = xch + lane * 8;
    const float* head = xch + (lane & ~(G - 1)) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) mine[e] = v[e];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = 8 * u + e;
      if (c < 2 * a.P) {
        const bool second = c >= a.P;
        const float2 w = cs[second ? c - a.P : c];
        const float o = head[second ? c - a.P : c + a.P];
        v[e] = second ? turned_second(o, v[e], w) : turned_first(v[e], o, w);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

struct Place { int u, sub, head; bool on; };
__device__ __forceinline__ Place place_of(const RotaryArgs& a) {
  const int slot = threadIdx.x >> a.lgG;
  Place p;
  p.u = threadIdx.x & ((1 << a.lgG) - 1);
  p.sub = slot / a.HB;
  p.head = blockIdx.y * a.HB + (slot - p.sub * a.HB);
  p.on = p.sub < a.R && p.head < a.h && p.u < a.U;
  // an idle lane reads a place that exists and stores nothing
  if (!p.on) { p.sub = 0; p.head = blockIdx.y * a.HB; }
  return p;
}
template <int MODE> __device__ __forceinline__ void load_gain(const RotaryArgs& a, const Place& p, float* g) {
  const float* src = p.head < a.q_heads ? a.q_gain : a.k_gain;
  const int row = p.head < a.q_heads ? p.head : p.head - a.q_heads;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = channel_of<MODE>(a, p.u, e);
    g[e] = (src && p.on && c < a.dh) ? src[(int64_t)row * a.gain_pitch + c] : 1.f;
  }
}

constexpr int UN = 4;                      // token rows in flight per lane: a tile's, all requested before its table is computed

template <class T, int MODE, bool VEC, bool NORM>
__global__ __launch_bounds__(256) void rotary_fwd_kernel(RotaryArgs a) {
  __shared__ float2 table[TABLE_PAIRS];
  __shared__ float xch[MODE == MODE_SPLIT_ANY ? 4 * 512 : 1];
  const Place p = place_of(a);
  const int64_t t0 = (int64_t)blockIdx.x * a.TB;
  const int tokens = (int)(a.n - t0 < a.TB ? a.n - t0 : a.TB);
  const int u = p.on ? p.u : 0;
  const T* x = reinterpret_cast<const T*>(a.x) + p.head * a.hpx;
  T* y = reinterpret_cast<T*>(a.y) + (int64_t)p.head * a.dh;
  const int64_t ldy = (int64_t)a.h * a.dh;
  const float inv_dh = 1.f / (float)a.dh;
  float g[8];
  if constexpr (NORM) load_gain<MODE>(a, p, g);
  Raw<T, VEC> raw[UN];
#pragma unroll
  for (int k = 0; k < UN; ++k) {
    const int t = k * a.R + p.sub;
    raw[k] = request_unit<T, MODE, VEC>(x + (t0 + (t < tokens ? t : tokens - 1)) * a.ldx, a, u);
  }
  fill_table(a, t0, tokens, table);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < UN; ++k) {
    const int t = k * a.R + p.sub, tc = t < tokens ? t : tokens - 1;
    float v[8];
    unpack<T, VEC>(raw[k], v);
    if constexpr (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += v[e] * v[e];
      ss = lanes_sum(p.u < a.U ? ss : 0.f, a.lgG);
      const float r = rsqrtf(ss * inv_dh + a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= r * g[e];
    }
    turn_unit<MODE>(a, p.u, table + tc * a.PT, v, xch + (threadIdx.x >> 6) * 512);
    if (p.on && t < tokens) store_unit<T, MODE, VEC>(y + (t0 + t) * ldy, a, u, v);
  }
}

// The gradient of the norm.  Workgroups walk the tiles with the grid's stride; a lane's share of the gain gradient stays in registers
// and leaves once, through LDS, as one partial row per workgroup (summed over the tokens in a fixed order; no atomics).  A lane's
// registers of a row are requested again for the next tile as soon as they are unpacked.
template <class T, int MODE, bool VEC>
__global__ __launch_bounds__(256) void qk_norm_rotary_bwd_kernel(RotaryArgs a) {
  __shared__ float2 tables[2][TABLE_PAIRS];
  __shared__ float xch[4 * 512];
  const Place p = place_of(a);
  const int u = p.on ? p.u : 0;
  const T* x = reinterpret_cast<const T*>(a.x) + p.head * a.hpx;
  const int64_t ldy = (int64_t)a.h * a.dh;
  const T* dy = reinterpret_cast<const T*>(a.dy) + (int64_t)p.head * a.dh;
  T* dx = reinterpret_cast<T*>(a.y) + (int64_t)p.head * a.dh;
  const float inv_dh = 1.f / (float)a.dh;
  float g[8], dg[8];
  load_gain<MODE>(a, p, g);
#pragma unroll
  for (int e = 0; e < 8; ++e) dg[e] = 0.f;
  Raw<T, VEC> rx[UN], rd[UN];
  auto request = [&](int64_t t0, int k) {
    const int64_t row = t0 + k * a.R + p.sub;
    const int64_t r = row < a.n ? row : a.n - 1;
    rx[k] = request_unit<T, MODE, VEC>(x + r * a.ldx, a, u);
    rd[k] = request_unit<T, MODE, VEC>(dy + r * ldy, a, u);
  };
  const int64_t step = (int64_t)gridDim.x * a.TB;
  float2* table = tables[0];
  float2* other = tables[1];
#pragma unroll
  for (int k = 0; k < UN; ++k) request((int64_t)blockIdx.x * a.TB, k);
  for (int64_t t0 = (int64_t)blockIdx.x * a.TB; t0 < a.n; t0 += step) {
    const int tokens = (int)(a.n - t0 < a.TB ? a.n - t0 : a.TB);
    fill_table(a, t0, tokens, table);
    __syncthreads();                       // one a tile: the table of the tile after the next is this one again
#pragma unroll
    for (int k = 0; k < UN; ++k) {
      const int t = k * a.R + p.sub, tc = t < tokens ? t : tokens - 1;
      float v[8], d[8];
      unpack<T, VEC>(rx[k], v);
      unpack<T, VEC>(rd[k], d);
      request(t0 + step, k);               // (behind the last tile: the last row again)
      turn_unit<MODE>(a, p.u, table + tc * a.PT, d, xch + (threadIdx.x >> 6) * 512);
      float ss = 0.f, st = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ss += v[e] * v[e];
        st += g[e] * d[e] * v[e];
      }
      ss = lanes_sum(p.u < a.U ? ss : 0.f, a.lgG);
      st = lanes_sum(p.u < a.U ? st : 0.f, a.lgG);
      const float r = rsqrtf(ss * inv_dh + a.eps), m = r * r * st * inv_dh;
      if (p.on && t < tokens) {
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dg[e] += d[e] * v[e] * r;
          o[e] = r * (g[e] * d[e] - v[e] * m);
        }
        store_unit<T, MODE, VEC>(dx + (t0 + t) * ldy, a, u, o);
      }
    }
    float2* const swap = table; table = other; other = swap;
  }
  if (!a.part) return;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 8; ++e) xch[threadIdx.x * 8 + e] = p.on ? dg[e] : 0.f;
  __syncthreads();
  // column (head of this workgroup, channel) = the sum of its R token rows; one gain for all heads: the sum over the heads of a side too
  const int G = 1 << a.lgG;
  const bool shared = a.gain_pitch == 0;
  const int cols = (shared ? 2 : a.HB) * G * 8;
  const int h0 = blockIdx.y * a.HB;
  float* out = a.part + (shared ? ((int64_t)blockIdx.x * gridDim.y + blockIdx.y) * 2 * a.dh : (int64_t)blockIdx.x * a.h * a.dh);
  for (int c = threadIdx.x; c < cols; c += 256) {
    const int which = c / (G * 8), w = c - which * G * 8, cu = w >> 3, e = w & 7;
    if (cu >= a.U) continue;
    const int ch = channel_of<MODE>(a, cu, e);
    if (ch >= a.dh) continue;
    float s = 0.f;
    if (shared) {
      const int lo = which ? a.q_heads - h0 : 0, hi = which ? a.HB : a.q_heads - h0;
      for (int hl = lo > 0 ? lo : 0; hl < hi && hl < a.HB; ++hl)
        for (int sub = 0; sub < a.R; ++sub) s += xch[(((sub * a.HB + hl) << a.lgG) + cu) * 8 + e];
      out[which * a.dh + ch] = s;
    } else if (h0 + which < a.h) {
      for (int sub = 0; sub < a.R; ++sub) s += xch[(((sub * a.HB + which) << a.lgG) + cu) * 8 + e];
      out[(h0 + which) * a.dh + ch] = s;
    }
  }
}

// gradient column = the sum of the partial rows: 4 columns a workgroup, 256 strips of rows, each in row order, then the strips in a fixed
// order
__global__ __launch_bounds__(1024) void gain_finish_kernel(const float* __restrict__ part, int rows, int cols, int q_cols,
                                                          float* __restrict__ dq_gain, float* __restrict__ dk_gain) {
  __shared__ double red[16][4];
  const int cl = threadIdx.x & 3, strip = threadIdx.x >> 2, c = blockIdx.x * 4 + cl;
  double s = 0.0;
  if (c < cols) {
    for (int r = strip; r < rows; r += 256 * 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = part[(int64_t)(r + 256 * k < rows ? r + 256 * k : r) * cols + c];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += r + 256 * k < rows ? (double)v[k] : 0.0;
    }
  }
#pragma unroll
  for (int k = 4; k < 64; k *= 2) s += __shfl_xor(s, k, 64);
  if ((threadIdx.x & 63) < 4) red[threadIdx.x >> 6][cl] = s;
  __syncthreads();
  if (threadIdx.x < 4 && c < cols) {
    double t = 0.0;
    for (int k = 0; k < 16; ++k) t += red[k][cl];
    if (c < q_cols) { if (dq_gain) dq_gain[c] = (float)t; }
    else if (dk_gain) dk_gain[c - q_cols] = (float)t;
  }
}

bool aligned16(const void* p, int64_t ld, int64_t hp, int es) {
  return ((uintptr_t)p & 15) == 0 && (ld * es) % 16 == 0 && (hp * es) % 16 == 0;
}

struct Shape { int U, lgG, HB, R, TB, gy; };
// Lanes and tiles.  HB heads x R token rows fill the 256 lanes; the tile holds at most TABLE_PAIRS cos / sin pairs, and so few tokens
// that about two workgroups per CU have work when the tensor is small.
Shape shape_of(int64_t n, int h, int dh, int PT) {
  Shape s;
  s.U = (dh + 7) / 8;
  s.lgG = 0;
  while ((1 << s.lgG) < s.U) ++s.lgG;
  const int slots = 256 >> s.lgG;
  s.gy = (h + slots - 1) / slots;
  s.HB = (h + s.gy - 1) / s.gy;
  s.R = slots / s.HB;
  const int64_t want = (n + 511) / 512;
  int64_t tb = (want + s.R - 1) / s.R * s.R;
  const int64_t most = s.R * UN;
  if (tb > most) tb = most;
  if (tb * PT > TABLE_PAIRS) tb = TABLE_PAIRS / PT;
  s.TB = (int)(tb < 1 ? 1 : tb);
  return s;
}

int fill_args(RotaryArgs& a, const void* x, int64_t ldx, int64_t hpx, int dtype, int64_t n, int h, int dh, const void* positions,
              int pos_kind, int64_t ldpos, const double* inv_freq, const int32_t* sections, int axes) {
  if (dtype != TMAE_F32 && dtype != TMAE_BF16) return TMAE_EDTYPE;
  if (n < 0 || h < 1 || h > 65535 || dh < 1 || dh > 512 || axes < 1 || axes > MAX_AXES || !sections || pos_kind < 0 || pos_kind > 2) return TMAE_EARG;
  if (n && (!x || !positions || !inv_freq)) return TMAE_EARG;
  if (ldx < 0 || hpx < 0 || ldpos < axes) return TMAE_EARG;
  int p = 0;
  for (int k = 0; k < MAX_AXES; ++k) {
    if (k < axes) {
      if (sections[k] < 1 || sections[k] > dh) return TMAE_EARG;
      p += sections[k];
    }
    a.sec_end[k] = k < axes ? p : 0x7fffffff;
  }
  if (2 * p > dh) return TMAE_EARG;
  a.x = x; a.ldx = ldx; a.hpx = hpx; a.n = n; a.h = h; a.dh = dh; a.q_heads = h;
  a.pos = positions; a.ldpos = ldpos; a.pos_kind = pos_kind; a.inv_freq = inv_freq; a.P = p; a.PT = (p + 3) & ~3;
  const Shape s = shape_of(n, h, dh, a.PT);
  a.U = s.U; a.lgG = s.lgG; a.HB = s.HB; a.R = s.R; a.TB = s.TB;
  if (n && ((n + s.TB - 1) / s.TB > 0x7fffffff || s.gy > 65535)) return TMAE_EARG;
  return TMAE_OK;
}

// (MODE, VEC): vector accesses need 16-byte rows and whole units; pairs (i, i + P) can then stay in one lane when P is a multiple of 4
template <int MODE, class F> void by_access(bool vec, F&& f) {
  if (vec) f(std::integral_constant<int, MODE>(), std::true_type());
  else f(std::integral_constant<int, MODE>(), std::false_type());
}
template <class F> void by_layout(const RotaryArgs& a, bool interleaved, bool vec, F&& f) {
  if (interleaved && a.P % 4 == 0) by_access<MODE_ADJACENT>(vec, f);
  else if (interleaved) by_access<MODE_ADJACENT_ANY>(vec, f);
  else if (vec && a.P % 4 == 0) f(std::integral_constant<int, MODE_SPLIT>(), std::true_type());
  else by_access<MODE_SPLIT_ANY>(vec, f);
}

template <class T, bool NORM> void launch_fwd(const RotaryArgs& a, bool interleaved, bool vec, hipStream_t stream) {
  const dim3 grid((unsigned)((a.n + a.TB - 1) / a.TB), (unsigned)((a.h + a.HB - 1) / a.HB));
  by_layout(a, interleaved, vec, [&](auto mode, auto v) {
    hipLaunchKernelGGL((rotary_fwd_kernel<T, decltype(mode)::value, decltype(v)::value, NORM>), grid, dim3(256), 0, stream, a);
  });
}
template <class T> void launch_bwd(const RotaryArgs& a, bool interleaved, bool vec, unsigned gx, hipStream_t stream) {
  const dim3 grid(gx, (unsigned)((a.h + a.HB - 1) / a.HB));
  by_layout(a, interleaved, vec, [&](auto mode, auto v) {
    hipLaunchKernelGGL((qk_norm_rotary_bwd_kernel<T, decltype(mode)::value, decltype(v)::value>), grid, dim3(256), 0, stream, a);
  });
}

// workgroups of the backward along the tokens: as many as are resident at once (3 per CU; with 4, a fourth of the float32 ones wait for a
// place: 20 k tokens of 16 heads of 72 in 70 us, not 56), fewer where the heads need more than one
unsigned bwd_blocks(int64_t n, int TB, int gy) {
  const int64_t tiles = (n + TB - 1) / TB;
  int64_t most = 768 / gy;
  if (most < 1) most = 1;
  return (unsigned)(tiles < most ? tiles : most);
}

}  // namespace

int tmae_rotary_axes(const void* x, int64_t ldx, int64_t hpx, int dtype, int64_t n, int h, int dh, const void* positions, int pos_kind,
                     int64_t ldpos, const double* inv_freq, const int32_t* sections, int axes, int interleaved, int inverse, void* y,
                     void* stream) {
  (void)hipGetLastError();
  RotaryArgs a = {};
  const int rc = fill_args(a, x, ldx, hpx, dtype, n, h, dh, positions, pos_kind, ldpos, inv_freq, sections, axes);
  if (rc != TMAE_OK) return rc;
  if (n == 0) return TMAE_OK;
  if (!y) return TMAE_EARG;
  a.y = y;
  a.sign = inverse ? -1.f : 1.f;
  const int es = dtype == TMAE_BF16 ? 2 : 4;
  const bool vec = dh % 8 == 0 && aligned16(x, ldx, hpx, es) && aligned16(y, 0, dh, es);
  if (dtype == TMAE_BF16) launch_fwd<__hip_bfloat16, false>(a, interleaved != 0, vec, (hipStream_t)stream);
  else launch_fwd<float, false>(a, interleaved != 0, vec, (hipStream_t)stream);
  return tmae_launch_status();
}

int tmae_qk_norm_rotary_fwd(const void* x, int64_t ldx, int64_t hpx, int dtype, int64_t n, int h, int q_heads, int dh,
                            const float* q_gain, const float* k_gain, int gain_per_head, float eps, const void* positions, int pos_kind,
                            int64_t ldpos, const double* inv_freq, const int32_t* sections, int axes, int interleaved, void* y,
                            void* stream) {
  (void)hipGetLastError();
  RotaryArgs a = {};
  const int rc = fill_args(a, x, ldx, hpx, dtype, n, h, dh, positions, pos_kind, ldpos, inv_freq, sections, axes);
  if (rc != TMAE_OK) return rc;
  if (q_heads < 0 || q_heads > h || !(eps >= 0.f)) return TMAE_EARG;
  if (n == 0) return TMAE_OK;
  if (!y) return TMAE_EARG;
  a.y = y; a.sign = 1.f; a.q_heads = q_heads; a.q_gain = q_gain; a.k_gain = k_gain; a.gain_pitch = gain_per_head ? dh : 0; a.eps = eps;
  const int es = dtype == TMAE_BF16 ? 2 : 4;
  const bool vec = dh % 8 == 0 && aligned16(x, ldx, hpx, es) && aligned16(y, 0, dh, es);
  if (dtype == TMAE_BF16) launch_fwd<__hip_bfloat16, true>(a, interleaved != 0, vec, (hipStream_t)stream);
  else launch_fwd<float, true>(a, interleaved != 0, vec, (hipStream_t)stream);
  return tmae_launch_status();
}

size_t tmae_qk_norm_rotary_bwd_workspace(int64_t n, int h, int dh, int pairs, int gain_per_head) {
  if (n <= 0 || h < 1 || dh < 1 || dh > 512 || pairs < 1) return 0;
  const Shape s = shape_of(n, h, dh, (pairs + 3) & ~3);
  const size_t rows = (size_t)bwd_blocks(n, s.TB, s.gy) * (gain_per_head ? 1 : s.gy);
  return tmae_align(rows * (gain_per_head ? (size_t)h * dh : (size_t)2 * dh) * sizeof(float));
}

int tmae_qk_norm_rotary_bwd(const void* x, int64_t ldx, int64_t hpx, const void* dy, int dtype, int64_t n, int h, int q_heads, int dh,
                            const float* q_gain, const float* k_gain, int gain_per_head, float eps, const void* positions, int pos_kind,
                            int64_t ldpos, const double* inv_freq, const int32_t* sections, int axes, int interleaved, void* dx,
                            float* dq_gain, float* dk_gain, void* ws, size_t ws_bytes, void* stream) {
  (void)hipGetLastError();
  RotaryArgs a = {};
  const int rc = fill_args(a, x, ldx, hpx, dtype, n, h, dh, positions, pos_kind, ldpos, inv_freq, sections, axes);
  if (rc != TMAE_OK) return rc;
  if (q_heads < 0 || q_heads > h || !(eps >= 0.f)) return TMAE_EARG;
  if (n && (!dy || !dx)) return TMAE_EARG;
  const bool want = dq_gain || dk_gain;
  a.dy = dy; a.y = dx; a.sign = -1.f; a.q_heads = q_heads; a.q_gain = q_gain; a.k_gain = k_gain; a.gain_pitch = gain_per_head ? dh : 0; a.eps = eps;
  const int gy = (h + a.HB - 1) / a.HB;
  const unsigned gx = n ? bwd_blocks(n, a.TB, gy) : 0;
  const int q_cols = gain_per_head ? q_heads * dh : dh, cols = gain_per_head ? h * dh : 2 * dh;
  const int rows = (int)(gx * (gain_per_head ? 1 : gy));
  if (want && n) {
    WsCarver c(ws, ws_bytes);
    a.part = c.take<float>((size_t)rows * cols);
    if (!c.ok || !a.part) return TMAE_EWS;
  }
  if (n) {
    const int es = dtype == TMAE_BF16 ? 2 : 4;
    const bool vec = dh % 8 == 0 && aligned16(x, ldx, hpx, es) && aligned16(dy, 0, dh, es) && aligned16(dx, 0, dh, es);
    if (dtype == TMAE_BF16) launch_bwd<__hip_bfloat16>(a, interleaved != 0, vec, gx, (hipStream_t)stream);
    else launch_bwd<float>(a, interleaved != 0, vec, gx, (hipStream_t)stream);
  }
  if (want)
    hipLaunchKernelGGL(gain_finish_kernel, dim3(tmae_cdiv(cols, 4)), dim3(1024), 0, (hipStream_t)stream, a.part, rows, cols, q_cols,
                       dq_gain, dk_gain);
  return tmae_launch_status();
}

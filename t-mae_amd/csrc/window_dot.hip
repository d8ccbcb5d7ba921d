// Scaled-dot-product attention inside 8x8 windows of the token grid.
//
//   P_ij = softmax_j(scale q_i . k_j) over the keys j of the query's window,  o_i = sum_j P_ij v_j;  a window without keys: o_i = 0
//   backward, P recomputed from the saved log2 of the softmax's denominator:
//   dV_j = sum_i P_ij dO_i,  dP_ij = dO_i . v_j,  dS_ij = scale P_ij (dP_ij - sum_j P_ij dP_ij),  dQ_i = sum_j dS_ij k_j,  dK_j = sum_i dS_ij q_i
//
// One wavefront per (window, head), tiles of 16 tokens on the float32 matrix instruction 16x16x4.  Its accumulator layout -- lane
// (g, i) = (lane >> 4, lane & 15) holds rows 4g .. 4g+3 of column i -- is also what its B operand takes, row 4g + r in step r: the
// probabilities go from one product into the next without leaving the registers.  Which of the two products' orders is wanted (the
// query or the key in the column) is had by exchanging the operands.
//
// A slot without a token stands for the window's first one: it is read, its probability is set to 0, and nothing is stored for it.
#include "common.h"
#include <type_traits>

namespace {

constexpr int WIN = 8;
constexpr int WL_HDR = 8;                  // the work list: tmae_window_worklist
constexpr float LOG2E = 1.4426950408889634f;

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct DotArgs {
  const void *q, *k, *v, *g;               // g: dO
  int64_t ldq, ldk, ldv, ldg;
  void *o, *dq, *dk, *dv;
  int64_t ldo, lddq, lddk, lddv;
  float* lse;                              // [mq, nhead]: log2 of sum_j 2^(c q.k_j), c = scale * log2(e)
  const int32_t *grid_q, *grid_k, *wl;
  int64_t mq, mk, nwin;
  int nhead, batch, ny, nx, Wy, Wx, s;
  float scale;
};

struct Window { int Tq, Tk; };

// The window's tokens in cell order, into toks[0] (queries) and toks[1] (keys); slots behind the last token repeat the first one.
// A row number outside the tensors counts as an empty cell.  False: the block has no window.
__device__ __forceinline__ bool find_window(const DotArgs& a, int cls, int (*toks)[64], Window& w) {
  const int lane = threadIdx.x & 63;
  int b, wcy, wcx;
  if (a.wl) {
    const int64_t cnt = a.wl[cls];
    if ((int64_t)blockIdx.x >= cnt || (int64_t)blockIdx.x >= a.nwin) return false;
    const int p = a.wl[WL_HDR + cls * a.nwin + blockIdx.x];
    b = p >> 16; wcx = (p >> 8) & 255; wcy = p & 255;
  } else {
    const unsigned u = blockIdx.x;
    wcy = (int)(u % (unsigned)a.Wy); wcx = (int)((u / (unsigned)a.Wy) % (unsigned)a.Wx); b = (int)(u / (unsigned)(a.Wy * a.Wx));
  }
  const int y = wcy * WIN - a.s + (lane >> 3), x = wcx * WIN - a.s + (lane & 7);
  const bool in = b >= 0 && b < a.batch && y >= 0 && y < a.ny && x >= 0 && x < a.nx;
  const int64_t cell = ((int64_t)b * a.ny + y) * a.nx + x;
  int tq = in ? a.grid_q[cell] : -1, tk = in ? a.grid_k[cell] : -1;
  if (tq >= a.mq) tq = -1;
  if (tk >= a.mk) tk = -1;
  const unsigned long long mq = __ballot(tq >= 0), mk = __ballot(tk >= 0), below = (1ull << lane) - 1ull;
  w.Tq = __popcll(mq);
  w.Tk = __popcll(mk);
  const int fq = mq ? __shfl(tq, __ffsll(mq) - 1, 64) : -1, fk = mk ? __shfl(tk, __ffsll(mk) - 1, 64) : -1;
  if (threadIdx.x < 64) {
    if (lane >= w.Tq) toks[0][lane] = fq;
    if (lane >= w.Tk) toks[1][lane] = fk;
    if (tq >= 0) toks[0][__popcll(mq & below)] = tq;
    if (tk >= 0) toks[1][__popcll(mk & below)] = tk;
  }
  return true;
}

// channels KD g .. KD g + KD - 1 of a token's head: what the lane contributes to a product over the channels
template <class T, int KD> __device__ __forceinline__ void load_frag(const T* p, float* f);
template <> __device__ __forceinline__ void load_frag<float, 4>(const float* p, float* f) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
}
template <> __device__ __forceinline__ void load_frag<float, 8>(const float* p, float* f) { load8<float>(p, f); }
template <> __device__ __forceinline__ void load_frag<float, 16>(const float* p, float* f) { load8<float>(p, f); load8<float>(p + 8, f + 8); }
template <> __device__ __forceinline__ void load_frag<__hip_bfloat16, 4>(const __hip_bfloat16* p, float* f) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  f[0] = __uint_as_float(u.x << 16); f[1] = __uint_as_float(u.x & 0xFFFF0000u);
  f[2] = __uint_as_float(u.y << 16); f[3] = __uint_as_float(u.y & 0xFFFF0000u);
}
template <> __device__ __forceinline__ void load_frag<__hip_bfloat16, 8>(const __hip_bfloat16* p, float* f) { load8<__hip_bfloat16>(p, f); }
template <> __device__ __forceinline__ void load_frag<__hip_bfloat16, 16>(const __hip_bfloat16* p, float* f) {
  load8<__hip_bfloat16>(p, f);
  load8<__hip_bfloat16>(p + 8, f + 8);
}
template <class T> __device__ __forceinline__ void store_four(T* p, const f32x4& v) {
#pragma unroll
  for (int r = 0; r < 4; ++r) st_f<T>(p + r, v[r]);
}

__device__ __forceinline__ float lanes4_sum(float v) { v += __shfl_xor(v, 16, 64); return v + __shfl_xor(v, 32, 64); }
__device__ __forceinline__ float lanes4_max(float v) { v = fmaxf(v, __shfl_xor(v, 16, 64)); return fmaxf(v, __shfl_xor(v, 32, 64)); }

template <int KD> __device__ __forceinline__ f32x4 product(const float* a, const float* b) {
  f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < KD; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
  return c;
}
// c[ct] += (tokens' channels as rows) x (b as columns): rows 16 ct .. +15 of the head's channels, contraction over the tile's tokens
template <class T, int CT>
__device__ __forceinline__ void accumulate(const T* base, int64_t ld, const int* toks, const f32x4& b, f32x4* c, int g, int i) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const T* row = base + (int64_t)toks[4 * g + r] * ld + i;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) c[ct] = __builtin_amdgcn_mfma_f32_16x16x4f32(ld_f<T>(row + 16 * ct), b[r], c[ct], 0, 0, 0);
  }
}
__device__ __forceinline__ void order_lds() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <class T, int DH>
__global__ __launch_bounds__(256, 2) void dot_fwd_kernel(DotArgs a, int cls) {
  constexpr int KD = DH / 4, CT = DH / 16;
  __shared__ int toks[2][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, i = lane & 15;
  Window win;
  if (!find_window(a, cls, toks, win)) return;
  __syncthreads();
  const int head = blockIdx.y * 4 + w;
  if (head >= a.nhead || win.Tq == 0) return;
  const int hoff = head * DH;
  T* out = (T*)a.o + hoff;
  if (win.Tk == 0) {
    if (lane < win.Tq) {
      T* o = out + (int64_t)toks[0][lane] * a.ldo;
      for (int c = 0; c < DH; ++c) st_f<T>(o + c, 0.f);
      a.lse[(int64_t)toks[0][lane] * a.nhead + head] = 0.f;
    }
    return;
  }
  const T *q = (const T*)a.q + hoff, *k = (const T*)a.k + hoff, *v = (const T*)a.v + hoff;
  const int nq = (win.Tq + 15) >> 4, nk = (win.Tk + 15) >> 4;
  const float c = a.scale * LOG2E;
  for (int qt = 0; qt < nq; ++qt) {
    const int64_t tq = toks[0][qt * 16 + i];
    float qf[KD];
    load_frag<T, KD>(q + tq * a.ldq + KD * g, qf);
    f32x4 st[4];
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      if (kt < nk) {
        float kf[KD];
        load_frag<T, KD>(k + (int64_t)toks[1][kt * 16 + i] * a.ldk + KD * g, kf);
        st[kt] = product<KD>(kf, qf);                                  // rows = keys, column = query i
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (kt * 16 + 4 * g + r >= win.Tk) st[kt][r] = -INFINITY;
          mx = fmaxf(mx, st[kt][r]);
        }
      }
    }
    mx = lanes4_max(mx) * c;
    float l = 0.f;
    f32x4 o[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) o[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      if (kt < nk) {
        f32x4 p;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[r] = kt * 16 + 4 * g + r < win.Tk ? __builtin_amdgcn_exp2f(fmaf(st[kt][r], c, -mx)) : 0.f;
          l += p[r];
        }
        accumulate<T, CT>(v, a.ldv, toks[1] + kt * 16, p, o, g, i);      // rows = channels, column = query i
      }
    }
    l = lanes4_sum(l);
    if (qt * 16 + i < win.Tq) {
      const float inv = 1.f / l;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) store_four<T>(out + tq * a.ldo + 16 * ct + 4 * g, o[ct] * inv);
      if (g == 0) a.lse[tq * a.nhead + head] = mx + __builtin_amdgcn_logf(l);          // v_log_f32: the logarithm to base 2
    }
  }
}

template <class T, int DH>
__global__ __launch_bounds__(256, 2) void dot_bwd_kernel(DotArgs a, int cls) {
  constexpr int KD = DH / 4, CT = DH / 16;
  __shared__ int toks[2][64];
  __shared__ float lse[4][64], dot[4][64];               // of the query slots: saved log2 denominator, sum_j P dP
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, i = lane & 15;
  Window win;
  if (!find_window(a, cls, toks, win)) return;
  __syncthreads();
  const int head = blockIdx.y * 4 + w;
  if (head >= a.nhead) return;
  const int hoff = head * DH;
  T *dq = (T*)a.dq + hoff, *dk = (T*)a.dk + hoff, *dv = (T*)a.dv + hoff;
  if (win.Tq == 0 || win.Tk == 0) {
    if (lane < win.Tq) {
      T* p = dq + (int64_t)toks[0][lane] * a.lddq;
      for (int c = 0; c < DH; ++c) st_f<T>(p + c, 0.f);
    }
    if (lane < win.Tk) {
      T *p = dk + (int64_t)toks[1][lane] * a.lddk, *r = dv + (int64_t)toks[1][lane] * a.lddv;
      for (int c = 0; c < DH; ++c) { st_f<T>(p + c, 0.f); st_f<T>(r + c, 0.f); }
    }
    return;
  }
  const T *q = (const T*)a.q + hoff, *k = (const T*)a.k + hoff, *v = (const T*)a.v + hoff, *gr = (const T*)a.g + hoff;
  const int nq = (win.Tq + 15) >> 4, nk = (win.Tk + 15) >> 4;
  const float c = a.scale * LOG2E;
  lse[w][lane] = a.lse[(int64_t)toks[0][lane] * a.nhead + head];
  order_lds();
  // dQ: the query in the column
  for (int qt = 0; qt < nq; ++qt) {
    const int64_t tq = toks[0][qt * 16 + i];
    const float ls = lse[w][qt * 16 + i];
    float qf[KD], gf[KD];
    load_frag<T, KD>(q + tq * a.ldq + KD * g, qf);
    load_frag<T, KD>(gr + tq * a.ldg + KD * g, gf);
    f32x4 p[4], dp[4], acc[CT];
    float d = 0.f;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      if (kt < nk) {
        const int64_t tk = toks[1][kt * 16 + i];
        float f[KD];
        load_frag<T, KD>(k + tk * a.ldk + KD * g, f);
        const f32x4 s = product<KD>(f, qf);
        load_frag<T, KD>(v + tk * a.ldv + KD * g, f);
        dp[kt] = product<KD>(f, gf);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[kt][r] = kt * 16 + 4 * g + r < win.Tk ? __builtin_amdgcn_exp2f(fmaf(s[r], c, -ls)) : 0.f;
          d += p[kt][r] * dp[kt][r];
        }
      }
    }
    d = lanes4_sum(d);
    if (g == 0) dot[w][qt * 16 + i] = d;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) acc[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      if (kt < nk) {
        f32x4 ds;
#pragma unroll
        for (int r = 0; r < 4; ++r) ds[r] = a.scale * p[kt][r] * (dp[kt][r] - d);
        accumulate<T, CT>(k, a.ldk, toks[1] + kt * 16, ds, acc, g, i);
      }
    }
    if (qt * 16 + i < win.Tq) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) store_four<T>(dq + tq * a.lddq + 16 * ct + 4 * g, acc[ct]);
    }
  }
  order_lds();
  // dK, dV: the key in the column
  for (int kt = 0; kt < nk; ++kt) {
    const int64_t tk = toks[1][kt * 16 + i];
    float kf[KD], vf[KD];
    load_frag<T, KD>(k + tk * a.ldk + KD * g, kf);
    load_frag<T, KD>(v + tk * a.ldv + KD * g, vf);
    f32x4 ak[CT], av[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) ak[ct] = av[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int qt = 0; qt < nq; ++qt) {
      const int64_t tq = toks[0][qt * 16 + i];
      float f[KD];
      load_frag<T, KD>(q + tq * a.ldq + KD * g, f);
      const f32x4 s = product<KD>(f, kf);                               // rows = queries, column = key i
      load_frag<T, KD>(gr + tq * a.ldg + KD * g, f);
      const f32x4 dp = product<KD>(f, vf);
      f32x4 p, ds;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int slot = qt * 16 + 4 * g + r;
        p[r] = slot < win.Tq ? __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse[w][slot])) : 0.f;
        ds[r] = a.scale * p[r] * (dp[r] - dot[w][slot]);
      }
      accumulate<T, CT>(gr, a.ldg, toks[0] + qt * 16, p, av, g, i);
      accumulate<T, CT>(q, a.ldq, toks[0] + qt * 16, ds, ak, g, i);
    }
    if (kt * 16 + i < win.Tk) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        store_four<T>(dk + tk * a.lddk + 16 * ct + 4 * g, ak[ct]);
        store_four<T>(dv + tk * a.lddv + 16 * ct + 4 * g, av[ct]);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------ bfloat16
// The same products on the bfloat16 matrix instructions.  A lane's piece of a token row -- FR = DH / 4 channels -- is as loaded the
// operand of the products over the channels (logits, dP).  The products over tokens need a tile by columns: its rows go through LDS
// (ds_read_b64_tr_b16 returns four rows of one column).  In the image of a row, position 4 a + b of 16-channel tile ct holds channel
// FR a + 4 ct + b, so that a lane ends with FR consecutive channels of one token and stores them at once.
//
// P and dS enter their products rounded to bfloat16 (2^-8 of each; sums, maxima and everything else stay float32): their error is
// that of the results' own rounding.
//
// A wave holds the NK key tiles of its window and walks the query tiles; NK is a template parameter, so no branch stands between a
// matrix instruction and its reader.  Windows of at most 16 tokens (three quarters of an outdoor scene's, with two fifths of the tokens):
// one wave takes up to four heads of the window at once, whose rows it requests together.

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int TILE_PITCH = 40;             // bytes per row of a 16x16 bfloat16 tile in LDS

__device__ __forceinline__ unsigned pack2(float a, float b) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
__device__ __forceinline__ s16x4 pack4(const f32x4& v) { return __builtin_bit_cast(s16x4, u32x2{pack2(v[0], v[1]), pack2(v[2], v[3])}); }
__device__ __forceinline__ s16x4 read_columns(const char* lds) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)lds);
}
// sum / maximum over the 4 lanes that share a column, in every one of them
__device__ __forceinline__ float column_sum(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float column_max(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <int FR> struct Piece { unsigned u[FR / 2]; };          // FR channels of a token
template <int FR> __device__ __forceinline__ Piece<FR> load_piece(const char* p) {
  Piece<FR> f;
  if constexpr (FR == 4) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    f.u[0] = v.x; f.u[1] = v.y;
  } else {
#pragma unroll
    for (int j = 0; j < FR / 8; ++j) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[j];
      f.u[4 * j] = v.x; f.u[4 * j + 1] = v.y; f.u[4 * j + 2] = v.z; f.u[4 * j + 3] = v.w;
    }
  }
  return f;
}
template <int FR> __device__ __forceinline__ void store_piece(char* p, const f32x4* v, float by) {
  unsigned u[FR / 2];
#pragma unroll
  for (int ct = 0; ct < FR / 4; ++ct) {
    u[2 * ct] = pack2(v[ct][0] * by, v[ct][1] * by);
    u[2 * ct + 1] = pack2(v[ct][2] * by, v[ct][3] * by);
  }
  if constexpr (FR == 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
  } else {
#pragma unroll
    for (int j = 0; j < FR / 8; ++j) reinterpret_cast<uint4*>(p)[j] = make_uint4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
  }
}
template <int FR> __device__ __forceinline__ f32x4 over_channels(const Piece<FR>& a, const Piece<FR>& b, f32x4 c) {
  if constexpr (FR == 4) {
    c = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < FR / 8; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
          __builtin_bit_cast(bf16x8, u32x4{a.u[4 * j], a.u[4 * j + 1], a.u[4 * j + 2], a.u[4 * j + 3]}),
          __builtin_bit_cast(bf16x8, u32x4{b.u[4 * j], b.u[4 * j + 1], b.u[4 * j + 2], b.u[4 * j + 3]}), c, 0, 0, 0);
  }
  return c;
}
// c += A B over the 16 tokens of one tile, or over the 32 of two (a third tile rides with zeros: one accumulator goes through products
// of one shape only -- a 16x16x16 right behind the 16x16x32 that it continues has read wrong values)
__device__ __forceinline__ f32x4 over_tokens(const s16x4& a, const s16x4& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 over_tokens(const s16x4& a0, const s16x4& a1, const s16x4& b0, const s16x4& b1, f32x4 c) {
  const s16x8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7), b = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <int DH> struct Image {            // rows of a head by token, read by columns
  static constexpr int FR = DH / 4, CT = DH / 16, PITCH = DH * 2 + 16, TILE = 16 * PITCH;
  static __device__ __forceinline__ void put(char* tile, int g, int i, const Piece<FR>& f) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) *reinterpret_cast<uint2*>(tile + i * PITCH + 32 * ct + 8 * g) = make_uint2(f.u[2 * ct], f.u[2 * ct + 1]);
  }
  static __device__ __forceinline__ s16x4 get(const char* tile, int g, int i, int ct) {
    return read_columns(tile + (4 * g + (i >> 2)) * PITCH + 32 * ct + 8 * (i & 3));
  }
};

// One window, one head: NK key tiles against nq query tiles.  toks: the window's token lists in LDS; lds: 16 NK rows of an image.
template <int DH, int NK>
__device__ __forceinline__ void fwd_window(const DotArgs& a, const int* tq_, const int* tk_, int Tq, int Tk, int head, char* lds) {
  using Im = Image<DH>;
  constexpr int FR = Im::FR, CT = Im::CT;
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
  const int64_t col = (int64_t)head * DH * 2 + FR * 2 * g;
  const char *q = (const char*)a.q + col, *k = (const char*)a.k + col, *v = (const char*)a.v + col;
  char* out = (char*)a.o + col;
  const int nq = (Tq + 15) >> 4;
  Piece<FR> kf[NK], vf[NK];
#pragma unroll
  for (int kt = 0; kt < NK; ++kt) {
    const int64_t t = tk_[kt * 16 + i];
    kf[kt] = load_piece<FR>(k + t * a.ldk * 2);
    vf[kt] = load_piece<FR>(v + t * a.ldv * 2);
  }
  int64_t tq = tq_[i];
  Piece<FR> qf = load_piece<FR>(q + tq * a.ldq * 2);
#pragma unroll
  for (int kt = 0; kt < NK; ++kt) Im::put(lds + kt * Im::TILE, g, i, vf[kt]);
  order_lds();
  s16x4 vc[NK][CT];
#pragma unroll
  for (int kt = 0; kt < NK; ++kt)
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) vc[kt][ct] = Im::get(lds + kt * Im::TILE, g, i, ct);
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 absent;                              // of the last key tile: -inf where there is no key
#pragma unroll
  for (int r = 0; r < 4; ++r) absent[r] = (NK - 1) * 16 + 4 * g + r < Tk ? 0.f : -INFINITY;
  const float c = a.scale * LOG2E;
  for (int qt = 0; qt < nq; ++qt) {
    const int64_t tnext = tq_[(qt + 1 < nq ? qt + 1 : qt) * 16 + i];
    const Piece<FR> qnext = load_piece<FR>(q + tnext * a.ldq * 2);
    f32x4 st[NK];
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < NK; ++kt) st[kt] = over_channels<FR>(kf[kt], qf, kt == NK - 1 ? absent : zero);
#pragma unroll
    for (int kt = 0; kt < NK; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, st[kt][r]);
    mx = column_max(mx) * c;
    float l = 0.f;
    s16x4 p[NK];
#pragma unroll
    for (int kt = 0; kt < NK; ++kt) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        st[kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[kt][r], c, -mx));
        l += st[kt][r];
      }
      p[kt] = pack4(st[kt]);
    }
    l = column_sum(l);
    f32x4 o[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      o[ct] = zero;
      if constexpr (NK >= 2) o[ct] = over_tokens(vc[0][ct], vc[1][ct], p[0], p[1], o[ct]);
      if constexpr (NK == 4) o[ct] = over_tokens(vc[2][ct], vc[3][ct], p[2], p[3], o[ct]);
      if constexpr (NK == 3) o[ct] = over_tokens(vc[2][ct], s16x4{0, 0, 0, 0}, p[2], s16x4{0, 0, 0, 0}, o[ct]);
      if constexpr (NK == 1) o[ct] = over_tokens(vc[0][ct], p[0], o[ct]);
    }
    const float inv = __builtin_amdgcn_rcpf(l);
    if (qt * 16 + i < Tq) {
      store_piece<FR>(out + tq * a.ldo * 2, o, inv);
      if (g == 0) a.lse[tq * a.nhead + head] = mx + __builtin_amdgcn_logf(l);
    }
    tq = tnext;
    qf = qnext;
  }
}

template <int DH, int NK>
__device__ __forceinline__ void bwd_window(const DotArgs& a, const int* tq_, const int* tk_, int Tq, int Tk, int head, char* lds) {
  using Im = Image<DH>;
  constexpr int FR = Im::FR, CT = Im::CT, TP = TILE_PITCH;
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
  const int64_t col = (int64_t)head * DH * 2 + FR * 2 * g;
  const char *q = (const char*)a.q + col, *k = (const char*)a.k + col, *v = (const char*)a.v + col, *gr = (const char*)a.g + col;
  const int nq = (Tq + 15) >> 4;
  Piece<FR> kf[NK], vf[NK];
#pragma unroll
  for (int kt = 0; kt < NK; ++kt) {
    const int64_t t = tk_[kt * 16 + i];
    kf[kt] = load_piece<FR>(k + t * a.ldk * 2);
    vf[kt] = load_piece<FR>(v + t * a.ldv * 2);
  }
  int64_t tq = tq_[i];
  Piece<FR> qf = load_piece<FR>(q + tq * a.ldq * 2), gf = load_piece<FR>(gr + tq * a.ldg * 2);
  float ls = a.lse[tq * a.nhead + head];
#pragma unroll
  for (int kt = 0; kt < NK; ++kt) Im::put(lds + kt * Im::TILE, g, i, kf[kt]);
  order_lds();
  s16x4 kc[NK][CT];
#pragma unroll
  for (int kt = 0; kt < NK; ++kt)
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) kc[kt][ct] = Im::get(lds + kt * Im::TILE, g, i, ct);
  order_lds();
  // from here on: the query tile's q and dO rows, and the P and dS tiles of every key tile
  char *qimg = lds, *gimg = lds + Im::TILE, *tiles = lds + 2 * Im::TILE;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 absent;
#pragma unroll
  for (int r = 0; r < 4; ++r) absent[r] = (NK - 1) * 16 + 4 * g + r < Tk ? 0.f : -INFINITY;
  const float c = a.scale * LOG2E;
  f32x4 dk[NK][CT], dv[NK][CT];
#pragma unroll
  for (int kt = 0; kt < NK; ++kt)
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) dk[kt][ct] = dv[kt][ct] = zero;
  for (int qt = 0; qt < nq; ++qt) {
    const int64_t tnext = tq_[(qt + 1 < nq ? qt + 1 : qt) * 16 + i];
    const Piece<FR> qnext = load_piece<FR>(q + tnext * a.ldq * 2), gnext = load_piece<FR>(gr + tnext * a.ldg * 2);
    const float lsnext = a.lse[tnext * a.nhead + head];
    Im::put(qimg, g, i, qf);
    Im::put(gimg, g, i, gf);
    order_lds();
    s16x4 qc[CT], gc[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      qc[ct] = Im::get(qimg, g, i, ct);
      gc[ct] = Im::get(gimg, g, i, ct);
    }
    order_lds();
    const float le = qt * 16 + i < Tq ? ls : INFINITY;           // no query: P = 0
    f32x4 p[NK], dp[NK];
    float d = 0.f;
#pragma unroll
    for (int kt = 0; kt < NK; ++kt) {
      p[kt] = over_channels<FR>(kf[kt], qf, kt == NK - 1 ? absent : zero);           // rows = keys, column = query i
      dp[kt] = over_channels<FR>(vf[kt], gf, zero);
    }
#pragma unroll
    for (int kt = 0; kt < NK; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[kt][r], c, -le));
        d = __builtin_fmaf(p[kt][r], dp[kt][r], d);
      }
    d = column_sum(d);
    s16x4 ds[NK];
#pragma unroll
    for (int kt = 0; kt < NK; ++kt) {
      f32x4 t;
#pragma unroll
      for (int r = 0; r < 4; ++r) t[r] = p[kt][r] * (dp[kt][r] - d);
      ds[kt] = pack4(t);
      *reinterpret_cast<s16x4*>(tiles + (2 * kt) * 16 * TP + i * TP + 8 * g) = pack4(p[kt]);
      *reinterpret_cast<s16x4*>(tiles + (2 * kt + 1) * 16 * TP + i * TP + 8 * g) = ds[kt];
    }
    order_lds();
    f32x4 dq[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      dq[ct] = zero;
      if constexpr (NK >= 2) dq[ct] = over_tokens(kc[0][ct], kc[1][ct], ds[0], ds[1], dq[ct]);
      if constexpr (NK == 4) dq[ct] = over_tokens(kc[2][ct], kc[3][ct], ds[2], ds[3], dq[ct]);
      if constexpr (NK == 3) dq[ct] = over_tokens(kc[2][ct], s16x4{0, 0, 0, 0}, ds[2], s16x4{0, 0, 0, 0}, dq[ct]);
      if constexpr (NK == 1) dq[ct] = over_tokens(kc[0][ct], ds[0], dq[ct]);
    }
#pragma unroll
    for (int kt = 0; kt < NK; ++kt) {
      const s16x4 pt = read_columns(tiles + (2 * kt) * 16 * TP + (4 * g + (i >> 2)) * TP + 8 * (i & 3));            // queries 4g.. of key i
      const s16x4 dt = read_columns(tiles + (2 * kt + 1) * 16 * TP + (4 * g + (i >> 2)) * TP + 8 * (i & 3));
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        dv[kt][ct] = over_tokens(gc[ct], pt, dv[kt][ct]);
        dk[kt][ct] = over_tokens(qc[ct], dt, dk[kt][ct]);
      }
    }
    order_lds();
    if (qt * 16 + i < Tq) store_piece<FR>((char*)a.dq + col + tq * a.lddq * 2, dq, a.scale);
    tq = tnext;
    qf = qnext;
    gf = gnext;
    ls = lsnext;
  }
#pragma unroll
  for (int kt = 0; kt < NK; ++kt)
    if (kt * 16 + i < Tk) {
      const int64_t t = tk_[kt * 16 + i];
      store_piece<FR>((char*)a.dk + col + t * a.lddk * 2, dk[kt], a.scale);
      store_piece<FR>((char*)a.dv + col + t * a.lddv * 2, dv[kt], 1.f);
    }
}

template <int DH, int NT> constexpr int lds_bytes(bool bwd) {            // of one wave
  const int image = NT * Image<DH>::TILE, rest = 2 * Image<DH>::TILE + NT * 2 * 16 * TILE_PITCH;
  return !bwd || image > rest ? image : rest;
}

// A window of up to 16 NT tokens per workgroup, a head per wave; without a work list (NT = 4) every window, empty ones included.
// Two waves per SIMD as the bound: 256 registers at most, and the matrix instructions then write plain vector registers.
template <int DH, int NT, bool BWD>
__global__ __launch_bounds__(256, 2) void dot_window_kernel(DotArgs a, int cls) {
  constexpr int BYTES = lds_bytes<DH, NT>(BWD);
  __shared__ int toks[2][64];
  __shared__ __attribute__((aligned(16))) char lds[4][BYTES];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  Window win;
  if (!find_window(a, cls, toks, win)) return;
  __syncthreads();
  const int head = blockIdx.y * 4 + w;
  if (head >= a.nhead) return;
  const int Tq = win.Tq < NT * 16 ? win.Tq : NT * 16, Tk = win.Tk < NT * 16 ? win.Tk : NT * 16;
  if (Tq == 0 || Tk == 0) {
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    if (lane < Tq) {
      uint4* o = reinterpret_cast<uint4*>(BWD ? (char*)a.dq + (toks[0][lane] * a.lddq + head * DH) * 2 : (char*)a.o + (toks[0][lane] * a.ldo + head * DH) * 2);
      for (int c = 0; c < DH / 8; ++c) o[c] = z;
    }
    if (BWD && lane < Tk) {
      uint4 *p = reinterpret_cast<uint4*>((char*)a.dk + (toks[1][lane] * a.lddk + head * DH) * 2),
            *r = reinterpret_cast<uint4*>((char*)a.dv + (toks[1][lane] * a.lddv + head * DH) * 2);
      for (int c = 0; c < DH / 8; ++c) { p[c] = z; r[c] = z; }
    }
    return;
  }
  const int nk = (Tk + 15) >> 4;
#define ONE(NK)                                                                     \
  if constexpr (BWD) bwd_window<DH, NK>(a, toks[0], toks[1], Tq, Tk, head, lds[w]); \
  else fwd_window<DH, NK>(a, toks[0], toks[1], Tq, Tk, head, lds[w])
  if (nk == 1) { ONE(1); }
  else if (NT == 2 || nk == 2) { ONE(2); }
  else if constexpr (NT == 4) {
    if (nk == 3) { ONE(3); } else { ONE(4); }
  }
#undef ONE
}

// Windows of at most 16 tokens: a window per wave, HG heads of it at a time.  Nothing is shared between the waves of a workgroup.
template <int DH> constexpr int heads_at_once() { return DH == 16 ? 4 : DH == 32 ? 2 : 1; }

template <int DH, bool BWD>
__global__ __launch_bounds__(256, 2) void dot_small_kernel(DotArgs a) {
  using Im = Image<DH>;
  constexpr int FR = Im::FR, CT = Im::CT, HG = heads_at_once<DH>(), TP = TILE_PITCH;
  constexpr int PER_HEAD = (BWD ? 3 : 1) * Im::TILE > (BWD ? 2 * 16 * TP : 0) ? (BWD ? 3 : 1) * Im::TILE : 2 * 16 * TP;
  __shared__ int toks_[4][2][16];
  __shared__ __attribute__((aligned(16))) char lds_[4][HG * PER_HEAD];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, i = lane & 15;
  // list 1 first (9 to 16 tokens), then list 0
  const int64_t e = (int64_t)blockIdx.x * 4 + w, n1 = a.wl[1] < a.nwin ? a.wl[1] : a.nwin, n0 = a.wl[0] < a.nwin ? a.wl[0] : a.nwin;
  if (e >= n1 + n0) return;
  const int packed = a.wl[WL_HDR + (e < n1 ? a.nwin + e : e - n1)];
  const int b = packed >> 16, wcx = (packed >> 8) & 255, wcy = packed & 255;
  const int y = wcy * WIN - a.s + (lane >> 3), x = wcx * WIN - a.s + (lane & 7);
  const bool in = b >= 0 && b < a.batch && y >= 0 && y < a.ny && x >= 0 && x < a.nx;
  const int64_t cell = ((int64_t)b * a.ny + y) * a.nx + x;
  int t0 = in ? a.grid_q[cell] : -1, t1 = in ? a.grid_k[cell] : -1;
  if (t0 >= a.mq) t0 = -1;
  if (t1 >= a.mk) t1 = -1;
  const unsigned long long m0 = __ballot(t0 >= 0), m1 = __ballot(t1 >= 0), below = (1ull << lane) - 1ull;
  const int Tq = min(__popcll(m0), 16), Tk = min(__popcll(m1), 16);
  if (Tq == 0 || Tk == 0) return;                        // (in no list: the rows are zeroed elsewhere)
  int (*toks)[16] = toks_[w];
  char* lds = lds_[w];
  const int f0 = __shfl(t0, __ffsll(m0) - 1, 64), f1 = __shfl(t1, __ffsll(m1) - 1, 64);
  if (lane < 16) { toks[0][lane] = f0; toks[1][lane] = f1; }
  order_lds();
  const int r0 = __popcll(m0 & below), r1 = __popcll(m1 & below);
  if (t0 >= 0 && r0 < 16) toks[0][r0] = t0;
  if (t1 >= 0 && r1 < 16) toks[1][r1] = t1;
  order_lds();
  const int64_t tq = toks[0][i], tk = toks[1][i];
  const float c = a.scale * LOG2E;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 absent;
#pragma unroll
  for (int r = 0; r < 4; ++r) absent[r] = 4 * g + r < Tk ? 0.f : -INFINITY;
  const int64_t at = FR * 2 * g;
  const char *q = (const char*)a.q + tq * a.ldq * 2 + at, *k = (const char*)a.k + tk * a.ldk * 2 + at, *v = (const char*)a.v + tk * a.ldv * 2 + at;
  const char* gr = BWD ? (const char*)a.g + tq * a.ldg * 2 + at : nullptr;
  for (int h0 = 0; h0 < a.nhead; h0 += HG) {
    Piece<FR> kf[HG], vf[HG], qf[HG], gf[HG];
    float ls[HG];
#pragma unroll
    for (int h = 0; h < HG; ++h) {
      const int hh = h0 + h < a.nhead ? h0 + h : a.nhead - 1;            // a head behind the last one: read twice, stored once
      kf[h] = load_piece<FR>(k + hh * DH * 2);
      vf[h] = load_piece<FR>(v + hh * DH * 2);
      qf[h] = load_piece<FR>(q + hh * DH * 2);
      if constexpr (BWD) {
        gf[h] = load_piece<FR>(gr + hh * DH * 2);
        ls[h] = a.lse[tq * a.nhead + hh];
      }
    }
    if constexpr (!BWD) {
#pragma unroll
      for (int h = 0; h < HG; ++h) Im::put(lds + h * PER_HEAD, g, i, vf[h]);
      order_lds();
      s16x4 vc[HG][CT], p[HG];
#pragma unroll
      for (int h = 0; h < HG; ++h)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) vc[h][ct] = Im::get(lds + h * PER_HEAD, g, i, ct);
      order_lds();
      f32x4 st[HG];
      float mx[HG], l[HG];
#pragma unroll
      for (int h = 0; h < HG; ++h) st[h] = over_channels<FR>(kf[h], qf[h], absent);
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        mx[h] = column_max(fmaxf(fmaxf(st[h][0], st[h][1]), fmaxf(st[h][2], st[h][3]))) * c;
        l[h] = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          st[h][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[h][r], c, -mx[h]));
          l[h] += st[h][r];
        }
        p[h] = pack4(st[h]);
      }
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        f32x4 o[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) o[ct] = over_tokens(vc[h][ct], p[h], zero);
        const float s = column_sum(l[h]);
        if (i < Tq && h0 + h < a.nhead) {
          store_piece<FR>((char*)a.o + tq * a.ldo * 2 + (h0 + h) * DH * 2 + at, o, __builtin_amdgcn_rcpf(s));
          if (g == 0) a.lse[tq * a.nhead + h0 + h] = mx[h] + __builtin_amdgcn_logf(s);
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        char* im = lds + h * PER_HEAD;
        Im::put(im, g, i, kf[h]);
        Im::put(im + Im::TILE, g, i, qf[h]);
        Im::put(im + 2 * Im::TILE, g, i, gf[h]);
      }
      order_lds();
      s16x4 kc[HG][CT], qc[HG][CT], gc[HG][CT], ds[HG], pb[HG];
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        const char* im = lds + h * PER_HEAD;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          kc[h][ct] = Im::get(im, g, i, ct);
          qc[h][ct] = Im::get(im + Im::TILE, g, i, ct);
          gc[h][ct] = Im::get(im + 2 * Im::TILE, g, i, ct);
        }
      }
      order_lds();
      f32x4 p[HG], dp[HG];
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        p[h] = over_channels<FR>(kf[h], qf[h], absent);
        dp[h] = over_channels<FR>(vf[h], gf[h], zero);
      }
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        const float le = i < Tq ? ls[h] : INFINITY;
        float d = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[h][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[h][r], c, -le));
          d = __builtin_fmaf(p[h][r], dp[h][r], d);
        }
        d = column_sum(d);
        f32x4 t;
#pragma unroll
        for (int r = 0; r < 4; ++r) t[r] = p[h][r] * (dp[h][r] - d);
        ds[h] = pack4(t);
        pb[h] = pack4(p[h]);
        char* im = lds + h * PER_HEAD;
        *reinterpret_cast<s16x4*>(im + i * TP + 8 * g) = pb[h];
        *reinterpret_cast<s16x4*>(im + 16 * TP + i * TP + 8 * g) = ds[h];
      }
      order_lds();
      s16x4 pt[HG], dt[HG];
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        const char* im = lds + h * PER_HEAD;
        pt[h] = read_columns(im + (4 * g + (i >> 2)) * TP + 8 * (i & 3));
        dt[h] = read_columns(im + 16 * TP + (4 * g + (i >> 2)) * TP + 8 * (i & 3));
      }
      order_lds();
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        f32x4 dq[CT], dk[CT], dv[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          dq[ct] = over_tokens(kc[h][ct], ds[h], zero);
          dv[ct] = over_tokens(gc[h][ct], pt[h], zero);
          dk[ct] = over_tokens(qc[h][ct], dt[h], zero);
        }
        const int64_t hcol = (int64_t)(h0 + h) * DH * 2 + at;
        if (h0 + h < a.nhead) {
          if (i < Tq) store_piece<FR>((char*)a.dq + tq * a.lddq * 2 + hcol, dq, a.scale);
          if (i < Tk) {
            store_piece<FR>((char*)a.dk + tk * a.lddk * 2 + hcol, dk, a.scale);
            store_piece<FR>((char*)a.dv + tk * a.lddv * 2 + hcol, dv, 1.f);
          }
        }
      }
    }
  }
}

// The windows that are in no list: zero rows for queries without a key (out, or dq) and for keys without a query (dk, dv).  One wave per
// window, a lane per cell.
__global__ __launch_bounds__(256) void dot_orphan_kernel(DotArgs a, char* q0, int64_t ldq0, char* k0, int64_t ldk0, char* k1, int64_t ldk1,
                                                        int row16) {
  const int lane = threadIdx.x & 63;
  const int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (u >= a.nwin) return;
  const int wcy = (int)(u % a.Wy), wcx = (int)((u / a.Wy) % a.Wx), b = (int)(u / ((int64_t)a.Wy * a.Wx));
  const int y = wcy * WIN - a.s + (lane >> 3), x = wcx * WIN - a.s + (lane & 7);
  const bool in = y >= 0 && y < a.ny && x >= 0 && x < a.nx;
  const int64_t cell = ((int64_t)b * a.ny + y) * a.nx + x;
  int tq = in ? a.grid_q[cell] : -1, tk = in ? a.grid_k[cell] : -1;
  if (tq >= a.mq) tq = -1;
  if (tk >= a.mk) tk = -1;
  const bool some_q = __ballot(tq >= 0) != 0, some_k = __ballot(tk >= 0) != 0;
  const uint4 z = make_uint4(0u, 0u, 0u, 0u);
  if (q0 && !some_k && tq >= 0)
    for (int c = 0; c < row16; ++c) reinterpret_cast<uint4*>(q0 + tq * ldq0)[c] = z;
  if (k0 && !some_q && tk >= 0)
    for (int c = 0; c < row16; ++c) {
      reinterpret_cast<uint4*>(k0 + tk * ldk0)[c] = z;
      reinterpret_cast<uint4*>(k1 + tk * ldk1)[c] = z;
    }
}

// blocks of a work list's class: class c > 0 windows hold more than 8 * 2^(c-1) tokens of one of the two frames
int64_t class_blocks(int cls, int64_t nwin, int64_t mq, int64_t mk) {
  const int64_t most = cls == 0 ? nwin : (mq + mk) / (cls == 1 ? 9 : cls == 2 ? 17 : 33);
  return most < nwin ? most : nwin;
}

bool rows_ok(const void* p, int64_t ld, int width, int es) {
  return p && ((uintptr_t)p & 15) == 0 && ld >= width && (ld * es) % 16 == 0;
}

int fill(DotArgs& a, int dtype, int64_t mq, int64_t mk, int nhead, int dh, const int32_t* grid_q, const int32_t* grid_k, int batch, int ny,
         int nx, int do_shift, float scale, const int32_t* worklist) {
  if (dtype != TMAE_F32 && dtype != TMAE_BF16) return TMAE_EDTYPE;
  if (mq < 0 || mk < 0 || mq > 0x7fffffff || mk > 0x7fffffff || nhead < 1 || nhead > 4096 || (dh != 16 && dh != 32 && dh != 64)) return TMAE_EARG;
  if (!grid_q || !grid_k || batch < 1 || ny < 1 || nx < 1 || (int64_t)ny * nx >= ((int64_t)1 << 31) ||
      (int64_t)batch * ny * nx >= ((int64_t)1 << 31) || !(scale > 0.f) || scale > 3e38f)
    return TMAE_EARG;
  a.Wy = (ny + WIN - 1) / WIN + 1; a.Wx = (nx + WIN - 1) / WIN + 1;
  if (worklist && (a.Wy > 255 || a.Wx > 255 || batch > 32767)) return TMAE_EARG;
  a.nwin = (int64_t)batch * a.Wy * a.Wx;
  if (a.nwin > 0x7fffffff) return TMAE_EARG;
  a.grid_q = grid_q; a.grid_k = grid_k; a.wl = worklist; a.mq = mq; a.mk = mk; a.nhead = nhead; a.batch = batch; a.ny = ny; a.nx = nx;
  a.s = do_shift ? WIN / 2 : WIN;
  a.scale = scale;
  return TMAE_OK;
}

template <class F> void by_head(int dh, F&& f) {
  if (dh == 16) f(std::integral_constant<int, 16>());
  else if (dh == 32) f(std::integral_constant<int, 32>());
  else f(std::integral_constant<int, 64>());
}
template <int DH, bool BWD> void launch_bf16(const DotArgs& a, hipStream_t stream) {
  const unsigned gy = (unsigned)((a.nhead + 3) / 4);
  if (!a.wl) {
    hipLaunchKernelGGL((dot_window_kernel<DH, 4, BWD>), dim3((unsigned)a.nwin, gy), dim3(256), 0, stream, a, 0);
    return;
  }
  const int64_t b3 = class_blocks(3, a.nwin, a.mq, a.mk), b2 = class_blocks(2, a.nwin, a.mq, a.mk);
  if (b3 > 0) hipLaunchKernelGGL((dot_window_kernel<DH, 4, BWD>), dim3((unsigned)b3, gy), dim3(256), 0, stream, a, 3);
  if (b2 > 0) hipLaunchKernelGGL((dot_window_kernel<DH, 2, BWD>), dim3((unsigned)b2, gy), dim3(256), 0, stream, a, 2);
  int64_t small = a.mq < a.mk ? a.mq : a.mk;             // a listed window holds a query and a key
  if (small > a.nwin) small = a.nwin;
  if (small > 0) hipLaunchKernelGGL((dot_small_kernel<DH, BWD>), dim3(tmae_cdiv(small, 4)), dim3(256), 0, stream, a);
}

template <class F> void by_class(const DotArgs& a, F&& f) {
  const unsigned gy = (unsigned)((a.nhead + 3) / 4);
  if (!a.wl) { f(dim3((unsigned)a.nwin, gy), 0); return; }
  for (int cls = 3; cls >= 0; --cls) {
    const int64_t blocks = class_blocks(cls, a.nwin, a.mq, a.mk);
    if (blocks > 0) f(dim3((unsigned)blocks, gy), cls);
  }
}

}  // namespace

int tmae_win_attn_dot_fwd(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, int dtype, int64_t mq,
                          int64_t mk, int nhead, int dh, const int32_t* grid_q, const int32_t* grid_k, int batch, int ny, int nx,
                          int do_shift, float scale, void* out, int64_t ldo, float* lse, const int32_t* worklist, void* stream) {
  (void)hipGetLastError();
  DotArgs a = {};
  const int rc = fill(a, dtype, mq, mk, nhead, dh, grid_q, grid_k, batch, ny, nx, do_shift, scale, worklist);
  if (rc != TMAE_OK) return rc;
  if (mq == 0) return TMAE_OK;
  const int es = dtype == TMAE_BF16 ? 2 : 4, d = nhead * dh;
  if (!rows_ok(q, ldq, d, es) || !rows_ok(out, ldo, d, es) || !lse || (mk && (!rows_ok(k, ldk, d, es) || !rows_ok(v, ldv, d, es)))) return TMAE_EARG;
  a.q = q; a.ldq = ldq; a.k = k; a.ldk = ldk; a.v = v; a.ldv = ldv; a.o = out; a.ldo = ldo; a.lse = lse;
  if (worklist && grid_q != grid_k)
    hipLaunchKernelGGL(dot_orphan_kernel, dim3(tmae_cdiv(a.nwin, 4)), dim3(256), 0, (hipStream_t)stream, a, (char*)out, ldo * es, nullptr,
                       (int64_t)0, nullptr, (int64_t)0, d * es / 16);
  by_head(dh, [&](auto w) {
    constexpr int DH = decltype(w)::value;
    if (dtype == TMAE_BF16) launch_bf16<DH, false>(a, (hipStream_t)stream);
    else
      by_class(a, [&](dim3 grid, int cls) {
        hipLaunchKernelGGL((dot_fwd_kernel<float, DH>), grid, dim3(256), 0, (hipStream_t)stream, a, cls);
      });
  });
  return tmae_launch_status();
}

int tmae_win_attn_dot_bwd(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, const void* dout,
                          int64_t lddo, const float* lse, int dtype, int64_t mq, int64_t mk, int nhead, int dh, const int32_t* grid_q,
                          const int32_t* grid_k, int batch, int ny, int nx, int do_shift, float scale, void* dq, int64_t lddq, void* dk,
                          int64_t lddk, void* dv, int64_t lddv, const int32_t* worklist, void* stream) {
  (void)hipGetLastError();
  DotArgs a = {};
  const int rc = fill(a, dtype, mq, mk, nhead, dh, grid_q, grid_k, batch, ny, nx, do_shift, scale, worklist);
  if (rc != TMAE_OK) return rc;
  if (mq == 0 && mk == 0) return TMAE_OK;
  const int es = dtype == TMAE_BF16 ? 2 : 4, d = nhead * dh;
  if (mq && (!rows_ok(q, ldq, d, es) || !rows_ok(dout, lddo, d, es) || !rows_ok(dq, lddq, d, es) || !lse)) return TMAE_EARG;
  if (mk && (!rows_ok(k, ldk, d, es) || !rows_ok(v, ldv, d, es) || !rows_ok(dk, lddk, d, es) || !rows_ok(dv, lddv, d, es))) return TMAE_EARG;
  a.q = q; a.ldq = ldq; a.k = k; a.ldk = ldk; a.v = v; a.ldv = ldv; a.g = dout; a.ldg = lddo; a.lse = const_cast<float*>(lse);
  a.dq = dq; a.lddq = lddq; a.dk = dk; a.lddk = lddk; a.dv = dv; a.lddv = lddv;
  if (worklist && grid_q != grid_k)
    hipLaunchKernelGGL(dot_orphan_kernel, dim3(tmae_cdiv(a.nwin, 4)), dim3(256), 0, (hipStream_t)stream, a, (char*)dq, lddq * es,
                       (char*)dk, lddk * es, (char*)dv, lddv * es, d * es / 16);
  by_head(dh, [&](auto w) {
    constexpr int DH = decltype(w)::value;
    if (dtype == TMAE_BF16) launch_bf16<DH, true>(a, (hipStream_t)stream);
    else
      by_class(a, [&](dim3 grid, int cls) {
        hipLaunchKernelGGL((dot_bwd_kernel<float, DH>), grid, dim3(256), 0, (hipStream_t)stream, a, cls);
      });
  });
  return tmae_launch_status();
}
